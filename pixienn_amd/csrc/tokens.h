// What the log probabilities of tokens leave for beam search.
#pragma once

#include "common.h"

namespace pxh {

size_t token_rows_workspace_bytes(long long rows, int vocab, int top);

// The `top` largest logits of every row, ids [rows][top] descending, the lowest index first among equal ones, and in sums the row's largest logit
// with the sum of exp(scale * (logit - largest)).  Logits are ordered as they are: times the scale, rounded, neighbours would be equal.  values:
// as many floats for its own use.  The arguments have been looked at.
int token_rows(const char* who, const void* logits, int type, long long rows, int vocab, long long stride, int top, float scale,
               float* values, int* ids, float2* sums, void* workspace, hipStream_t s);

}  // namespace pxh
