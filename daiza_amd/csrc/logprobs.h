// logprobs.h — log probabilities of rows of logits on the device (logprobs.hip), for the entry points on contexts.
#pragma once
#include "common.h"

namespace dz {

constexpr int kLogprobTop = 64;  // most alternatives

// Bytes of work memory, and the launches: see dz_logprobs_dev.  The arguments are checked by the caller.
size_t logprobs_work(int n, int64_t vocab, int top);
int logprobs(const void* logits, int64_t ld, int type, int n, int vocab, const int32_t* tokens, int top, float* logp, float* entropy,
             int32_t* top_ids, float* top_logp, void* work, hipStream_t s);

}  // namespace dz
