// The two places of prioritized replay that need the host's pow (host_pow.h), as enqueued on a stream (tree.hip).
#pragma once
#include "host_pow.h"
#include "tree_dev.h"

namespace samx {

// memory.py:370-379: n TD errors -> their leaves in the stage (n values); max_priority and the asserts -> state
int per_leaves_enqueue(const float* td, const int64_t* idxs, int64_t n, int64_t cap, int64_t num_entries, double alpha,
                       int64_t num_demos, double demos_eps, PerState* state, const int64_t* geom, const PowStage& s,
                       hipStream_t st);
// memory.py:301-309: the bases per_sample_body left in the stage (B + 1 values) -> the importance weights
int per_weights_enqueue(const PowStage& s, int64_t B, double beta, double* iws, float* iws32, hipStream_t st);

}  // namespace samx
