// pow(x, y) of the HOST C library for numbers that a kernel made, in stream order: the kernel writes them into pinned
// host memory (a PowStage), a host function on the stream calls pow on each, the next kernel reads the results.
// Prioritized replay needs it: `priority ** alpha` and `(n * prob) ** -beta` (memory.py:301,308,341-342,376-377) reach
// the host's pow in the reference, and the sampled indices of every later step depend on its last bit, which no other
// implementation of pow reproduces.  All of it only enqueues and can be captured into a graph.
#pragma once
#include "samx_common.h"
#include <math.h>

namespace samx {

// Pinned doubles, written and read by kernels, one owner at a time.
struct PowStage {
    double* x = nullptr;
    int slot = -1;          // >= 0: a slot of the pool, given back by host_pow_done; -1: held by a captured graph
};

// The exponents pow is called with here.
inline bool pow_exponent_ok(double y) { return fabs(y) >= 0x1p-65 && fabs(y) < 0x1p63; }

// x[i] = pow(x[i], y): what the host function does
void host_pow_values(double* x, int64_t n, double y);

// n doubles.  Outside a capture: a pool slot whose last use on the GPU is over.  Under capture the memory has to live as
// long as the graph, so it belongs to `owner`, a buffer that the call writes: calls that share it race on it anyway.
int host_pow_stage(const void* owner, int64_t n, hipStream_t st, PowStage* s);
// x[i] = pow(x[i], y) on the host, behind the work on `st`
int host_pow_run(const PowStage& s, int64_t n, double y, hipStream_t st);
// the last kernel that uses the stage has been enqueued
int host_pow_done(const PowStage& s, hipStream_t st);

}  // namespace samx
