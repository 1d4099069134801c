// k_decay.h -- what the sources of decay attention share: the operands of one run of the recurrence (k_decay.hip says which
// four runs a training step consists of) and the launchers, one source for each element type.
#pragma once
#include "pxg_ops.h"

struct DecayRun {
    pxg_sequence x, y, z;      // operands: widths E, E, F
    const float* init;         // state before the first step (of the run's direction), element (e, f) at e * init_e + f * init_f
    float* fin;                // state behind the last one, same layout
    int64_t init_e, init_f;
    void* out;                 // [batch][steps][heads][F]
    int E, F;
    int reverse;               // steps taken from the last to the first; then init joins the first step without decay
    int wide;                  // every row can be read 16 bytes and written four values at a time
    float* carry;              // states between segments, [batch * heads][segments - 1][E][F] (and the slopes behind them)
    // gradient of log_decay (the run of dq): q's rows, the gradient of the final state, one partial sum per (batch * heads, segment)
    pxg_sequence dot;
    const float* grad_fin;
    double* partial;
};

struct DecayRuns {
    DecayRun run[3];
    int64_t steps;
    int batch, heads;
    const float* log_decay;
    const void* lengths;
    int lengths_are_64;
    int segments, segment_chunks;      // the time axis in so many pieces of so many chunks, each a workgroup of its own
};

__device__ __forceinline__ int64_t decay_length(const DecayRuns& s, int b)
{
    if (!s.lengths) return s.steps;
    const int64_t n = s.lengths_are_64 ? ((const int64_t*)s.lengths)[b] : (int64_t)((const int32_t*)s.lengths)[b];
    return n < 0 ? 0 : n > s.steps ? s.steps : n;
}

// exp(n log_a): what the product's rounding takes is given back, for it would be the same in every chunk
__device__ __forceinline__ float decay_over(float n, float log_a)
{
    const float p = n * log_a, lost = fmaf(n, log_a, -p), w = expf(p);
    return w > 0.f && w < INFINITY ? fmaf(w, lost, w) : w;
}

constexpr int DECAY_CHUNK = 32;        // steps

// the width that a head's are padded to
constexpr int decay_width(int e, int f)
{
    const int w = e > f ? e : f;
    return w <= 16 ? 16 : w <= 32 ? 32 : w <= 64 ? 64 : 128;
}

// `n` runs, the first `slopes` of them (none or one) with dS/dlog_decay; states_only: nothing but `carry` is written
int decay_launch_f32(const DecayRuns& a, int n, int slopes, bool states_only, hipStream_t stream);
int decay_launch_bf16(const DecayRuns& a, int n, int slopes, bool states_only, hipStream_t stream);
int decay_launch_f16(const DecayRuns& a, int n, int slopes, bool states_only, hipStream_t stream);
