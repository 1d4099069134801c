// k_decay.hip -- linear attention with one decay per head, over whole sequences (forward, backward) and for single steps.
//
//   S_t = a S_(t-1) + k_t v_t^T,   o_t = q_t S_t,   a = exp(log_decay[head])
//
// The four outputs of a training step are the same recurrence with other operands (x: read against the state, y and z: written
// into it), two of them over the steps backwards:
//   o  = run(x q,  y k,  z v)                         dq = run(x do, y v,  z k)            with S^T as its state
//   dk = run(x v,  y do, z q) backwards               dv = run(x k,  y q,  z do) backwards  with R = dL/dS as their state
// and the gradient of log_decay is sum_t do_t . (q_t D_t) + <dL/dS_T, D_T> with D = dS/dlog_decay = a (D + S) carried beside S
// in the run of dq: no difference of large sums, however long the sequence.
//
// The runs themselves are in k_decay_chunk.h.
#include "k_decay.h"

namespace {

// carry[s] becomes the state in front of segment s + 1: each segment's own, plus what came before it, decayed over its length;
// the slopes behind the states decay and grow with the distance.  Bound by reading and
// writing the states: 128 pairs x 6 states of 64 x 64 6.5 us, three runs of them with slopes 12.4.
constexpr int AT_ONCE = 8;

__global__ __launch_bounds__(256) void k_decay_join(const DecayRuns a, int slope_runs)
{
    const DecayRun& r = a.run[blockIdx.z];
    const int64_t size = (int64_t)r.E * r.F, bh = blockIdx.x, n = a.segments - 1;
    const int64_t slopes = (int64_t)a.batch * a.heads * n * size;
    const int i = blockIdx.y * 256 + threadIdx.x;
    if (i >= size) return;
    const int used = (int)((uint32_t)(decay_length(a, (int)bh / a.heads) + DECAY_CHUNK - 1) / DECAY_CHUNK);
    const float steps = (float)a.segment_chunks * (float)DECAY_CHUNK, decay = decay_over(steps, a.log_decay[(int)bh % a.heads]);
    const bool slope = (int)blockIdx.z < slope_runs;
    float* c = r.carry + bh * n * size + i;
    float S = c[0], G = slope ? c[slopes] : 0.f;
    // state s is read by segment s + 1, if that has chunks
    const auto needed = [&](int s) { return s < n && (s + 1) * a.segment_chunks < used; };
    for (int s = 1; needed(s); s += AT_ONCE) {                                 // the loads of some, then the chain through them
        float own[AT_ONCE], own_slope[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) {
            own[j] = needed(s + j) ? c[(s + j) * size] : 0.f;
            own_slope[j] = slope && needed(s + j) ? c[slopes + (s + j) * size] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++)
            if (needed(s + j)) {
                G = fmaf(decay, G + steps * S, own_slope[j]);
                S = fmaf(decay, S, own[j]);
                c[(s + j) * size] = S;
                if (slope) c[slopes + (s + j) * size] = G;
            }
    }
}

// grad_log_decay[h] = the sum of the partial sums [batch][heads][segments], in a fixed order
__global__ __launch_bounds__(256) void k_decay_sum(const double* partial, int64_t batch, int heads, int segments, float* out)
{
    __shared__ double red[256];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < batch * segments; i += 256)
        sum += partial[(i / segments * heads + blockIdx.x) * segments + i % segments];
    red[threadIdx.x] = sum;
    __syncthreads();
    for (int w = 128; w; w >>= 1) {
        if (threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[blockIdx.x] = (float)red[0];
}

int launch(const DecayRuns& a, int dtype, int n, int slopes, bool states_only, hipStream_t stream)
{
    switch (dtype) {
    case PXG_DT_F32: return decay_launch_f32(a, n, slopes, states_only, stream);
    case PXG_DT_BF16: return decay_launch_bf16(a, n, slopes, states_only, stream);
    default: return decay_launch_f16(a, n, slopes, states_only, stream);
    }
}

int launch_runs(const DecayRuns& a, int dtype, int n, int slopes, hipStream_t stream)
{
    if (a.segments > 1) {
        const int rc = launch(a, dtype, n, slopes, true, stream);
        if (rc != PXG_OK) return rc;
        const dim3 grid(a.batch * a.heads, (a.run[0].E * a.run[0].F + 255) / 256, n);
        k_decay_join<<<grid, 256, 0, stream>>>(a, slopes);
        if (hipGetLastError() != hipSuccess) return PXG_E_HIP;
    }
    return launch(a, dtype, n, slopes, false, stream);
}

// One step.  The state is read once and written once, 8 dk dv bytes for 5 dk dv operations: bandwidth is all there is.  P threads
// have a (sequence, head) pair, each four columns of every (4 P / columns)-th row, four rows in flight; their parts of o meet in
// shared memory.  A pair of up to 32 x 32 takes a wave (four of them a workgroup, so that small states fill a CU), a larger one a
// workgroup.  2 048 x 8 states of 64 x 64, bf16 rows, nine tenths of them active: 100 us, 4.9 TB/s, what a copy reaches; one stream of
// 4 heads 4.2, a launch.  (One column a thread: 183.)
template <typename T, int P>
__global__ __launch_bounds__(256) void k_decay_step(const pxg_decay a)
{
    constexpr int PAIRS = 256 / P, ROWS = 4;
    __shared__ float qs[PAIRS][PXG_DECAY_MAX_WIDTH], ks[PAIRS][PXG_DECAY_MAX_WIDTH];
    __shared__ __attribute__((aligned(16))) float parts[PAIRS][P][4];
    const int own = threadIdx.x / P, t = threadIdx.x % P, dk = a.dk, dv = a.dv;
    const int64_t pairs = a.batch * a.heads, pair = (int64_t)blockIdx.x * PAIRS + own;
    const bool there = pair < pairs;
    const int64_t b = there ? pair / a.heads : 0, h = there ? pair % a.heads : 0;
    const bool active = there && !(a.lengths && !((const uint8_t*)a.lengths)[b]);
    const int groups = (dv + 3) / 4, every = P / groups, col = t % groups * 4, first = t / groups;       // groups <= 32 <= P
    const bool works = active && first < every;
    float* const S = a.final_state + (there ? pair : 0) * dk * dv + col;
    const bool wide = dv % 4 == 0 && (uintptr_t)a.final_state % 16 == 0;
    const auto load = [&](int e) {
        float4 s = {};
        if (wide) s = *(const float4*)(S + e * dv);
        else {
            s.x = S[e * dv];
            if (col + 1 < dv) s.y = S[e * dv + 1];
            if (col + 2 < dv) s.z = S[e * dv + 2];
            if (col + 3 < dv) s.w = S[e * dv + 3];
        }
        return s;
    };
    float4 s[ROWS];
    if (works)
#pragma unroll
        for (int n = 0; n < ROWS; n++)
            if (first + n * every < dk) s[n] = load(first + n * every);
    if (active) {
        const T* q = (const T*)a.q.data + b * a.q.batch_stride + h * a.q.head_stride;
        const T* k = (const T*)a.k.data + b * a.k.batch_stride + h * a.k.head_stride;
        for (int e = t; e < dk; e += P) qs[own][e] = pxg_to_f32(q[e]), ks[own][e] = pxg_to_f32(k[e]);
    }
    float v[4] = {}, o[4] = {};
    float decay = 0.f;
    if (works) {
        const T* at = (const T*)a.v.data + b * a.v.batch_stride + h * a.v.head_stride + col;
#pragma unroll
        for (int n = 0; n < 4; n++)
            if (col + n < dv) v[n] = pxg_to_f32(at[n]);
        decay = expf(a.log_decay[h]);
    }
    __syncthreads();
    if (works)
        for (int e0 = first; e0 < dk; e0 += ROWS * every) {
            float4 next[ROWS];
#pragma unroll
            for (int n = 0; n < ROWS; n++)
                if (e0 + (n + ROWS) * every < dk) next[n] = load(e0 + (n + ROWS) * every);
#pragma unroll
            for (int n = 0; n < ROWS; n++) {
                const int e = e0 + n * every;
                if (e >= dk) break;
                const float ke = ks[own][e], qe = qs[own][e];
                const float4 now = {fmaf(decay, s[n].x, ke * v[0]), fmaf(decay, s[n].y, ke * v[1]), fmaf(decay, s[n].z, ke * v[2]),
                                    fmaf(decay, s[n].w, ke * v[3])};
                if (wide) *(float4*)(S + e * dv) = now;
                else {
                    S[e * dv] = now.x;
                    if (col + 1 < dv) S[e * dv + 1] = now.y;
                    if (col + 2 < dv) S[e * dv + 2] = now.z;
                    if (col + 3 < dv) S[e * dv + 3] = now.w;
                }
                o[0] = fmaf(qe, now.x, o[0]), o[1] = fmaf(qe, now.y, o[1]), o[2] = fmaf(qe, now.z, o[2]), o[3] = fmaf(qe, now.w, o[3]);
            }
#pragma unroll
            for (int n = 0; n < ROWS; n++) s[n] = next[n];
        }
    *(float4*)parts[own][t] = float4{o[0], o[1], o[2], o[3]};
    __syncthreads();
    if (there)
        for (int f = t; f < dv; f += P) {
            float sum = 0.f;
            for (int n = 0; n < every; n++) sum += parts[own][n * groups + f / 4][f % 4];
            ((T*)a.out)[pair * dv + f] = pxg_from_f32<T>(active ? sum : 0.f);
        }
}

template <typename T> void launch_step(const pxg_decay& a, hipStream_t stream)
{
    const int64_t pairs = a.batch * a.heads;
    if ((int64_t)a.dk * a.dv <= 1024) k_decay_step<T, 64><<<(unsigned)((pairs + 3) / 4), 256, 0, stream>>>(a);
    else k_decay_step<T, 256><<<(unsigned)pairs, 256, 0, stream>>>(a);
}

bool bad_shape(const pxg_decay* a)
{
    return !a || a->struct_bytes != sizeof(pxg_decay) || a->dtype < PXG_DT_F32 || a->dtype > PXG_DT_F16 || a->batch < 0 ||
           a->steps < 0 || a->steps > INT32_MAX || a->heads < 1 || a->heads > PXG_DECAY_MAX_PAIRS || a->dk < 1 || a->dk > PXG_DECAY_MAX_WIDTH || a->dv < 1 ||
           a->dv > PXG_DECAY_MAX_WIDTH || a->batch > PXG_DECAY_MAX_PAIRS / a->heads;
}

// a pointer may be missing only where nothing is read or written through it
bool bad_operands(const pxg_decay* a)
{
    const bool any = a->batch > 0 && a->steps > 0;
    return !a->log_decay || (any && (!a->q.data || !a->k.data || !a->v.data));
}

// How the time axis is cut.  The cost of segments is a second reading of y and z, their gain waves that hide each other's latency:
// a pass takes them where its (sequence, head) pairs come to no more than 1 024 waves (four for each CU), and enough of them for
// 4 096 (forward) or 2 048 (backward, which has three runs to do), of at least four chunks each (eight where that fills a quarter
// of the card by itself: 1 024 pairs x 300 steps x 16 wide f32 31 -> 47).  Forward / backward in us, uncut
// and cut: 128 pairs x 2 000 steps x 64 wide bf16 113 / 263 -> 61 / 190, 256 pairs (the limit) 113 / 287 -> 98 / 293, 384 pairs
// 129 / 361 -> 146 / 475; 256 pairs x 16 wide f32 (one wave each) 171 / 418 -> 71 / 201.
struct Cut {
    int segments, chunks;
};

Cut cut_of(const pxg_decay* a, bool backward)
{
    const int width = decay_width(a->dk, a->dv);
    const int64_t chunks = (a->steps + DECAY_CHUNK - 1) / DECAY_CHUNK;
    const int64_t waves = a->batch * a->heads * (width / 16);
    int64_t segments = 1;
    if (waves > 0 && waves <= (backward ? 1023 : 1024)) segments = ((backward ? 2048 : 4096) + waves - 1) / waves;
    const int64_t least = waves > 256 ? 8 : 4;                 // chunks of a segment
    if (segments > chunks / least) segments = chunks / least;
    if (segments < 1) segments = 1;
    const int64_t each = segments > 1 ? (chunks + segments - 1) / segments : chunks > 0 ? chunks : 1;
    Cut c = {(int)(segments > 1 ? (chunks + each - 1) / each : 1), (int)each};
    return c;
}

int64_t carry_values(const pxg_decay* a, const Cut& c)
{
    return a->batch * a->heads * (c.segments - 1) * a->dk * a->dv;
}

DecayRuns runs_of(const pxg_decay* a, const Cut& c)
{
    DecayRuns s = {};
    s.steps = a->steps, s.batch = (int)a->batch, s.heads = a->heads;
    s.log_decay = a->log_decay, s.lengths = a->lengths, s.lengths_are_64 = a->lengths_are_64;
    s.segments = c.segments, s.segment_chunks = c.chunks;
    return s;
}

// rows that can be read 16 bytes at a time, in whole groups of eight elements, a chunk of them within 32 bits of one another
bool wide(const pxg_sequence& s, int width, int dtype)
{
    const int64_t unit = dtype == PXG_DT_F32 ? 4 : 8;
    return (uintptr_t)s.data % 16 == 0 && width % 8 == 0 && s.batch_stride % unit == 0 && s.step_stride % unit == 0 &&
           s.head_stride % unit == 0 && s.step_stride >= 0 && s.step_stride < 1 << 24;
}

void finish_run(DecayRun& r, int dtype)
{
    r.wide = wide(r.x, r.E, dtype) && wide(r.y, r.E, dtype) && wide(r.z, r.F, dtype) && (!r.partial || wide(r.dot, r.F, dtype)) && (uintptr_t)r.out % 16 == 0;
}

}  // namespace

extern "C" int64_t pxg_decay_workspace_bytes(const pxg_decay* a, int32_t backward)
{
    if (bad_shape(a)) return PXG_E_INVALID;
    const Cut c = cut_of(a, backward != 0);
    // the states between segments (backward: of three runs, and the slopes of one), the partial sums of grad_log_decay
    return backward ? (int64_t)sizeof(double) * a->batch * a->heads * c.segments + (int64_t)sizeof(float) * 4 * carry_values(a, c)
                    : (int64_t)sizeof(float) * carry_values(a, c);
}

extern "C" int pxg_decay_forward(const pxg_decay* a, void* stream)
{
    if (bad_shape(a) || bad_operands(a)) return PXG_E_INVALID;
    if (a->batch == 0) return PXG_OK;
    if (a->steps > 0 && !a->out) return PXG_E_INVALID;
    const int64_t bytes = pxg_decay_workspace_bytes(a, 0);
    if (a->workspace_bytes < bytes || (bytes > 0 && (!a->workspace || (uintptr_t)a->workspace % 8))) return PXG_E_INVALID;
    DecayRuns s = runs_of(a, cut_of(a, false));
    DecayRun& r = s.run[0];
    r.x = a->q, r.y = a->k, r.z = a->v;
    r.init = a->initial_state, r.fin = a->final_state, r.init_e = a->dv, r.init_f = 1;
    r.out = a->out, r.E = a->dk, r.F = a->dv;
    r.carry = (float*)a->workspace;
    finish_run(r, a->dtype);
    (void)hipGetLastError();                     // what an earlier call left is not this call's
    return launch_runs(s, a->dtype, 1, 0, (hipStream_t)stream);
}

extern "C" int pxg_decay_backward(const pxg_decay* a, void* stream)
{
    if (bad_shape(a) || bad_operands(a)) return PXG_E_INVALID;
    const bool any = a->batch > 0 && a->steps > 0;
    if (any && (!a->grad_q || !a->grad_k || !a->grad_v || !a->grad_out.data)) return PXG_E_INVALID;
    const int64_t bytes = pxg_decay_workspace_bytes(a, 1);
    if (a->workspace_bytes < bytes || (bytes > 0 && (!a->workspace || (uintptr_t)a->workspace % 8))) return PXG_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    (void)hipGetLastError();                     // what an earlier call left is not this call's
    const Cut c = cut_of(a, true);
    DecayRuns s = runs_of(a, c);
    double* const partial = (double*)a->workspace;
    int rc = PXG_OK;
    if (a->batch > 0) {
        DecayRun &dq = s.run[0], &dk = s.run[1], &dv = s.run[2];
        dq.x = a->grad_out, dq.y = a->v, dq.z = a->k;
        dq.init = a->initial_state, dq.init_e = 1, dq.init_f = a->dv;
        dq.out = a->grad_q, dq.E = a->dv, dq.F = a->dk;
        if (a->grad_log_decay) dq.dot = a->q, dq.grad_fin = a->grad_final_state, dq.partial = partial;
        dk.x = a->v, dk.y = a->grad_out, dk.z = a->q, dk.reverse = 1;
        dk.init = a->grad_final_state, dk.init_e = 1, dk.init_f = a->dv;
        dk.out = a->grad_k, dk.E = a->dv, dk.F = a->dk;
        dv.x = a->k, dv.y = a->q, dv.z = a->grad_out, dv.reverse = 1;
        dv.init = a->grad_final_state, dv.fin = a->grad_initial_state, dv.init_e = a->dv, dv.init_f = 1;
        dv.out = a->grad_v, dv.E = a->dk, dv.F = a->dv;
        dq.carry = (float*)(partial + a->batch * a->heads * c.segments);                                      // states and slopes
        dk.carry = dq.carry + 2 * carry_values(a, c), dv.carry = dk.carry + carry_values(a, c);
        for (DecayRun& r : s.run) finish_run(r, a->dtype);
        rc = launch_runs(s, a->dtype, 3, a->grad_log_decay ? 1 : 0, st);
    }
    if (rc == PXG_OK && a->grad_log_decay) {
        k_decay_sum<<<a->heads, 256, 0, st>>>(partial, a->batch, a->heads, c.segments, a->grad_log_decay);
        if (hipGetLastError() != hipSuccess) rc = PXG_E_HIP;
    }
    return rc;
}

extern "C" int pxg_decay_step(const pxg_decay* a, void* stream)
{
    if (bad_shape(a) || a->steps != 1 || bad_operands(a)) return PXG_E_INVALID;
    if (a->batch == 0) return PXG_OK;
    if (!a->out || !a->final_state) return PXG_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    (void)hipGetLastError();                     // what an earlier call left is not this call's
    switch (a->dtype) {
    case PXG_DT_F32: launch_step<float>(*a, st); break;
    case PXG_DT_BF16: launch_step<pxg_bf16>(*a, st); break;
    default: launch_step<pxg_f16>(*a, st);
    }
    return hipGetLastError() == hipSuccess ? PXG_OK : PXG_E_HIP;
}
