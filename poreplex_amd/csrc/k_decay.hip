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
#include "pxg_ops.h"

namespace {

struct DecayRun {
    pxg_sequence x, y, z;      // operands: widths E, E, F
    const float* init;         // state before the first step (of the run's direction), element (e, f) at e * init_e + f * init_f
    float* fin;                // state behind the last one, same layout
    int64_t init_e, init_f;
    void* out;                 // [batch][steps][heads][F]
    int E, F;
    int reverse;               // steps taken from the last to the first; then init joins the first step without decay
    // gradient of log_decay (the run of dq): q's rows, the gradient of the final state, one partial sum per (batch, head)
    pxg_sequence dot;
    const float* grad_fin;
    float* partial;
};

struct DecayShape {
    int64_t steps;
    int batch, heads;
    const float* log_decay;
    const void* lengths;
    int lengths_are_64;
};

__device__ __forceinline__ int64_t decay_length(const DecayShape& s, int b)
{
    if (!s.lengths) return s.steps;
    const int64_t n = s.lengths_are_64 ? ((const int64_t*)s.lengths)[b] : (int64_t)((const int32_t*)s.lengths)[b];
    return n < 0 ? 0 : n > s.steps ? s.steps : n;
}

// One step after the other, the state in shared memory: thread f owns column f.
template <typename T, bool DER>
__global__ __launch_bounds__(128) void k_decay_serial(DecayRun r, DecayShape s)
{
    extern __shared__ float lds[];
    const int f = threadIdx.x, b = blockIdx.x / s.heads, h = blockIdx.x % s.heads;
    float* S = lds;
    float* D = S + r.E * r.F;
    float* xs = D + (DER ? r.E * r.F : 0);
    float* ys = xs + r.E;
    const int64_t len = decay_length(s, b), base = (int64_t)blockIdx.x * r.E * r.F;
    const float a = expf(s.log_decay[h]);
    const T* x = (const T*)r.x.data + b * r.x.batch_stride + h * r.x.head_stride;
    const T* y = (const T*)r.y.data + b * r.y.batch_stride + h * r.y.head_stride;
    const T* z = (const T*)r.z.data + b * r.z.batch_stride + h * r.z.head_stride;
    T* out = (T*)r.out + ((int64_t)b * s.steps * s.heads + h) * r.F;
    const int64_t out_step = (int64_t)s.heads * r.F;
    if (f < r.F)
        for (int e = 0; e < r.E; e++) {
            S[e * r.F + f] = r.init ? r.init[base + e * r.init_e + f * r.init_f] : 0.f;
            if (DER) D[e * r.F + f] = 0.f;
        }
    float part = 0.f;
    for (int64_t u = 0; u < len; u++) {
        const int64_t t = r.reverse ? len - 1 - u : u;
        for (int e = f; e < r.E; e += blockDim.x) {
            xs[e] = pxg_to_f32(x[t * r.x.step_stride + e]);
            ys[e] = pxg_to_f32(y[t * r.y.step_stride + e]);
        }
        __syncthreads();
        if (f < r.F) {
            const float zf = pxg_to_f32(z[t * r.z.step_stride + f]), decay = r.reverse && u == 0 ? 1.f : a;
            float o = 0.f, d = 0.f;
            for (int e = 0; e < r.E; e++) {
                const float old = S[e * r.F + f], now = fmaf(decay, old, ys[e] * zf);
                S[e * r.F + f] = now;
                o = fmaf(xs[e], now, o);
                if (DER) {
                    const float dn = decay * (D[e * r.F + f] + old);
                    D[e * r.F + f] = dn;
                    d = fmaf(xs[e], dn, d);
                }
            }
            out[t * out_step + f] = pxg_from_f32<T>(o);
            if (DER) {
                const T* q = (const T*)r.dot.data + b * r.dot.batch_stride + h * r.dot.head_stride;
                part = fmaf(pxg_to_f32(q[t * r.dot.step_stride + f]), d, part);
            }
        }
        __syncthreads();
    }
    if (f < r.F) {
        for (int64_t t = len; t < s.steps; t++) out[t * out_step + f] = pxg_from_f32<T>(0.f);
        for (int e = 0; e < r.E; e++) {
            if (r.fin) r.fin[base + e * r.init_e + f * r.init_f] = r.reverse && len ? a * S[e * r.F + f] : S[e * r.F + f];
            if (DER && r.grad_fin) part = fmaf(r.grad_fin[base + e * r.init_e + f * r.init_f], D[e * r.F + f], part);
        }
    }
    if (DER) {
        __syncthreads();
        xs[f] = f < r.F ? part : 0.f;
        __syncthreads();
        if (f == 0) {
            float sum = 0.f;
            for (int i = 0; i < (int)blockDim.x; i++) sum += xs[i];
            r.partial[blockIdx.x] = sum;
        }
    }
}

// grad_log_decay[h] = sum over the batch (and whatever else lies between) of the partial sums, in a fixed order
__global__ __launch_bounds__(256) void k_decay_sum(const float* partial, int64_t n, int heads, float* out)
{
    __shared__ double red[256];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 256) sum += (double)partial[i * heads + blockIdx.x];
    red[threadIdx.x] = sum;
    __syncthreads();
    for (int w = 128; w; w >>= 1) {
        if (threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[blockIdx.x] = (float)red[0];
}

template <typename T>
int launch_run(const DecayRun& r, const DecayShape& s, hipStream_t stream)
{
    const size_t state = (size_t)r.E * r.F * sizeof(float), rows = (2 * (size_t)r.E + 128) * sizeof(float);
    if (r.partial)
        k_decay_serial<T, true><<<s.batch * s.heads, 128, 2 * state + rows, stream>>>(r, s);
    else
        k_decay_serial<T, false><<<s.batch * s.heads, 128, state + rows, stream>>>(r, s);
    return hipGetLastError() == hipSuccess ? PXG_OK : PXG_E_HIP;
}

int run(const DecayRun& r, const DecayShape& s, int dtype, hipStream_t stream)
{
    switch (dtype) {
    case PXG_DT_F32: return launch_run<float>(r, s, stream);
    case PXG_DT_BF16: return launch_run<pxg_bf16>(r, s, stream);
    default: return launch_run<pxg_f16>(r, s, stream);
    }
}

// One step: the state is read once and written once, which is all the time this takes.
template <typename T>
__global__ __launch_bounds__(128) void k_decay_step(pxg_decay a)
{
    const int f = threadIdx.x, b = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
    if (f >= a.dv) return;
    T* out = (T*)a.out + (int64_t)blockIdx.x * a.dv;
    if (a.lengths && !((const uint8_t*)a.lengths)[b]) {
        out[f] = pxg_from_f32<T>(0.f);
        return;
    }
    const T* q = (const T*)a.q.data + b * a.q.batch_stride + h * a.q.head_stride;
    const T* k = (const T*)a.k.data + b * a.k.batch_stride + h * a.k.head_stride;
    const float v = pxg_to_f32(((const T*)a.v.data + b * a.v.batch_stride + h * a.v.head_stride)[f]);
    float* S = a.final_state + (int64_t)blockIdx.x * a.dk * a.dv + f;
    const float decay = expf(a.log_decay[h]);
    float o = 0.f;
    for (int e = 0; e < a.dk; e++, S += a.dv) {
        const float now = fmaf(decay, *S, pxg_to_f32(k[e]) * v);
        *S = now;
        o = fmaf(pxg_to_f32(q[e]), now, o);
    }
    out[f] = pxg_from_f32<T>(o);
}

bool bad_shape(const pxg_decay* a)
{
    return !a || a->struct_bytes != sizeof(pxg_decay) || a->dtype < PXG_DT_F32 || a->dtype > PXG_DT_F16 || a->batch < 0 ||
           a->steps < 0 || a->steps > INT32_MAX || a->heads < 1 || a->dk < 1 || a->dk > PXG_DECAY_MAX_WIDTH || a->dv < 1 ||
           a->dv > PXG_DECAY_MAX_WIDTH || a->batch > INT32_MAX / a->heads;
}

// a pointer may be missing only where nothing is read or written through it
bool bad_operands(const pxg_decay* a)
{
    const bool any = a->batch > 0 && a->steps > 0;
    return !a->log_decay || (any && (!a->q.data || !a->k.data || !a->v.data));
}

DecayShape shape_of(const pxg_decay* a)
{
    DecayShape s = {a->steps, (int)a->batch, a->heads, a->log_decay, a->lengths, a->lengths_are_64};
    return s;
}

}  // namespace

extern "C" int64_t pxg_decay_workspace_bytes(const pxg_decay* a, int32_t backward)
{
    if (bad_shape(a)) return PXG_E_INVALID;
    return backward ? a->batch * a->heads * (int64_t)sizeof(float) : 0;
}

extern "C" int pxg_decay_forward(const pxg_decay* a, void* stream)
{
    if (bad_shape(a) || bad_operands(a)) return PXG_E_INVALID;
    if (a->batch == 0) return PXG_OK;
    if (a->steps > 0 && !a->out) return PXG_E_INVALID;
    DecayRun r = {};
    r.x = a->q, r.y = a->k, r.z = a->v;
    r.init = a->initial_state, r.fin = a->final_state, r.init_e = a->dv, r.init_f = 1;
    r.out = a->out, r.E = a->dk, r.F = a->dv;
    return run(r, shape_of(a), a->dtype, (hipStream_t)stream);
}

extern "C" int pxg_decay_backward(const pxg_decay* a, void* stream)
{
    if (bad_shape(a) || bad_operands(a)) return PXG_E_INVALID;
    const bool any = a->batch > 0 && a->steps > 0;
    if (any && (!a->grad_q || !a->grad_k || !a->grad_v || !a->grad_out.data)) return PXG_E_INVALID;
    if (a->workspace_bytes < pxg_decay_workspace_bytes(a, 1) || (a->batch > 0 && !a->workspace)) return PXG_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    const DecayShape s = shape_of(a);
    int rc = PXG_OK;
    if (a->batch > 0) {
        DecayRun dq = {}, dk = {}, dv = {};
        dq.x = a->grad_out, dq.y = a->v, dq.z = a->k;
        dq.init = a->initial_state, dq.init_e = 1, dq.init_f = a->dv;
        dq.out = a->grad_q, dq.E = a->dv, dq.F = a->dk;
        if (a->grad_log_decay) dq.dot = a->q, dq.grad_fin = a->grad_final_state, dq.partial = (float*)a->workspace;
        dk.x = a->v, dk.y = a->grad_out, dk.z = a->q, dk.reverse = 1;
        dk.init = a->grad_final_state, dk.init_e = 1, dk.init_f = a->dv;
        dk.out = a->grad_k, dk.E = a->dv, dk.F = a->dk;
        dv.x = a->k, dv.y = a->q, dv.z = a->grad_out, dv.reverse = 1;
        dv.init = a->grad_final_state, dv.fin = a->grad_initial_state, dv.init_e = a->dv, dv.init_f = 1;
        dv.out = a->grad_v, dv.E = a->dk, dv.F = a->dv;
        rc = run(dq, s, a->dtype, st);
        if (rc == PXG_OK) rc = run(dk, s, a->dtype, st);
        if (rc == PXG_OK) rc = run(dv, s, a->dtype, st);
    }
    if (rc == PXG_OK && a->grad_log_decay) {
        k_decay_sum<<<a->heads, 256, 0, st>>>((const float*)a->workspace, a->batch, a->heads, a->grad_log_decay);
        if (hipGetLastError() != hipSuccess) rc = PXG_E_HIP;
    }
    return rc;
}

extern "C" int pxg_decay_step(const pxg_decay* a, void* stream)
{
    if (bad_shape(a) || a->steps != 1 || bad_operands(a)) return PXG_E_INVALID;
    if (a->batch == 0) return PXG_OK;
    if (!a->out || !a->final_state) return PXG_E_INVALID;
    const int blocks = (int)a->batch * a->heads;
    hipStream_t st = (hipStream_t)stream;
    switch (a->dtype) {
    case PXG_DT_F32: k_decay_step<float><<<blocks, 128, 0, st>>>(*a); break;
    case PXG_DT_BF16: k_decay_step<pxg_bf16><<<blocks, 128, 0, st>>>(*a); break;
    default: k_decay_step<pxg_f16><<<blocks, 128, 0, st>>>(*a);
    }
    return hipGetLastError() == hipSuccess ? PXG_OK : PXG_E_HIP;
}
