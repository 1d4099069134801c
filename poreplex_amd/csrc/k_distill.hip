// k_distill.hip -- learning from another network's answers: the largest logits of a teacher's rows, and the distillation loss of
// a student against them with its gradient.
//
// Teacher: p over the k listed classes and ONE class for all others, from values / temperature and rest (natural log units).
// Student: z = log sum_v exp(x_v / temperature); q_i = exp(x_i / temperature - z) of a listed class, q_r the sum over the others.
//   L = temperature^2 sum_i p_i (log p_i - log q_i),   dL/dx_v = temperature (q_v - p_v)            v listed
//                                                      dL/dx_v = temperature q_v (1 - p_r / q_r)    v unlisted
// The sum over the classes is taken in float32 against its own maximum; the k + 1 shares of a row are combined in float64, where
// the difference of nearly equal unlisted shares (few listed classes, a high temperature) keeps its digits.
#include "pxg_ops.h"

namespace {

constexpr int THREADS = 256;

// floats in the order of their values as unsigned integers: -0 as +0, NaN above everything
__device__ __forceinline__ uint32_t order_of(float x)
{
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float value_of(uint32_t key)
{
    return key == 0xffffffffu ? __uint_as_float(0x7fc00000u) : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// exp((x - base) / temperature): the factor log2(e) / temperature as a sum of two floats, so that the exponent of a far
// element is off by its own rounding only
struct Scale {
    float hi, lo;
};

__device__ __forceinline__ Scale scale_of(float temperature)
{
    const double c = 1.4426950408889634074 / (double)temperature;
    Scale s;
    s.hi = (float)c;
    s.lo = (float)(c - (double)s.hi);
    return s;
}

__device__ __forceinline__ float exp_from(float x, float base, Scale s)
{
    const float d = x - base;
    return __builtin_amdgcn_exp2f(fmaf(d, s.hi, d * s.lo));
}

template <typename V, typename F> __device__ __forceinline__ V block_reduce(V v, V* lds, F f)
{
    __syncthreads();
    lds[threadIdx.x] = v;
    __syncthreads();
    for (int w = THREADS / 2; w; w >>= 1) {
        if ((int)threadIdx.x < w) lds[threadIdx.x] = f(lds[threadIdx.x], lds[threadIdx.x + w]);
        __syncthreads();
    }
    return lds[0];
}

struct MaxOf { template <typename V> __device__ V operator()(V a, V b) const { return a > b ? a : b; } };
struct SumOf { template <typename V> __device__ V operator()(V a, V b) const { return a + b; } };

template <typename T>
__global__ __launch_bounds__(THREADS) void k_top(int64_t classes, const T* logits, int64_t row_stride, int k, float temperature,
                                                T* values, int32_t* indices, float* rest)
{
    __shared__ unsigned long long red[THREADS];
    __shared__ float redf[THREADS];
    const int64_t row = blockIdx.x;
    const T* x = logits + row * row_stride;
    // (order, classes - index) of the last one chosen: the next is the largest pair below it
    unsigned long long last = ~0ull;
    for (int i = 0; i < k; i++) {
        unsigned long long best = 0;
        for (int64_t v = threadIdx.x; v < classes; v += THREADS) {
            const unsigned long long key = (unsigned long long)order_of(pxg_to_f32(x[v])) << 32 | (uint32_t)(classes - v);
            if (key < last && key > best) best = key;
        }
        last = block_reduce(best, red, MaxOf());
        if (threadIdx.x == 0) {
            const int64_t v = classes - (int64_t)(last & 0xffffffffu);
            values[row * k + i] = x[v];
            indices[row * k + i] = (int32_t)v;
        }
    }
    uint32_t most = 0;
    for (int64_t v = threadIdx.x; v < classes; v += THREADS) {
        const unsigned long long key = (unsigned long long)order_of(pxg_to_f32(x[v])) << 32 | (uint32_t)(classes - v);
        if (key < last && (uint32_t)(key >> 32) > most) most = (uint32_t)(key >> 32);
    }
    most = (uint32_t)block_reduce((unsigned long long)most, red, MaxOf());
    const float base = value_of(most);
    const Scale s = scale_of(temperature);
    float sum = 0.f;
    for (int64_t v = threadIdx.x; v < classes; v += THREADS) {
        const float f = pxg_to_f32(x[v]);
        const unsigned long long key = (unsigned long long)order_of(f) << 32 | (uint32_t)(classes - v);
        if (key < last) sum += exp_from(f, base, s);
    }
    sum = block_reduce(sum, redf, SumOf());
    if (threadIdx.x == 0)
        rest[row] = most == 0 || base == -INFINITY ? -INFINITY : base == INFINITY ? INFINITY
                                                   : (float)((double)base / (double)temperature + log((double)sum));
}

__device__ __forceinline__ double number_at(const void* p, int64_t i, int dtype)
{
    return dtype == PXG_DT_F32 ? (double)((const float*)p)[i]
         : dtype == PXG_DT_BF16 ? (double)(float)((const pxg_bf16*)p)[i] : (double)(float)((const pxg_f16*)p)[i];
}

// A row's listed classes in shared memory: index (-1: empty place or an earlier place holds the class; then `share` is 0 and the
// first place has the sum) and the teacher's share.
struct Listed {
    int64_t index[PXG_TOP_MAX_K];
    double share[PXG_TOP_MAX_K], raw[PXG_TOP_MAX_K], rest_share;
    int bad, none;
};

__device__ void read_teacher(const pxg_distill& a, int64_t row, Listed& l, double* red)
{
    const int i = threadIdx.x;
    double t = -INFINITY;
    int64_t index = -1;
    if (i == 0) l.bad = 0;
    __syncthreads();
    if (i < a.k) {
        index = a.indices_are_64 ? ((const int64_t*)a.indices)[row * a.k + i] : ((const int32_t*)a.indices)[row * a.k + i];
        if (index < -1 || index >= a.classes) l.bad = 1, index = -1;
        else if (index >= 0) t = number_at(a.values, row * a.k + i, a.value_dtype) / (double)a.temperature;
        l.index[i] = index;
    }
    const double rest = a.rest ? (double)a.rest[row] : -INFINITY;
    double base = block_reduce(t, red, MaxOf());
    if (rest > base) base = rest;
    const double e = t == -INFINITY ? 0.0 : exp(t - base), er = rest == -INFINITY ? 0.0 : exp(rest - base);
    const double total = block_reduce(e, red, SumOf()) + er;
    if (i < a.k) l.raw[i] = total > 0.0 || total != total ? e / total : 0.0;
    if (i == 0) l.rest_share = total > 0.0 || total != total ? er / total : 0.0, l.none = total == 0.0;
    __syncthreads();
    // every thread takes every barrier: the first place of a class takes the shares of all of them
    double sum = 0.0;
    bool first = index >= 0;
    for (int j = 0; i < a.k && index >= 0 && j < a.k; j++)
        if (l.index[j] == index) {
            if (j < i) first = false;
            sum += l.raw[j];
        }
    __syncthreads();
    if (i < a.k) {
        l.share[i] = first ? sum : 0.0;
        if (!first) l.index[i] = -1;
    }
    __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(THREADS) void k_distill_forward(pxg_distill a)
{
    __shared__ Listed l;
    __shared__ double red[THREADS];
    __shared__ float redf[THREADS];
    const int64_t row = blockIdx.x;
    const double w = a.weight ? (double)a.weight[row] : 1.0;
    float* stats = a.stats + row * 4;
    if (w != 0.0) read_teacher(a, row, l, red);
    if (w == 0.0 || (l.none && !l.bad)) {
        if (threadIdx.x == 0) {
            a.row_loss[row] = 0.f;
            stats[0] = stats[1] = stats[2] = stats[3] = 0.f;
        }
        return;
    }
    const T* x = (const T*)a.logits + row * a.row_stride;
    const Scale s = scale_of(a.temperature);
    float most = -INFINITY, sum = 0.f;
    for (int64_t v = threadIdx.x; v < a.classes; v += THREADS) {
        bool listed = false;
        for (int i = 0; i < a.k; i++) listed |= l.index[i] == v;
        const float f = pxg_to_f32(x[v]);
        if (!listed && (f > most || f != f)) most = f;
    }
    const float base_u = block_reduce(most, redf, MaxOf());
    for (int64_t v = threadIdx.x; v < a.classes; v += THREADS) {
        bool listed = false;
        for (int i = 0; i < a.k; i++) listed |= l.index[i] == v;
        const float f = pxg_to_f32(x[v]);
        if (!listed && f != -INFINITY) sum += exp_from(f, base_u, s);
    }
    const double sum_u = block_reduce(sum, redf, SumOf());
    // the k + 1 shares
    const int i = threadIdx.x;
    const bool mine = i < a.k && l.index[i] >= 0;
    const double xi = mine ? (double)pxg_to_f32(x[l.index[i]]) : -INFINITY;
    double base = block_reduce(xi, red, MaxOf());
    if ((double)base_u > base) base = base_u;
    const double tau = a.temperature, u = sum_u == 0.0 ? 0.0 : sum_u * exp(((double)base_u - base) / tau);
    const double total = block_reduce(mine ? exp((xi - base) / tau) : 0.0, red, SumOf()) + u;
    const double log_total = log(total);
    double term = 0.0;
    if (mine && l.share[i] != 0.0) term = l.share[i] * (log(l.share[i]) - ((xi - base) / tau - log_total));
    double loss = block_reduce(term, red, SumOf());
    if (i == 0) {
        const double pr = l.rest_share;
        if (pr != 0.0) loss += pr * (log(pr) - (log(sum_u) + ((double)base_u - base) / tau - log_total));
        if (l.bad) loss = NAN;
        a.row_loss[row] = (float)(w * tau * tau * loss);
        stats[0] = base_u;
        stats[1] = sum_u == 0.0 ? 0.f : (float)((u / total - pr) / sum_u);
        stats[2] = (float)base;
        stats[3] = l.bad ? NAN : (float)total;
    }
}

__global__ __launch_bounds__(THREADS) void k_distill_sum(const float* row_loss, int64_t rows, int mean, float* loss)
{
    __shared__ double red[THREADS];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += THREADS) sum += (double)row_loss[i];
    sum = block_reduce(sum, red, SumOf());
    if (threadIdx.x == 0) *loss = (float)(mean ? sum / (double)rows : sum);
}

template <typename T>
__global__ __launch_bounds__(THREADS) void k_distill_backward(pxg_distill a)
{
    __shared__ Listed l;
    __shared__ double red[THREADS];
    const int64_t row = blockIdx.x;
    const double w = a.weight ? (double)a.weight[row] : 1.0;
    const float* stats = a.stats + row * 4;
    const float base_u = stats[0], c = stats[1], base = stats[2], total = stats[3];
    T* g = (T*)a.grad_logits + row * a.classes;
    if (w == 0.0 || total == 0.f) {
        for (int64_t v = threadIdx.x; v < a.classes; v += THREADS) g[v] = pxg_from_f32<T>(0.f);
        return;
    }
    read_teacher(a, row, l, red);
    const double tau = a.temperature;
    const double factor = w * tau * (double)a.grad_loss[a.grad_per_row ? row : 0] / (a.mean && !a.grad_per_row ? (double)a.rows : 1.0);
    const T* x = (const T*)a.logits + row * a.row_stride;
    const Scale s = scale_of(a.temperature);
    const float fc = l.bad ? NAN : (float)(factor * c);
    for (int64_t v = threadIdx.x; v < a.classes; v += THREADS) {
        int at = -1;
        for (int i = 0; i < a.k; i++)
            if (l.index[i] == v) at = i;
        const float f = pxg_to_f32(x[v]);
        float r;
        if (at < 0)
            r = f == -INFINITY ? 0.f * fc : exp_from(f, base_u, s) * fc;
        else
            r = (float)(factor * (exp(((double)f - (double)base) / tau) / (double)total - l.share[at]));
        g[v] = pxg_from_f32<T>(r);
    }
}

bool bad_call(const pxg_distill* a)
{
    return !a || a->struct_bytes != sizeof(pxg_distill) || a->dtype < PXG_DT_F32 || a->dtype > PXG_DT_F16 ||
           a->value_dtype < PXG_DT_F32 || a->value_dtype > PXG_DT_F16 || a->rows < 0 || a->rows > INT32_MAX || a->classes < 1 ||
           a->classes > INT32_MAX || a->k < 0 || a->k > PXG_TOP_MAX_K || !(a->temperature > 0.f) ||
           a->temperature > 3.0e38f || (a->rows > 0 && (!a->logits || !a->stats || (a->k > 0 && (!a->values || !a->indices))));
}

}  // namespace

extern "C" int pxg_top_logits(int32_t dtype, int64_t rows, int64_t classes, const void* logits, int64_t row_stride, int32_t k,
                              float temperature, void* values, int32_t* indices, float* rest, void* stream)
{
    if (dtype < PXG_DT_F32 || dtype > PXG_DT_F16 || rows < 0 || rows > INT32_MAX || classes < 1 || classes > INT32_MAX || k < 1 ||
        k > PXG_TOP_MAX_K || k > classes || !(temperature > 0.f) || temperature > 3.0e38f)
        return PXG_E_INVALID;
    if (rows == 0) return PXG_OK;
    if (!logits || !values || !indices || !rest) return PXG_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    const int n = (int)rows;
    switch (dtype) {
    case PXG_DT_F32:
        k_top<float><<<n, THREADS, 0, st>>>(classes, (const float*)logits, row_stride, k, temperature, (float*)values, indices, rest);
        break;
    case PXG_DT_BF16:
        k_top<pxg_bf16><<<n, THREADS, 0, st>>>(classes, (const pxg_bf16*)logits, row_stride, k, temperature, (pxg_bf16*)values,
                                               indices, rest);
        break;
    default:
        k_top<pxg_f16><<<n, THREADS, 0, st>>>(classes, (const pxg_f16*)logits, row_stride, k, temperature, (pxg_f16*)values,
                                              indices, rest);
    }
    return hipGetLastError() == hipSuccess ? PXG_OK : PXG_E_HIP;
}

extern "C" int pxg_distill_forward(const pxg_distill* a, void* stream)
{
    if (bad_call(a) || (a->rows > 0 && !a->row_loss)) return PXG_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    const int n = (int)a->rows;
    if (n) {
        switch (a->dtype) {
        case PXG_DT_F32: k_distill_forward<float><<<n, THREADS, 0, st>>>(*a); break;
        case PXG_DT_BF16: k_distill_forward<pxg_bf16><<<n, THREADS, 0, st>>>(*a); break;
        default: k_distill_forward<pxg_f16><<<n, THREADS, 0, st>>>(*a);
        }
        if (hipGetLastError() != hipSuccess) return PXG_E_HIP;
    }
    if (a->loss) {
        k_distill_sum<<<1, THREADS, 0, st>>>(a->row_loss, a->rows, a->mean, a->loss);
        if (hipGetLastError() != hipSuccess) return PXG_E_HIP;
    }
    return PXG_OK;
}

extern "C" int pxg_distill_backward(const pxg_distill* a, void* stream)
{
    if (bad_call(a)) return PXG_E_INVALID;
    if (a->rows == 0) return PXG_OK;
    if (!a->grad_loss || !a->grad_logits) return PXG_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    const int n = (int)a->rows;
    switch (a->dtype) {
    case PXG_DT_F32: k_distill_backward<float><<<n, THREADS, 0, st>>>(*a); break;
    case PXG_DT_BF16: k_distill_backward<pxg_bf16><<<n, THREADS, 0, st>>>(*a); break;
    default: k_distill_backward<pxg_f16><<<n, THREADS, 0, st>>>(*a);
    }
    return hipGetLastError() == hipSuccess ? PXG_OK : PXG_E_HIP;
}
