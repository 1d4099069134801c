// k_distill.hip -- learning from another network's answers: the largest logits of a teacher's rows, and the distillation loss of
// a student against them with its gradient.
//
// Teacher: p over the k listed classes and ONE class for all others, from values / temperature and rest (natural log units).
// Student: z = log sum_v exp(x_v / temperature); q_i = exp(x_i / temperature - z) of a listed class, q_r the sum over the others.
//   L = temperature^2 sum_i p_i (log p_i - log q_i),   dL/dx_v = temperature (q_v - p_v)            v listed
//                                                      dL/dx_v = temperature q_v (1 - p_r / q_r)    v unlisted
// The sum over the classes is taken in float32 against its own running maximum, in one pass over the row; the k + 1 shares of a
// row are combined in float64, where the difference of nearly equal unlisted shares (few listed classes, a high temperature)
// keeps its digits.
//
// All of them are bound by reading the logits once (and writing the gradient once): a row belongs to one wave, to four or to
// sixteen, by its length and the number of rows, and every lane reads 16 bytes at a time, four times before it computes.
//   4 096 x 32 768 bf16, k = 32:      loss 59 to 86 us (4.5 to 3.1 TB/s), gradient 89 (6.0)
//   1 023 x 131 071 f32, k = 100:     loss 117 to 153 (4.6 to 3.5), gradient 211 (5.1), where a copy of 2 GiB reaches 4.9
//   2 047 x 50 001 bf16, k = 64:      the largest logits 63 (3.3): exponentials and comparisons fill half of the time, loads are
//                                     waited for in the other
//   10 000 x 5 f32 and 256 x 5 f32:   3.6, and 9.6 + 2.3 + 4.4: launches and the latency of a few dependent reductions
#include "pxg_ops.h"
#include <type_traits>

namespace {

constexpr int AHEAD = 4;                      // 16-byte loads of a lane in flight

// ---- a group of G threads (one wave, or the whole workgroup) that shares a row ------------------------------------------------
template <int G> __device__ __forceinline__ void group_sync()
{
    if constexpr (G == 64) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

// rows in the order of the workgroups, which lie in a grid of two axes where one would hold 2^32 threads or more
template <int G> __device__ __forceinline__ int64_t row_of()
{
    const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    return G <= 64 ? block * (256 / G) + threadIdx.x / G : block;
}

struct MaxOf { template <typename V> __device__ V operator()(V a, V b) const { return a > b ? a : b; } };
struct SumOf { template <typename V> __device__ V operator()(V a, V b) const { return a + b; } };

// every thread gets the result; `lds` holds G / 64 values and may be used again at once
template <int G, typename V, typename F> __device__ __forceinline__ V group_reduce(V v, V* lds, F f)
{
#pragma unroll
    for (int m = 32; m; m >>= 1) v = f(v, __shfl_xor(v, m));
    if constexpr (G > 64) {
        __syncthreads();
        if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < G / 64; w++) v = f(v, lds[w]);
    }
    return v;
}

// ---- numbers --------------------------------------------------------------------------------------------------------------------
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
// element is off by its own rounding only.  Of half-precision rows one float is enough: they are off by more themselves.  Both
// parts are above 0: x may be -inf.
struct Scale {
    float hi, lo;
};

template <typename T> __device__ __forceinline__ Scale scale_of(float temperature)
{
    const double c = 1.4426950408889634074 / (double)temperature;
    Scale s = {(float)c, 0.f};
    if (sizeof(T) == 4) {
        if ((double)s.hi >= c) s.hi = __uint_as_float(__float_as_uint(s.hi) - 1);
        s.lo = fmaxf((float)(c - (double)s.hi), 0x1p-149f);       // (0 from temperatures of 1e29 or so on)
    }
    return s;
}

template <typename T> __device__ __forceinline__ float exp_from(float x, float base, Scale s)
{
    const float d = x - base;
    return __builtin_amdgcn_exp2f(sizeof(T) == 2 ? d * s.hi : fmaf(d, s.hi, d * s.lo));
}

// the larger one, or NaN if either is
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A thread's sum of exponentials against the largest of them so far.  (NaN among them: the sum is NaN.)
template <typename T> struct RunningSum {
    float base = -3.402823466e38f, sum = 0.f;

    __device__ __forceinline__ void raise(float most, Scale s)
    {
        if (most > base) sum *= exp_from<T>(base, most, s), base = most;
    }
    template <int N> __device__ __forceinline__ void add(const float (&v)[N], float most, Scale s)
    {
        raise(most, s);
#pragma unroll
        for (int e = 0; e < N; e++) sum += exp_from<T>(v[e], base, s);
    }
};

// 16 bytes of a row, which may begin anywhere; -inf behind its end
template <typename T> struct Unit {
    static constexpr int n = 16 / sizeof(T);
    T v[n];
};

template <typename T> __device__ __forceinline__ Unit<T> load_whole(const T* x, int64_t unit)
{
    Unit<T> u;
    __builtin_memcpy(&u, x + unit * Unit<T>::n, sizeof u);
    return u;
}

template <typename T> __device__ __forceinline__ Unit<T> load_unit(const T* x, int64_t unit, int64_t classes)
{
    constexpr int n = Unit<T>::n;
    if ((unit + 1) * n <= classes) return load_whole(x, unit);
    Unit<T> u;
#pragma unroll
    for (int e = 0; e < n; e++) u.v[e] = unit * n + e < classes ? x[unit * n + e] : (T)-INFINITY;
    return u;
}

// Calls f(units, first unit, step) for this thread's units of a row, AHEAD at a time and step apart, as long as all of them are
// whole (loads without a branch between them, so that all are on their way at once), then g(unit, its number) for those that are
// left, the last of which may be cut.
template <int G, typename T, typename F, typename L>
__device__ __forceinline__ void each_units(const T* x, int64_t classes, int t, F f, L g)
{
    constexpr int n = Unit<T>::n;
    const int64_t whole = classes / n, units = (classes + n - 1) / n;
    int64_t i = t;
    for (; i - t + G * AHEAD <= whole; i += G * AHEAD) {
        Unit<T> u[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) u[a] = load_whole(x, i + a * G);
        f(u, i);
    }
    for (; i < units; i += G) g(load_unit(x, i, classes), i);
}

// calls f(first class, floats) for the units of a row that are this thread's
template <int G, typename T, typename F> __device__ __forceinline__ void each_unit(const T* x, int64_t classes, int t, F f)
{
    constexpr int n = Unit<T>::n;
    const auto one = [&](const Unit<T>& u, int64_t unit) {
        float v[n];
#pragma unroll
        for (int e = 0; e < n; e++) v[e] = pxg_to_f32(u.v[e]);
        f(unit * n, v);
    };
    each_units<G>(x, classes, t, [&](const Unit<T>* u, int64_t unit) {
#pragma unroll
        for (int a = 0; a < AHEAD; a++) one(u[a], unit + a * G);
    }, one);
}

// ---- the largest logits ---------------------------------------------------------------------------------------------------------
// One pass.  Each of the threads knows the largest of its own elements so far; the k-th largest of these 64 to 256 maxima is a bound
// that at least k elements reach, and only so many more of evenly spread ones (k = 128 of 256: 177).  The bound is raised as the row
// goes by, at the first tiles of 4 units a thread and then ever more rarely.  A unit below the bound is added to the sum of the rest
// at once; the number of any other is noted, some hundred of them in a row of any length.  These are looked at again with the last
// bound: what reaches it is ranked by counting, and all but the first k join the sum.  Rows with more than these lists hold (plateaus
// of equal values, rows that only ascend, rows full of NaN) take their bound by bisection instead, reading the row again and again.
// Masked rows: what is -inf or the type's lowest number is below every bound.  While fewer than k threads have met more than that,
// the bound is looked for at every tile; where the row's other numbers do not fill the list, its first k classes have as many of the
// masked ones as it needs (in rows that hold both kinds of them perhaps not: bisection).  2 047 x 50 001 bf16, k = 64, all but 40 or
// 1 000 of the classes masked, or half: 46 to 56 us (57 of evenly spread ones; by bisection 2 000).
//   2 047 x 50 001 bf16, k = 64: reading the row a second time for the sum, from whatever cache has it, took 101 us, keeping it in
//   registers (which leaves room for few workgroups) 222, collecting elements instead of units' numbers 88.
template <int G> struct alignas(16) TopShared {
    static constexpr int parts = G < 256 ? G : 256, notes = G == 64 ? 256 : 2048;       // more than evenly spread rows need
    static constexpr int room = G == 64 ? 256 : 1024;
    unsigned long long cand[room];              // (order, ~class): no two are equal
    uint32_t most[G];
    double redd[G / 64];
    long long redi[G / 64];
    float redf[G / 64];
    int red[G / 64];
    uint32_t note[notes];
    int count, noted;
    uint32_t bound;
};

template <int G, typename T>
__global__ __launch_bounds__(G == 64 ? 256 : G)
void k_top(int64_t rows, int64_t classes, const T* logits, int64_t row_stride, int k, float temperature, T* values, int32_t* indices,
           float* rest)
{
    constexpr int GROUPS = G == 64 ? 4 : 1, n = Unit<T>::n, PARTS = TopShared<G>::parts, EACH = G / PARTS, CAND = TopShared<G>::room;
    __shared__ TopShared<G> shared[GROUPS];
    const int64_t row = row_of<G>();
    if (row >= rows) return;                    // a whole wave, or nobody
    TopShared<G>& s = shared[G == 64 ? threadIdx.x / 64 : 0];
    const int t = threadIdx.x % G;
    const T* x = logits + row * row_stride;
    const Scale scale = scale_of<T>(temperature);
    if (t == 0) s.count = s.noted = 0;

    constexpr float LOWEST = sizeof(T) == 4 ? -3.402823466e38f : std::is_same<T, pxg_f16>::value ? -65504.f : -3.3895313892515355e38f;
    const uint32_t MASKED = order_of(LOWEST);
    float largest = -INFINITY, bound = 0.f;
    const auto search = [&](auto parts) {       // the k-th largest of `most`: one wave, bit by bit; one that is a little low will do
        constexpr int P = decltype(parts)::value;
        if (t < 64) {
            uint32_t o[P / 64];
#pragma unroll
            for (int j = 0; j < P / 64; j++) o[j] = s.most[t + 64 * j];
            uint32_t key = 0;
            for (int bit = 31; bit >= 14; bit--) {
                const uint32_t more = key | 1u << bit;
                int c = 0;
#pragma unroll
                for (int j = 0; j < P / 64; j++) c += __popcll(__ballot(o[j] >= more));
                if (c >= k) key = more;
            }
            if (t == 0) s.bound = key;
        }
        group_sync<G>();
    };
    const auto raise_bound = [&] {              // the k-th largest of the threads' maxima
        float m = largest;
#pragma unroll
        for (int w = 1; w < EACH; w *= 2) m = larger(m, __shfl_xor(m, w));
        group_sync<G>();
        if (t % EACH == 0) s.most[t / EACH] = order_of(m);
        group_sync<G>();
        search(std::integral_constant<int, PARTS>());
        uint32_t key = s.bound;
        if (EACH > 1 && key <= MASKED) {         // a few hundred numbers in a row lie with a few threads: each for itself
            group_sync<G>();
            s.most[t] = order_of(largest);
            group_sync<G>();
            search(std::integral_constant<int, G>());
            key = s.bound;
        }
        bound = value_of(key > MASKED ? key : MASKED + 1);
    };
    RunningSum<T> sum;
    const auto take = [&](const float (&v)[n], int64_t unit) {
        float here = v[0];
#pragma unroll
        for (int e = 1; e < n; e++) here = larger(here, v[e]);
        if (here < bound) {                     // nearly every unit
            sum.add(v, here, scale);
        } else if (unit * n < classes) {
            const int at = atomicAdd(&s.noted, 1);
            if (at < TopShared<G>::notes) s.note[at] = (uint32_t)unit;
        }
    };
    if (classes < (int64_t)G * n) {             // one element after the other: min(G, classes) threads have some, k at least
        for (int64_t v = t; v < classes; v += G) largest = larger(largest, pxg_to_f32(x[v]));
        raise_bound();
        each_unit<G>(x, classes, t, [&](int64_t first, const float (&v)[n]) { take(v, first / n); });
    } else {
        constexpr int64_t TILE = G * AHEAD;
        const int64_t whole = classes / n, units = (classes + n - 1) / n;
        int tile = 0, next = 0;
        int64_t i = t;
        const auto numbers = [&](const Unit<T>& u, float (&v)[n]) {
#pragma unroll
            for (int e = 0; e < n; e++) v[e] = pxg_to_f32(u.v[e]);
        };
        for (; i - t < units; i += TILE) {
            Unit<T> u[AHEAD];
            if (i - t + TILE <= whole) {
#pragma unroll
                for (int a = 0; a < AHEAD; a++) u[a] = load_whole(x, i + a * G);
            } else {
#pragma unroll
                for (int a = 0; a < AHEAD; a++) u[a] = load_unit(x, i + a * G, classes);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; a++) {
                float v[n];
                numbers(u[a], v);
#pragma unroll
                for (int e = 0; e < n; e++) largest = larger(largest, v[e]);
            }
            if (tile == next || s.bound <= MASKED) {          // tiles 0, 1, 2, 3, 4, 6, 9, 13, ...
                if (tile == next) next += next / 2 + (next < 2 ? 1 : 0);
                raise_bound();
            }
            tile++;
#pragma unroll
            for (int a = 0; a < AHEAD; a++) {
                float v[n];
                numbers(u[a], v);
                take(v, i + a * G);
            }
        }
    }
    if (classes >= (int64_t)G * n) raise_bound();
    group_sync<G>();
    const int noted = s.noted;
    bool listed = noted <= TopShared<G>::notes;
    float most = -INFINITY;                     // of what is below the bound in the noted units
    if (listed)
        for (int i = t; i < noted; i += G) {
            const int64_t unit = s.note[i];
            const Unit<T> u = load_unit(x, unit, classes);
#pragma unroll
            for (int e = 0; e < n; e++) {
                const float v = pxg_to_f32(u.v[e]);
                if (v < bound) {
                    most = fmaxf(most, v);
                } else if (unit * n + e < classes) {
                    const int at = atomicAdd(&s.count, 1);
                    if (at < CAND) s.cand[at] = (unsigned long long)order_of(v) << 32 | (uint32_t)~(uint32_t)(unit * n + e);
                }
            }
        }
    group_sync<G>();
    int found = listed ? s.count : CAND + 1;
    double listed_lowest = 0.0;                 // of the sum so far
    if (found < k) {                            // all that was summed is masked: the first ones fill the list
        const bool lowest = group_reduce<G>((int)(sum.sum > 0.f || most > -INFINITY), s.red, MaxOf());
        const float fill = lowest ? LOWEST : -INFINITY;
        const int need = k - found;
        group_sync<G>();
        for (int i = t; i < k; i += G) {
            if (pxg_to_f32(x[i]) != fill) continue;
            int before = 0;
            for (int j = 0; j < i; j++) before += pxg_to_f32(x[j]) == fill;
            if (before < need) s.cand[atomicAdd(&s.count, 1)] = (unsigned long long)order_of(fill) << 32 | (uint32_t)~(uint32_t)i;
        }
        group_sync<G>();
        found = s.count == k ? k : CAND + 1;
        listed_lowest = lowest ? need : 0;
    }
    bool no_number = false;                     // among the rest (bisection only: otherwise it is a candidate)
    if (found > CAND) {
        // the largest key that k elements reach, bit by bit; then the smallest class below which enough of the ties lie
        const auto count = [&](auto is) {
            int c = 0;
            each_unit<G>(x, classes, t, [&](int64_t first, const float (&v)[n]) {
#pragma unroll
                for (int e = 0; e < n; e++)
                    if (first + e < classes && is(order_of(v[e]), (uint32_t)(first + e))) c++;
            });
            return group_reduce<G>(c, s.red, SumOf());
        };
        uint32_t key = 0;
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t more = key | 1u << bit;
            if (count([&](uint32_t o, uint32_t) { return o >= more; }) >= k) key = more;
        }
        const int need = k - count([&](uint32_t o, uint32_t) { return o > key; });
        uint32_t low = 0, high = (uint32_t)classes;                 // count(low) < need <= count(high)
        while (high - low > 1) {
            const uint32_t mid = low + (high - low) / 2;
            if (count([&](uint32_t o, uint32_t c) { return o == key && c < mid; }) >= need) high = mid;
            else low = mid;
        }
        found = k, listed = false, most = -INFINITY, listed_lowest = 0.0;
        if (t == 0) s.count = 0;
        group_sync<G>();
        sum = RunningSum<T>();
        bool strange = false;
        each_unit<G>(x, classes, t, [&](int64_t first, const float (&v)[n]) {
            float left[n], most = -INFINITY;
#pragma unroll
            for (int e = 0; e < n; e++) {
                const uint32_t o = order_of(v[e]);
                const bool chosen = first + e < classes && (o > key || (o == key && (uint32_t)(first + e) < high));
                if (chosen) s.cand[atomicAdd(&s.count, 1)] = (unsigned long long)o << 32 | (uint32_t)~(uint32_t)(first + e);
                left[e] = chosen ? -INFINITY : v[e];
                most = fmaxf(most, left[e]), strange |= left[e] != left[e];
            }
            sum.add(left, most, scale);
        });
        no_number = group_reduce<G>((int)strange, s.red, MaxOf());
        group_sync<G>();
    }
    // What is noted comes in another order in every run: its sum is taken in whole multiples of 2^-44 of the largest term, which no
    // order changes.
    const auto whole_part = [](double part) { return (long long)rint(part * 0x1p44); };
    const float base = group_reduce<G>(fmaxf(sum.base, most), s.redf, MaxOf());
    double below = group_reduce<G>(sum.sum == 0.f ? 0.0 : (double)sum.sum * (double)exp_from<T>(sum.base, base, scale), s.redd, SumOf());
    if (listed) {
        long long parts = 0;
        for (int i = t; i < noted; i += G) {
            const Unit<T> u = load_unit(x, s.note[i], classes);
#pragma unroll
            for (int e = 0; e < n; e++) {
                const float v = pxg_to_f32(u.v[e]);
                if (v < bound) parts += whole_part(exp_from<T>(v, base, scale));
            }
        }
        below += (double)group_reduce<G>(parts, s.redi, SumOf()) * 0x1p-44;
    }
    below -= listed_lowest;                     // (each counts 1: nothing larger is in the sum)
    // rank the candidates; the first k are the answer, the rest join the sum against the largest of them
    long long extra = 0;
    const bool left = found > k;
    int rank[(CAND + G - 1) / G];
#pragma unroll
    for (int a = 0; a < (CAND + G - 1) / G; a++) {
        const int i = t + a * G;
        int ahead = 0;
        if (i < found) {
            const unsigned long long key = s.cand[i];
#pragma unroll 4
            for (int j = 0; j < found; j++) ahead += s.cand[j] > key;
            if (ahead < k) {
                const int64_t at = (int64_t)(uint32_t)~(uint32_t)key;
                values[row * k + ahead] = x[at];
                indices[row * k + ahead] = (int32_t)at;
            } else if (ahead == k) {
                s.bound = (uint32_t)(key >> 32);
            }
        }
        rank[a] = ahead;
    }
    float top = base;
    if (left) {
        group_sync<G>();
        top = value_of(s.bound);
        if (__builtin_isfinite(top)) {
#pragma unroll
            for (int a = 0; a < (CAND + G - 1) / G; a++)
                if (t + a * G < found && rank[a] >= k)
                    extra += whole_part(exp(((double)value_of((uint32_t)(s.cand[t + a * G] >> 32)) - (double)top) / (double)temperature));
        }
        extra = group_reduce<G>(extra, s.redi, SumOf());
    }
    if (t == 0) {
        double r;
        if (left && !__builtin_isfinite(top)) r = top;                     // -inf: so is all the rest
        else if (left) r = (double)top / temperature + log((double)extra * 0x1p-44 + (below > 0.0 ? below * exp(((double)base - top) / temperature) : 0.0));
        else if (no_number) r = NAN;
        else if (base == INFINITY) r = INFINITY;
        else r = below > 0.0 ? (double)base / temperature + log(below) : -INFINITY;
        rest[row] = (float)r;
    }
}

// Rows of up to 64 classes: a lane for each of them, so that nothing is noted or searched for; an element's place is the number of
// those ahead of it.  10 000 x 5 f32, k = 3: 3.6 us, with a wave for a row 8.5.
template <int G, typename T>
__global__ __launch_bounds__(256)
void k_top_narrow(int64_t rows, int64_t classes, const T* logits, int64_t row_stride, int k, float temperature, T* values,
                  int32_t* indices, float* rest)
{
    const int64_t row = row_of<G>();
    const int lane = threadIdx.x % G;
    const bool there = row < rows, in = there && lane < classes;
    const T raw = in ? logits[row * row_stride + lane] : (T)0.f;
    const float v = pxg_to_f32(raw);
    const uint32_t o = in ? order_of(v) : 0;                      // below every number's
    int ahead = 0;
#pragma unroll
    for (int j = 0; j < G; j++) {
        const uint32_t other = __shfl(o, j, G);
        ahead += other > o || (other == o && j < lane);
    }
    const bool left = in && ahead >= k;
    if (in && !left) values[row * k + ahead] = raw, indices[row * k + ahead] = lane;
    float top = left ? v : -INFINITY;
#pragma unroll
    for (int m = G / 2; m; m >>= 1) top = larger(top, __shfl_xor(top, m));
    const bool finite = __builtin_isfinite(top);
    float sum = left && finite ? exp_from<float>(v, top, scale_of<float>(temperature)) : 0.f;
#pragma unroll
    for (int m = G / 2; m; m >>= 1) sum += __shfl_xor(sum, m);
    // (no number or +inf among the rest; -inf: nothing else)
    if (there && lane == 0) rest[row] = finite ? (float)((double)top / temperature + log((double)sum)) : top;
}

// ---- the loss -------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ double number_at(const void* p, int64_t i, int dtype)
{
    return dtype == PXG_DT_F32 ? (double)((const float*)p)[i]
         : dtype == PXG_DT_BF16 ? (double)(float)((const pxg_bf16*)p)[i] : (double)(float)((const pxg_f16*)p)[i];
}

// Which classes of a row are listed: one bit for each 16-byte unit of the row (more units share a bit in rows of more than
// 32 768 of them), and a table of the units that hold listed classes.
template <int G> struct Marks {
    static constexpr int words = G == 64 ? 64 : 1024, slots = 256;
    uint32_t filter[words];
    int32_t unit[slots];
    uint32_t mask[slots];

    __device__ void clear(int t)
    {
        for (int i = t; i < words; i += G) filter[i] = 0;
        for (int i = t; i < slots; i += G) unit[i] = -1, mask[i] = 0;
    }
    static __device__ int slot_of(int32_t u) { return (int)((uint32_t)u * 2654435761u >> 24); }
    __device__ void add(int64_t index, int n)                     // at most PXG_TOP_MAX_K of them: there is always a free slot
    {
        const int32_t u = (int32_t)(index / n);
        atomicOr(&filter[(u >> 5) & (words - 1)], 1u << (u & 31));
        for (int s = slot_of(u);; s = (s + 1) & (slots - 1)) {
            const int32_t was = atomicCAS(&unit[s], -1, u);
            if (was == -1 || was == u) {
                atomicOr(&mask[s], 1u << (index % n));
                return;
            }
        }
    }
    __device__ __forceinline__ uint32_t of(int32_t u) const
    {
        if (!(filter[(u >> 5) & (words - 1)] >> (u & 31) & 1)) return 0;
        for (int s = slot_of(u);; s = (s + 1) & (slots - 1)) {
            const int32_t is = unit[s];
            if (is == u) return mask[s];
            if (is < 0) return 0;
        }
    }
};

template <int G> struct LossShared {
    Marks<G> marks;
    int32_t index[PXG_TOP_MAX_K];               // -1: an empty place, or an earlier one holds the class
    double share[PXG_TOP_MAX_K];
    double redd[G / 64];
    float redf[G / 64];
};

// `stats` of a row: the unlisted classes' maximum, the factor of their exponentials in the gradient, whether the row counts (0: no,
// 1: yes, NaN: it names what is no class), unused, then q - p of each place (+inf: no class's first place)
constexpr int STATS = 4;

// The classes are everybody's; what there is one of for each listed class, and every sum over those, is the first wave's, which
// needs no barrier for it (with the whole workgroup at eight such sums a row of 2 000 classes took twice as long).
template <int G, typename T>
__global__ __launch_bounds__(G == 64 ? 256 : G) void k_distill_forward(const pxg_distill a)
{
    constexpr int GROUPS = G == 64 ? 4 : 1, n = Unit<T>::n, PLACES = PXG_TOP_MAX_K / 64;
    __shared__ LossShared<G> shared[GROUPS];
    const int64_t row = row_of<G>();
    if (row >= a.rows) return;
    LossShared<G>& s = shared[G == 64 ? threadIdx.x / 64 : 0];
    const int t = threadIdx.x % G, k = a.k;
    float* stats = a.stats + row * (STATS + k);
    const double w = a.weight ? (double)a.weight[row] : 1.0, tau = a.temperature;
    const T* x = (const T*)a.logits + row * a.row_stride;
    if (w == 0.0) {                                               // the whole group
        if (t == 0) stats[2] = 0.f, a.row_loss[row] = 0.f;
        return;
    }
    s.marks.clear(t);
    group_sync<G>();
    double value[PLACES], xi[PLACES], rest = -INFINITY;
    int32_t index[PLACES];
    bool bad = false;
    if (t < 64) {
        rest = a.rest ? (double)a.rest[row] : -INFINITY;
#pragma unroll
        for (int p = 0; p < PLACES; p++) {
            const int i = t + p * 64;
            value[p] = xi[p] = -INFINITY, index[p] = -1;
            if (i >= k) continue;
            const int64_t at = row * k + i, is = a.indices_are_64 ? ((const int64_t*)a.indices)[at] : ((const int32_t*)a.indices)[at];
            if (is < -1 || is >= a.classes) bad = true;
            else index[p] = (int32_t)is;
            s.index[i] = index[p];
            if (index[p] < 0) continue;
            s.marks.add(index[p], n);
            value[p] = number_at(a.values, at, a.value_dtype) / tau;
            xi[p] = (double)pxg_to_f32(x[index[p]]);
        }
    }
    group_sync<G>();

    // the student's unlisted classes: running maximum and sum
    const Scale scale = scale_of<T>(a.temperature);
    RunningSum<T> sum_u;
    const auto numbers = [&](const Unit<T>& u, int64_t unit, float* v) {
        const uint32_t mask = s.marks.of((int32_t)unit);
#pragma unroll
        for (int e = 0; e < n; e++) v[e] = pxg_to_f32(u.v[e]);
        if (mask)
#pragma unroll
            for (int e = 0; e < n; e++)
                if (mask >> e & 1) v[e] = -INFINITY;
    };
    each_units<G>(x, a.classes, t, [&](const Unit<T>* u, int64_t unit) {
        float v[AHEAD][n], next = -INFINITY;
#pragma unroll
        for (int b = 0; b < AHEAD; b++) {
            numbers(u[b], unit + b * G, v[b]);
#pragma unroll
            for (int e = 0; e < n; e++) next = larger(next, v[b][e]);
        }
        sum_u.raise(next, scale);
#pragma unroll
        for (int b = 0; b < AHEAD; b++)
#pragma unroll
            for (int e = 0; e < n; e++) sum_u.sum += exp_from<T>(v[b][e], sum_u.base, scale);
    }, [&](const Unit<T>& u, int64_t unit) {
        float v[n], next = -INFINITY;
        numbers(u, unit, v);
#pragma unroll
        for (int e = 0; e < n; e++) next = larger(next, v[e]);
        sum_u.add(v, next, scale);
    });
    // (what has none keeps its sum of 0 whatever its exponent says)
    float all_u = group_reduce<64>(sum_u.base, s.redf, MaxOf());
    double unlisted = group_reduce<64>(sum_u.sum == 0.f ? 0.0 : (double)sum_u.sum * (double)exp_from<T>(sum_u.base, all_u, scale),
                                       s.redd, SumOf());
    if constexpr (G > 64) {
        if (t % 64 == 0) s.redf[t / 64] = all_u, s.redd[t / 64] = unlisted;
        __syncthreads();
        if (t >= 64) return;
        const float most = t < G / 64 ? s.redf[t] : -INFINITY;
        const double sum = t < G / 64 ? s.redd[t] : 0.0;
        all_u = group_reduce<64>(most, s.redf, MaxOf());
        unlisted = group_reduce<64>(sum == 0.0 ? 0.0 : sum * (double)exp_from<T>(most, all_u, scale), s.redd, SumOf());
    }

    // the first wave.  The teacher's shares
    bad = __any(bad);
    double most = -INFINITY, sum = 0.0;
#pragma unroll
    for (int p = 0; p < PLACES; p++) most = value[p] > most ? value[p] : most;
    double top = group_reduce<64>(most, s.redd, MaxOf());
    top = rest > top ? rest : top;
#pragma unroll
    for (int p = 0; p < PLACES; p++) {
        value[p] = value[p] == -INFINITY ? 0.0 : exp(value[p] - top);
        sum += value[p];
    }
    const double rest_exp = rest == -INFINITY ? 0.0 : exp(rest - top);
    const double total_p = group_reduce<64>(sum, s.redd, SumOf()) + rest_exp;
    if (total_p == 0.0 && !bad) {
        if (t == 0) stats[2] = 0.f, a.row_loss[row] = 0.f;
        return;
    }
    const double p_rest = rest_exp / total_p;
#pragma unroll
    for (int p = 0; p < PLACES; p++)
        if (t + p * 64 < k) s.share[t + p * 64] = value[p] / total_p;
    group_sync<64>();
    // a class that is listed more than once: its first place takes all its shares
    double share[PLACES];
    bool first[PLACES];
#pragma unroll
    for (int p = 0; p < PLACES; p++) {
        const int i = t + p * 64;
        share[p] = 0.0, first[p] = index[p] >= 0;
        if (index[p] >= 0)
            for (int j = 0; j < k; j++)
                if (s.index[j] == index[p]) {
                    if (j < i) first[p] = false;
                    share[p] += s.share[j];
                }
    }

    // the k + 1 shares
    double base = -INFINITY;
#pragma unroll
    for (int p = 0; p < PLACES; p++) {
        if (!first[p]) xi[p] = -INFINITY;
        base = xi[p] > base ? xi[p] : base;
    }
    base = group_reduce<64>(base, s.redd, MaxOf());
    if (unlisted != 0.0 && !((double)all_u <= base)) base = all_u;
    double listed = 0.0;
#pragma unroll
    for (int p = 0; p < PLACES; p++) {
        xi[p] = (xi[p] - base) / tau;
        listed += first[p] ? exp(xi[p]) : 0.0;
    }
    const double far_u = ((double)all_u - base) / tau;
    const double u = unlisted == 0.0 ? 0.0 : unlisted * exp(far_u);
    const double total = group_reduce<64>(listed, s.redd, SumOf()) + u, log_total = log(total);
    double term = 0.0;
#pragma unroll
    for (int p = 0; p < PLACES; p++) {
        const int i = t + p * 64;
        if (first[p] && share[p] != 0.0) term += share[p] * (log(share[p]) - (xi[p] - log_total));
        if (i < k) stats[STATS + i] = first[p] ? (float)(exp(xi[p]) / total - share[p]) : INFINITY;
    }
    double loss = group_reduce<64>(term, s.redd, SumOf());
    if (t == 0) {
        if (p_rest != 0.0) loss += p_rest * (log(p_rest) - (log(unlisted) + far_u - log_total));
        if (bad) loss = NAN;
        a.row_loss[row] = (float)(w * tau * tau * loss);
        stats[0] = all_u;
        stats[1] = unlisted == 0.0 ? 0.f : (float)((u / total - p_rest) / unlisted);
        stats[2] = bad ? NAN : 1.f;
        stats[3] = 0.f;
    }
}

// One workgroup, in a fixed order, eight loads ahead of the additions (4 096 rows 3.9 us, one after the other 5.6; 16 384 rows 6.2).
__global__ __launch_bounds__(1024) void k_distill_sum(const float* row_loss, int64_t rows, int mean, float* loss)
{
    constexpr int AT_ONCE = 8;
    __shared__ double red[16];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += 1024 * AT_ONCE) {
        float v[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) v[j] = i + j * 1024 < rows ? row_loss[i + j * 1024] : 0.f;
#pragma unroll
        for (int j = 0; j < AT_ONCE; j++) sum += (double)v[j];
    }
    sum = group_reduce<1024>(sum, red, SumOf());
    if (threadIdx.x == 0) *loss = (float)(mean ? sum / (double)rows : sum);
}

template <int G, typename T>
__global__ __launch_bounds__(G == 64 ? 256 : G) void k_distill_backward(const pxg_distill a)
{
    constexpr int GROUPS = G == 64 ? 4 : 1, n = Unit<T>::n;
    __shared__ Marks<G> shared[GROUPS];
    const int64_t row = row_of<G>();
    if (row >= a.rows) return;
    Marks<G>& marks = shared[G == 64 ? threadIdx.x / 64 : 0];
    const int t = threadIdx.x % G, k = a.k;
    const float* stats = a.stats + row * (STATS + k);
    const float counts = stats[2], base_u = stats[0], c = stats[1];
    const T* x = (const T*)a.logits + row * a.row_stride;
    T* g = (T*)a.grad_logits + row * a.classes;
    const double w = a.weight ? (double)a.weight[row] : 1.0;
    const double factor = counts == 0.f ? 0.0
        : counts * w * (double)a.temperature * (double)a.grad_loss[a.grad_per_row ? row : 0] / (a.mean && !a.grad_per_row ? (double)a.rows : 1.0);
    const float fc = counts == 0.f ? 0.f : (float)(factor * c);
    const Scale scale = scale_of<T>(a.temperature);
    if (counts != 0.f) {
        marks.clear(t);
        group_sync<G>();
        for (int i = t; i < k; i += G) {
            const float d = stats[STATS + i];
            if (d == INFINITY) continue;
            const int64_t at = row * k + i, index = a.indices_are_64 ? ((const int64_t*)a.indices)[at] : ((const int32_t*)a.indices)[at];
            if (index < 0 || index >= a.classes) continue;        // not what the forward pass saw: no place in this row
            marks.add(index, n);
            g[index] = pxg_from_f32<T>((float)(factor * (double)d));
        }
        group_sync<G>();
    }
    if (counts == 0.f) {
        const int64_t units = (a.classes + n - 1) / n;
        Unit<T> zero;
#pragma unroll
        for (int e = 0; e < n; e++) zero.v[e] = pxg_from_f32<T>(0.f);
        for (int64_t i = t; i < units; i += G) {
            if ((i + 1) * n <= a.classes) __builtin_memcpy(g + i * n, &zero, sizeof zero);
            else
                for (int64_t v = i * n; v < a.classes; v++) g[v] = pxg_from_f32<T>(0.f);
        }
        return;
    }
    const auto one = [&](const Unit<T>& u, int64_t unit) {
        Unit<T> r;
#pragma unroll
        for (int e = 0; e < n; e++) r.v[e] = pxg_from_f32<T>(exp_from<T>(pxg_to_f32(u.v[e]), base_u, scale) * fc);
        const uint32_t mask = marks.of((int32_t)unit);
        if (mask == 0 && (unit + 1) * n <= a.classes) {
            __builtin_memcpy(g + unit * n, &r, sizeof r);
        } else {
#pragma unroll
            for (int e = 0; e < n; e++)
                if (!(mask >> e & 1) && unit * n + e < a.classes) g[unit * n + e] = r.v[e];
        }
    };
    each_units<G>(x, a.classes, t, [&](const Unit<T>* u, int64_t unit) {
#pragma unroll
        for (int b = 0; b < AHEAD; b++) one(u[b], unit + b * G);
    }, one);
}

// The threads that share a row: a wave for short ones, a workgroup of four waves, sixteen where there are too few long rows to
// fill the card with less (one row of 131 071 f32, loss and gradient: 70 us with four, 48 with sixteen; 400 rows: 148 and 154).
// Many rows of up to 16 KB are better off with a wave each, too (16 384 rows, loss and gradient with one wave / four: 1 200 f16 79 /
// 112 us, 5 000 f16 150 / 170, 8 000 f16 217 / 218, 5 000 f32 258 / 230; 2 048 x 3 305 f16 29 / 27, 512 rows 23 / 18).
int threads_of(int64_t rows, int64_t classes, size_t element)
{
    if (classes <= 1024 || (rows >= 4096 && classes * (int64_t)element <= 16384)) return 64;
    return rows < 256 && classes > 16384 ? 1024 : 256;
}

dim3 blocks_of(int64_t rows, int threads)
{
    const int64_t each = threads <= 64 ? 256 / threads : 1, n = (rows + each - 1) / each, x = n < 1 << 21 ? n : 1 << 21;
    return dim3((unsigned)x, (unsigned)((n + x - 1) / x));
}

template <typename T>
void launch_top(int64_t rows, int64_t classes, const void* logits, int64_t row_stride, int k, float temperature, void* values,
                int32_t* indices, float* rest, hipStream_t st)
{
    const auto narrow = [&](auto lanes) {
        constexpr int G = decltype(lanes)::value;
        k_top_narrow<G, T><<<blocks_of(rows, G), 256, 0, st>>>(rows, classes, (const T*)logits, row_stride, k, temperature, (T*)values,
                                                               indices, rest);
    };
    if (classes <= 8) return narrow(std::integral_constant<int, 8>());
    if (classes <= 16) return narrow(std::integral_constant<int, 16>());
    if (classes <= 32) return narrow(std::integral_constant<int, 32>());
    if (classes <= 64) return narrow(std::integral_constant<int, 64>());
    // A wave holds up to 32 (twice as many threads as are to be chosen), and serves many rows of up to 64 KB better than a workgroup
    // each (k = 4, four waves / one: 2 048 x 5 000 f32 22 / 14 us, 16 384 x 16 000 f16 159 / 110, 16 384 x 16 000 f32 201 / 188,
    // 16 384 x 32 000 f32 354 / 364, 1 024 x 5 000 f16 12 / 11, 256 x 5 000 f32 11 / 11, 256 x 16 000 f32 14 / 19).  Two waves hold
    // up to 64, and are better than four in the same way (k = 64, four / two: 2 047 x 50 001 bf16 72 / 62, 2 047 x 50 001 f32
    // 100 / 95, 16 384 x 2 000 f32 110 / 84, 16 384 x 8 000 f32 161 / 165, 16 384 x 20 000 f32 282 / 315, 512 x 20 000 bf16 19 / 24).
    const bool short_rows = classes * (int64_t)sizeof(T) <= 65536;
    const int g = k <= 32 && (classes <= 1024 || (rows >= 2048 && short_rows)) ? 64
                : k <= 64 && rows >= 1024 && (short_rows || rows < 8192) ? 128
                : rows < 256 && classes > 16384 ? 1024 : 256;
    const dim3 blocks = blocks_of(rows, g);
    switch (g) {
    case 64: k_top<64, T><<<blocks, 256, 0, st>>>(rows, classes, (const T*)logits, row_stride, k, temperature, (T*)values, indices, rest); break;
    case 128: k_top<128, T><<<blocks, 128, 0, st>>>(rows, classes, (const T*)logits, row_stride, k, temperature, (T*)values, indices, rest); break;
    case 256: k_top<256, T><<<blocks, 256, 0, st>>>(rows, classes, (const T*)logits, row_stride, k, temperature, (T*)values, indices, rest); break;
    default: k_top<1024, T><<<blocks, 1024, 0, st>>>(rows, classes, (const T*)logits, row_stride, k, temperature, (T*)values, indices, rest);
    }
}

template <typename T> void launch_forward(const pxg_distill& a, hipStream_t st)
{
    const int g = threads_of(a.rows, a.classes, sizeof(T));
    const dim3 blocks = blocks_of(a.rows, g);
    switch (g) {
    case 64: k_distill_forward<64, T><<<blocks, 256, 0, st>>>(a); break;
    case 256: k_distill_forward<256, T><<<blocks, 256, 0, st>>>(a); break;
    default: k_distill_forward<1024, T><<<blocks, 1024, 0, st>>>(a);
    }
}

template <typename T> void launch_backward(const pxg_distill& a, hipStream_t st)
{
    const int g = threads_of(a.rows, a.classes, sizeof(T));
    const dim3 blocks = blocks_of(a.rows, g);
    switch (g) {
    case 64: k_distill_backward<64, T><<<blocks, 256, 0, st>>>(a); break;
    case 256: k_distill_backward<256, T><<<blocks, 256, 0, st>>>(a); break;
    default: k_distill_backward<1024, T><<<blocks, 1024, 0, st>>>(a);
    }
}

// below the least normal number its reciprocal is no float32 (scale_of): 0 times that would be NaN
bool bad_temperature(float t) { return !(t >= 1.17549435e-38f && t <= 3.0e38f); }

bool bad_call(const pxg_distill* a)
{
    return !a || a->struct_bytes != sizeof(pxg_distill) || a->dtype < PXG_DT_F32 || a->dtype > PXG_DT_F16 ||
           a->value_dtype < PXG_DT_F32 || a->value_dtype > PXG_DT_F16 || a->rows < 0 || a->rows > INT32_MAX || a->classes < 1 ||
           a->classes > INT32_MAX || a->k < 0 || a->k > PXG_TOP_MAX_K || bad_temperature(a->temperature) ||
           (a->rows > 0 && (!a->logits || !a->stats || (a->k > 0 && (!a->values || !a->indices))));
}

}  // namespace

extern "C" int pxg_top_logits(int32_t dtype, int64_t rows, int64_t classes, const void* logits, int64_t row_stride, int32_t k,
                              float temperature, void* values, int32_t* indices, float* rest, void* stream)
{
    if (dtype < PXG_DT_F32 || dtype > PXG_DT_F16 || rows < 0 || rows > INT32_MAX || classes < 1 || classes > INT32_MAX || k < 1 ||
        k > PXG_TOP_MAX_K || k > classes || bad_temperature(temperature))
        return PXG_E_INVALID;
    if (rows == 0) return PXG_OK;
    if (!logits || !values || !indices || !rest) return PXG_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    (void)hipGetLastError();                     // what an earlier call left is not this call's
    switch (dtype) {
    case PXG_DT_F32: launch_top<float>(rows, classes, logits, row_stride, k, temperature, values, indices, rest, st); break;
    case PXG_DT_BF16: launch_top<pxg_bf16>(rows, classes, logits, row_stride, k, temperature, values, indices, rest, st); break;
    default: launch_top<pxg_f16>(rows, classes, logits, row_stride, k, temperature, values, indices, rest, st);
    }
    return hipGetLastError() == hipSuccess ? PXG_OK : PXG_E_HIP;
}

extern "C" int pxg_distill_forward(const pxg_distill* a, void* stream)
{
    if (bad_call(a) || (a->rows > 0 && !a->row_loss)) return PXG_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    (void)hipGetLastError();                     // what an earlier call left is not this call's
    if (a->rows) {
        switch (a->dtype) {
        case PXG_DT_F32: launch_forward<float>(*a, st); break;
        case PXG_DT_BF16: launch_forward<pxg_bf16>(*a, st); break;
        default: launch_forward<pxg_f16>(*a, st);
        }
        if (hipGetLastError() != hipSuccess) return PXG_E_HIP;
    }
    if (a->loss) {
        k_distill_sum<<<1, 1024, 0, st>>>(a->row_loss, a->rows, a->mean, a->loss);
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
    (void)hipGetLastError();                     // what an earlier call left is not this call's
    switch (a->dtype) {
    case PXG_DT_F32: launch_backward<float>(*a, st); break;
    case PXG_DT_BF16: launch_backward<pxg_bf16>(*a, st); break;
    default: launch_backward<pxg_f16>(*a, st);
    }
    return hipGetLastError() == hipSuccess ? PXG_OK : PXG_E_HIP;
}
