// k_decay_chunk.h -- the recurrence of decay attention on the matrix cores, in chunks of C steps (k_decay_{f32,bf16,f16}.hip).
//
// Inside a chunk, with the state S_in in front of it and local steps i, j = 0 .. C-1:
//   o_i   = sum_{j <= i} a^(i-j) (x_i . y_j) z_j + a^(i+1) x_i S_in
//   S_out = a^C S_in + sum_j a^(C-1-j) y_j z_j^T
// One workgroup takes one (sequence, head) and walks its chunks; wave w owns 16 columns of the state for all its rows, in the
// accumulators of its matrix instructions from the first chunk to the last.  Shared memory holds the rows of a chunk and the
// weights P[i][j] = a^(i-j) (x_i . y_j), which the waves compute tile by tile for each other:
//   * P is computed transposed, y_j . x_i, so that a lane holds four consecutive j of one i: 8 bytes to write, and to read again as
//     an operand.  The k axis of a product may be permuted if both operands are: an operand of 32 is two pieces of four out of two
//     tiles of 16, which is also how the state's accumulators lie, so x S takes them as its operand without a detour.
//   * operands that run over the steps (z for the weights, y and z for the state) are read transposed from row-major shared
//     memory by ds_read_b64_tr_b16.
//   * results are computed transposed as well, o^T[f][i]: a lane has four consecutive columns of one row to write, and the factor
//     a^(i+1) is one number per lane.
//
// Precision.  A matrix instruction takes bfloat16 operands and adds in float32.  A float32 number is the sum of three bfloat16
// ("planes"), a float16 number of two, both exactly: products of planes p, q are taken for p + q <= 2, which leaves 2^-24.
// What is computed in float32 and goes into a product is split in the same way.  The weighted z that the state is made of takes three
// planes, and so do state and slope in the run that gives the gradient of log_decay.  The weights P, and the state as an operand
// against x in all other runs, take three where the result is float32 and two (2^-18 left of each term) where it is rounded to half
// precision: the errors against 64 bits are those of one rounding then as well (128 x 2 000 x 8 x 64: f16 2.074e-4, bf16 1.659e-3
// either way), and three planes everywhere took 588 us instead of 537 (1 x 100 003 x 8 x 128 f16) and 221 instead of 210 (training
// 16 x 2 000 x 8 x 64 bf16).  The state itself is float32 from the first chunk to the last.
//
// The gradient of log_decay: inside a chunk sum_{j < i} (i - j) P_ij (q_i . z_j), a second product of rows beside P; from earlier
// chunks q_i . (x_i dS/dlog_decay), with the slope G = dS/dlog_decay carried like the state.
//
// A sequence's steps are aligned to the END of its chunks: the first chunk begins with `pad` empty rows, so that no later factor
// depends on the length.
//
// 0 * inf: a weight of 0 (j > i) does not keep a z that is no finite number out of a matrix product.  Staging looks for such z;
// a chunk that has one takes its diagonal products row by row, with later rows' z left out.
//
// What bounds it.  128 x 2 000 x 8 heads of 64, bf16, ragged: 241 us, 3.7 TB/s of rows (3.9 where all have 2 000 steps); rows of one
// head, 128 bytes at a stride of 1 KB, can be read and written at 4.3 to 4.4, a copy reaches 4.9.  Waits are 53 % of a wave's time,
// vector units 36 % busy, matrix units 13 %.  One sequence of 100 003 x 8 x 128, f16, 530 us: about a third for the states between 64
// segments and their join, the rest for the rows: of a wave's time 62 % are waits (two barriers a chunk, and chains of products
// behind shared memory), matrix instructions fill 28 %, shared memory is busy for 56 %.
// Why 32 steps: with 64 the triangle costs twice the products and half as many segments fit; no case was faster.
// Tried and slower: two buffers of shared memory, chunks fetched two ahead (f16 608 -> 818: registers), rows padded so that no
// two lanes meet on a bank (conflicts halved, 534 -> 547; 16 x 2 000 x 8 x 64 bf16 training 206 -> 278).
#pragma once
#include "k_decay.h"
#include <type_traits>

namespace decay {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef pxg_f32x4 f32x4;

template <typename T> struct Type;
template <> struct Type<float> { static constexpr int planes = 3, code = PXG_DT_F32; };
template <> struct Type<pxg_f16> { static constexpr int planes = 2, code = PXG_DT_F16; };
template <> struct Type<pxg_bf16> { static constexpr int planes = 1, code = PXG_DT_BF16; };

struct No { static constexpr bool value = false; };
struct Yes { static constexpr bool value = true; };
static constexpr No no;
static constexpr Yes yes;

template <int D> struct Shape {
    static constexpr int waves = D / 16, threads = 64 * waves;
    static constexpr int row = D + 8;                          // of shared memory: 16 bytes more, an odd number of 16-byte units
    static constexpr int kb = D == 16 ? 1 : D / 32, et = D / 16;
};

__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pair(float a, float b)    // one conversion for two
{
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ float low_of(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high_of(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

__device__ __forceinline__ f32x4 widen(bf16x4 v)
{
    const uint2 u = __builtin_bit_cast(uint2, v);
    return f32x4{low_of(u.x), high_of(u.x), low_of(u.y), high_of(u.y)};
}

// Products of planes, the small ones first.  Heads of 16 fill half of an instruction's k axis: two products share one.
template <int NU, int NV, int LIMIT> __device__ __forceinline__ f32x4 plane_products(const bf16x8* u, const bf16x8* v, f32x4 acc)
{
#pragma unroll
    for (int p = NU - 1; p >= 0; p--)
#pragma unroll
        for (int n = 0; n < NV; n++)
            if (p + n <= LIMIT) acc = mfma(u[p], v[n], acc);
    return acc;
}
template <int NU, int NV, int LIMIT> __device__ __forceinline__ f32x4 plane_products(const bf16x4* u, const bf16x4* v, f32x4 acc)
{
    bf16x4 wait_u = {}, wait_v = {};
    bool waits = false;
#pragma unroll
    for (int p = NU - 1; p >= 0; p--)
#pragma unroll
        for (int n = 0; n < NV; n++)
            if (p + n <= LIMIT) {
                if (waits) acc = mfma(join(wait_u, u[p]), join(wait_v, v[n]), acc);
                else wait_u = u[p], wait_v = v[n];
                waits = !waits;
            }
    if (waits) acc = mfma(join(wait_u, bf16x4{}), join(wait_v, bf16x4{}), acc);
    return acc;
}

// four floats into N planes, the largest part first
template <int N> __device__ __forceinline__ void split(f32x4 v, bf16x4* p)
{
#pragma unroll
    for (int n = 0; n < N; n++) {
        const uint2 u = {pair(v[0], v[1]), pair(v[2], v[3])};
        p[n] = __builtin_bit_cast(bf16x4, u);
        if (n + 1 < N) v -= widen(p[n]);
    }
}

// 4 rows x 16 columns of row-major shared memory, transposed: lane li of its group of 16 gets column li, four rows.  `p` points
// at row li / 4, columns 4 (li % 4) of the block.
__device__ __forceinline__ bf16x4 read_transposed(const __bf16* p)
{
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
    return __builtin_bit_cast(bf16x4, v);
}

// eight elements of a row on their way into shared memory
template <typename T> struct Piece { T v[8]; };

template <typename T> __device__ __forceinline__ Piece<T> load_wide(const T* at)
{
    Piece<T> p;
    __builtin_memcpy(&p, __builtin_assume_aligned(at, 16), sizeof p);
    return p;
}

template <typename T> __device__ __forceinline__ Piece<T> load_narrow(const T* row, int col, int width)
{
    Piece<T> p = {};
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (col + e < width) p.v[e] = row[col + e];
    return p;
}

template <typename T> __device__ __forceinline__ void clear_unless(bool keep, Piece<T>& p)
{
    uint4 w[sizeof p / 16];
    __builtin_memcpy(w, &p, sizeof p);
#pragma unroll
    for (auto& v : w) v.x = keep ? v.x : 0, v.y = keep ? v.y : 0, v.z = keep ? v.z : 0, v.w = keep ? v.w : 0;
    __builtin_memcpy(&p, w, sizeof p);
}

template <typename T, int PLANE> __device__ __forceinline__ void store_piece(const Piece<T>& p, __bf16* at)
{
    if constexpr (Type<T>::planes == 1) {
        *(uint4*)at = __builtin_bit_cast(uint4, p);
    } else {
        bf16x4 lo[3], hi[3];
        const f32x4 a = {(float)p.v[0], (float)p.v[1], (float)p.v[2], (float)p.v[3]};
        const f32x4 b = {(float)p.v[4], (float)p.v[5], (float)p.v[6], (float)p.v[7]};
        split<Type<T>::planes>(a, lo), split<Type<T>::planes>(b, hi);
#pragma unroll
        for (int n = 0; n < Type<T>::planes; n++) *(bf16x8*)(at + n * PLANE) = join(lo[n], hi[n]);
    }
}

// the largest magnitude's bits of a piece, two 16-bit halves at a time
template <typename T> __device__ __forceinline__ uint32_t magnitude(const Piece<T>& p, uint32_t so_far)
{
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    uint32_t w[sizeof p / 4];
    __builtin_memcpy(w, &p, sizeof p);
#pragma unroll
    for (uint32_t v : w) {
        if constexpr (sizeof(T) == 4) {
            v &= 0x7fffffffu;
            so_far = so_far > v ? so_far : v;
        } else {
            v &= 0x7fff7fffu;
            so_far = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, so_far), __builtin_bit_cast(u16x2, v)));
        }
    }
    return so_far;
}

template <typename T> __device__ __forceinline__ bool finite_magnitude(uint32_t m)
{
    if constexpr (sizeof(T) == 4) return m < 0x7f7f8000u;       // from here on the first plane is infinite
    const uint32_t limit = Type<T>::code == PXG_DT_BF16 ? 0x7f80u : 0x7c00u;
    return (m & 0xffffu) < limit && m >> 16 < limit;
}

// workgroups of neighbouring heads on one XCD, which they leave through one L2: `n` ids dealt out round-robin over 8
__device__ __forceinline__ int xcd_order(int id, int n)
{
    const int each = n / 8, more = n % 8, x = id % 8;
    return x * each + (x < more ? x : more) + id / 8;
}

// waves of a SIMD that the registers are to leave room for
constexpr int waves_wanted(int planes, int width, bool slope, bool states_only)
{
    if (states_only) return 3;
    if (slope || (planes == 3 && (width == 16 || width == 128))) return 2;
    return planes < 3 && width >= 64 ? 4 : 3;
}

// Shared memory of one workgroup, as separate arrays: what is written to one does not hold up what is read from another.
#define DECAY_SHARED(T, D, SLOPE, STATES_ONLY)                                                                                          \
    constexpr int SETS = STATES_ONLY ? 2 : SLOPE ? 4 : 3, CHUNK = DECAY_CHUNK;                                     \
    constexpr int WEIGHT_PLANES = STATES_ONLY || D == 16 ? 0 : Type<T>::planes == 3 ? 3 : 2;                                          \
    __shared__ __attribute__((aligned(16))) __bf16 tile[SETS * Type<T>::planes * CHUNK * Shape<D>::row];                              \
    __shared__ __attribute__((aligned(16))) __bf16 weights[WEIGHT_PLANES ? WEIGHT_PLANES * CHUNK * (CHUNK + 8) : 8];                  \
    __shared__ float pw[CHUNK + 1];                                                                                                   \
    __shared__ double sums[Shape<D>::waves];                                                                                          \
    __shared__ int strange[2]

template <typename T, int D, bool SLOPE, bool STATES_ONLY, bool WIDE>
__device__ __forceinline__ void walk_chunks(const DecayRuns& a, const DecayRun& r, __bf16* const tile, __bf16* const weights,
                                            float* const pw, double* const sums, int* const strange)
{
    using Sh = Shape<D>;
    constexpr int NP = Type<T>::planes, C = DECAY_CHUNK, CT = C / 16, ET = Sh::et, KB = Sh::kb;
    constexpr int ROW = Sh::row, PLANE = C * ROW, N = Sh::threads, W = Sh::waves, PIECES = C * (D / 8) / N;
    constexpr int KEEP = NP == 3 ? 2 : 1;                     // products of planes p + q <= KEEP go into the result (Precision, above)
    constexpr int PROW = C + 8, PPLANE = C * PROW;            // of the weights
    constexpr int SLOPE_PLANES = 3;
    constexpr bool OUT = !STATES_ONLY, DOT = SLOPE && OUT;
    // The state and its slope are rounded once a chunk where a chunk's sums are taken apart from them: float32 training 256 x 300 x 4
    // x 16 has 0.6 of the error in the gradient of log_decay, at the same speed.  Half-precision rows gain nothing (208 -> 237 us).
    constexpr bool APART = SLOPE && NP == 3;
    constexpr int KEEP_S = DOT ? 2 : KEEP;                    // of the state against x: the gradient of log_decay is made of them, too
    static_assert(PIECES * N == C * (D / 8), "whole pieces");
    static_assert(C == 32, "a chunk is one operand of a matrix instruction: two tiles of 16 steps");
    const int bh = xcd_order(blockIdx.x, gridDim.x), b = bh / a.heads, h = bh % a.heads, seg = blockIdx.y;
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, g = lane / 16, li = lane % 16, f0 = wave * 16;
    const int E = r.E, F = r.F;
    const bool works = f0 < F;                                // the others only stage and compute weights
    const int64_t len = decay_length(a, b), base = (int64_t)bh * E * F;
    const int64_t chunks = (len + C - 1) / C, c_first = (int64_t)seg * a.segment_chunks;
    const int64_t c_last = chunks < c_first + a.segment_chunks ? chunks : c_first + a.segment_chunks;
    const int pad = (int)(chunks * C - len), reverse = r.reverse;

    if (OUT) {                                                // rows behind the sequence, dealt out over the segments
        for (int64_t t = len + seg * W + wave; t < a.steps; t += a.segments * W) {
            T* out = (T*)r.out + (((int64_t)b * a.steps + t) * a.heads + h) * F;
            for (int f = lane; f < F; f += 64) out[f] = pxg_from_f32<T>(0.f);
        }
    }
    if (STATES_ONLY && c_first + a.segment_chunks >= chunks) return;            // nothing behind it waits for its state
    if (c_first >= chunks && !(seg == 0 && chunks == 0)) {
        if (SLOPE && tid == 0) r.partial[(int64_t)bh * a.segments + seg] = 0.0;
        return;
    }

    const float log_a = a.log_decay[h];
    // More steps than the sequence has lie between no two of its rows, only between the empty ones in front (whose zeros a decay
    // that grows out of float32 would turn into NaN: one step, log_decay = 3): 0 for those.
    for (int n = tid; n <= C; n += N) pw[n] = n == 0 ? 1.f : n <= len ? decay_over((float)n, log_a) : 0.f;
    if (tid < 2) strange[tid] = 0;
    __syncthreads();
    // factors of one lane: inside a diagonal tile, for tiles further off, for the state (index: step 4 g + s of a tile)
    f32x4 w_diag, w_off, w_state;
    float tiles[CT];                                          // and for whole tiles
#pragma unroll
    for (int n = 0; n < CT; n++) tiles[n] = pw[16 * n];
#pragma unroll
    for (int s = 0; s < 4; s++) {
        const int d = li - 4 * g - s;
        w_diag[s] = d >= 0 ? pw[d] : 0.f;
        w_off[s] = pw[16 + d];
        w_state[s] = pw[15 - 4 * g - s];
    }

    // the state: rows 4 g + k of each tile of 16, column li of this wave's sixteen
    f32x4 S[ET], G[SLOPE ? ET : 1];
    const bool from_carry = seg > 0 && OUT;
    const int64_t at_carry = ((int64_t)bh * (a.segments - 1) + seg - 1) * E * F;
    const int64_t slopes = (int64_t)a.batch * a.heads * (a.segments - 1) * E * F;
    const float* const start = from_carry ? r.carry + at_carry : seg == 0 && r.init ? r.init + base : nullptr;
    const int start_e = from_carry ? F : (int)r.init_e, start_f = from_carry ? 1 : (int)r.init_f;
#pragma unroll
    for (int t = 0; t < ET; t++) {
        S[t] = f32x4{};
        if constexpr (SLOPE) G[t] = f32x4{};
    }
    if (start) {
#pragma unroll
        for (int t = 0; t < ET; t++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int e = t * 16 + 4 * g + k, f = f0 + li;
                const bool in = e < E && f < F;
                const int at = in ? e * start_e + f * start_f : 0;
                const float v = start[at];
                S[t][k] = in ? v : 0.f;
                if constexpr (SLOPE)
                    if (from_carry) {
                        const float w = start[slopes + at];
                        G[t][k] = in ? w : 0.f;
                    }
            }
    }

    // What is loaded for the next chunk stays in registers while this one is computed: the loads take no branch (rows in front of
    // the sequence and columns behind the width read something that is there, and are cleared on their way to shared memory).  From
    // the second chunk on a lane's place in the chunk is a constant offset from its first step.
    const T* const x = (const T*)r.x.data + b * r.x.batch_stride + h * r.x.head_stride;
    const T* const y = (const T*)r.y.data + b * r.y.batch_stride + h * r.y.head_stride;
    const T* const z = (const T*)r.z.data + b * r.z.batch_stride + h * r.z.head_stride;
    const T* const q = DOT ? (const T*)r.dot.data + b * r.dot.batch_stride + h * r.dot.head_stride : nullptr;
    Piece<T> px[OUT ? PIECES : 1], py[PIECES], pz[PIECES], pq[DOT ? PIECES : 1];
    uint32_t ox[PIECES], oy[PIECES], oz[PIECES], oq[PIECES];                    // in elements
#pragma unroll
    for (int n = 0; n < PIECES; n++) {
        const int at = tid + n * N, col = at % (D / 8) * 8, row = reverse ? C - 1 - at / (D / 8) : at / (D / 8);
        const uint32_t ce = col < E ? col : 0, cf = col < F ? col : 0;
        ox[n] = row * (uint32_t)r.x.step_stride + ce, oy[n] = row * (uint32_t)r.y.step_stride + ce;
        oz[n] = row * (uint32_t)r.z.step_stride + cf, oq[n] = DOT ? row * (uint32_t)r.dot.step_stride + cf : 0;
    }
    const auto fetch = [&](int64_t c) {
#pragma unroll
        for (int n = 0; n < PIECES; n++) {
            const int at = tid + n * N, col = at % (D / 8) * 8;
            int64_t u = c * C + at / (D / 8) - pad;
            u = u > 0 ? u : 0;
            const int64_t t = reverse ? len - 1 - u : u;
            if constexpr (WIDE) {
                const int ce = col < E ? col : 0, cf = col < F ? col : 0;
                py[n] = load_wide(y + t * r.y.step_stride + ce);
                pz[n] = load_wide(z + t * r.z.step_stride + cf);
                if constexpr (OUT) px[n] = load_wide(x + t * r.x.step_stride + ce);
                if constexpr (DOT) pq[n] = load_wide(q + t * r.dot.step_stride + cf);
            } else {
                py[n] = load_narrow(y + t * r.y.step_stride, col, E);
                pz[n] = load_narrow(z + t * r.z.step_stride, col, F);
                if constexpr (OUT) px[n] = load_narrow(x + t * r.x.step_stride, col, E);
                if constexpr (DOT) pq[n] = load_narrow(q + t * r.dot.step_stride, col, F);
            }
        }
    };
    const auto fetch_next = [&](int64_t c) {
        if constexpr (WIDE) {
            const int64_t t = reverse ? len - (c + 1) * C + pad : c * C - pad;
            const T *xs = x + t * r.x.step_stride, *ys = y + t * r.y.step_stride, *zs = z + t * r.z.step_stride;
            const T* qs = DOT ? q + t * r.dot.step_stride : nullptr;
#pragma unroll
            for (int n = 0; n < PIECES; n++) {
                py[n] = load_wide(ys + oy[n]);
                pz[n] = load_wide(zs + oz[n]);
                if constexpr (OUT) px[n] = load_wide(xs + ox[n]);
                if constexpr (DOT) pq[n] = load_wide(qs + oq[n]);
            }
        } else {
            fetch(c);
        }
    };
    // steps 16 n .. of a tile, columns 32 k .. as an operand, permuted (heads of 16: half an operand)
    using Operand = std::conditional_t<D == 16, bf16x4, bf16x8>;
    const auto block = [&](const __bf16* of, int n, int k, int p) {
        const __bf16* at = of + p * PLANE + (n * 16 + li) * ROW + k * 32 + 4 * g;
        if constexpr (D == 16) return *(const bf16x4*)at;
        else return join(*(const bf16x4*)at, *(const bf16x4*)(at + 16));
    };
    // x_i . y_j, transposed, for tiles n and m of 16 steps
    const auto products = [&](const __bf16* of_j, const __bf16* of_i, int m, int n) {
        f32x4 acc = {};
#pragma unroll
        for (int k = 0; k < KB; k++) {
            Operand u[NP], v[NP];
#pragma unroll
            for (int p = 0; p < NP; p++) u[p] = block(of_j, m, k, p), v[p] = block(of_i, n, k, p);
            acc = plane_products<NP, NP, 2>(u, v, acc);
        }
        return acc;
    };
    __bf16 *const ty = tile, *const tz = tile + NP * PLANE, *const tx = tile + (OUT ? 2 * NP * PLANE : 0), *const tq = tile + (DOT ? 3 * NP * PLANE : 0);
    const int at_tr = (4 * g + li / 4) * ROW + li % 4 * 4;    // of a lane in a 16 x 16 block that is read transposed
    const bool narrow = E < D || F < D;
    float part = 0.f;                                         // of one chunk; `total` of all
    double total = 0.0;

    const auto stage = [&](int64_t c) {                       // what was fetched, into shared memory
        if (narrow || c == 0) {
#pragma unroll
            for (int n = 0; n < PIECES; n++) {
                const int at = tid + n * N, col = at % (D / 8) * 8;
                const bool live = c > 0 || at / (D / 8) >= pad;
                clear_unless(live && col < E, py[n]);
                clear_unless(live && col < F, pz[n]);
                if constexpr (OUT) clear_unless(live && col < E, px[n]);
                if constexpr (DOT) clear_unless(live && col < F, pq[n]);
            }
        }
        uint32_t most = 0;
#pragma unroll
        for (int n = 0; n < PIECES; n++) {
            const int at = tid + n * N, o = at / (D / 8) * ROW + at % (D / 8) * 8;
            store_piece<T, PLANE>(py[n], tile + o);
            store_piece<T, PLANE>(pz[n], tile + NP * PLANE + o);
            if constexpr (OUT) {
                store_piece<T, PLANE>(px[n], tile + 2 * NP * PLANE + o);
                most = magnitude(pz[n], most);
            }
            if constexpr (DOT) store_piece<T, PLANE>(pq[n], tile + 3 * NP * PLANE + o);
        }
        if (OUT && !finite_magnitude<T>(most)) strange[c & 1] = 1;
    };

    if (c_first < c_last) {
        fetch(c_first);
        stage(c_first);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                       // the state is there (vmcnt 0): no wait for it, and the rows behind it, in the loop
    for (int64_t c = c_first; c < c_last; c++) {
        __syncthreads();                                      // the chunk's rows are there
        if (c + 1 < c_last) fetch_next(c + 1);
        if (tid == 0) strange[(c + 1) & 1] = 0;
        const int skip = c == 0 ? pad + (reverse && seg == 0 ? 1 : 0) : 0;      // steps by which the state's decay is short

        constexpr int TILES = CT * (CT + 1) / 2;
        bf16x4 own[W == 1 ? TILES : 1][KEEP + 1];
        if constexpr (OUT) {
            // the weights, each wave its tiles
#pragma unroll
            for (int turn = 0; turn < (TILES + W - 1) / W; turn++) {
                const int n = W == 1 ? turn : wave + turn * W;
                if (n >= TILES) break;
                const int it = n < 1 ? 0 : 1, jt = n - it;               // two tiles of 16: (0, 0), (1, 0), (1, 1)
                f32x4 acc = products(ty, tx, jt, it);
                if (it == jt) {
#pragma unroll
                    for (int s = 0; s < 4; s++) acc[s] = li >= 4 * g + s ? acc[s] * w_diag[s] : 0.f;
                } else {
                    acc *= w_off;
                }
                bf16x4 u[KEEP + 1];
                split<KEEP + 1>(acc, u);
#pragma unroll
                for (int p = 0; p <= KEEP; p++) {
                    if constexpr (W == 1) own[turn][p] = u[p];
                    else *(bf16x4*)(weights + p * PPLANE + (it * 16 + li) * PROW + jt * 16 + 4 * g) = u[p];
                }
                if constexpr (DOT) {
                    const f32x4 d = products(tz, tq, jt, it);
#pragma unroll
                    for (int s = 0; s < 4; s++) {
                        const int away = 16 * (it - jt) + li - 4 * g - s;
                        if (away > 0) part = fmaf((float)away * acc[s], d[s], part);
                    }
                }
            }
        }
        f32x4 o[OUT ? CT : 1];
        if (OUT && works) {
            // x S: what the steps in front of the chunk leave in each row
            f32x4 d[DOT ? CT : 1];
#pragma unroll
            for (int it = 0; it < CT; it++) {
                o[it] = f32x4{};
                if constexpr (DOT) d[it] = f32x4{};
            }
#pragma unroll
            for (int k = 0; k < KB; k++) {
                Operand su[KEEP_S + 1], gu[SLOPE ? SLOPE_PLANES : 1];
                const auto operand = [&](const f32x4* of, auto planes, Operand* to) {
                    constexpr int M = decltype(planes)::value;
                    bf16x4 u[M], v[M];
                    split<M>(of[D == 16 ? 0 : 2 * k], u);
                    if constexpr (D > 16) {
                        split<M>(of[2 * k + 1], v);
#pragma unroll
                        for (int p = 0; p < M; p++) to[p] = join(u[p], v[p]);
                    } else {
#pragma unroll
                        for (int p = 0; p < M; p++) to[p] = u[p];
                    }
                };
                operand(S, std::integral_constant<int, KEEP_S + 1>(), su);
                if constexpr (DOT) operand(G, std::integral_constant<int, SLOPE_PLANES>(), gu);
#pragma unroll
                for (int it = 0; it < CT; it++) {
                    Operand xb[NP];
#pragma unroll
                    for (int p = 0; p < NP; p++) xb[p] = block(tx, it, k, p);
                    o[it] = plane_products<KEEP_S + 1, NP, KEEP_S>(su, xb, o[it]);
                    if constexpr (DOT) d[it] = plane_products<SLOPE_PLANES, NP, SLOPE_PLANES - 1>(gu, xb, d[it]);
                }
            }
#pragma unroll
            for (int it = 0; it < CT; it++) {
                const int ahead = it * 16 + li + 1 - skip;    // steps from the state in front of the chunk to this lane's row
                const float w = pw[ahead > 0 ? ahead : 0];
                if constexpr (DOT) {
                    const f32x4 slope = (d[it] + o[it] * (float)ahead) * w;
                    f32x4 row = {};
#pragma unroll
                    for (int p = NP - 1; p >= 0; p--) row += widen(*(const bf16x4*)(tq + p * PLANE + (it * 16 + li) * ROW + f0 + 4 * g));
                    if (ahead > 0)
#pragma unroll
                        for (int s = 0; s < 4; s++) part = fmaf(row[s], slope[s], part);
                }
                o[it] *= w;
            }
        }
        if (works) {
            // the state behind the chunk
            const float decay = pw[C - skip];
            if constexpr (!APART) {
#pragma unroll
                for (int t = 0; t < ET; t++) {
                    if constexpr (SLOPE) G[t] = (G[t] + S[t] * (float)(C - skip)) * decay;
                    S[t] *= decay;
                }
            }
            bf16x8 zw[3], zs[SLOPE ? SLOPE_PLANES : 1];
            bf16x4 u[CT][3], v[CT][SLOPE ? SLOPE_PLANES : 1];
#pragma unroll
            for (int jt = 0; jt < CT; jt++) {
                const __bf16* at = tz + jt * 16 * ROW + f0 + at_tr;
                f32x4 value = widen(read_transposed(at + (NP - 1) * PLANE));
#pragma unroll
                for (int n = NP - 2; n >= 0; n--) value += widen(read_transposed(at + n * PLANE));
                value *= w_state;
                if (jt < CT - 1) value *= tiles[CT - 1 - jt];
                split<3>(value, u[jt]);
                if constexpr (SLOPE) {
#pragma unroll
                    for (int n = 0; n < 4; n++) value[n] *= (float)(C - 1 - jt * 16 - 4 * g - n);
                    split<SLOPE_PLANES>(value, v[jt]);
                }
            }
#pragma unroll
            for (int p = 0; p < 3; p++) zw[p] = join(u[0][p], u[1][p]);
            if constexpr (SLOPE)
#pragma unroll
                for (int p = 0; p < SLOPE_PLANES; p++) zs[p] = join(v[0][p], v[1][p]);
#pragma unroll
            for (int t = 0; t < ET; t++) {
                bf16x8 yt[NP];
#pragma unroll
                for (int n = 0; n < NP; n++) {
                    const __bf16* at = ty + n * PLANE + t * 16 + at_tr;
                    yt[n] = join(read_transposed(at), read_transposed(at + 16 * ROW));
                }
                f32x4 sum = {}, slope = {};
                if constexpr (!APART) {
                    sum = S[t];
                    if constexpr (SLOPE) slope = G[t];
                }
#pragma unroll
                for (int p = 2; p >= 0; p--)
#pragma unroll
                    for (int n = 0; n < NP; n++)
                        if (p + n <= 2) sum = mfma(yt[n], zw[p], sum);
                if constexpr (SLOPE) {
#pragma unroll
                    for (int p = SLOPE_PLANES - 1; p >= 0; p--)
#pragma unroll
                        for (int n = 0; n < NP; n++)
                            if (p + n < SLOPE_PLANES) slope = mfma(yt[n], zs[p], slope);
                    G[t] = APART ? (G[t] + S[t] * (float)(C - skip)) * decay + slope : slope;
                }
                S[t] = APART ? S[t] * decay + sum : sum;
            }
        }
        if constexpr (OUT && W > 1) __syncthreads();          // the weights are there
        if (OUT && works) {
            // P z
            const auto add_rows = [&](int it, auto careful) {
                bf16x8 wp[KEEP + 1], zb[NP];
#pragma unroll
                for (int p = 0; p <= KEEP; p++) {
                    if constexpr (W == 1) {
                        const int n = it * (it + 1) / 2;
                        wp[p] = join(own[n][p], it > 0 ? own[n + 1][p] : bf16x4{});
                    } else {
                        const __bf16* at = weights + p * PPLANE + (it * 16 + li) * PROW + 4 * g;
                        wp[p] = join(*(const bf16x4*)at, it > 0 ? *(const bf16x4*)(at + 16) : bf16x4{});
                    }
                }
#pragma unroll
                for (int n = 0; n < NP; n++) {
                    const __bf16* at = tz + n * PLANE + f0 + at_tr;
                    zb[n] = join(read_transposed(at), read_transposed(at + 16 * ROW));
                }
                const auto add = [&](const bf16x8* zz, f32x4 to) {
#pragma unroll
                    for (int p = KEEP; p >= 0; p--)
#pragma unroll
                        for (int n = 0; n < NP; n++)
                            if (p + n <= KEEP) to = mfma(zz[n], wp[p], to);
                    return to;
                };
                if constexpr (decltype(careful)::value) {
                    // one row of the tile at a time, without the z of the rows behind it
                    const f32x4 before = o[it];
#pragma unroll 1
                    for (int i = 0; i < 16; i++) {
                        bf16x8 zz[NP];
#pragma unroll
                        for (int n = 0; n < NP; n++)
#pragma unroll
                            for (int m = 0; m < 8; m++) {
                                const int j = (m / 4 - it) * 16 + 4 * g + m % 4;             // from the tile's first row
                                zz[n][m] = j <= i ? zb[n][m] : (__bf16)0.f;
                            }
                        const f32x4 one = add(zz, before);
                        if (li == i) o[it] = one;
                    }
                } else {
                    o[it] = add(zb, o[it]);
                }
            };
            if (strange[c & 1]) {
#pragma unroll
                for (int it = 0; it < CT; it++) add_rows(it, yes);
            } else {
#pragma unroll
                for (int it = 0; it < CT; it++) add_rows(it, no);
            }
        }
        if constexpr (DOT) total += (double)part, part = 0.f;
        const auto write = [&] {
            if (!OUT || !works) return;
            // rows of the result: four columns of this lane's step
            const int64_t first = reverse ? len - 1 - c * C + pad : c * C - pad;
            T* const out = (T*)r.out + (((int64_t)b * a.steps + first) * a.heads + h) * F + f0 + 4 * g;
            const int64_t out_step = (int64_t)(reverse ? -a.heads : a.heads) * F;
#pragma unroll
            for (int it = 0; it < CT; it++) {
                if (c == 0 && it * 16 + li < pad) continue;   // in front of the sequence
                T* const at = out + (it * 16 + li) * out_step;
                const int f = f0 + 4 * g;
                if constexpr (WIDE) {
                    if (f < F) {
                        struct alignas(4 * sizeof(T)) Four { T v[4]; } four;
#pragma unroll
                        for (int k = 0; k < 4; k++) four.v[k] = pxg_from_f32<T>(o[it][k]);
                        *(Four*)at = four;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (f + k < F) at[k] = pxg_from_f32<T>(o[it][k]);
                }
            }
        };
        if (c + 1 == c_last) {
            write();
            break;
        }
        // staged before the stores: the wait for what was fetched is no wait for them
        __syncthreads();
        stage(c + 1);
        write();
    }

    // where the state goes: to the next segment, or behind the sequence
    const bool last = c_last == chunks;
    const int64_t to_carry = ((int64_t)bh * (a.segments - 1) + seg) * E * F;
    const float end = reverse && len > 0 ? pw[1] : 1.f;       // S before the first step is the gradient's a R
    float* const fin = STATES_ONLY ? r.carry + to_carry : last && r.fin ? r.fin + base : nullptr;
    const int fin_e = STATES_ONLY ? F : (int)r.init_e, fin_f = STATES_ONLY ? 1 : (int)r.init_f;
    if (fin) {
#pragma unroll
        for (int t = 0; t < ET; t++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int e = t * 16 + 4 * g + k, f = f0 + li;
                if (e < E && f < F) {
                    fin[e * fin_e + f * fin_f] = STATES_ONLY ? S[t][k] : end * S[t][k];
                    if constexpr (STATES_ONLY && SLOPE) fin[slopes + e * fin_e + f * fin_f] = G[t][k];
                }
            }
    }
    if constexpr (DOT) {
        if (last && r.grad_fin) {
#pragma unroll
            for (int t = 0; t < ET; t++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int e = t * 16 + 4 * g + k, f = f0 + li;
                    const bool in = e < E && f < F;
                    const float v = r.grad_fin[base + (in ? e * (int)r.init_e + f * (int)r.init_f : 0)];
                    part = fmaf(in ? v : 0.f, G[t][k], part);
                }
        }
    }
    if constexpr (DOT) {
        total += (double)part;
#pragma unroll
        for (int m = 32; m; m >>= 1) total += __shfl_xor(total, m);
        if (lane == 0) sums[wave] = total;
        __syncthreads();
        if (tid == 0) {
            double sum = 0.0;
            for (int i = 0; i < W; i++) sum += sums[i];
            r.partial[(int64_t)bh * a.segments + seg] = sum;
        }
    }
}

template <typename T, int D, bool SLOPE, bool STATES_ONLY, bool WIDE>
__global__ __launch_bounds__(Shape<D>::threads, waves_wanted(Type<T>::planes, D, SLOPE, STATES_ONLY))
void k_chunks(const DecayRuns a, const int first_run)
{
    DECAY_SHARED(T, D, SLOPE, STATES_ONLY);
    const DecayRun r = a.run[first_run + blockIdx.z];
    walk_chunks<T, D, SLOPE, STATES_ONLY, WIDE>(a, r, tile, weights, pw, sums, strange);
}

// run 0 with slopes beside the others
template <typename T, int D, bool STATES_ONLY, bool WIDE>
__global__ __launch_bounds__(Shape<D>::threads, waves_wanted(Type<T>::planes, D, true, STATES_ONLY))
void k_mixed_chunks(const DecayRuns a)
{
    DECAY_SHARED(T, D, true, STATES_ONLY);
    const DecayRun r = a.run[blockIdx.z];
    if (blockIdx.z == 0) walk_chunks<T, D, true, STATES_ONLY, WIDE>(a, r, tile, weights, pw, sums, strange);
    else walk_chunks<T, D, false, STATES_ONLY, WIDE>(a, r, tile, weights, pw, sums, strange);
}

// The first `slopes` of the `n` runs (none or one) carry slopes.
template <typename T, int D, bool STATES_ONLY, bool WIDE> int launch_width(const DecayRuns& a, int n, int slopes, hipStream_t stream)
{
    const dim3 block(Shape<D>::threads);
    const auto grid = [&](int runs) { return dim3(a.batch * a.heads, STATES_ONLY ? a.segments - 1 : a.segments, runs); };
    // side by side where the others do not lose waves to the registers that slopes take
    if (slopes && n > slopes && !(Type<T>::planes == 2 && D == 128)) {
        k_mixed_chunks<T, D, STATES_ONLY, WIDE><<<grid(n), block, 0, stream>>>(a);
    } else {
        if (slopes) k_chunks<T, D, true, STATES_ONLY, WIDE><<<grid(slopes), block, 0, stream>>>(a, 0);
        if (hipPeekAtLastError() == hipSuccess && n > slopes)
            k_chunks<T, D, false, STATES_ONLY, WIDE><<<grid(n - slopes), block, 0, stream>>>(a, slopes);
    }
    return hipGetLastError() == hipSuccess ? PXG_OK : PXG_E_HIP;
}

template <typename T, int D> int launch_rows(const DecayRuns& a, int n, int slopes, bool states_only, hipStream_t stream)
{
    bool wide = true;
    for (int i = 0; i < n; i++) wide &= a.run[i].wide != 0;
    if (states_only) return wide ? launch_width<T, D, true, true>(a, n, slopes, stream) : launch_width<T, D, true, false>(a, n, slopes, stream);
    return wide ? launch_width<T, D, false, true>(a, n, slopes, stream) : launch_width<T, D, false, false>(a, n, slopes, stream);
}

template <typename T> int launch(const DecayRuns& a, int n, int slopes, bool states_only, hipStream_t stream)
{
    switch (decay_width(a.run[0].E, a.run[0].F)) {
    case 16: return launch_rows<T, 16>(a, n, slopes, states_only, stream);
    case 32: return launch_rows<T, 32>(a, n, slopes, states_only, stream);
    case 64: return launch_rows<T, 64>(a, n, slopes, states_only, stream);
    default: return launch_rows<T, 128>(a, n, slopes, states_only, stream);
    }
}

}  // namespace decay
