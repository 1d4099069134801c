// k_decay_chunk.h -- the recurrence of decay attention on the matrix cores, in chunks of C steps (k_decay_{f32,bf16,f16}.hip).
//
// Inside a chunk, with the state S_in in front of it and local steps i, j = 0 .. C-1:
//   o_i   = sum_{j <= i} a^(i-j) (x_i . y_j) z_j + a^(i+1) x_i S_in
//   S_out = a^C S_in + sum_j a^(C-1-j) y_j z_j^T
// One workgroup takes one (sequence, head) and walks its chunks; wave w owns 16 (128-wide: 32) columns of the state for all its
// rows, in the accumulators of its matrix instructions from the first chunk to the last.  Nothing but the x, y, z rows of a chunk
// is in shared memory, and nothing crosses waves:
//   * the weights are computed transposed, P^T[j][i] = y_j . x_i, so that a lane holds four consecutive j of one i: which is how
//     the next product wants its operand.  The k axis of a product may be permuted if both operands are, so an operand of 32
//     is two accumulator tiles of 16 side by side.  The state's accumulators serve as the operand of x S the same way.
//   * operands that run over the steps (z for the weights, y and z for the state) are read transposed from row-major shared
//     memory by ds_read_b64_tr_b16.
//   * results are computed transposed as well, o^T[f][i]: a lane has four consecutive columns of one row to write, and the factor
//     a^(i+1) is one number per lane.
// Every wave computes all of P^T for itself.  That is C^2 E products four times instead of once; handing P around through shared
// memory would cost the barriers and the traffic that the permutation saves.
//
// Precision.  A matrix instruction takes bfloat16 operands and adds in float32.  A float32 number is the sum of three bfloat16
// ("planes"), a float16 number of two, both exactly: products of planes p, q are taken for p + q <= 2, which leaves 2^-24.
// What is computed in float32 and goes into a product (P, S, the weighted z) is split in the same way: into three planes where the
// result is float32, into two (2^-17 left) where it is rounded to half precision; the state itself always takes three.
//
// A sequence's steps are aligned to the END of its chunks: the first chunk begins with `pad` empty rows, so that no later factor
// depends on the length.
//
// 0 * inf: a weight of 0 (j > i) does not keep a z that is no finite number out of a matrix product.  Staging looks for such z;
// a chunk that has one takes its diagonal products row by row, with later rows' z left out.
#pragma once
#include "k_decay.h"

namespace decay {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef pxg_f32x4 f32x4;

template <typename T> struct Type;
template <> struct Type<float> { static constexpr int planes = 3, code = PXG_DT_F32; };
template <> struct Type<pxg_f16> { static constexpr int planes = 2, code = PXG_DT_F16; };
template <> struct Type<pxg_bf16> { static constexpr int planes = 1, code = PXG_DT_BF16; };

template <int D> struct Shape {
    static constexpr int waves = D == 16 ? 1 : D == 32 ? 2 : 4, slices = D == 128 ? 2 : 1, threads = 64 * waves;
    static constexpr int row = D + 8;                          // of shared memory: 16 bytes more, an odd number of 16-byte units
    static constexpr int kb = D == 16 ? 1 : D / 32, et = D / 16;
};

__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// four floats into N planes, the largest part first
template <int N> __device__ __forceinline__ void split(f32x4 v, bf16x4* p)
{
#pragma unroll
    for (int n = 0; n < N; n++) {
        p[n] = __builtin_convertvector(v, bf16x4);
        if (n + 1 < N) v -= __builtin_convertvector(p[n], f32x4);
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

template <typename T> __device__ __forceinline__ bool finite_piece(const Piece<T>& p)
{
    bool ok = true;
#pragma unroll
    for (int e = 0; e < 8; e++) ok &= __builtin_isfinite((float)p.v[e]);
    return ok;
}

// workgroups of neighbouring heads on one XCD, which they leave through one L2: `n` ids dealt out round-robin over 8
__device__ __forceinline__ int xcd_order(int id, int n)
{
    const int each = n / 8, more = n % 8, x = id % 8;
    return x * each + (x < more ? x : more) + id / 8;
}

template <typename T, int D, bool SLOPE, bool STATES_ONLY, bool WIDE>
__global__ __launch_bounds__(Shape<D>::threads) void k_chunks(const DecayRuns a, const int first_run)
{
    using Sh = Shape<D>;
    constexpr int NP = Type<T>::planes, C = decay_chunk(Type<T>::code, D), CT = C / 16, SL = Sh::slices, ET = Sh::et, KB = Sh::kb;
    constexpr int ROW = Sh::row, PLANE = C * ROW, N = Sh::threads, PIECES = C * (D / 8) / N;
    constexpr int KEEP = NP == 3 || SLOPE ? 2 : 1;            // products of planes p + q <= KEEP go into the result
    static_assert(PIECES * N == C * (D / 8), "whole pieces");
    __shared__ __attribute__((aligned(16))) __bf16 tile[(STATES_ONLY ? 2 : 3) * NP * PLANE];
    __shared__ float pw[C + 1];
    __shared__ int strange[2];
    __bf16* const ty = tile;
    __bf16* const tz = tile + NP * PLANE;
    __bf16* const tx = tile + (STATES_ONLY ? 0 : 2 * NP * PLANE);

    const DecayRun& r = a.run[first_run + blockIdx.z];
    const int bh = xcd_order(blockIdx.x, gridDim.x), b = bh / a.heads, h = bh % a.heads, seg = blockIdx.y;
    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64, g = lane / 16, li = lane % 16;
    const int E = r.E, F = r.F;
    const bool works = wave * SL * 16 < F;                    // the others only stage
    const int64_t len = decay_length(a, b), base = (int64_t)bh * E * F;
    const int64_t chunks = (len + C - 1) / C, c_first = (int64_t)seg * a.segment_chunks;
    const int64_t c_last = chunks < c_first + a.segment_chunks ? chunks : c_first + a.segment_chunks;
    const int pad = (int)(chunks * C - len), reverse = r.reverse;

    if (!STATES_ONLY) {                                       // rows behind the sequence, dealt out over the segments
        for (int64_t t = len + seg * Sh::waves + wave; t < a.steps; t += a.segments * Sh::waves) {
            T* out = (T*)r.out + (((int64_t)b * a.steps + t) * a.heads + h) * F;
            for (int f = lane; f < F; f += 64) out[f] = pxg_from_f32<T>(0.f);
        }
    }
    if (STATES_ONLY && c_first + a.segment_chunks >= chunks) return;            // nothing behind it waits for its state
    if (c_first >= chunks && !(seg == 0 && chunks == 0)) {
        if (SLOPE && tid == 0) r.partial[(int64_t)bh * a.segments + seg] = 0.f;
        return;
    }

    const float log_a = a.log_decay[h];
    for (int n = tid; n <= C; n += N) pw[n] = n ? expf((float)n * log_a) : 1.f;
    if (tid < 2) strange[tid] = 0;
    __syncthreads();
    // factors of one lane: inside a diagonal tile, for tiles further off, for the state (index r: step 4 g + r of a tile)
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

    // the state: rows 4 g + r of each tile of 16, column li of each slice
    f32x4 S[SL][ET], G[SLOPE ? SL : 1][SLOPE ? ET : 1];
    const bool from_carry = seg > 0 && !STATES_ONLY;
    const int64_t at_carry = ((int64_t)bh * (a.segments - 1) + seg - 1) * E * F;
    const int64_t slopes = (int64_t)a.batch * a.heads * (a.segments - 1) * E * F;
#pragma unroll
    for (int s = 0; s < SL; s++)
#pragma unroll
        for (int t = 0; t < ET; t++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int e = t * 16 + 4 * g + k, f = (wave * SL + s) * 16 + li;
                const bool in = e < E && f < F;
                float v = 0.f;
                if (in && from_carry) v = r.carry[at_carry + e * F + f];
                else if (in && seg == 0 && r.init) v = r.init[base + e * r.init_e + f * r.init_f];
                S[s][t][k] = v;
                if constexpr (SLOPE) G[s][t][k] = in && from_carry ? r.carry[slopes + at_carry + e * F + f] : 0.f;
            }

    const T* const x = (const T*)r.x.data + b * r.x.batch_stride + h * r.x.head_stride;
    const T* const y = (const T*)r.y.data + b * r.y.batch_stride + h * r.y.head_stride;
    const T* const z = (const T*)r.z.data + b * r.z.batch_stride + h * r.z.head_stride;
    // What is loaded for the next chunk stays in registers while this one is computed: the loads take no branch (rows in front of
    // the sequence and columns behind the width read something that is there, and are cleared on their way to shared memory).
    Piece<T> px[STATES_ONLY ? 1 : PIECES], py[PIECES], pz[PIECES];
    const auto fetch = [&](int64_t c) {
#pragma unroll
        for (int n = 0; n < PIECES; n++) {
            const int at = tid + n * N, col = at % (D / 8) * 8;
            int64_t u = c * C + at / (D / 8) - pad;
            u = u > 0 ? u : 0;
            const int64_t t = reverse ? len - 1 - u : u;
            if constexpr (WIDE) {
                py[n] = load_wide(y + t * r.y.step_stride + (col < E ? col : 0));
                pz[n] = load_wide(z + t * r.z.step_stride + (col < F ? col : 0));
                if constexpr (!STATES_ONLY) px[n] = load_wide(x + t * r.x.step_stride + (col < E ? col : 0));
            } else {
                py[n] = load_narrow(y + t * r.y.step_stride, col, E);
                pz[n] = load_narrow(z + t * r.z.step_stride, col, F);
                if constexpr (!STATES_ONLY) px[n] = load_narrow(x + t * r.x.step_stride, col, E);
            }
        }
    };
    const auto x_block = [&](int it, int k, int p) {          // x of steps it * 16 .., columns 32 k .. as an operand, permuted
        const __bf16* at = tx + p * PLANE + (it * 16 + li) * ROW + k * 32 + 4 * g;
        return join(*(const bf16x4*)at, D == 16 ? bf16x4{} : *(const bf16x4*)(at + (D == 16 ? 0 : 16)));
    };
    const auto y_block = [&](int jt, int k, int p) {
        const __bf16* at = ty + p * PLANE + (jt * 16 + li) * ROW + k * 32 + 4 * g;
        return join(*(const bf16x4*)at, D == 16 ? bf16x4{} : *(const bf16x4*)(at + (D == 16 ? 0 : 16)));
    };
    const int at_tr = (4 * g + li / 4) * ROW + li % 4 * 4;    // of a lane in a 16 x 16 block that is read transposed
    float part = 0.f;

    if (c_first < c_last) fetch(c_first);
    for (int64_t c = c_first; c < c_last; c++) {
        const int odd = (int)(c & 1);
        __syncthreads();
        bool fine = true;
#pragma unroll
        for (int n = 0; n < PIECES; n++) {
            const int at = tid + n * N, col = at % (D / 8) * 8, o = at / (D / 8) * ROW + col;
            const bool live = c > 0 || at / (D / 8) >= pad;
            clear_unless(live && col < E, py[n]);
            clear_unless(live && col < F, pz[n]);
            if constexpr (!STATES_ONLY) clear_unless(live && col < E, px[n]);
            store_piece<T, PLANE>(py[n], ty + o);
            store_piece<T, PLANE>(pz[n], tz + o);
            if constexpr (!STATES_ONLY) {
                store_piece<T, PLANE>(px[n], tx + o);
                fine &= finite_piece(pz[n]);
            }
        }
        if (!STATES_ONLY && !fine) strange[odd] = 1;
        if (c + 1 < c_last) fetch(c + 1);
        __syncthreads();
        const int skip = c == 0 ? pad + (reverse && seg == 0 ? 1 : 0) : 0;      // steps by which the state's decay is short
        const bool odd_values = !STATES_ONLY && strange[odd];
        if (tid == 0) strange[odd ^ 1] = 0;
        if (!works) continue;

        if constexpr (!STATES_ONLY) {
            // the state as an operand: two tiles of rows side by side, in planes
            bf16x8 sp[SL][KB][KEEP + 1], gp[SLOPE ? SL : 1][SLOPE ? KB : 1][KEEP + 1];
#pragma unroll
            for (int s = 0; s < SL; s++)
#pragma unroll
                for (int k = 0; k < KB; k++) {
                    bf16x4 u[KEEP + 1], v[KEEP + 1] = {};
                    split<KEEP + 1>(S[s][2 * k], u);
                    if constexpr (D > 16) split<KEEP + 1>(S[s][2 * k + 1], v);
#pragma unroll
                    for (int p = 0; p <= KEEP; p++) sp[s][k][p] = join(u[p], v[p]);
                    if constexpr (SLOPE) {
                        split<KEEP + 1>(G[s][2 * k], u);
                        if constexpr (D > 16) split<KEEP + 1>(G[s][2 * k + 1], v);
#pragma unroll
                        for (int p = 0; p <= KEEP; p++) gp[s][k][p] = join(u[p], v[p]);
                    }
                }
#pragma unroll
            for (int it = 0; it < CT; it++) {
                bf16x8 xb[KB][NP];
#pragma unroll
                for (int k = 0; k < KB; k++)
#pragma unroll
                    for (int p = 0; p < NP; p++) xb[k][p] = x_block(it, k, p);
                f32x4 o[SL], d[SLOPE ? SL : 1];
                const int ahead = it * 16 + li + 1 - skip;    // steps from the state in front of the chunk to this lane's row
                const float w = pw[ahead > 0 ? ahead : 0];
#pragma unroll
                for (int s = 0; s < SL; s++) {
                    f32x4 acc = {}, slope = {};
#pragma unroll
                    for (int k = 0; k < KB; k++)
#pragma unroll
                        for (int p = KEEP; p >= 0; p--)
#pragma unroll
                            for (int q = 0; q < NP; q++)
                                if (p + q <= KEEP) {
                                    acc = mfma(sp[s][k][p], xb[k][q], acc);
                                    if constexpr (SLOPE) slope = mfma(gp[s][k][p], xb[k][q], slope);
                                }
                    o[s] = acc * w;
                    if constexpr (SLOPE) d[s] = (slope + acc * (float)ahead) * w;
                }
#pragma unroll
                for (int k = 0; k <= it / 2; k++) {           // 32 earlier steps at a time
                    f32x4 weight[2], far[2];
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const int jt = 2 * k + half;
                        f32x4 acc = {};
                        if (jt <= it) {
#pragma unroll
                            for (int m = 0; m < KB; m++)
#pragma unroll
                                for (int p = NP - 1; p >= 0; p--) {
                                    const bf16x8 yb = y_block(jt, m, p);
#pragma unroll
                                    for (int q = 0; q < NP; q++)
                                        if (p + q <= 2) acc = mfma(yb, xb[m][q], acc);
                                }
                            if (jt == it) {
#pragma unroll
                                for (int s = 0; s < 4; s++) acc[s] = li >= 4 * g + s ? acc[s] * w_diag[s] : 0.f;
                            } else {
                                acc *= w_off;
                                if (it - jt > 1) acc *= tiles[it - jt - 1];
                            }
                        }
                        weight[half] = acc;
                        if constexpr (SLOPE)
#pragma unroll
                            for (int s = 0; s < 4; s++) far[half][s] = acc[s] * (float)(16 * (it - jt) + li - 4 * g - s);
                    }
                    bf16x4 u[KEEP + 1], v[KEEP + 1];
                    bf16x8 wp[KEEP + 1], fp[SLOPE ? KEEP + 1 : 1];
                    split<KEEP + 1>(weight[0], u), split<KEEP + 1>(weight[1], v);
#pragma unroll
                    for (int p = 0; p <= KEEP; p++) wp[p] = join(u[p], v[p]);
                    if constexpr (SLOPE) {
                        split<KEEP + 1>(far[0], u), split<KEEP + 1>(far[1], v);
#pragma unroll
                        for (int p = 0; p <= KEEP; p++) fp[p] = join(u[p], v[p]);
                    }
#pragma unroll
                    for (int s = 0; s < SL; s++) {
                        const int f0 = (wave * SL + s) * 16;
                        bf16x8 zb[NP];
#pragma unroll
                        for (int q = 0; q < NP; q++) {
                            const __bf16* at = tz + q * PLANE + k * 32 * ROW + f0 + at_tr;
                            zb[q] = join(read_transposed(at), read_transposed(at + 16 * ROW));
                        }
                        const auto add = [&](const bf16x8* zz, f32x4& to, f32x4& to_slope) {
#pragma unroll
                            for (int p = KEEP; p >= 0; p--)
#pragma unroll
                                for (int q = 0; q < NP; q++)
                                    if (p + q <= KEEP) {
                                        to = mfma(zz[q], wp[p], to);
                                        if constexpr (SLOPE) to_slope = mfma(zz[q], fp[p], to_slope);
                                    }
                        };
                        if (odd_values && k == it / 2) {
                            // one row of the tile at a time, without the z of the rows behind it
                            f32x4 sum = o[s], sum_slope = d[SLOPE ? s : 0];
#pragma unroll 1
                            for (int i = 0; i < 16; i++) {
                                bf16x8 zz[NP];
#pragma unroll
                                for (int q = 0; q < NP; q++)
#pragma unroll
                                    for (int n = 0; n < 8; n++) {
                                        const int j = (n / 4 - it % 2) * 16 + 4 * g + n % 4;     // from the tile's first row
                                        zz[q][n] = j <= i ? zb[q][n] : (__bf16)0.f;
                                    }
                                f32x4 one = o[s], one_slope = d[SLOPE ? s : 0];
                                add(zz, one, one_slope);
                                if (li == i) sum = one, sum_slope = one_slope;
                            }
                            o[s] = sum;
                            if constexpr (SLOPE) d[s] = sum_slope;
                        } else {
                            add(zb, o[s], d[SLOPE ? s : 0]);
                        }
                    }
                }
                // rows of the result: four columns of this lane's step
                const int64_t u = c * C + it * 16 + li - pad, t = reverse ? len - 1 - u : u;
                if (u >= 0) {
                    const int64_t row = ((int64_t)b * a.steps + t) * a.heads + h;
#pragma unroll
                    for (int s = 0; s < SL; s++) {
                        const int f = (wave * SL + s) * 16 + 4 * g;
                        T* out = (T*)r.out + row * F + f;
                        if constexpr (WIDE) {
                            if (f < F) {
                                struct alignas(4 * sizeof(T)) Four { T v[4]; } four;
#pragma unroll
                                for (int k = 0; k < 4; k++) four.v[k] = pxg_from_f32<T>(o[s][k]);
                                *(Four*)out = four;
                            }
                        } else {
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                if (f + k < F) out[k] = pxg_from_f32<T>(o[s][k]);
                        }
                        if constexpr (SLOPE) {
                            const T* q = (const T*)r.dot.data + b * r.dot.batch_stride + t * r.dot.step_stride + h * r.dot.head_stride + f;
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                if (WIDE ? f < F : f + k < F) part = fmaf((float)q[k], d[s][k], part);
                        }
                    }
                }
            }
        }

        // the state behind the chunk
        const float decay = pw[C - skip];
#pragma unroll
        for (int s = 0; s < SL; s++)
#pragma unroll
            for (int t = 0; t < ET; t++) {
                if constexpr (SLOPE) G[s][t] = (G[s][t] + S[s][t] * (float)(C - skip)) * decay;
                S[s][t] *= decay;
            }
#pragma unroll
        for (int k = 0; k < C / 32; k++) {
            bf16x8 zw[SL][3], zs[SLOPE ? SL : 1][3];
#pragma unroll
            for (int s = 0; s < SL; s++) {
                bf16x4 u[2][3], v[2][3];
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const int jt = 2 * k + half;
                    const __bf16* at = tz + jt * 16 * ROW + (wave * SL + s) * 16 + at_tr;
                    f32x4 value = __builtin_convertvector(read_transposed(at), f32x4);
#pragma unroll
                    for (int q = 1; q < NP; q++) value += __builtin_convertvector(read_transposed(at + q * PLANE), f32x4);
                    value *= w_state;
                    if (jt < CT - 1) value *= tiles[CT - 1 - jt];
                    split<3>(value, u[half]);
                    if constexpr (SLOPE) {
#pragma unroll
                        for (int n = 0; n < 4; n++) value[n] *= (float)(C - 1 - jt * 16 - 4 * g - n);
                        split<3>(value, v[half]);
                    }
                }
#pragma unroll
                for (int p = 0; p < 3; p++) {
                    zw[s][p] = join(u[0][p], u[1][p]);
                    if constexpr (SLOPE) zs[s][p] = join(v[0][p], v[1][p]);
                }
            }
#pragma unroll
            for (int t = 0; t < ET; t++) {
                bf16x8 yt[NP];
#pragma unroll
                for (int q = 0; q < NP; q++) {
                    const __bf16* at = ty + q * PLANE + k * 32 * ROW + t * 16 + at_tr;
                    yt[q] = join(read_transposed(at), read_transposed(at + 16 * ROW));
                }
#pragma unroll
                for (int s = 0; s < SL; s++)
#pragma unroll
                    for (int p = 2; p >= 0; p--)
#pragma unroll
                        for (int q = 0; q < NP; q++)
                            if (p + q <= 2) {
                                S[s][t] = mfma(yt[q], zw[s][p], S[s][t]);
                                if constexpr (SLOPE) G[s][t] = mfma(yt[q], zs[s][p], G[s][t]);
                            }
            }
        }
    }

    // where the state goes: to the next segment, or behind the sequence
    const bool last = c_last == chunks;
    const int64_t to_carry = ((int64_t)bh * (a.segments - 1) + seg) * E * F;
    const float end = reverse && len > 0 ? pw[1] : 1.f;       // S before the first step is the gradient's a R
#pragma unroll
    for (int s = 0; s < SL; s++)
#pragma unroll
        for (int t = 0; t < ET; t++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int e = t * 16 + 4 * g + k, f = (wave * SL + s) * 16 + li;
                if (e >= E || f >= F) continue;
                if constexpr (STATES_ONLY) {
                    r.carry[to_carry + e * F + f] = S[s][t][k];
                    if constexpr (SLOPE) r.carry[slopes + to_carry + e * F + f] = G[s][t][k];
                } else if (last) {
                    const int64_t at = base + e * r.init_e + f * r.init_f;
                    if (r.fin) r.fin[at] = end * S[s][t][k];
                    if constexpr (SLOPE)
                        if (r.grad_fin) part = fmaf(r.grad_fin[at], G[s][t][k], part);
                }
            }
    if constexpr (SLOPE && !STATES_ONLY) {
#pragma unroll
        for (int m = 32; m; m >>= 1) part += __shfl_xor(part, m);
        __syncthreads();
        if (lane == 0) pw[wave] = part;
        __syncthreads();
        if (tid == 0) {
            float sum = 0.f;
            for (int i = 0; i < Sh::waves; i++) sum += pw[i];
            r.partial[(int64_t)bh * a.segments + seg] = sum;
        }
    }
}

template <typename T, int D, bool WIDE>
int launch_width(const DecayRuns& a, int first, int n, bool slope, bool states_only, hipStream_t stream)
{
    const dim3 grid(a.batch * a.heads, states_only ? a.segments - 1 : a.segments, n), block(Shape<D>::threads);
    if (states_only) {
        if (slope) k_chunks<T, D, true, true, WIDE><<<grid, block, 0, stream>>>(a, first);
        else k_chunks<T, D, false, true, WIDE><<<grid, block, 0, stream>>>(a, first);
    } else {
        if (slope) k_chunks<T, D, true, false, WIDE><<<grid, block, 0, stream>>>(a, first);
        else k_chunks<T, D, false, false, WIDE><<<grid, block, 0, stream>>>(a, first);
    }
    return hipGetLastError() == hipSuccess ? PXG_OK : PXG_E_HIP;
}

template <typename T, int D> int launch_rows(const DecayRuns& a, int first, int n, bool slope, bool states_only, hipStream_t stream)
{
    bool wide = true;
    for (int i = first; i < first + n; i++) wide &= a.run[i].wide != 0;
    return wide ? launch_width<T, D, true>(a, first, n, slope, states_only, stream)
                : launch_width<T, D, false>(a, first, n, slope, states_only, stream);
}

template <typename T> int launch(const DecayRuns& a, int first, int n, bool slope, bool states_only, hipStream_t stream)
{
    switch (decay_width(a.run[first].E, a.run[first].F)) {
    case 16: return launch_rows<T, 16>(a, first, n, slope, states_only, stream);
    case 32: return launch_rows<T, 32>(a, first, n, slope, states_only, stream);
    case 64: return launch_rows<T, 64>(a, first, n, slope, states_only, stream);
    default: return launch_rows<T, 128>(a, first, n, slope, states_only, stream);
    }
}

}  // namespace decay
