// Causal attention of packed sequences (fmlh_attention_packed, fmlh_attention_packed_backward):
// sequences of different lengths one behind the other in the rows of q, k and v, with n_head
// query heads on n_kv_head key heads.  With G = n_head / n_kv_head, "row" rho of a sequence and
// key head is query rho / G of query head kv * G + rho % G, so that the heads of a group share
// every key and value they read.
//
//   s_ij = scale q_i . k_j for the keys j <= i + kl - ql (ql, kl: the sequence's queries and keys),
//   p = softmax over j, o_i = sum_j p_ij v_j, lse_i = log sum_j exp(s_ij);
//   backward, with d_i = do_i . o_i:  dv_j = sum_i p_ij do_i,
//   ds_ij = p_ij (do_i . v_j - d_i) scale, dq_i = sum_j ds_ij k_j, dk_j = sum_i ds_ij q_i.
//
// No score matrix is stored: keys (forward, dq) or rows (dk, dv) stream through LDS in tiles and a
// softmax keeps a running maximum and sum per row; the backward pass forms p from lse.  The sums over
// a group's heads stay in the work-group that owns the keys: no atomics, results do not depend on
// the order of work-groups.
//
// Masked scores are replaced before they are used, but 0 * v of a masked infinite or NaN v would
// still reach a sum on the matrix cores: tiles that hold a masked pair and a value that is not
// finite are multiplied element by element instead.
#include "attention_packed_device.h"

#include <algorithm>

namespace fmlh {

namespace {

// NaN where a value is infinite or NaN, else 0.
__device__ __forceinline__ float not_finite(floatx4 v) { return (v[0] + v[1] + v[2] + v[3]) * 0.f; }

// Copies rows [first, first + R) of a matrix (row stride rs) into LDS rows of LD floats, DP of
// them filled; rows from `rows` on are zero.  Returns NaN where a value is not finite.
template <int R, int DP, int LD>
__device__ __forceinline__ float stage_rows(float* lds, const float* base, size_t rs, uint32_t first, uint32_t rows, int dim,
                                            bool vec) {
    constexpr int U = DP / 4;
    float bad = 0.f;
    for (int e = threadIdx.x; e < R * U; e += 256) {
        const uint32_t r = first + e / U;
        const int d = 4 * (e % U);
        floatx4 v = {0.f, 0.f, 0.f, 0.f};
        if (r < rows) v = load4(base + (size_t)r * rs, d, dim, vec);
        bad += not_finite(v);
        *reinterpret_cast<floatx4*>(lds + (e / U) * LD + d) = v;
    }
    return bad;
}

// S (32 x 32) = A B^T over DP dims: A's rows from LDS (row stride LD), B's row of lane column c in
// registers (dims h DP / 2 ..).  The matrix core's two k of a step are dims u and DP / 2 + u.
template <int DP, int LD>
__device__ __forceinline__ floatx16 lds_rows_product(const float* lds_rows, const float (&b)[DP / 2], int h, int c) {
    floatx16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
    const float* row = lds_rows + c * LD + h * (DP / 2);
#pragma unroll
    for (int u = 0; u < DP / 2; u += 4) {
        const floatx4 x = *reinterpret_cast<const floatx4*>(row + u);
#pragma unroll
        for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], b[u + e], s, 0, 0, 0);
    }
    return s;
}

// acc (dims x 32 columns) += X^T w, X 32 rows in LDS, w their 32 x 32 weights in accumulator layout.
template <int DP, int LD>
__device__ __forceinline__ void add_product(floatx16 (&acc)[DP / 32], const float* lds_rows, const floatx16& w, int h, int c) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const float* x = lds_rows + acc_row(r, h) * LD + c;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) acc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[32 * i], w[r], acc[i], 0, 0, 0);
    }
}

// ---- few rows over many keys -------------------------------------------------------------------

// Single tokens over a cache: with RT rows (the heads of a group, a few queries) the keys' and values'
// bytes are the work.  A work-group takes a tile of RT rows of one (sequence, key head) and one of
// the ranges its keys are cut into; LPK lanes hold a key (NF float4 each), 64 / LPK keys per
// wave and step, kUnroll steps in flight.  Every lane group keeps its own maximum, sum and output
// over its keys; they are joined over the wave and the work-group once, at the end.

// A tile with one range writes its rows, otherwise their (maximum, sum, output) go to the workspace
// and are joined by attn_packed_join_kernel in range order.
// Sum over the LPK lanes of a key (4, 8 or 16, inside a DPP row): every lane holds it afterwards.
template <int LPK>
__device__ __forceinline__ float key_sum(float x) {
    x += dpp_move<0xB1, 0xf>(0.f, x);  // quad_perm [1, 0, 3, 2]
    x += dpp_move<0x4E, 0xf>(0.f, x);  // quad_perm [2, 3, 0, 1]
    if (LPK >= 8) x += dpp_move<0x141, 0xf>(0.f, x);   // row_half_mirror
    if (LPK >= 16) x += dpp_move<0x140, 0xf>(0.f, x);  // row_mirror
    return x;
}

template <int LPK, int NF, int RT>
__global__ __launch_bounds__(256) void attn_packed_few_kernel(PackedAttn a, float* __restrict__ out, float* __restrict__ lse,
                                                              const float* __restrict__ q, const float* __restrict__ k,
                                                              const float* __restrict__ v, float* __restrict__ ws, uint32_t budget) {
    constexpr int KPW = 64 / LPK, UN = RT * NF >= 8 ? 2 : 4, STEP = 4 * KPW * UN, W = 4 * LPK * NF;
    __shared__ float join_ml[4][RT][2];
    __shared__ __attribute__((aligned(16))) float join_o[4][RT][W];
    Work w;
    if (!find_work<false, false>(a, RT, budget, blockIdx.x, &w)) return;
    const RowTile tl = row_tile(a, w, RT);
    if (w.range >= tl.ranges) return;
    const Span sp = w.sp;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LPK, slot = wave * KPW + lane / LPK;
    const int dim = a.head_dim, group = a.group, kv = blockIdx.y;
    const int rows = tl.rows, rho0 = tl.rho0, shift = tl.shift, k_begin = tl.k_begin, k_end = tl.k_end;
    const float* kb = k + (size_t)sp.k0 * a.k_rs + (size_t)kv * a.k_hs;
    const float* vb = v + (size_t)sp.k0 * a.v_rs + (size_t)kv * a.v_hs;
    const float factor = a.scale * kLog2e;

    floatx4 qr[RT][NF], o[RT][NF];
    float m[RT], l[RT];
    int limit[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int rho = min(rho0 + t, rows - 1);
        const float* row = q + (size_t)(sp.q0 + rho / group) * a.q_rs + (size_t)(kv * group + rho % group) * dim;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            qr[t][f] = load4(row, 4 * (sub + LPK * f), dim, a.vec);
            o[t][f] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
        m[t] = -INFINITY;
        l[t] = 0.f;
        limit[t] = rho / group + shift;
    }
    for (int j0 = k_begin; j0 < k_end; j0 += STEP) {
        floatx4 kx[UN][NF], vx[UN][NF];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const size_t j = min(j0 + u * 4 * KPW + slot, k_end - 1);
#pragma unroll
            for (int f = 0; f < NF; ++f) kx[u][f] = load4(kb + j * a.k_rs, 4 * (sub + LPK * f), dim, a.vec);
#pragma unroll
            for (int f = 0; f < NF; ++f) vx[u][f] = load4(vb + j * a.v_rs, 4 * (sub + LPK * f), dim, a.vec);
        }
        const bool all = j0 + STEP <= min(k_end, rho0 / group + shift + 1);  // every row sees every key of the step
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            float s[UN], top = m[t];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                float d = 0.f;
#pragma unroll
                for (int f = 0; f < NF; ++f)
#pragma unroll
                    for (int e = 0; e < 4; ++e) d += qr[t][f][e] * kx[u][f][e];
                s[u] = key_sum<LPK>(d) * factor;
                if (!all && j0 + u * 4 * KPW + slot > min(limit[t], k_end - 1)) s[u] = -INFINITY;
                top = fmaxf(top, s[u]);
            }
            const float base = top == -INFINITY ? 0.f : top;
            const float corr = exp2f(m[t] - base);
            m[t] = top;
            l[t] *= corr;
#pragma unroll
            for (int f = 0; f < NF; ++f) o[t][f] *= corr;
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const float p = exp2f(s[u] - base);
                l[t] += p;
                if (all) {
#pragma unroll
                    for (int f = 0; f < NF; ++f) o[t][f] += p * vx[u][f];
                } else if (j0 + u * 4 * KPW + slot <= min(limit[t], k_end - 1)) {  // 0 * v of a masked v that is not finite
#pragma unroll
                    for (int f = 0; f < NF; ++f) o[t][f] += p * vx[u][f];
                }
            }
        }
    }
    // Join the lane groups of the wave, then the waves.
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float top = m[t];
#pragma unroll
        for (int d = LPK; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
        const float corr = exp2f(m[t] - (top == -INFINITY ? 0.f : top));
        float sum = l[t] * corr;
#pragma unroll
        for (int f = 0; f < NF; ++f) o[t][f] *= corr;
#pragma unroll
        for (int d = LPK; d < 64; d <<= 1) {
            sum += __shfl_xor(sum, d);
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[t][f][e] += __shfl_xor(o[t][f][e], d);
        }
        if (lane < LPK) {
#pragma unroll
            for (int f = 0; f < NF; ++f) *reinterpret_cast<floatx4*>(&join_o[wave][t][4 * (sub + LPK * f)]) = o[t][f];
            if (lane == 0) {
                join_ml[wave][t][0] = top;
                join_ml[wave][t][1] = sum;
            }
        }
    }
    __syncthreads();
    const Partials part = partials(ws, gridDim.y, kv, gridDim.x, w.item0 + w.range, RT, dim);
    for (int e = threadIdx.x; e < RT * (W / 4); e += 256) {
        const int t = e / (W / 4), d = 4 * (e % (W / 4)), rho = rho0 + t;
        if (rho >= rows) continue;
        float top = -INFINITY;
        for (int i = 0; i < 4; ++i) top = fmaxf(top, join_ml[i][t][0]);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        floatx4 x = {0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < 4; ++i) {
            const float corr = exp2f(join_ml[i][t][0] - base);
            sum += join_ml[i][t][1] * corr;
            x += *reinterpret_cast<const floatx4*>(&join_o[i][t][d]) * corr;
        }
        const size_t head = (size_t)kv * group + rho % group, row = sp.q0 + rho / group;
        const size_t at = head * a.q_rows + row;
        if (tl.ranges == 1) {
            const float inv = rho / group + shift < 0 || sp.kl == 0 ? 0.f : 1.0f / sum;
            store4(out + row * a.o_rs + head * dim, d, dim, a.vec, x * inv);
            if (lse && d == 0) lse[at] = (top + log2f(sum)) * kLn2;
        } else {
            store4(part.o + t * dim, d, dim, false, x);
            if (d == 0) {
                part.ml[2 * t] = top;
                part.ml[2 * t + 1] = sum;
            }
        }
    }
}

// Joins the ranges of the rows whose keys were cut into more than one: a wave per row, four rows of a
// tile per work-group; the ranges' outputs are added in range order.
template <int TILE>
__global__ __launch_bounds__(256) void attn_packed_join_kernel(PackedAttn a, float* __restrict__ out, float* __restrict__ lse,
                                                               float* __restrict__ ws, uint32_t budget, uint32_t items) {
    Work w;
    if (!find_work<false, true>(a, TILE, budget, blockIdx.x, &w)) return;
    const RowTile tl = row_tile(a, w, TILE);
    const int lane = threadIdx.x & 63, t = blockIdx.z * 4 + (threadIdx.x >> 6), rho = tl.rho0 + t;
    if (tl.ranges == 1 || rho > tl.last) return;
    const int dim = a.head_dim, group = a.group, kv = blockIdx.y;
    const size_t head = (size_t)kv * group + rho % group, row = w.sp.q0 + rho / group;
    const Partials part = partials(ws, gridDim.y, kv, items, w.item0, TILE, dim);
    float top = -INFINITY;
    for (int z = lane; z < tl.ranges; z += 64) top = fmaxf(top, part.ml[2 * (z * TILE + t)]);
    top = wave_max(top);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x[2] = {0.f, 0.f};
    for (int z0 = 0; z0 < tl.ranges; z0 += 64) {
        const int z = z0 + lane;
        float corr = 0.f;
        if (z < tl.ranges) {
            corr = exp2f(part.ml[2 * (z * TILE + t)] - base);
            sum += part.ml[2 * (z * TILE + t) + 1] * corr;
        }
        const int n = min(64, tl.ranges - z0);
        for (int i0 = 0; i0 < n; i0 += 8) {
            float y[8][2];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    y[i][e] = lane + 64 * e < dim ? part.o[((size_t)min(z0 + i0 + i, tl.ranges - 1) * TILE + t) * dim + lane + 64 * e] : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float c = __shfl(corr, i0 + i);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (i0 + i < n) x[e] += y[i][e] * c;
            }
        }
    }
    sum = wave_sum(sum);
    const float inv = rho / group + tl.shift < 0 ? 0.f : 1.0f / sum;
    float* dst = out + row * a.o_rs + head * dim;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < dim) dst[lane + 64 * e] = x[e] * inv;
    if (lse && lane == 0) lse[head * a.q_rows + row] = (top + log2f(sum)) * kLn2;
}

// ---- forward ---------------------------------------------------------------------------------

// A work-group per 128 rows of one (sequence, key head), 32 per wave, a row per lane column c; the
// products are taken transposed, S^T = K Q^T and O^T += V^T P^T, so that a lane's probabilities
// are the matrix core's operand as they stand.
template <int DP>
__global__ __launch_bounds__(256) void attn_packed_kernel(PackedAttn a, float* __restrict__ out, float* __restrict__ lse,
                                                          const float* __restrict__ q, const float* __restrict__ k,
                                                          const float* __restrict__ v, float* __restrict__ ws, uint32_t budget) {
    constexpr int KT = 32, KL = DP + 4, VL = DP + 8;
    __shared__ __attribute__((aligned(16))) float ks[KT * KL];
    __shared__ __attribute__((aligned(16))) float vs[KT * VL];
    __shared__ int bad_tile;  // the last tile whose values are not all finite, + 1
    const int kv = blockIdx.x % a.n_kv;
    Work w;
    if (!find_work<false, false>(a, kRowsPerWG, budget, blockIdx.x / a.n_kv, &w)) return;
    const RowTile tl = row_tile(a, w, kRowsPerWG);
    if (w.range >= tl.ranges) return;
    const Span sp = w.sp;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, c = lane & 31;
    const int dim = a.head_dim, group = a.group, rows = tl.rows, shift = tl.shift, k_begin = tl.k_begin, k_end = tl.k_end;
    const int rho = tl.rho0 + wave * kRowsPerWave + c;
    const bool live = rho < rows;
    const int qi = (live ? rho : rows - 1) / group, head = kv * group + (live ? rho : rows - 1) % group;
    const int limit = qi + shift;  // last key this row sees
    const float* kb = k + (size_t)sp.k0 * a.k_rs + (size_t)kv * a.k_hs;
    const float* vb = v + (size_t)sp.k0 * a.v_rs + (size_t)kv * a.v_hs;

    float qr[DP / 2];
    const float* q_row = q + (size_t)(sp.q0 + qi) * a.q_rs + (size_t)head * dim;
#pragma unroll
    for (int u = 0; u < DP / 2; u += 4) {
        const floatx4 x = load4(q_row, h * (DP / 2) + u, dim, a.vec);
#pragma unroll
        for (int e = 0; e < 4; ++e) qr[u + e] = x[e];
    }
    floatx16 o[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float factor = a.scale * kLog2e;
    if (threadIdx.x == 0) bad_tile = 0;
    for (int t0 = k_begin; t0 < k_end; t0 += KT) {
        __syncthreads();
        stage_rows<KT, DP, KL>(ks, kb, a.k_rs, t0, k_end, dim, a.vec);
        if (stage_rows<KT, DP, VL>(vs, vb, a.v_rs, t0, k_end, dim, a.vec) != 0.f) bad_tile = t0 + 1;
        __syncthreads();
        floatx16 s = lds_rows_product<DP, KL>(ks, qr, h, c);
        uint32_t seen = 0;
        float top = m;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] *= factor;
            if (t0 + acc_row(r, h) <= min(limit, k_end - 1)) {
                seen |= 1u << r;
                top = fmaxf(top, s[r]);
            } else {
                s[r] = -INFINITY;
            }
        }
        top = fmaxf(top, __shfl_xor(top, 32));
        const float base = top == -INFINITY ? 0.f : top;  // nothing seen, or scores of -inf alone
        const float corr = exp2f(m - base);
        m = top;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = exp2f(s[r] - base);
            sum += s[r];
        }
        l = l * corr + sum;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] *= corr;
        if (bad_tile == t0 + 1 && __ballot(seen != 0xffffu)) add_seen<DP>(o, s, seen, h, c, DP, true, [&](int n) { return vs + n * VL; });
        else add_product<DP, VL>(o, vs, s, h, c);
    }
    l += __shfl_xor(l, 32);
    if (!live) return;
    const size_t at = (size_t)head * a.q_rows + sp.q0 + qi;
    float inv = limit < 0 || sp.kl == 0 ? 0.f : 1.0f / l;
    float* dst = out + (size_t)(sp.q0 + qi) * a.o_rs + (size_t)head * dim;
    int vec = a.vec;
    if (tl.ranges > 1) {
        const int t = rho - tl.rho0;
        const Partials part = partials(ws, a.n_kv, kv, gridDim.x / a.n_kv, w.item0 + w.range, kRowsPerWG, dim);
        inv = 1.0f;
        dst = part.o + t * dim;
        vec = 0;
        if (h == 0) {
            part.ml[2 * t] = m;
            part.ml[2 * t + 1] = l;
        }
    } else if (lse && h == 0) {
        lse[at] = (m + log2f(l)) * kLn2;
    }
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            floatx4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = o[i][4 * u + e] * inv;
            store4(dst, 32 * i + 8 * u + 4 * h, dim, vec, x);
        }
}

// ---- backward --------------------------------------------------------------------------------

// dq, and d_i of every row for the kernel below: work-groups and lanes as in the forward pass,
// dQ^T += K^T dS^T.
template <int DP>
__global__ __launch_bounds__(256) void attn_packed_dq_kernel(PackedAttn a, float* __restrict__ dq, float* __restrict__ delta,
                                                             const float* __restrict__ dout, const float* __restrict__ out,
                                                             const float* __restrict__ lse, const float* __restrict__ q,
                                                             const float* __restrict__ k, const float* __restrict__ v) {
    constexpr int KT = 32, LD = DP + 4;
    __shared__ __attribute__((aligned(16))) float ks[KT * LD];
    __shared__ __attribute__((aligned(16))) float vs[KT * LD];
    __shared__ int bad_tile;
    const int kv = blockIdx.x % a.n_kv;
    Work w;
    if (!find_work<false, true>(a, kRowsPerWG, 0, blockIdx.x / a.n_kv, &w)) return;
    const RowTile tl = row_tile(a, w, kRowsPerWG);
    const Span sp = w.sp;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, c = lane & 31;
    const int dim = a.head_dim, group = a.group, rows = tl.rows, shift = tl.shift, nkeys = tl.nkeys;
    const int rho = tl.rho0 + wave * kRowsPerWave + c;
    const bool live = rho < rows;
    const int qi = (live ? rho : rows - 1) / group, head = kv * group + (live ? rho : rows - 1) % group;
    const int limit = qi + shift;  // last key this row sees
    const float* kb = k + (size_t)sp.k0 * a.k_rs + (size_t)kv * a.k_hs;
    const float* vb = v + (size_t)sp.k0 * a.v_rs + (size_t)kv * a.v_hs;

    float qr[DP / 2], gr[DP / 2];
    const float* q_row = q + (size_t)(sp.q0 + qi) * a.q_rs + (size_t)head * dim;
    const float* g_row = dout + (size_t)(sp.q0 + qi) * a.o_rs + (size_t)head * dim;
    const float* o_row = out + (size_t)(sp.q0 + qi) * a.o_rs + (size_t)head * dim;
    float d = 0.f;
#pragma unroll
    for (int u = 0; u < DP / 2; u += 4) {
        const int at = h * (DP / 2) + u;
        const floatx4 x = load4(q_row, at, dim, a.vec), g = load4(g_row, at, dim, a.vec), y = load4(o_row, at, dim, a.vec);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            qr[u + e] = x[e];
            gr[u + e] = g[e];
            d += g[e] * y[e];
        }
    }
    d += __shfl_xor(d, 32);
    const size_t stat = (size_t)head * a.q_rows + sp.q0 + qi;
    if (live && h == 0) delta[stat] = d;
    const float lse2 = lse[stat] * kLog2e;
    floatx16 acc[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    const float factor = a.scale * kLog2e;
    if (threadIdx.x == 0) bad_tile = 0;
    for (int t0 = 0; t0 < nkeys; t0 += KT) {
        __syncthreads();
        if (stage_rows<KT, DP, LD>(ks, kb, a.k_rs, t0, nkeys, dim, a.vec) != 0.f) bad_tile = t0 + 1;
        stage_rows<KT, DP, LD>(vs, vb, a.v_rs, t0, nkeys, dim, a.vec);
        __syncthreads();
        const floatx16 s = lds_rows_product<DP, LD>(ks, qr, h, c);
        floatx16 ds = lds_rows_product<DP, LD>(vs, gr, h, c);
        uint32_t seen = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const bool on = t0 + acc_row(r, h) <= limit;
            ds[r] = on ? exp2f(s[r] * factor - lse2) * (ds[r] - d) * a.scale : 0.f;
            seen |= (on ? 1u : 0u) << r;
        }
        if (bad_tile == t0 + 1 && __ballot(seen != 0xffffu)) add_seen<DP>(acc, ds, seen, h, c, DP, true, [&](int n) { return ks + n * LD; });
        else add_product<DP, LD>(acc, ks, ds, h, c);
    }
    if (!live) return;
    float* dst = dq + (size_t)(sp.q0 + qi) * a.q_rs + (size_t)head * dim;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u)
            store4(dst, 32 * i + 8 * u + 4 * h, dim, a.vec,
                   floatx4{acc[i][4 * u], acc[i][4 * u + 1], acc[i][4 * u + 2], acc[i][4 * u + 3]});
}

// dk and dv: a work-group per 128 keys of one (sequence, key head), 32 per wave, a key per lane
// column, K and V in registers; the rows of the group's heads stream through LDS, one head after
// the other: S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS.
template <int DP>
__global__ __launch_bounds__(256) void attn_packed_dkv_kernel(PackedAttn a, float* __restrict__ dk, float* __restrict__ dv,
                                                              const float* __restrict__ delta, const float* __restrict__ dout,
                                                              const float* __restrict__ lse, const float* __restrict__ q,
                                                              const float* __restrict__ k, const float* __restrict__ v) {
    constexpr int RT = 32, LD = DP + 4;
    __shared__ __attribute__((aligned(16))) float qs[RT * LD];
    __shared__ __attribute__((aligned(16))) float gs[RT * LD];
    __shared__ __attribute__((aligned(16))) float stats[2][RT];
    __shared__ int bad_tile;
    const int kv = blockIdx.x % a.n_kv;
    Work w;
    if (!find_work<true, true>(a, kRowsPerWG, 0, blockIdx.x / a.n_kv, &w)) return;
    const Span sp = w.sp;
    const int tile = w.tile;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, c = lane & 31;
    const int dim = a.head_dim, group = a.group;
    const int key = tile * kRowsPerWG + wave * kRowsPerWave + c;
    const bool live = key < (int)sp.kl;
    const int shift = (int)sp.kl - (int)sp.ql;
    const size_t row = sp.k0 + (live ? key : (int)sp.kl - 1);
    float kr[DP / 2], vr[DP / 2];
#pragma unroll
    for (int u = 0; u < DP / 2; u += 4) {
        const int at = h * (DP / 2) + u;
        const floatx4 x = load4(k + row * a.k_rs + (size_t)kv * a.k_hs, at, dim, a.vec);
        const floatx4 y = load4(v + row * a.v_rs + (size_t)kv * a.v_hs, at, dim, a.vec);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            kr[u + e] = x[e];
            vr[u + e] = y[e];
        }
    }
    floatx16 ak[DP / 32], av[DP / 32];
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) ak[i][r] = av[i][r] = 0.f;
    const float factor = a.scale * kLog2e;
    if (threadIdx.x == 0) bad_tile = 0;
    const int first = max(0, tile * kRowsPerWG - shift) / RT * RT;  // the first row that sees a key of the tile
    int pass = 0;
    for (int g = 0; g < group; ++g) {
        const int head = kv * group + g;
        const float* qb = q + (size_t)sp.q0 * a.q_rs + (size_t)head * dim;
        const float* gb = dout + (size_t)sp.q0 * a.o_rs + (size_t)head * dim;
        const size_t stat = (size_t)head * a.q_rows + sp.q0;
        for (int i0 = first; i0 < (int)sp.ql; i0 += RT) {
            ++pass;
            __syncthreads();
            float bad = stage_rows<RT, DP, LD>(qs, qb, a.q_rs, i0, sp.ql, dim, a.vec);
            bad += stage_rows<RT, DP, LD>(gs, gb, a.o_rs, i0, sp.ql, dim, a.vec);
            if (threadIdx.x < RT) {
                const bool in = i0 + threadIdx.x < sp.ql;
                stats[0][threadIdx.x] = in ? lse[stat + i0 + threadIdx.x] * kLog2e : 0.f;
                stats[1][threadIdx.x] = in ? delta[stat + i0 + threadIdx.x] : 0.f;
            }
            if (bad != 0.f) bad_tile = pass;
            __syncthreads();
            floatx16 p = lds_rows_product<DP, LD>(qs, kr, h, c);
            floatx16 ds = lds_rows_product<DP, LD>(gs, vr, h, c);
            uint32_t seen = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = acc_row(r, h);
                const bool on = key <= i0 + i + shift && i0 + i < (int)sp.ql;
                p[r] = on ? exp2f(p[r] * factor - stats[0][i]) : 0.f;
                ds[r] = on ? p[r] * (ds[r] - stats[1][i]) * a.scale : 0.f;
                seen |= (on ? 1u : 0u) << r;
            }
            if (bad_tile == pass && __ballot(seen != 0xffffu)) {
                add_seen<DP>(av, p, seen, h, c, DP, true, [&](int n) { return gs + n * LD; });
                add_seen<DP>(ak, ds, seen, h, c, DP, true, [&](int n) { return qs + n * LD; });
            } else {
                add_product<DP, LD>(av, gs, p, h, c);
                add_product<DP, LD>(ak, qs, ds, h, c);
            }
        }
    }
    if (!live) return;
    float* dkr = dk + row * a.k_rs + (size_t)kv * a.k_hs;
    float* dvr = dv + row * a.v_rs + (size_t)kv * a.v_hs;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int at = 32 * i + 8 * u + 4 * h;
            store4(dkr, at, dim, a.vec, floatx4{ak[i][4 * u], ak[i][4 * u + 1], ak[i][4 * u + 2], ak[i][4 * u + 3]});
            store4(dvr, at, dim, a.vec, floatx4{av[i][4 * u], av[i][4 * u + 1], av[i][4 * u + 2], av[i][4 * u + 3]});
        }
}

// ---- host ------------------------------------------------------------------------------------

// A launch's threads stay inside 32 bits.
constexpr uint32_t kMaxRows = 1u << 30, kMaxSeqs = 1u << 22;

int check_shape(const char* fn, const fmlh_packed_attention* s) {
    FMLH_REQUIRE(s != nullptr, "%s: null shape", fn);
    FMLH_REQUIRE(s->n_head >= 1 && s->n_kv_head >= 1 && s->n_head % s->n_kv_head == 0 && s->n_head <= 65535,
                 "%s: %u query heads on %u key heads (a multiple, up to 65535)", fn, s->n_head, s->n_kv_head);
    FMLH_REQUIRE(s->head_dim >= 1 && s->head_dim <= 128, "%s: head_dim %u outside 1..128", fn, s->head_dim);
    FMLH_REQUIRE(s->q_rows <= kMaxRows && s->k_rows <= kMaxRows, "%s: more than 2^30 rows", fn);
    FMLH_REQUIRE(s->n_seq <= kMaxSeqs, "%s: more than 2^22 sequences", fn);
    FMLH_REQUIRE((uint64_t)s->q_rows * (s->n_head / s->n_kv_head) <= kMaxRows, "%s: more than 2^30 rows of a group", fn);
    FMLH_REQUIRE(s->scale == s->scale && s->scale - s->scale == 0.f, "%s: scale is not finite", fn);
    const size_t row = (size_t)s->n_head * s->head_dim;
    FMLH_REQUIRE(s->q_rs >= row && s->o_rs >= row, "%s: rows of q (%zu) and out (%zu) hold %zu floats", fn, s->q_rs, s->o_rs,
                 row);
    FMLH_REQUIRE(s->k_rs >= s->head_dim && s->v_rs >= s->head_dim, "%s: row strides of k (%zu) and v (%zu) below head_dim", fn,
                 s->k_rs, s->v_rs);
    FMLH_REQUIRE(s->n_kv_head == 1 || (s->k_hs >= s->head_dim && s->v_hs >= s->head_dim),
                 "%s: head strides of k (%zu) and v (%zu) below head_dim", fn, s->k_hs, s->v_hs);
    for (size_t x : {s->q_rs, s->o_rs, s->k_rs, s->v_rs, s->k_hs, s->v_hs})
        FMLH_REQUIRE(x < (size_t(1) << 32), "%s: a stride of %zu floats", fn, x);
    FMLH_REQUIRE(s->n_seq == 0 || (s->q_off && s->k_off), "%s: null offsets", fn);
    return FMLH_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

PackedAttn make_args(const fmlh_packed_attention* s) {
    PackedAttn a{};
    a.n_seq = s->n_seq;
    a.q_rows = s->q_rows;
    a.k_rows = s->k_rows;
    a.group = s->n_head / s->n_kv_head;
    a.n_kv = s->n_kv_head;
    a.head_dim = s->head_dim;
    a.scale = s->scale;
    a.q_off = s->q_off;
    a.k_off = s->k_off;
    a.k_len = s->k_len;
    a.q_rs = s->q_rs;
    a.k_rs = s->k_rs;
    a.v_rs = s->v_rs;
    a.o_rs = s->o_rs;
    a.k_hs = s->k_hs;
    a.v_hs = s->v_hs;
    a.vec = s->head_dim % 4 == 0 && ((s->q_rs | s->k_rs | s->v_rs | s->o_rs) & 3) == 0 &&
            (s->n_kv_head == 1 || ((s->k_hs | s->v_hs) & 3) == 0);
    return a;
}

uint32_t row_tiles(const PackedAttn& a, uint32_t per) { return (uint32_t)(((uint64_t)a.q_rows * a.group) / per) + a.n_seq; }
uint32_t key_tiles(const PackedAttn& a) { return a.k_rows / kRowsPerWG + a.n_seq; }

// Sequences of fewer keys are not cut: joining the ranges costs a launch of 5 us.
constexpr uint64_t kCutKeys = 512;

// Keys that a sequence has room for, on average (a cache in slabs holds a head's rows one behind the other).
uint64_t keys_per_sequence(const PackedAttn& a) {
    const uint64_t n = a.k_rows / a.n_seq;
    return a.k_hs > a.k_rs ? n / a.n_kv : n;
}

// How the forward pass cuts its work, by the sizes alone (lengths are the device's to know).
struct ForwardPlan {
    int per;          // rows per tile: kRowsPerWG, or at most 8 for attn_packed_few_kernel
    uint32_t tiles;   // at most, for a key head
    uint32_t budget;  // ranges to cut the tiles' keys into, for a key head; 0: none
};

ForwardPlan plan_forward(const PackedAttn& a) {
    ForwardPlan p;
    const uint64_t rows = (uint64_t)a.q_rows * a.group;  // of a key head
    const uint64_t per_seq = rows / a.n_seq;
    p.per = per_seq > 8 ? kRowsPerWG : per_seq > 4 ? 8 : per_seq > 2 ? 4 : per_seq > 1 ? 2 : 1;
    p.tiles = row_tiles(a, p.per);
    const uint64_t about = std::max<uint64_t>(a.n_seq, (rows + p.per - 1) / p.per) * a.n_kv;
    const uint64_t want = p.per <= 8 ? 1024 : 512;  // work-groups that keep the device busy
    p.budget = 2 * about <= want && keys_per_sequence(a) >= kCutKeys ? (uint32_t)(want / a.n_kv) : 0;
    return p;
}

// Work-groups of a launch, all key heads': its threads stay inside 32 bits.
constexpr uint64_t kMaxGroups = 1u << 23;

// How the backward pass cuts the rows that a tile of keys sees.
int plan_parts(const PackedAttn& a) {
    const uint64_t tiles = std::max<uint64_t>(std::min(a.n_seq, key_tiles(a)), a.k_rows / kRowsPerWG) * a.n_kv;
    const uint64_t want = 1024;          // work-groups that keep the device busy although early keys see more rows than late ones
    const size_t most = size_t(1) << 26;  // floats of partial sums
    const uint64_t fit = std::max<uint64_t>(1, most / std::max<size_t>(1, attn_split_part_floats(a, key_tiles(a))));
    // A part has some tiles of rows to do on average.
    const uint64_t steps = (uint64_t)a.q_rows / a.n_seq * a.group / 160;
    return (int)std::min<uint64_t>({16, fit, std::max<uint64_t>(1, steps), std::max<uint64_t>(1, want / std::max<uint64_t>(1, tiles))});
}

size_t deltas(const PackedAttn& a) { return ((size_t)a.n_kv * a.group * a.q_rows + 3) / 4 * 4; }  // d_i, in whole 16 bytes

size_t workspace(const PackedAttn& a, bool backward) {
    if (a.n_seq == 0) return 0;
    const ForwardPlan p = plan_forward(a);
    const size_t forward = p.budget ? (size_t)a.n_kv * (p.tiles + p.budget) * p.per * (a.head_dim + 2) : 0;
    if (!backward) return forward;
    const int parts = plan_parts(a);
    return std::max(forward, deltas(a) + (parts > 1 ? parts * attn_split_part_floats(a, key_tiles(a)) : 0));
}

}  // namespace

}  // namespace fmlh

using namespace fmlh;

#define FMLH_BY_DIM(LAUNCH)                        \
    do {                                           \
        if (a.head_dim <= 32) LAUNCH(32);          \
        else if (a.head_dim <= 64) LAUNCH(64);     \
        else if (a.head_dim <= 96) LAUNCH(96);     \
        else LAUNCH(128);                          \
    } while (0)

extern "C" {

int fmlh_attention_packed_workspace(const fmlh_packed_attention* shape, int backward, size_t* floats) {
    FMLH_REQUIRE(floats != nullptr, "fmlh_attention_packed_workspace: null output pointer");
    FMLH_TRY(check_shape("fmlh_attention_packed_workspace", shape));
    *floats = workspace(make_args(shape), backward != 0);
    return FMLH_OK;
}

int fmlh_attention_packed(const fmlh_packed_attention* shape, float* out, float* lse, const float* q, const float* k,
                          const float* v, float* ws, size_t ws_floats) {
    const char* fn = "fmlh_attention_packed";
    FMLH_TRY(check_shape(fn, shape));
    if (shape->n_seq == 0 || shape->q_rows == 0) return FMLH_OK;
    FMLH_REQUIRE(out && q, "%s: null pointer", fn);
    FMLH_REQUIRE(shape->k_rows == 0 || (k && v), "%s: null keys or values", fn);
    FMLH_TRY(ensure_init());
    PackedAttn a = make_args(shape);
    const size_t need = workspace(a, false);
    FMLH_REQUIRE(need == 0 || (ws && ws_floats >= need), "%s: a workspace of %zu floats is needed", fn, need);
    a.vec = a.vec && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out);
    const ForwardPlan plan = plan_forward(a);
    const uint32_t items = plan.tiles + plan.budget;
    FMLH_REQUIRE((uint64_t)items * a.n_kv <= kMaxGroups, "%s: more than 2^23 tiles of rows", fn);
    if (plan.per <= 8) {
        const dim3 grid(items, a.n_kv);
#define FMLH_FEW(LPK, NF, RT) \
    hipLaunchKernelGGL((attn_packed_few_kernel<LPK, NF, RT>), grid, dim3(256), 0, stream(), a, out, lse, q, k, v, ws, plan.budget)
#define FMLH_FEW_ROWS(LPK, NF)                       \
    do {                                             \
        if (plan.per == 1) FMLH_FEW(LPK, NF, 1);      \
        else if (plan.per == 2) FMLH_FEW(LPK, NF, 2); \
        else if (plan.per == 4) FMLH_FEW(LPK, NF, 4); \
        else FMLH_FEW(LPK, NF, 8);                    \
    } while (0)
        if (a.head_dim <= 16) FMLH_FEW_ROWS(4, 1);
        else if (a.head_dim <= 32) FMLH_FEW_ROWS(8, 1);
        else if (a.head_dim <= 64) FMLH_FEW_ROWS(16, 1);
        else FMLH_FEW_ROWS(16, 2);
#undef FMLH_FEW_ROWS
#undef FMLH_FEW
        FMLH_LAUNCHED("attn_packed_few_kernel");
    } else if (!getenv("FMLH_PLAIN")) {
        FMLH_TRY(attn_split_forward(a, items, plan.budget, out, lse, q, k, v, ws, stream()));
    } else {
#define FMLH_LAUNCH(DP)                                                                                                \
    hipLaunchKernelGGL(attn_packed_kernel<DP>, dim3(items * a.n_kv), dim3(256), 0, stream(), a, out, lse, q, k, v, ws, \
                       plan.budget)
        FMLH_BY_DIM(FMLH_LAUNCH);
#undef FMLH_LAUNCH
        FMLH_LAUNCHED("attn_packed_kernel");
    }
    if (plan.budget) {
#define FMLH_JOIN(TILE)                                                                                                      \
    hipLaunchKernelGGL(attn_packed_join_kernel<TILE>, dim3(plan.tiles, a.n_kv, (TILE + 3) / 4), dim3(256), 0, stream(), a, out, \
                       lse, ws, plan.budget, items)
        switch (plan.per) {
            case 1: FMLH_JOIN(1); break;
            case 2: FMLH_JOIN(2); break;
            case 4: FMLH_JOIN(4); break;
            case 8: FMLH_JOIN(8); break;
            default: FMLH_JOIN(kRowsPerWG); break;
        }
#undef FMLH_JOIN
        FMLH_LAUNCHED("attn_packed_join_kernel");
    }
    return FMLH_OK;
}

int fmlh_attention_packed_backward(const fmlh_packed_attention* shape, float* dq, float* dk, float* dv, const float* dout,
                                   const float* out, const float* lse, const float* q, const float* k, const float* v,
                                   float* ws, size_t ws_floats) {
    const char* fn = "fmlh_attention_packed_backward";
    FMLH_TRY(check_shape(fn, shape));
    if (shape->n_seq == 0 || (shape->q_rows == 0 && shape->k_rows == 0)) return FMLH_OK;
    FMLH_REQUIRE(shape->q_rows == 0 || (dq && dout && out && lse && q), "%s: null pointer", fn);
    FMLH_REQUIRE(shape->k_rows == 0 || (dk && dv && k && v), "%s: null pointer", fn);
    FMLH_TRY(ensure_init());
    PackedAttn a = make_args(shape);
    const int parts = plan_parts(a);
    const size_t need = deltas(a) + (parts > 1 ? parts * attn_split_part_floats(a, key_tiles(a)) : 0);
    FMLH_REQUIRE(need == 0 || (ws && ws_floats >= need), "%s: a workspace of %zu floats is needed", fn, need);
    FMLH_REQUIRE((uint64_t)std::max(row_tiles(a, kRowsPerWG), key_tiles(a)) * a.n_kv <= kMaxGroups, "%s: more than 2^23 tiles of rows or keys", fn);
    a.vec = a.vec && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(dout) && aligned16(dq) &&
            aligned16(dk) && aligned16(dv);
    FMLH_REQUIRE((uintptr_t)ws % 16 == 0, "%s: the workspace is not 16-byte aligned", fn);
    if (!getenv("FMLH_PLAIN")) {
        if (shape->q_rows) FMLH_TRY(attn_split_dq(a, row_tiles(a, kRowsPerWG), dq, ws, dout, out, lse, q, k, v, stream()));
        if (shape->k_rows) FMLH_TRY(attn_split_dkv(a, key_tiles(a), parts, dk, dv, ws, dout, lse, q, k, v, ws + deltas(a), stream()));
        return FMLH_OK;
    }
    if (shape->q_rows) {
        const dim3 grid(row_tiles(a, kRowsPerWG) * a.n_kv);
#define FMLH_LAUNCH(DP) \
    hipLaunchKernelGGL(attn_packed_dq_kernel<DP>, grid, dim3(256), 0, stream(), a, dq, ws, dout, out, lse, q, k, v)
        FMLH_BY_DIM(FMLH_LAUNCH);
#undef FMLH_LAUNCH
        FMLH_LAUNCHED("attn_packed_dq_kernel");
    }
    if (shape->k_rows) {
        const dim3 grid(key_tiles(a) * a.n_kv);
#define FMLH_LAUNCH(DP) \
    hipLaunchKernelGGL(attn_packed_dkv_kernel<DP>, grid, dim3(256), 0, stream(), a, dk, dv, ws, dout, lse, q, k, v)
        FMLH_BY_DIM(FMLH_LAUNCH);
#undef FMLH_LAUNCH
        FMLH_LAUNCHED("attn_packed_dkv_kernel");
    }
    return FMLH_OK;
}

}  // extern "C"
