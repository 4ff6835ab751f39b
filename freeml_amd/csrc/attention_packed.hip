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
#include "attention_packed.h"
#include "bf16_split.h"

#include <algorithm>

namespace fmlh {

namespace {

constexpr int kRowsPerWave = 32;
constexpr int kRowsPerWG = 4 * kRowsPerWave;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ uint32_t clamp_row(int32_t v, uint32_t rows) {
    return v < 0 ? 0u : min((uint32_t)v, rows);
}

// A sequence's rows: offsets outside [0, rows] or falling are cut to what lies inside.
struct Span {
    uint32_t q0, ql, k0, kl;
};

__device__ __forceinline__ Span load_span(const PackedAttn& a, uint32_t s) {
    Span p;
    p.q0 = clamp_row(a.q_off[s], a.q_rows);
    const uint32_t q1 = clamp_row(a.q_off[s + 1], a.q_rows);
    p.ql = q1 > p.q0 ? q1 - p.q0 : 0u;
    p.k0 = clamp_row(a.k_off[s], a.k_rows);
    const uint32_t k1 = clamp_row(a.k_off[s + 1], a.k_rows);
    p.kl = k1 > p.k0 ? k1 - p.k0 : 0u;
    if (a.k_len) p.kl = min(p.kl, (uint32_t)max(a.k_len[s], 0));
    return p;
}

// The sequence that tile `t` of the launch falls to, where sequence s has ceil(count_s / per) tiles
// (count: its keys, or its rows of all heads of a group): every wave scans the offsets, 64
// sequences at a time.  Returns false for tiles behind the last sequence (the grid holds
// sum / per + n_seq tiles, never fewer than there are).
template <bool KEYS>
__device__ __forceinline__ bool find_tile(const PackedAttn& a, uint32_t per, uint32_t t, Span* span, uint32_t* tile,
                                          uint32_t* tiles) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (uint32_t base = 0; base < a.n_seq; base += 64) {
        const uint32_t s = base + lane;
        uint32_t n = 0;
        if (s < a.n_seq) {
            const Span p = load_span(a, s);
            n = (uint32_t)(((uint64_t)(KEYS ? p.kl : p.ql) * (KEYS ? 1u : a.group) + per - 1) / per);
        }
        uint32_t upto = n;  // inclusive scan
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(upto, d);
            if (lane >= (uint32_t)d) upto += o;
        }
        const uint64_t hit = __ballot(before + upto > t);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const uint32_t first = before + __shfl(upto - n, l);
            *tiles = __shfl(n, l);
            *tile = t - first;
            *span = load_span(a, base + l);
            return true;
        }
        before += __shfl(upto, 63);
    }
    return false;
}

// Dims 4 u .. 4 u + 3 of a row, zeros past head_dim.
__device__ __forceinline__ floatx4 load4(const float* row, int d, int dim, bool vec) {
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
    if (vec) {
        if (d < dim) v = *reinterpret_cast<const floatx4*>(row + d);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < dim) v[e] = row[d + e];
    }
    return v;
}

__device__ __forceinline__ void store4(float* row, int d, int dim, bool vec, floatx4 v) {
    if (vec) {
        if (d < dim) *reinterpret_cast<floatx4*>(row + d) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < dim) row[d + e] = v[e];
    }
}

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

// Register r of a lane's 32 x 32 accumulator is row 8 (r / 4) + 4 h + r % 4 of it.
__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// S (32 x 32) = A B^T over DP dims: A's rows from LDS (row stride LD), B's row of lane column c in
// registers (dims h DP / 2 ..).  The matrix core's two k of a step are dims u and DP / 2 + u.
template <int DP, int LD>
__device__ __forceinline__ floatx16 rows_product(const float* lds_rows, const float (&b)[DP / 2], int h, int c) {
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

// The same element by element, over the pairs `seen` names only (bit r of lane (h, c): row
// acc_row(r, h), column c).  Rolled up: it runs for tiles that are rare.
template <int DP, int LD>
__device__ __forceinline__ void add_seen(floatx16 (&acc)[DP / 32], const float* lds_rows, const floatx16& w, uint32_t seen, int h,
                                         int c) {
#pragma unroll 1
    for (int n = 0; n < 32; ++n) {
        const int r = n >> 1, from = c + 32 * (n & 1);
        float mine = 0.f;
#pragma unroll
        for (int t = 0; t < 16; ++t) mine = t == r ? w[t] : mine;
        const float p = __shfl(mine, from);
        const bool on = (__shfl((int)seen, from) >> r) & 1;
        const float* x = lds_rows + acc_row(r, n & 1) * LD;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][e] += on ? p * x[32 * i + acc_row(e, h)] : 0.f;
    }
}

// ---- forward ---------------------------------------------------------------------------------

// A work-group per 128 rows of one (sequence, key head), 32 per wave, a row per lane column c; the
// products are taken transposed, S^T = K Q^T and O^T += V^T P^T, so that a lane's probabilities
// are the matrix core's operand as they stand.
template <int DP>
__global__ __launch_bounds__(256) void attn_packed_kernel(PackedAttn a, float* __restrict__ out, float* __restrict__ lse,
                                                          const float* __restrict__ q, const float* __restrict__ k,
                                                          const float* __restrict__ v) {
    constexpr int KT = 32, KL = DP + 4, VL = DP + 8;
    __shared__ __attribute__((aligned(16))) float ks[KT * KL];
    __shared__ __attribute__((aligned(16))) float vs[KT * VL];
    __shared__ int bad_tile;  // the last tile whose values are not all finite, + 1
    Span sp;
    uint32_t tile, tiles;
    if (!find_tile<false>(a, kRowsPerWG, blockIdx.x, &sp, &tile, &tiles)) return;
    tile = tiles - 1 - tile;  // longest first
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, c = lane & 31;
    const int dim = a.head_dim, group = a.group, kv = blockIdx.y;
    const uint32_t rows = sp.ql * group;
    const uint32_t rho0 = tile * kRowsPerWG, rho = rho0 + wave * kRowsPerWave + c;
    const bool live = rho < rows;
    const uint32_t qi = (live ? rho : rows - 1) / group;
    const int head = kv * group + (live ? rho : rows - 1) % group;
    const int shift = (int)sp.kl - (int)sp.ql;
    const int limit = (int)qi + shift;  // last key this row sees
    const uint32_t last_qi = min(rho0 + kRowsPerWG - 1, rows - 1) / group;
    const int nkeys = min((int)last_qi + shift + 1, (int)sp.kl);  // keys the work-group needs
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
    for (int t0 = 0; t0 < nkeys; t0 += KT) {
        __syncthreads();
        stage_rows<KT, DP, KL>(ks, kb, a.k_rs, t0, nkeys, dim, a.vec);
        if (stage_rows<KT, DP, VL>(vs, vb, a.v_rs, t0, nkeys, dim, a.vec) != 0.f) bad_tile = t0 + 1;
        __syncthreads();
        floatx16 s = rows_product<DP, KL>(ks, qr, h, c);
        uint32_t seen = 0;
        float top = m;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] *= factor;
            if (t0 + acc_row(r, h) <= limit) {
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
        if (bad_tile == t0 + 1 && __ballot(seen != 0xffffu)) add_seen<DP, VL>(o, vs, s, seen, h, c);
        else add_product<DP, VL>(o, vs, s, h, c);
    }
    l += __shfl_xor(l, 32);
    if (!live) return;
    const float inv = limit < 0 || sp.kl == 0 ? 0.f : 1.0f / l;
    float* dst = out + (size_t)(sp.q0 + qi) * a.o_rs + (size_t)head * dim;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            floatx4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = o[i][4 * u + e] * inv;
            store4(dst, 32 * i + 8 * u + 4 * h, dim, a.vec, x);
        }
    if (lse && h == 0) lse[(size_t)head * a.q_rows + sp.q0 + qi] = (m + log2f(l)) * kLn2;
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
    Span sp;
    uint32_t tile, tiles;
    if (!find_tile<false>(a, kRowsPerWG, blockIdx.x, &sp, &tile, &tiles)) return;
    tile = tiles - 1 - tile;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, c = lane & 31;
    const int dim = a.head_dim, group = a.group, kv = blockIdx.y;
    const uint32_t rows = sp.ql * group;
    const uint32_t rho0 = tile * kRowsPerWG, rho = rho0 + wave * kRowsPerWave + c;
    const bool live = rho < rows;
    const uint32_t qi = (live ? rho : rows - 1) / group;
    const int head = kv * group + (live ? rho : rows - 1) % group;
    const int shift = (int)sp.kl - (int)sp.ql;
    const int limit = (int)qi + shift;
    const uint32_t last_qi = min(rho0 + kRowsPerWG - 1, rows - 1) / group;
    const int nkeys = min((int)last_qi + shift + 1, (int)sp.kl);
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
        const floatx16 s = rows_product<DP, LD>(ks, qr, h, c);
        floatx16 ds = rows_product<DP, LD>(vs, gr, h, c);
        uint32_t seen = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const bool on = t0 + acc_row(r, h) <= limit;
            ds[r] = on ? exp2f(s[r] * factor - lse2) * (ds[r] - d) * a.scale : 0.f;
            seen |= (on ? 1u : 0u) << r;
        }
        if (bad_tile == t0 + 1 && __ballot(seen != 0xffffu)) add_seen<DP, LD>(acc, ks, ds, seen, h, c);
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
    Span sp;
    uint32_t tile, tiles;
    if (!find_tile<true>(a, kRowsPerWG, blockIdx.x, &sp, &tile, &tiles)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, c = lane & 31;
    const int dim = a.head_dim, group = a.group, kv = blockIdx.y;
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
    const int first = max(0, (int)tile * kRowsPerWG - shift) / RT * RT;  // the first row that sees a key of the tile
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
            floatx16 p = rows_product<DP, LD>(qs, kr, h, c);
            floatx16 ds = rows_product<DP, LD>(gs, vr, h, c);
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
                add_seen<DP, LD>(av, gs, p, seen, h, c);
                add_seen<DP, LD>(ak, qs, ds, seen, h, c);
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

uint32_t row_tiles(const PackedAttn& a) { return (uint32_t)(((uint64_t)a.q_rows * a.group) / kRowsPerWG) + a.n_seq; }
uint32_t key_tiles(const PackedAttn& a) { return a.k_rows / kRowsPerWG + a.n_seq; }

size_t workspace(const PackedAttn& a, uint32_t n_head, bool backward) {
    return backward ? (size_t)n_head * a.q_rows : 0;  // d_i
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
    *floats = workspace(make_args(shape), shape->n_head, backward != 0);
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
    const size_t need = workspace(a, shape->n_head, false);
    FMLH_REQUIRE(need == 0 || (ws && ws_floats >= need), "%s: a workspace of %zu floats is needed", fn, need);
    a.vec = a.vec && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out);
    const dim3 grid(row_tiles(a), shape->n_kv_head);
#define FMLH_LAUNCH(DP) hipLaunchKernelGGL(attn_packed_kernel<DP>, grid, dim3(256), 0, stream(), a, out, lse, q, k, v)
    FMLH_BY_DIM(FMLH_LAUNCH);
#undef FMLH_LAUNCH
    FMLH_LAUNCHED("attn_packed_kernel");
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
    const size_t need = workspace(a, shape->n_head, true);
    FMLH_REQUIRE(need == 0 || (ws && ws_floats >= need), "%s: a workspace of %zu floats is needed", fn, need);
    a.vec = a.vec && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(dout) && aligned16(dq) &&
            aligned16(dk) && aligned16(dv);
    if (shape->q_rows) {
        const dim3 grid(row_tiles(a), shape->n_kv_head);
#define FMLH_LAUNCH(DP) \
    hipLaunchKernelGGL(attn_packed_dq_kernel<DP>, grid, dim3(256), 0, stream(), a, dq, ws, dout, out, lse, q, k, v)
        FMLH_BY_DIM(FMLH_LAUNCH);
#undef FMLH_LAUNCH
        FMLH_LAUNCHED("attn_packed_dq_kernel");
    }
    if (shape->k_rows) {
        const dim3 grid(key_tiles(a), shape->n_kv_head);
#define FMLH_LAUNCH(DP) \
    hipLaunchKernelGGL(attn_packed_dkv_kernel<DP>, grid, dim3(256), 0, stream(), a, dk, dv, ws, dout, lse, q, k, v)
        FMLH_BY_DIM(FMLH_LAUNCH);
#undef FMLH_LAUNCH
        FMLH_LAUNCHED("attn_packed_dkv_kernel");
    }
    return FMLH_OK;
}

}  // extern "C"
