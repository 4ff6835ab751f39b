// The packed attention kernels on the bf16 matrix cores: forward, dq, and dk / dv (attention_packed.hip
// has the formulas and the layout of tiles and lanes).
//
// Every operand is written exactly as three bf16 parts (bf16_split.h) and the six part products of
// weight 2^-16 and more are summed in fp32 by v_mfma_f32_32x32x16_bf16: 6 x 32 clocks per 32 x 32 x 16
// block where the fp32 matrix cores need 512.
//   * Operands are staged times 2^24, so that every part of every fp32 number is zero or normal; sums
//     carry 2^48 and are taken back.  What leaves the range at the upper end (elements from 2^104, sums
//     from 2^80), and infinities and NaN, masked ones included, show as a result that is not finite:
//     that wave does its rows or keys again, on the fp32 matrix cores and element by element, from memory.
//   * A tile's rows lie in LDS as bf16 planes, 16-byte units of 8 dims: unit o of row r at o ^ swz(r), so
//     that 8 lanes on one unit of 8 rows touch distinct banks.  Products over the dims read them by
//     row; products over the rows read them transposed (ds_read_b64_tr_b16: lanes 4 r .. 4 r + 3 of 16
//     name 16 dims of row r, lane i gets dim i of 4 rows), so one copy serves both.
//   * A lane's accumulator registers 8 t .. 8 t + 7 are rows 16 t + 4 h + {0..3, 8..11} of its column:
//     taking the rows in this order as the 8 k of a half makes probabilities and their gradients
//     the next product's operand without leaving the registers.
//   * A tile's rows are requested into registers while the tile before them is multiplied, by buffer loads whose
//     range check gives the zeros behind a sequence or a head (with the zeros chosen after an ordinary load every
//     such tile waited for its values: 48 queries over 500 .. 4000 keys, 16 heads of 80 on 4, 41.4 us, 37.5 so).
//
// What bounds them: at 8 x 4096 rows, 16 heads of 64, the forward pass runs at 178 TFLOP/s of the 234 that a
// sixth of a large bf16 product is (matrix cores 54% and vector units 60% of the clocks, which the power
// limit holds at 1.9 GHz); the fp32 matrix cores' 151 would leave 97.  The backward pass forms seven products
// for the five that have to be (S and dP twice, so that no sum crosses work-groups): 131 TFLOP/s of the five,
// 184 of the seven.  Short sequences are bound by the chain of one wave: offsets, loads, S, softmax, P V, 10 us for one tile.
// Measured and not kept: the next tile's S among this one's softmax, in program order or by scheduling
// groups (D 64 -2 .. +4%, D 128 +9%, shorter sequences 5 - 10% slower); pairs of waves for dq up to
// head_dim 64 (8 x 4096 rows, 16 heads: 5.76 ms for the pass, 5.22); keys cut into ranges from 256 tiles on.
#include "attention_packed_device.h"

namespace fmlh {

namespace {

constexpr float kUp = 0x1p24f, kDown2 = 0x1p-48f;

template <int DP>
struct Shape {
    static constexpr int U = DP / 8;      // 16-byte units per row and plane
    static constexpr int KS = DP / 16;    // steps of a product over the dims
    static constexpr int NB = DP / 32;    // blocks of 32 dims
    __device__ static __forceinline__ int swz(int r) { return U % 8 == 0 ? (r & 7) : ((r >> 2) & 3); }
};

// R rows of a matrix in the registers of NT threads (a thread's share) and from there as planes in LDS.
template <int R, int DP, bool VEC, int NT = 256>
struct Stage {
    static constexpr int U = DP / 8, N = (R * U + NT - 1) / NT;
    floatx4 x[N][2];
    // Rows first .. of a matrix at base (64-bit, uniform), row stride rs; rows from `rows` on (rows > first) and
    // dims from `dim` on are zeros.  VEC: by buffer loads, whose range check gives the zeros, so that no value is
    // waited for here; offsets stay inside 31 bits (kMaxVecStride).
    __device__ __forceinline__ void load(const float* base, size_t rs, int first, int rows, int dim) {
        const int t = threadIdx.x & (NT - 1);
        const float* tile = base + (size_t)first * rs;
        const int left = min(rows - first, R);
        if constexpr (VEC) {
            const int stride = (int)rs * 4, bytes = __builtin_amdgcn_readfirstlane((left - 1) * stride + 4 * dim);
            const uint64_t start = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)((uint64_t)tile >> 32)) << 32 |
                                   (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint64_t)tile);
            const __amdgpu_buffer_rsrc_t buffer = __builtin_amdgcn_make_buffer_rsrc((float*)start, 0, bytes, 0x00020000);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int u = t + NT * i, d = 8 * (u % U), at = u / U * stride + 4 * d;
                x[i][0] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(buffer, d < dim ? at : bytes, 0, 0));
                x[i][1] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(buffer, d + 4 < dim ? at + 16 : bytes, 0, 0));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int u = min(t + NT * i, R * U - 1), r = u / U, d = 8 * (u % U);
                const bool on = r < left;
                const float* row = tile + (size_t)(on ? r : 0) * rs;
                x[i][0] = load4_padded<false>(row, d, dim, on);
                x[i][1] = load4_padded<false>(row, d + 4, dim, on);
            }
        }
    }
    __device__ __forceinline__ void store(uintx4* planes) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = (threadIdx.x & (NT - 1)) + NT * i, r = u / U;
            if (R * U % NT != 0 && u >= R * U) break;
            const float v[8] = {x[i][0][0], x[i][0][1], x[i][0][2], x[i][0][3], x[i][1][0], x[i][1][1], x[i][1][2], x[i][1][3]};
            uintx4 p[3];
            split8(v, p, kUp);
#pragma unroll
            for (int q = 0; q < 3; ++q) planes[(q * R + r) * U + ((u % U) ^ Shape<DP>::swz(r))] = p[q];
        }
    }
};

// Row `row` of a tile as the matrix core's operand of dims 16 st + 8 h ..
template <int R, int DP>
__device__ __forceinline__ bf16x8 row_operand(const uintx4* planes, int q, int row, int st, int h) {
    constexpr int U = DP / 8;
    return __builtin_bit_cast(bf16x8, planes[(q * R + row) * U + ((2 * st + h) ^ Shape<DP>::swz(row))]);
}

// Dim 32 i + lane % 32 of rows row0 + 4 h + {0..3, 8..11} of a tile.
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));
template <int R, int DP>
__device__ __forceinline__ bf16x8 column_operand(const uintx4* planes, int q, int row0, int i, int lane) {
    constexpr int U = DP / 8;
    const int row = row0 + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int unit = 4 * i + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
    auto at = [&](int r) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_shortx4*)(planes + (q * R + r) * U + (unit ^ Shape<DP>::swz(r))) + (lane & 1));
    };
    const shortx4 lo = at(row), hi = at(row + 8);
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A lane's row as operand of products over the dims: dims 16 st + 8 h .. of every step, three parts.
template <int DP, bool VEC>
__device__ __forceinline__ void load_operand(bf16x8 (&p)[3][DP / 16], const float* row, int h, int dim) {
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) {
        const floatx4 a = load4_padded<VEC>(row, 16 * st + 8 * h, dim, true), b = load4_padded<VEC>(row, 16 * st + 8 * h + 4, dim, true);
        const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        uintx4 u[3];
        split8(v, u, kUp);
#pragma unroll
        for (int q = 0; q < 3; ++q) p[q][st] = __builtin_bit_cast(bf16x8, u[q]);
    }
}

// s (32 rows x 32 columns) = tile rows row0 .. row0 + 31 times the lanes' columns, over the dims.
template <int R, int DP>
__device__ __forceinline__ floatx16 tile_product(const uintx4* planes, int row0, const bf16x8 (&b)[3][DP / 16], int h, int c) {
    floatx16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int st = 0; st < DP / 16; ++st) {
        bf16x8 a[3];
#pragma unroll
        for (int q = 0; q < 3; ++q) a[q] = row_operand<R, DP>(planes, q, row0 + c, st, h);
#pragma unroll
        for (int q = 0; q < 6; ++q) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[kSplitA[q]], b[kSplitB[q]][st], s, 0, 0, 0);
    }
    return s;
}

// acc (dims x 32 columns) += (tile rows row0 .. row0 + 15)^T times their weights x, x times 2^24.
template <int R, int DP>
__device__ __forceinline__ void tile_add16(floatx16 (&acc)[DP / 32], const uintx4* planes, int row0, const float (&x)[8], int lane) {
    uintx4 u[3];
    split8(x, u, kUp);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
        bf16x8 a[3];
#pragma unroll
        for (int q = 0; q < 3; ++q) a[q] = column_operand<R, DP>(planes, q, row0, i, lane);
#pragma unroll
        for (int q = 0; q < 6; ++q)
            acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[kSplitA[q]], __builtin_bit_cast(bf16x8, u[kSplitB[q]]), acc[i], 0, 0, 0);
    }
}
template <int R, int DP>
__device__ __forceinline__ void tile_add(floatx16 (&acc)[DP / 32], const uintx4* planes, int row0, const floatx16& w, int lane) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = w[8 * t + e];
        tile_add16<R, DP>(acc, planes, row0 + 16 * t, x, lane);
    }
}

// Whether a value of the wave's accumulators is infinite or NaN.
template <int N>
__device__ __forceinline__ bool any_not_finite(const floatx16 (&acc)[N]) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad |= !(fabsf(acc[i][r]) < INFINITY);
    return __ballot(bad) != 0;
}

// LDS accesses of the work-group's waves are done; requested loads stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }  // below 2^-126: zero

// ---- forward ---------------------------------------------------------------------------------

// Output, maximum and sum of 32 rows again, from memory (a wave whose results are not finite).
template <int DP>
struct Redone {
    floatx16 x[DP / 32];
    float top, l;
};
template <int DP>
__device__ __noinline__ void redo_rows(Redone<DP>& result, const PackedAttn& a, const float* kb, const float* vb, const float* q_row,
                                       int k_begin, int k_end, int limit, int last_limit) {
    const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31;
    const float factor = a.scale * kLog2e;
    floatx16 o[DP / 32];
    clear(o);
    float top = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int t0 = k_begin; t0 < k_end && t0 <= last_limit; t0 += 32) {
        floatx16 s = rows_product<DP>(kb + (size_t)min(t0 + c, k_end - 1) * a.k_rs, q_row, a.head_dim, a.vec, h);
        uint32_t seen = 0;
        float mt = top;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const bool on = t0 + acc_row(r, h) <= limit;
            seen |= (on ? 1u : 0u) << r;
            s[r] = on ? s[r] * factor : -INFINITY;
            mt = fmaxf(mt, s[r]);
        }
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        const float base = mt == -INFINITY ? 0.f : mt, corr = fast_exp2(top - base);
        top = mt;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = fast_exp2(s[r] - base);
            sum += s[r];
        }
        l = l * corr + sum;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] *= corr;
        add_seen<DP>(o, s, seen, h, c, a.head_dim, a.vec, [&](int n) { return vb + (size_t)min(t0 + n, k_end - 1) * a.v_rs; });
    }
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) result.x[i] = o[i];
    result.top = top;
    result.l = l;
}

// PER rows per work-group: four waves of 32, or two pairs (64), whose second waves take the second half of every
// tile of keys and hand over their maxima, sums and outputs at the end.
template <int DP, bool VEC, int PER>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1) void attn_split_kernel(PackedAttn a, float* __restrict__ out, float* __restrict__ lse,
                                                            const float* __restrict__ q, const float* __restrict__ k,
                                                            const float* __restrict__ v, float* __restrict__ ws, uint32_t budget) {
    constexpr int KT = 64, U = DP / 8, NB = DP / 32, WAVES = PER / kRowsPerWave, KB = KT / 32 * WAVES / 4;
    __shared__ uintx4 planes[2][3 * KT * U];
    uintx4 *const kp = planes[0], *const vp = planes[1];
    const int kv = blockIdx.x % a.n_kv;
    Work w;
    if (!find_work<false, false>(a, PER, budget, blockIdx.x / a.n_kv, &w)) return;
    const RowTile tl = row_tile(a, w, PER);
    if (w.range >= tl.ranges) return;
    const Span sp = w.sp;
    const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31;
    const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all % WAVES, part0 = all / WAVES * KB * 32;
    const int dim = a.head_dim, group = a.group, rows = tl.rows, shift = tl.shift, k_begin = tl.k_begin, k_end = tl.k_end;
    const bool vec = a.vec;
    const int rho0 = tl.rho0 + wave * kRowsPerWave, rho = rho0 + c;
    const bool live = rho < rows;
    const int qi = (live ? rho : rows - 1) / group, head = kv * group + (live ? rho : rows - 1) % group;
    const int limit = min(qi + shift, k_end - 1);  // last key of the range that this row sees
    // Over the wave's rows (uniform): the first row's limit, and the last one's.
    const int first_limit = min(rho0, rows - 1) / group + shift;
    const int last_limit = rho0 < rows ? (min(rho0 + kRowsPerWave, rows) - 1) / group + shift : -1;
    const float* kb = k + (size_t)sp.k0 * a.k_rs + (size_t)kv * a.k_hs;
    const float* vb = v + (size_t)sp.k0 * a.v_rs + (size_t)kv * a.v_hs;
    const float* q_row = q + (size_t)(sp.q0 + qi) * a.q_rs + (size_t)head * dim;

    Stage<KT, DP, VEC> ks, vs;
    if (k_begin < k_end) {
        ks.load(kb, a.k_rs, k_begin, k_end, dim);
        vs.load(vb, a.v_rs, k_begin, k_end, dim);
    }
    bf16x8 qp[3][DP / 16];
    load_operand<DP, VEC>(qp, q_row, h, dim);
    floatx16 o[NB];
    clear(o);
    float top = -INFINITY, l = 0.f;  // the running maximum of the raw products, the sum of exponentials
    // A softmax step over 32 keys at t0 of products s, exponent factor f (its sign decides which product is largest).
    auto softmax = [&](floatx16* s, int blocks, int t0, float f) {
        const bool edge = t0 + 32 * blocks - 1 > min(first_limit, k_end - 1);
        float mt = top;
        for (int j = 0; j < blocks; ++j) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[j][r] *= f;
                if (edge && t0 + 32 * j + acc_row(r, h) > limit) s[j][r] = -INFINITY;
                mt = fmaxf(mt, s[j][r]);
            }
        }
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        const float base = mt == -INFINITY ? 0.f : mt;
        const float corr = fast_exp2(top - base);
        top = mt;
        float sum = 0.f;
        for (int j = 0; j < blocks; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[j][r] = fast_exp2(s[j][r] - base);
                sum += s[j][r];
            }
        l = l * corr + sum;
        if (__ballot(corr != 1.0f)) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][r] *= corr;
        }
    };
    const float factor = a.scale * kLog2e;
    for (int t0 = k_begin; t0 < k_end; t0 += KT) {
        lds_barrier();
        ks.store(kp);
        vs.store(vp);
        if (t0 + KT < k_end) {
            ks.load(kb, a.k_rs, t0 + KT, k_end, dim);
            vs.load(vb, a.v_rs, t0 + KT, k_end, dim);
        }
        lds_barrier();
        if (t0 + part0 > min(last_limit, k_end - 1)) continue;  // no row of the wave sees its keys of the tile
        floatx16 s[KB];
#pragma unroll
        for (int j = 0; j < KB; ++j) s[j] = tile_product<KT, DP>(kp, part0 + 32 * j, qp, h, c);
        softmax(s, KB, t0 + part0, factor * kDown2);
#pragma unroll
        for (int j = 0; j < KB; ++j) tile_add<KT, DP>(o, vp, part0 + 32 * j, s[j], lane);
    }
    if constexpr (WAVES == 2) {
        __syncthreads();  // the planes are free: the second waves' results pass through them
        floatx4* const pass = reinterpret_cast<floatx4*>(&planes[0][0]) + wave * (4 * NB + 1) * 64 + lane;
        if (part0) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) pass[(4 * i + u) * 64] = floatx4{o[i][4 * u], o[i][4 * u + 1], o[i][4 * u + 2], o[i][4 * u + 3]};
            pass[4 * NB * 64] = floatx4{top, l, 0.f, 0.f};
        }
        __syncthreads();
        if (part0) return;
        const floatx4 other = pass[4 * NB * 64];
        const float both = fmaxf(top, other[0]), base = both == -INFINITY ? 0.f : both;
        const float mine = fast_exp2(top - base), theirs = fast_exp2(other[0] - base);
        top = both;
        l = l * mine + other[1] * theirs;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const floatx4 x = pass[(4 * i + u) * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][4 * u + e] = o[i][4 * u + e] * mine + x[e] * theirs;
            }
    }
    float unit = kDown2;
    if (any_not_finite(o)) {
        unit = 1.0f;
        Redone<DP> r;  // a copy: o itself stays in registers
        redo_rows<DP>(r, a, kb, vb, q_row, k_begin, k_end, limit, last_limit);
#pragma unroll
        for (int i = 0; i < NB; ++i) o[i] = r.x[i];
        top = r.top;
        l = r.l;
    }
    l += __shfl_xor(l, 32);
    if (!live) return;
    float inv = qi + shift < 0 || sp.kl == 0 ? 0.f : 1.0f / l;
    float* dst = out + (size_t)(sp.q0 + qi) * a.o_rs + (size_t)head * dim;
    bool dst_vec = vec;
    if (tl.ranges > 1) {
        const int t = rho - tl.rho0;
        const Partials part = partials(ws, a.n_kv, kv, gridDim.x / a.n_kv, w.item0 + w.range, PER, dim);
        inv = 1.0f;
        dst = part.o + t * padded_dim(dim);
        dst_vec = true;
        if (h == 0) {
            part.ml[2 * t] = top;
            part.ml[2 * t + 1] = l;
        }
    } else if (lse && h == 0) {
        lse[(size_t)head * a.q_rows + sp.q0 + qi] = (top + log2f(l)) * kLn2;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            floatx4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = o[i][4 * u + e] * unit * inv;
            store4(dst, 32 * i + 8 * u + 4 * h, dim, dst_vec, x);
        }
}

// ---- backward --------------------------------------------------------------------------------

// dq / scale of 32 rows again, from memory.
template <int DP>
__device__ __noinline__ void redo_dq(Redone<DP>& result, const PackedAttn& a, const float* kb, const float* vb, const float* q_row,
                                     const float* g_row, float lse2, float d, int nkeys, int limit, int last_limit) {
    const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31;
    floatx16 acc[DP / 32];
    clear(acc);
#pragma unroll 1
    for (int t0 = 0; t0 < nkeys && t0 <= last_limit; t0 += 32) {
        const size_t row = min(t0 + c, nkeys - 1);
        floatx16 s = rows_product<DP>(kb + row * a.k_rs, q_row, a.head_dim, a.vec, h);
        const floatx16 dp = rows_product<DP>(vb + row * a.v_rs, g_row, a.head_dim, a.vec, h);
        uint32_t seen = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const bool on = t0 + acc_row(r, h) <= min(limit, nkeys - 1);
            seen |= (on ? 1u : 0u) << r;
            s[r] = on ? fast_exp2(fmaf(s[r], a.scale * kLog2e, -lse2)) * (dp[r] - d) : 0.f;
        }
        add_seen<DP>(acc, s, seen, h, c, a.head_dim, a.vec, [&](int n) { return kb + (size_t)min(t0 + n, nkeys - 1) * a.k_rs; });
    }
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) result.x[i] = acc[i];
}

// The two waves of a pair hand 32 x 32 values to one another through LDS as their accumulators lie.
struct Exchange {
    floatx4 x[4][64];
    __device__ __forceinline__ void put(const floatx16& v, int lane) {
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u][lane] = floatx4{v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]};
    }
    __device__ __forceinline__ floatx16 get(int lane) const {
        floatx16 v;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * u + e] = x[u][lane][e];
        return v;
    }
};

// The sums of 32 keys again, from memory (a wave whose results are not finite).
template <int DP>
__device__ __noinline__ void redo_dkv(Redone<DP>& result, const PackedAttn& a, const Span& sp, int kv, int second, int key0,
                                         int first, int tiles, int it0, int it1, int rt, const float* delta, const float* dout,
                                         const float* lse, const float* q, const float* k_row, const float* v_row) {
    const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31, ql = sp.ql, shift = (int)sp.kl - (int)sp.ql;
    floatx16 acc[DP / 32];
    clear(acc);
#pragma unroll 1
    for (int block = it0 * (rt / 32); block < it1 * (rt / 32); ++block) {
        const int it = block / (rt / 32), head = kv * a.group + it / tiles, i0 = (first + it % tiles) * rt + 32 * (block % (rt / 32));
        if (key0 > i0 + 31 + shift || i0 >= ql) continue;
        const float* qb = q + (size_t)sp.q0 * a.q_rs + (size_t)head * a.head_dim;
        const float* gb = dout + (size_t)sp.q0 * a.o_rs + (size_t)head * a.head_dim;
        const size_t at = (size_t)head * a.q_rows + sp.q0;
        const size_t mine = min(i0 + c, ql - 1);
        floatx16 s = rows_product<DP>(qb + mine * a.q_rs, k_row, a.head_dim, a.vec, h);
        const floatx16 dp = rows_product<DP>(gb + mine * a.o_rs, v_row, a.head_dim, a.vec, h);
        uint32_t seen = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = i0 + acc_row(r, h), j = min(i, ql - 1);
            const bool on = i < ql && key0 + c <= i + shift;
            seen |= (on ? 1u : 0u) << r;
            const float p = fast_exp2(fmaf(s[r], a.scale * kLog2e, -lse[at + j] * kLog2e));
            s[r] = on ? (second ? p * (dp[r] - delta[at + j]) : p) : 0.f;
        }
        const float* base = second ? qb : gb;
        const size_t rs = second ? a.q_rs : a.o_rs;
        add_seen<DP>(acc, s, seen, h, c, a.head_dim, a.vec, [&](int n) { return base + (size_t)min(i0 + n, ql - 1) * rs; });
    }
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) result.x[i] = acc[i];
}

// Keys of a sequence from which on a work-group of the backward pass has four pairs of waves.
constexpr uint32_t kLongKeys = 1536;

// Tiles of the backward pass: 64 rows or keys in LDS at head_dim 33 .. 64, else 32 (LDS at 128 would hold no more;
// at 32 it leaves room for two work-groups).
template <int DP>
constexpr int kBackTile = DP == 64 ? 64 : 32;

// P: pairs of waves per work-group.
template <int DP, int P>
struct BackwardLds {
    static constexpr int T = kBackTile<DP>;
    uintx4 planes[2][3 * T * (DP / 8)];
    Exchange exchange[T / 32][P];
    __attribute__((aligned(16))) float stats[2][T];
};

// dq of a tile of rows, two waves for each 32 of them (as in the forward pass a row per lane column):
//   the first S^T = K Q^T and p, the second dP^T = V dO^T - d; each hands half of its keys' values to the
// other, forms dS of the other half and adds K^T dS over it: dQ^T is the sum of the two.
template <int DP, bool VEC, int P>
__device__ __forceinline__ void dq_tile(BackwardLds<DP, P>& lds, const PackedAttn& a, uint32_t index, float* __restrict__ dq,
                                        const float* __restrict__ delta, const float* __restrict__ dout, const float* __restrict__ lse,
                                        const float* __restrict__ q, const float* __restrict__ k, const float* __restrict__ v) {
    constexpr int KT = kBackTile<DP>, NB = DP / 32, kTile = 32 * P;
    const int kv = index % a.n_kv;
    Work w;
    if (!find_work<false, true>(a, kTile, 0, index / a.n_kv, &w)) return;
    const RowTile tl = row_tile(a, w, kTile);
    const Span sp = w.sp;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
    const int pair = wave % P, second = wave / P;
    const int dim = a.head_dim, group = a.group, rows = tl.rows, shift = tl.shift, nkeys = tl.nkeys;
    const int rho0 = tl.rho0 + pair * kRowsPerWave, rho = rho0 + c;
    const bool live = rho < rows;
    const int qi = (live ? rho : rows - 1) / group, head = kv * group + (live ? rho : rows - 1) % group;
    const int limit = qi + shift;
    const int first_limit = min(rho0, rows - 1) / group + shift;
    const int last_limit = rho0 < rows ? (min(rho0 + kRowsPerWave, rows) - 1) / group + shift : -1;
    const float* kb = k + (size_t)sp.k0 * a.k_rs + (size_t)kv * a.k_hs;
    const float* vb = v + (size_t)sp.k0 * a.v_rs + (size_t)kv * a.v_hs;
    const float* q_row = q + (size_t)(sp.q0 + qi) * a.q_rs + (size_t)head * dim;
    const float* g_row = dout + (size_t)(sp.q0 + qi) * a.o_rs + (size_t)head * dim;

    // The first waves stage K, the others V.
    Stage<KT, DP, VEC, 64 * P> keys;
    const float* const base = second ? vb : kb;
    const size_t rs = second ? a.v_rs : a.k_rs;
    if (nkeys > 0) keys.load(base, rs, 0, nkeys, dim);
    const size_t stat = (size_t)head * a.q_rows + sp.q0 + qi;
    const float lse2 = lse[stat] * kLog2e, d = delta[stat];
    bf16x8 own[3][DP / 16];  // Q's, dO's parts
    load_operand<DP, VEC>(own, second ? g_row : q_row, h, dim);
    floatx16 acc[NB];
    clear(acc);
    const float factor = a.scale * kLog2e;
    for (int t0 = 0; t0 < nkeys; t0 += KT) {
        lds_barrier();
        keys.store(lds.planes[second]);
        if (t0 + KT < nkeys) keys.load(base, rs, t0 + KT, nkeys, dim);
        lds_barrier();
        floatx16 s[KT / 32];
#pragma unroll
        for (int j = 0; j < KT / 32; ++j) {
            if (t0 + 32 * j > last_limit) continue;  // no row of the wave sees the block
            s[j] = tile_product<KT, DP>(lds.planes[second], 32 * j, own, h, c);
            const bool edge = t0 + 32 * j + 31 > first_limit;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float x = second ? fmaf(s[j][r], kDown2, -d) : fast_exp2(fmaf(s[j][r], factor * kDown2, -lse2));
                s[j][r] = edge && t0 + 32 * j + acc_row(r, h) > limit ? 0.f : x;
            }
            Exchange& ex = lds.exchange[j][pair];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                ex.x[2 * second + u][lane] = second ? floatx4{s[j][4 * u], s[j][4 * u + 1], s[j][4 * u + 2], s[j][4 * u + 3]}
                                                    : floatx4{s[j][4 * u + 8], s[j][4 * u + 9], s[j][4 * u + 10], s[j][4 * u + 11]};
            }
        }
        lds_barrier();
#pragma unroll
        for (int j = 0; j < KT / 32; ++j) {
            if (t0 + 32 * j > last_limit) continue;
            const Exchange& ex = lds.exchange[j][pair];
            const floatx4 y0 = ex.x[2 - 2 * second][lane], y1 = ex.x[3 - 2 * second][lane];
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (second ? s[j][8 + e] : s[j][e]) * (e < 4 ? y0[e & 3] : y1[e & 3]);
            tile_add16<KT, DP>(acc, lds.planes[0], 32 * j + 16 * second, x, lane);
        }
    }
    // The second waves' sums, a block of 32 dims at a time.
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        lds_barrier();
        if (second) lds.exchange[0][pair].put(acc[i], lane);
        lds_barrier();
        if (!second) acc[i] += lds.exchange[0][pair].get(lane);
    }
    if (second) return;
    float unit = kDown2;
    if (any_not_finite(acc)) {
        unit = 1.0f;
        Redone<DP> r;
        redo_dq<DP>(r, a, kb, vb, q_row, g_row, lse2, d, nkeys, limit, last_limit);
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = r.x[i];
    }
    if (!live) return;
    float* dst = dq + (size_t)(sp.q0 + qi) * a.q_rs + (size_t)head * dim;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            floatx4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = acc[i][4 * u + e] * unit * a.scale;
            store4(dst, 32 * i + 8 * u + 4 * h, dim, a.vec, x);
        }
}

// dq of a tile of rows, a wave for each 32 of them, as in the forward pass: S^T = K Q^T, dP^T = V dO^T,
// dQ^T += K^T dS^T.
template <int DP, bool VEC, int P>
__device__ __forceinline__ void dq_tile_alone(BackwardLds<DP, P>& lds, const PackedAttn& a, uint32_t index, float* __restrict__ dq,
                                              const float* __restrict__ delta, const float* __restrict__ dout, const float* __restrict__ lse,
                                              const float* __restrict__ q, const float* __restrict__ k, const float* __restrict__ v) {
    constexpr int KT = kBackTile<DP>, NB = DP / 32, kTile = 64 * P, NT = 64 * P;
    const int kv = index % a.n_kv;
    Work w;
    if (!find_work<false, true>(a, kTile, 0, index / a.n_kv, &w)) return;
    const RowTile tl = row_tile(a, w, kTile);
    const Span sp = w.sp;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
    const int second = wave / P;
    const int dim = a.head_dim, group = a.group, rows = tl.rows, shift = tl.shift, nkeys = tl.nkeys;
    const int rho0 = tl.rho0 + wave * kRowsPerWave, rho = rho0 + c;
    const bool live = rho < rows;
    const int qi = (live ? rho : rows - 1) / group, head = kv * group + (live ? rho : rows - 1) % group;
    const int limit = qi + shift;
    const int first_limit = min(rho0, rows - 1) / group + shift;
    const int last_limit = rho0 < rows ? (min(rho0 + kRowsPerWave, rows) - 1) / group + shift : -1;
    const float* kb = k + (size_t)sp.k0 * a.k_rs + (size_t)kv * a.k_hs;
    const float* vb = v + (size_t)sp.k0 * a.v_rs + (size_t)kv * a.v_hs;
    const float* q_row = q + (size_t)(sp.q0 + qi) * a.q_rs + (size_t)head * dim;
    const float* g_row = dout + (size_t)(sp.q0 + qi) * a.o_rs + (size_t)head * dim;

    // The first waves stage K, the others V.
    Stage<KT, DP, VEC, NT> keys;
    const float* const base = second ? vb : kb;
    const size_t rs = second ? a.v_rs : a.k_rs;
    if (nkeys > 0) keys.load(base, rs, 0, nkeys, dim);
    const size_t stat = (size_t)head * a.q_rows + sp.q0 + qi;
    const float lse2 = lse[stat] * kLog2e, d = delta[stat];
    bf16x8 qp[3][DP / 16], gp[3][DP / 16];
    load_operand<DP, VEC>(qp, q_row, h, dim);
    load_operand<DP, VEC>(gp, g_row, h, dim);
    floatx16 acc[NB];
    clear(acc);
    const float factor = a.scale * kLog2e;
    for (int t0 = 0; t0 < nkeys; t0 += KT) {
        lds_barrier();
        keys.store(lds.planes[second]);
        if (t0 + KT < nkeys) keys.load(base, rs, t0 + KT, nkeys, dim);
        lds_barrier();
#pragma unroll
        for (int j = 0; j < KT / 32; ++j) {
            if (t0 + 32 * j > last_limit) continue;  // no row of the wave sees the block
            floatx16 s = tile_product<KT, DP>(lds.planes[0], 32 * j, qp, h, c);
            const floatx16 dp = tile_product<KT, DP>(lds.planes[1], 32 * j, gp, h, c);
            const bool edge = t0 + 32 * j + 31 > first_limit;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float x = fast_exp2(fmaf(s[r], factor * kDown2, -lse2)) * fmaf(dp[r], kDown2, -d);
                s[r] = edge && t0 + 32 * j + acc_row(r, h) > limit ? 0.f : x;
            }
            tile_add<KT, DP>(acc, lds.planes[0], 32 * j, s, lane);
        }
    }
    float unit = kDown2;
    if (any_not_finite(acc)) {
        unit = 1.0f;
        Redone<DP> r;
        redo_dq<DP>(r, a, kb, vb, q_row, g_row, lse2, d, nkeys, limit, last_limit);
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = r.x[i];
    }
    if (!live) return;
    float* dst = dq + (size_t)(sp.q0 + qi) * a.q_rs + (size_t)head * dim;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            floatx4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = acc[i][4 * u + e] * unit * a.scale;
            store4(dst, 32 * i + 8 * u + 4 * h, dim, a.vec, x);
        }
}

// dk and dv: a work-group per tile of keys of one (sequence, key head), a key per lane column; the rows of
// the group's heads stream through LDS.  Two waves share 32 keys (keeping K and V parts and both sums
// in one wave's registers spilled at head_dim 128: 4.9 ms for two sequences of 3000 .. 4096, 16 heads on 2; 1.8 so):
//   the first   S = Q K^T, p, dV^T += dO^T P     holds K and dV,
//   the second  dP = dO V^T, dS, dK^T += Q^T dS  holds V and dK and takes p from the first.
// Where there are few such tiles, their rows are cut into parts (whole tiles of rows, of all heads in
// order); the parts' sums go to the workspace and attn_split_dkv_join_kernel adds them in order.
template <int DP, bool VEC, int P>
__device__ __forceinline__ void dkv_tile(BackwardLds<DP, P>& lds, const PackedAttn& a, uint32_t index, uint32_t tiles_all, int part, int parts,
                                         float* __restrict__ dk, float* __restrict__ dv, const float* __restrict__ delta,
                                         const float* __restrict__ dout, const float* __restrict__ lse, const float* __restrict__ q,
                                         const float* __restrict__ k, const float* __restrict__ v, float* __restrict__ sums) {
    constexpr int RT = kBackTile<DP>, NB = DP / 32, kTile = 32 * P, NT = 64 * P;
    auto& planes = lds.planes;      // Q, dO
    auto& exchange = lds.exchange;
    auto& stats = lds.stats;        // lse (base 2), d
    const int kv = index % a.n_kv;
    Work w;
    if (!find_work<true, true>(a, kTile, 0, index / a.n_kv, &w)) return;
    const Span sp = w.sp;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
    const int pair = wave % P, second = wave / P;
    const int dim = a.head_dim, group = a.group;
    const bool vec = a.vec;
    const int key0 = w.tile * kTile + pair * kRowsPerWave, key = key0 + c;
    const bool live = key < (int)sp.kl;
    const int shift = (int)sp.kl - (int)sp.ql, ql = sp.ql;
    const size_t row = sp.k0 + (live ? key : (int)sp.kl - 1);
    const float* k_row = k + row * a.k_rs + (size_t)kv * a.k_hs;
    const float* v_row = v + row * a.v_rs + (size_t)kv * a.v_hs;
    // The tiles of rows that see a key of the work-group, over the group's heads, and this part of them.
    const int first = max(0, (int)w.tile * kTile - shift) / RT, tiles = max(0, (ql + RT - 1) / RT - first);
    const int64_t total = (int64_t)tiles * group;
    const int it0 = (int)(total * part / parts), it1 = (int)(total * (part + 1) / parts);

    bf16x8 own[3][DP / 16];  // K's, V's parts
    load_operand<DP, VEC>(own, second ? v_row : k_row, h, dim);
    floatx16 acc[NB];  // dV^T, dK^T
    clear(acc);
    // The first waves stage Q and lse, the others dO and d.
    Stage<RT, DP, VEC, NT> rows;
    float stat = 0.f;
    const float* const rows_base = second ? dout + (size_t)sp.q0 * a.o_rs : q + (size_t)sp.q0 * a.q_rs;
    const float* const stat_base = second ? delta : lse;
    const size_t rows_rs = second ? a.o_rs : a.q_rs;
    auto load = [&](int it) {
        const int head = kv * group + it / tiles, i0 = (first + it % tiles) * RT;
        rows.load(rows_base + (size_t)head * dim, rows_rs, i0, ql, dim);
        const int i = i0 + (threadIdx.x & (NT - 1));
        if ((threadIdx.x & (NT - 1)) < RT) stat = i < ql ? stat_base[(size_t)head * a.q_rows + sp.q0 + i] * (second ? 1.0f : kLog2e) : 0.f;
    };
    const float factor = a.scale * kLog2e;
    if (it0 < it1) load(it0);
    for (int it = it0; it < it1; ++it) {
        const int i0 = (first + it % tiles) * RT;
        lds_barrier();
        rows.store(planes[second]);
        if ((threadIdx.x & (NT - 1)) < RT) stats[second][threadIdx.x & (NT - 1)] = stat;
        if (it + 1 < it1) load(it + 1);
        lds_barrier();
        floatx16 s[RT / 32];
        // Blocks of 32 rows: none of a block's rows may see the wave's keys, or not all of them all.
        auto needed = [&](int j) { return key0 <= i0 + 32 * j + 31 + shift; };
        auto hidden = [&](int j, int r) { return key > i0 + 32 * j + r + shift; };
#pragma unroll
        for (int j = 0; j < RT / 32; ++j) {
            if (!needed(j)) continue;
            s[j] = tile_product<RT, DP>(planes[second], 32 * j, own, h, c);
            if (second) continue;
            const bool edge = key0 + kRowsPerWave - 1 > i0 + 32 * j + shift;
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const floatx4 m = *reinterpret_cast<const floatx4*>(&stats[0][32 * j + acc_row(r, h)]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = fast_exp2(fmaf(s[j][r + e], factor * kDown2, -m[e]));
                    s[j][r + e] = edge && hidden(j, acc_row(r, h) + e) ? 0.f : p;
                }
            }
            exchange[j][pair].put(s[j], lane);
        }
        lds_barrier();
#pragma unroll
        for (int j = 0; j < RT / 32; ++j) {
            if (!needed(j)) continue;
            if (second) {
                const floatx16 p = exchange[j][pair].get(lane);
                const bool edge = key0 + kRowsPerWave - 1 > i0 + 32 * j + shift;
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const floatx4 d = *reinterpret_cast<const floatx4*>(&stats[1][32 * j + acc_row(r, h)]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = p[r + e] * fmaf(s[j][r + e], kDown2, -d[e]);
                        s[j][r + e] = edge && hidden(j, acc_row(r, h) + e) ? 0.f : x;
                    }
                }
            }
            tile_add<RT, DP>(acc, planes[1 - second], 32 * j, s[j], lane);
        }
    }
    float unit = kDown2;
    if (any_not_finite(acc)) {
        unit = 1.0f;
        Redone<DP> r;
        redo_dkv<DP>(r, a, sp, kv, second, key0, first, tiles, it0, it1, RT, delta, dout, lse, q, k_row, v_row);
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = r.x[i];
    }
    if (!live) return;
    float* dst = second ? dk + row * a.k_rs + (size_t)kv * a.k_hs : dv + row * a.v_rs + (size_t)kv * a.v_hs;
    bool dst_vec = vec;
    int width = dim;
    if (parts > 1) {
        const size_t tile = (size_t)part * tiles_all + (size_t)w.tile0 * a.n_kv + kv;
        dst = sums + ((tile * 2 + 1 - second) * kTile + key - w.tile * kTile) * DP;
        dst_vec = true;
        width = DP;
    }
    const float by = second ? a.scale : 1.0f;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            floatx4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = acc[i][4 * u + e] * unit * by;
            store4(dst, 32 * i + 8 * u + 4 * h, width, dst_vec, x);
        }
}

// The backward pass in one launch: the tiles of dk and dv first (they take longest), then those of dq,
// which need nothing of them.
template <int DP, bool VEC, int P>
__global__ __launch_bounds__(128 * P, DP == 32 ? 3 : 2) void attn_split_backward_kernel(
    PackedAttn a, uint32_t key_groups, int parts, float* __restrict__ dq, float* __restrict__ dk, float* __restrict__ dv,
    const float* __restrict__ delta, const float* __restrict__ dout, const float* __restrict__ lse, const float* __restrict__ q,
    const float* __restrict__ k, const float* __restrict__ v, float* __restrict__ sums) {
    __shared__ BackwardLds<DP, P> lds;
    if (blockIdx.x < key_groups * parts)
        dkv_tile<DP, VEC, P>(lds, a, blockIdx.x % key_groups, key_groups, blockIdx.x / key_groups, parts, dk, dv, delta, dout, lse, q, k, v, sums);
    else if constexpr (DP <= 64)
        dq_tile_alone<DP, VEC, P>(lds, a, blockIdx.x - key_groups * parts, dq, delta, dout, lse, q, k, v);
    else
        dq_tile<DP, VEC, P>(lds, a, blockIdx.x - key_groups * parts, dq, delta, dout, lse, q, k, v);
}

// d_i = do_i . o_i of every row and head: LPR lanes each.
template <int LPR>
__global__ __launch_bounds__(256) void attn_split_delta_kernel(PackedAttn a, float* __restrict__ delta, const float* __restrict__ dout,
                                                               const float* __restrict__ out) {
    const uint32_t heads = a.n_kv * a.group, lane = threadIdx.x % LPR;
    const uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / LPR;
    const uint32_t row = (uint32_t)(i / heads), head = (uint32_t)(i % heads);
    float d = 0.f;
    if (row < a.q_rows) {
        const size_t at = (size_t)row * a.o_rs + (size_t)head * a.head_dim;
        for (int e = 4 * lane; e < a.head_dim; e += 4 * LPR) {
            const floatx4 x = load4(dout + at, e, a.head_dim, a.vec), y = load4(out + at, e, a.head_dim, a.vec);
#pragma unroll
            for (int j = 0; j < 4; ++j) d += x[j] * y[j];
        }
    }
#pragma unroll
    for (int m = 1; m < LPR; m <<= 1) d += __shfl_xor(d, m);
    if (row < a.q_rows && lane == 0) delta[(size_t)head * a.q_rows + row] = d;
}

// dk and dv of a tile of keys: its parts added in order.
template <int DP, int P>
__global__ __launch_bounds__(256) void attn_split_dkv_join_kernel(PackedAttn a, float* __restrict__ dk, float* __restrict__ dv,
                                                                  const float* __restrict__ part, int parts) {
    constexpr int kTile = 32 * P;
    const int kv = blockIdx.x % a.n_kv;
    Work w;
    if (!find_work<true, true>(a, kTile, 0, blockIdx.x / a.n_kv, &w)) return;
    const int keys = min((int)w.sp.kl - (int)w.tile * kTile, kTile), dim = a.head_dim;
    const size_t stride = (size_t)gridDim.x * 2 * kTile * DP;
    const float* p = part + ((size_t)w.tile0 * a.n_kv + kv) * 2 * kTile * DP;
    constexpr int N = 2 * kTile * (DP / 4);
    for (int e = blockIdx.y * 256 + threadIdx.x; e < N; e += 256 * gridDim.y) {
        const int which = e / (N / 2), key = e % (N / 2) / (DP / 4), d = 4 * (e % (DP / 4));
        if (key >= keys || d >= dim) continue;
        floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int z = 0; z < parts; ++z) x += *reinterpret_cast<const floatx4*>(p + z * stride + 4 * (size_t)e);
        const size_t row = w.sp.k0 + (size_t)w.tile * kTile + key;
        store4(which ? dv + row * a.v_rs + (size_t)kv * a.v_hs : dk + row * a.k_rs + (size_t)kv * a.k_hs, d, dim, a.vec, x);
    }
}

}  // namespace

int attn_split_forward(const PackedAttn& a, int per, uint32_t items, uint32_t budget, float* out, float* lse, const float* q, const float* k,
                       const float* v, float* ws, hipStream_t s) {
    const dim3 grid(items * a.n_kv);
#define FMLH_LAUNCH_PER(DP, PER)                                                                                                \
    hipLaunchKernelGGL((a.vec ? attn_split_kernel<DP, true, PER> : attn_split_kernel<DP, false, PER>), grid, dim3(256), 0, s, a, \
                       out, lse, q, k, v, ws, budget)
#define FMLH_LAUNCH(DP)                              \
    do {                                             \
        if (per == kRowsPerWG) FMLH_LAUNCH_PER(DP, kRowsPerWG); \
        else FMLH_LAUNCH_PER(DP, kRowsPerWG / 2);    \
    } while (0)
    if (a.head_dim <= 32) FMLH_LAUNCH(32);
    else if (a.head_dim <= 64) FMLH_LAUNCH(64);
    else if (a.head_dim <= 96) FMLH_LAUNCH(96);
    else FMLH_LAUNCH(128);
#undef FMLH_LAUNCH
#undef FMLH_LAUNCH_PER
    FMLH_LAUNCHED("attn_split_kernel");
    return FMLH_OK;
}

// Pairs of waves per work-group of the backward pass.  At head_dim up to 64 a work-group of two holds half a
// CU, and two of them are seldom in the same step: 64 x 128 rows, 12 heads of 64, take 116 us with two
// pairs, 151 with four; 32 x 512 375 and 408; 24 x 100 .. 2048, 12 heads on 4, 583 and 640.  Long sequences gain by staging
// a tile for more keys: 8 x 2048, 12 heads, 1100 and 1040, 8 x 4096, 16 heads, 5.75 ms and 5.22.  At head_dim 32 two
// fit three times (8 x 4096, 16 heads, 3.05 ms, four pairs 3.15); beyond 64 four pairs, whose staging takes half the registers
// (4 x 4096, 16 heads of 128, 5.6 ms, with two 10.4).
int attn_split_pairs(const PackedAttn& a) {
    return a.head_dim > 64 ? 4 : a.head_dim <= 32 ? 2 : a.k_rows / a.n_seq >= kLongKeys ? 4 : 2;
}
int attn_split_dq_rows(const PackedAttn& a) { return (a.head_dim <= 64 ? 64 : 32) * attn_split_pairs(a); }
int attn_split_back_rows(const PackedAttn& a) { return 32 * attn_split_pairs(a); }

size_t attn_split_part_floats(const PackedAttn& a, uint32_t tiles) {
    const size_t dp = a.head_dim <= 32 ? 32 : a.head_dim <= 64 ? 64 : a.head_dim <= 96 ? 96 : 128;
    return (size_t)tiles * a.n_kv * 2 * attn_split_back_rows(a) * dp;
}

int attn_split_backward(const PackedAttn& a, uint32_t row_tiles, uint32_t key_tiles, int parts, float* dq, float* dk, float* dv,
                        float* delta, const float* dout, const float* out, const float* lse, const float* q, const float* k,
                        const float* v, float* sums, hipStream_t s) {
    constexpr int kLanes = 16;
    const uint64_t items = (uint64_t)a.q_rows * a.n_kv * a.group;
    if (items) {
        hipLaunchKernelGGL(attn_split_delta_kernel<kLanes>, dim3((unsigned)((items * kLanes + 255) / 256)), dim3(256), 0, s, a, delta, dout, out);
        FMLH_LAUNCHED("attn_split_delta_kernel");
    }
    const uint32_t key_groups = key_tiles * a.n_kv;
    const dim3 grid(key_groups * parts + row_tiles * a.n_kv);
#define FMLH_LAUNCH_P(DP, P)                                                                                                            \
    do {                                                                                                                                \
        hipLaunchKernelGGL((a.vec ? attn_split_backward_kernel<DP, true, P> : attn_split_backward_kernel<DP, false, P>), grid,          \
                           dim3(128 * P), 0, s, a, key_groups, parts, dq, dk, dv, delta, dout, lse, q, k, v, sums);                      \
        FMLH_LAUNCHED("attn_split_backward_kernel");                                                                                    \
        if (parts > 1) {                                                                                                                \
            hipLaunchKernelGGL((attn_split_dkv_join_kernel<DP, P>), dim3(key_groups, 8), dim3(256), 0, s, a, dk, dv, sums, parts);       \
            FMLH_LAUNCHED("attn_split_dkv_join_kernel");                                                                                \
        }                                                                                                                               \
    } while (0)
    const bool two = attn_split_pairs(a) == 2;
    if (a.head_dim <= 32) {
        FMLH_LAUNCH_P(32, 2);
    } else if (a.head_dim <= 64) {
        if (two) FMLH_LAUNCH_P(64, 2);
        else FMLH_LAUNCH_P(64, 4);
    } else if (a.head_dim <= 96) {
        FMLH_LAUNCH_P(96, 4);
    } else {
        FMLH_LAUNCH_P(128, 4);
    }
#undef FMLH_LAUNCH_P
    return FMLH_OK;
}

}  // namespace fmlh
