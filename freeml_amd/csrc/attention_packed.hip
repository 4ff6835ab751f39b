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
// Here: a few rows over many keys, the joining of ranges of keys, plans and entry points.  Tiles of
// 64 and 128 rows and the backward pass are in attention_packed_split.hip.
#include "attention_packed_device.h"

#include <algorithm>

namespace fmlh {

namespace {

// ---- few rows over many keys -------------------------------------------------------------------

// Single tokens over a cache: with RT rows (the heads of a group, a few queries) the keys' and values'
// bytes are the work.  A work-group takes a tile of RT rows of one (sequence, key head) and one of
// the ranges its keys are cut into; LPK lanes hold a key (NF float4 each), 64 / LPK keys per
// wave and step, UN steps in flight.  Every lane group keeps its own maximum, sum and output over its
// keys; they are joined over the wave and the work-group once, at the end.  A tile with one range
// writes its rows, otherwise their (maximum, sum, output) go to the workspace and are joined by
// attn_packed_join_kernel in range order.
// The bytes bound it: one token on 8 x 2048 .. 32768 keys, 32 heads of 128 on 8 (750 MB), 162 us, 4.6 TB/s where a copy
// reaches 5.05; ranges of a fixed share of a sequence instead of a fixed length took 306 us.

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
            store4(part.o + t * padded_dim(dim), d, dim, true, x);
            if (d == 0) {
                part.ml[2 * t] = top;
                part.ml[2 * t + 1] = sum;
            }
        }
    }
}

// Joins the ranges of the rows whose keys were cut into more than one: a wave per row, the ranges'
// outputs added in range order.  A work-group takes four rows of a tile at a time; about 2048 of them are
// launched, since each has to find its tile first.
template <int TILE>
__global__ __launch_bounds__(256) void attn_packed_join_kernel(PackedAttn a, float* __restrict__ out, float* __restrict__ lse,
                                                               float* __restrict__ ws, uint32_t budget, uint32_t items) {
    Work w;
    if (!find_work<false, true>(a, TILE, budget, blockIdx.x, &w)) return;
    const RowTile tl = row_tile(a, w, TILE);
    if (tl.ranges == 1) return;
    const int lane = threadIdx.x & 63, dim = a.head_dim, group = a.group, kv = blockIdx.y;
    const Partials part = partials(ws, gridDim.y, kv, items, w.item0, TILE, dim);
    for (int t = blockIdx.z * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); tl.rho0 + t <= tl.last; t += 4 * gridDim.z) {
        const int rho = tl.rho0 + t;
        const size_t head = (size_t)kv * group + rho % group, row = w.sp.q0 + rho / group;
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
                        y[i][e] = lane + 64 * e < dim ? part.o[((size_t)min(z0 + i0 + i, tl.ranges - 1) * TILE + t) * padded_dim(dim) + lane + 64 * e] : 0.f;
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
    // The split kernels carry scale 2^-48 in one factor.
    const float size = s->scale < 0 ? -s->scale : s->scale;
    FMLH_REQUIRE(size == 0.f || (size >= 0x1p-60f && size <= 0x1p60f), "%s: scale %g is neither 0 nor of 2^-60 .. 2^60", fn,
                 (double)s->scale);
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
            (s->n_kv_head == 1 || ((s->k_hs | s->v_hs) & 3) == 0) &&
            std::max({s->q_rs, s->k_rs, s->v_rs, s->o_rs}) <= kMaxVecStride;
    return a;
}

uint32_t row_tiles(const PackedAttn& a, uint32_t per) { return (uint32_t)(((uint64_t)a.q_rows * a.group) / per) + a.n_seq; }
uint32_t key_tiles(const PackedAttn& a) { return a.k_rows / attn_split_back_rows(a) + a.n_seq; }

// Sequences of fewer keys are not cut: joining the ranges costs a launch of 5 us.
constexpr uint64_t kCutKeys = 512;

// Keys that a sequence has room for, on average (a cache in slabs holds a head's rows one behind the other).
uint64_t keys_per_sequence(const PackedAttn& a) {
    const uint64_t n = a.k_rows / a.n_seq;
    return a.k_hs > a.k_rs ? n / a.n_kv : n;
}

// How the forward pass cuts its work, by the sizes alone (lengths are the device's to know).
struct ForwardPlan {
    int per;          // rows per tile: kRowsPerWG or half of it, or at most 8 for attn_packed_few_kernel
    uint32_t tiles;   // at most, for a key head
    uint32_t budget;  // ranges to cut the tiles' keys into, for a key head; 0: none
};

ForwardPlan plan_forward(const PackedAttn& a) {
    ForwardPlan p;
    const uint64_t rows = (uint64_t)a.q_rows * a.group;  // of a key head
    const uint64_t per_seq = rows / a.n_seq;
    p.per = per_seq > 8 ? kRowsPerWG : per_seq > 4 ? 8 : per_seq > 2 ? 4 : per_seq > 1 ? 2 : 1;
    const uint64_t about = std::max<uint64_t>(a.n_seq, (rows + p.per - 1) / p.per) * a.n_kv;
    const bool prompts = 2 * (uint64_t)a.q_rows > keys_per_sequence(a) * a.n_seq, enough = keys_per_sequence(a) >= kCutKeys;
    // Work-groups to aim at (one that finds no range left costs its start).  Few rows: what keeps the memory busy.
    // Tiles of rows: two per CU are at work at once up to head_dim 64, and 512 end together (31 queries over 8 x 2000 ..
    // 32000 keys, 8 heads of 64: 95 us, with 768 121, with 1024 105).  Whole prompts leave the ranges behind a tile's
    // last row empty (4096 rows, 8 heads of 64: 188 with 512, 154 with 768; 1500 rows, 8 heads of 128: 104, 87
    // with 768 or 1024).
    const uint64_t want = p.per <= 8 ? 1024 : prompts ? 768 : 512;
    // Tiles up to which cutting pays.  Prompts: 2048 rows, 8 heads of 64 (128 tiles), 66 us cut, 76 whole; 16 heads
    // 96 and 82; 4 x 1024 rows, 8 heads of 128 (256), 147 and 94.
    const uint64_t few = p.per <= 8 ? 512 : prompts ? 128 : 256;
    p.budget = about <= few && enough ? (uint32_t)(want / a.n_kv) : 0;
    // Half the rows a tile, the keys shared by pairs of waves, where whole tiles leave CUs empty or ending early: 16 x
    // 20 .. 256 rows, 6 heads (126 tiles), 13.6 us, 17.0 with all rows; 4 x 1024, 12 heads (384), 65 and 82.  Short rows
    // lose where tiles are many (32 x 256, 6 heads, 384 tiles, 31.6 and 27.8), long ones too (16 x 512, 8 heads, 512, 49 and 44).
    if (p.per == kRowsPerWG && !p.budget && about <= (enough ? 400 : 256)) p.per = kRowsPerWG / 2;
    p.tiles = row_tiles(a, p.per);
    return p;
}

// Work-groups of a launch, all key heads': its threads stay inside 32 bits.
constexpr uint64_t kMaxGroups = 1u << 23;

// How the backward pass cuts the rows that a tile of keys sees.
int plan_parts(const PackedAttn& a) {
    const uint64_t tiles = std::max<uint64_t>(a.n_seq, a.k_rows / attn_split_back_rows(a)) * a.n_kv;
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
    const size_t forward = p.budget ? (size_t)a.n_kv * (p.tiles + p.budget) * p.per * (padded_dim(a.head_dim) + 2) : 0;
    if (!backward) return forward;
    const int parts = plan_parts(a);
    return std::max(forward, deltas(a) + (parts > 1 ? parts * attn_split_part_floats(a, key_tiles(a)) : 0));
}

}  // namespace

}  // namespace fmlh

using namespace fmlh;

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
    FMLH_REQUIRE(need == 0 || (uintptr_t)ws % 16 == 0, "%s: the workspace is not 16-byte aligned", fn);
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
    } else {
        FMLH_TRY(attn_split_forward(a, plan.per, items, plan.budget, out, lse, q, k, v, ws, stream()));
    }
    if (plan.budget) {
#define FMLH_JOIN(TILE)                                                                                                      \
    hipLaunchKernelGGL(attn_packed_join_kernel<TILE>, dim3(plan.tiles, a.n_kv, std::clamp<uint32_t>(2048 / (plan.tiles * a.n_kv), 1, (TILE + 3) / 4)), dim3(256), 0, stream(), a, out, \
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
    FMLH_REQUIRE(((uint64_t)row_tiles(a, attn_split_dq_rows(a)) + (uint64_t)key_tiles(a) * parts) * a.n_kv <= kMaxGroups / 2 &&
                     (uint64_t)a.q_rows * shape->n_head <= (uint64_t(1) << 27),
                 "%s: more than 2^22 tiles of rows and keys, or 2^27 rows of heads", fn);
    a.vec = a.vec && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(dout) && aligned16(dq) &&
            aligned16(dk) && aligned16(dv);
    FMLH_REQUIRE((uintptr_t)ws % 16 == 0, "%s: the workspace is not 16-byte aligned", fn);
    return attn_split_backward(a, shape->q_rows ? row_tiles(a, attn_split_dq_rows(a)) : 0, shape->k_rows ? key_tiles(a) : 0, parts, dq, dk, dv, ws,
                               dout, out, lse, q, k, v, ws + deltas(a), stream());
}

}  // extern "C"
