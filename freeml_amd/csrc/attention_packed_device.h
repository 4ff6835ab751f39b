// Device helpers of the packed attention kernels (attention_packed.hip, attention_packed_split.hip).
#pragma once

#include "attention_packed.h"
#include "bf16_split.h"

namespace fmlh {
namespace {

constexpr int kRowsPerWave = 32;
constexpr int kRowsPerWG = 4 * kRowsPerWave;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ uint32_t clamp_row(int32_t v, uint32_t rows) { return v < 0 ? 0u : min((uint32_t)v, rows); }

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

// Wave-wide integer scan (inclusive), sum and maximum, with wave_reduce's lane shifts.
template <class Op>
__device__ __forceinline__ int wave_scan_int(int v, int identity, Op op) {
#define FMLH_STEP(CTRL, ROWS) v = op(v, __builtin_amdgcn_update_dpp(identity, v, CTRL, ROWS, 0xf, false))
    FMLH_STEP(0x111, 0xf);
    FMLH_STEP(0x112, 0xf);
    FMLH_STEP(0x114, 0xf);
    FMLH_STEP(0x118, 0xf);
    FMLH_STEP(0x142, 0xa);
    FMLH_STEP(0x143, 0xc);
#undef FMLH_STEP
    return v;
}
__device__ __forceinline__ int wave_prefix_int(int v) {
    return wave_scan_int(v, 0, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_sum_int(int v) { return __builtin_amdgcn_readlane(wave_prefix_int(v), 63); }
__device__ __forceinline__ int wave_max_int(int v) {
    return __builtin_amdgcn_readlane(wave_scan_int(v, -0x7fffffff, [](int a, int b) { return max(a, b); }), 63);
}

// What a work-group does: tile `tile` of a sequence's `tiles`, and of the `ranges` that the sequence's
// keys are cut into (`per` keys each) number `range`.  tile0 / item0: the tile's number, and that of
// its first range, over all sequences.
struct Work {
    Span sp;
    uint32_t tile, tiles, tile0, item0;
    int range, ranges, per;
};

constexpr uint32_t kAtOnce = 512;  // work-groups of attention kernels on the device at once

// Finds work number `index`, counted in tiles (BY_TILE) or in (tile, range) items.  Sequence s has
// ceil(count_s / per_tile) tiles -- count: its keys (KEYS) or its rows of all heads of a group --
// and every one of them its keys' ranges.  `budget` ranges are spread over all tiles: one has the
// keys of all tiles / budget, so that long sequences are cut and short ones are not (budget 0: none
// is), and at least 128, or 256 for tiles of more rows: those start and end in the time of 256 keys
// (48 queries of 16 heads of 80 on 4 over 500 .. 4000 keys: 44 us with 128, 40 with 256).
// Every wave scans the offsets, 64 sequences at a time.  False behind the last sequence: grids hold
// sum / per_tile + n_seq tiles and budget items more, never fewer than there are.
// Up to 64 sequences whose keys are not cut come in the order of their work, most first over all of
// them, where the launch has more work-groups than run at once (below, finding the order only costs
// 1 us): a tile's level falls by one from each to the next, and work number `index` lies on the
// highest level T with more than index tiles on it and above.  (4 x 3584 rows, 8 heads of 64: sequence by
// sequence 478 us, so 350.)
template <bool KEYS, bool BY_TILE>
__device__ __forceinline__ bool find_work(const PackedAttn& a, uint32_t per_tile, uint32_t budget, uint32_t index, Work* w) {
    const uint32_t lane = threadIdx.x & 63;
    auto tiles_of = [&](const Span& p) {
        return (uint32_t)(((uint64_t)(KEYS ? p.kl : p.ql) * (KEYS ? 1u : a.group) + per_tile - 1) / per_tile);
    };
    Span p{};
    w->per = 0x40000000;
    if (budget) {
        // Keys of all tiles, in integers, so that every work-group and launch has the same: sums of 20 bits and of
        // the rest (cut launches have at most about 1000 tiles, so 2^41 keys of a sequence's).
        uint64_t keys = 0;
        for (uint32_t base = 0; base < a.n_seq; base += 64) {
            p = Span{};
            if (base + lane < a.n_seq) p = load_span(a, base + lane);
            const uint64_t x = (uint64_t)tiles_of(p) * p.kl;
            keys += wave_sum_int((int)(x & 0xfffff)) + ((uint64_t)wave_sum_int((int)(x >> 20)) << 20);
        }
        // An equal share, rounded up to whole `least`: 1 + 2^-18 covers the roundings of this quotient.
        const int least = per_tile <= 8 ? 128 : 256;
        const float share = __fmul_rn(__fmul_rn((float)keys, 1.0f + 0x1p-18f), __builtin_amdgcn_rcpf((float)(budget * least)));
        w->per = max(1, (int)ceilf(fminf(share, 0x1p30f / least))) * least;
    }
    if (!budget && a.n_seq <= 64 && gridDim.x > kAtOnce) {
        if (lane < a.n_seq) p = load_span(a, lane);
        const int n = tiles_of(p);  // at most 2^23, and a level 2^24: sums over 64 lanes stay inside 32 bits
        // Keys that a sequence's last tile sees (rows that see its first tile), in tiles.
        const int top = (int)min(KEYS ? (uint64_t)p.ql / per_tile : (uint64_t)p.kl * a.group / per_tile, (uint64_t)1 << 24);
        auto above = [&](int T) { return (uint32_t)wave_sum_int(min(max(top - T + 1, 0), n)); };  // tiles of level T and more
        int lo = -wave_max_int(n - top), hi = wave_max_int(top) + 1;  // above(lo) holds all, above(hi) none
        if (above(lo) <= index) return false;
        while (hi - lo > 1) {
            const int mid = lo + (hi - lo) / 2;
            if (above(mid) > index) lo = mid;
            else hi = mid;
        }
        const bool on = top - lo >= 0 && top - lo < n;
        const uint64_t level = __ballot(on);
        const uint32_t r = index - above(hi), mine = __builtin_popcountll(level & ((1ull << lane) - 1));
        const int l = __builtin_ctzll(__ballot(on && mine == r));
        const uint32_t upto = wave_prefix_int(n);
        w->sp.q0 = __builtin_amdgcn_readlane(p.q0, l);
        w->sp.ql = __builtin_amdgcn_readlane(p.ql, l);
        w->sp.k0 = __builtin_amdgcn_readlane(p.k0, l);
        w->sp.kl = __builtin_amdgcn_readlane(p.kl, l);
        w->tiles = __builtin_amdgcn_readlane(n, l);
        w->tile = __builtin_amdgcn_readlane(KEYS ? top - lo : n - 1 - (top - lo), l);
        w->tile0 = w->item0 = __builtin_amdgcn_readlane(upto - n, l) + w->tile;
        w->range = 0;
        w->ranges = 1;
        return true;
    }
    uint32_t tiles_before = 0, items_before = 0;
    for (uint32_t base = 0; base < a.n_seq; base += 64) {
        if (!budget || a.n_seq > 64) {
            p = Span{};
            if (base + lane < a.n_seq) p = load_span(a, base + lane);
        }
        const uint32_t n = tiles_of(p), r = max(1u, (p.kl + (uint32_t)w->per - 1) / (uint32_t)w->per), items = n * r;
        const uint32_t upto_t = wave_prefix_int(n), upto_i = wave_prefix_int(items);
        const uint64_t hit = __ballot((BY_TILE ? tiles_before + upto_t : items_before + upto_i) > index);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            w->sp.q0 = __builtin_amdgcn_readlane(p.q0, l);
            w->sp.ql = __builtin_amdgcn_readlane(p.ql, l);
            w->sp.k0 = __builtin_amdgcn_readlane(p.k0, l);
            w->sp.kl = __builtin_amdgcn_readlane(p.kl, l);
            w->tiles = __builtin_amdgcn_readlane(n, l);
            w->ranges = __builtin_amdgcn_readlane(r, l);
            const uint32_t first_t = tiles_before + __builtin_amdgcn_readlane(upto_t - n, l);
            const uint32_t first_i = items_before + __builtin_amdgcn_readlane(upto_i - items, l);
            w->tile = BY_TILE ? index - first_t : (index - first_i) / w->ranges;
            if (!KEYS) w->tile = w->tiles - 1 - w->tile;  // the last rows see the most keys: they start first
            w->range = BY_TILE ? 0 : (index - first_i) % w->ranges;
            w->tile0 = first_t + w->tile;
            w->item0 = first_i + w->tile * w->ranges;
            return true;
        }
        tiles_before += __builtin_amdgcn_readlane(upto_t, 63);
        items_before += __builtin_amdgcn_readlane(upto_i, 63);
    }
    return false;
}

// The rows of a tile of the forward and dq kernels, and the keys of its range.
struct RowTile {
    int rows, rho0, last;        // rows of the sequence and group; the tile's first and last
    int shift, nkeys;            // kl - ql; keys that the tile's last row sees
    int k_begin, k_end, ranges;  // this range's keys; ranges that hold any of the tile's (at least 1)
};

__device__ __forceinline__ RowTile row_tile(const PackedAttn& a, const Work& w, int per_tile) {
    RowTile t;
    t.rows = w.sp.ql * a.group;
    t.rho0 = w.tile * per_tile;
    t.last = min(t.rho0 + per_tile, t.rows) - 1;
    t.shift = (int)w.sp.kl - (int)w.sp.ql;
    t.nkeys = min(t.last / a.group + t.shift + 1, (int)w.sp.kl);
    t.ranges = t.nkeys <= w.per ? 1 : (t.nkeys + w.per - 1) / w.per;  // of one length, about
    const int each = t.ranges == 1 ? t.nkeys : ((t.nkeys + t.ranges - 1) / t.ranges + 63) / 64 * 64;
    t.k_begin = w.range * each;
    t.k_end = min(t.nkeys, t.k_begin + each);
    return t;
}

// Partial results of a tile's ranges in the workspace (16-byte aligned): outputs of every row, in whole
// 16 bytes, then maxima and sums.
struct Partials {
    float *o, *ml;
};
__host__ __device__ __forceinline__ int padded_dim(int dim) { return (dim + 3) & ~3; }
__device__ __forceinline__ Partials partials(float* ws, uint32_t n_kv, uint32_t kv, uint32_t items, uint32_t item, int per_tile, int dim) {
    const size_t rows = (size_t)n_kv * items * per_tile, at = ((size_t)kv * items + item) * per_tile;
    return Partials{ws + at * padded_dim(dim), ws + rows * padded_dim(dim) + 2 * at};
}

// Dims d .. d + 3 of a row, zeros past head_dim.
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

// Dims d .. d + 3 where at least d + 3 < DP; VEC: from memory without a branch, whatever lies past
// head_dim replaced by zeros.
template <bool VEC>
__device__ __forceinline__ floatx4 load4_padded(const float* row, int d, int dim, bool on) {
    if constexpr (VEC) {
        const bool in = on && d < dim;
        const floatx4 x = *reinterpret_cast<const floatx4*>(row + (in ? d : 0));
        floatx4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = in ? x[e] : 0.f;
        return v;
    } else {
        floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (on && d + e < dim) v[e] = row[d + e];
        return v;
    }
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

// Register r of a lane's 32 x 32 accumulator is row 8 (r / 4) + 4 h + r % 4 of it (h = lane / 32).
__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// acc (dims x 32 columns) += X^T w element by element over the pairs `seen` names only (bit r of lane
// (h, c): row acc_row(r, h), column c): nothing of a row that a column does not see reaches it, not
// even 0 * infinity.  row(n): where row n of X lies.  Rolled up: it runs for data that is rare.
template <int DP, class Row>
__device__ __forceinline__ void add_seen(floatx16 (&acc)[DP / 32], const floatx16& w, uint32_t seen, int h, int c, int dim, bool vec,
                                         Row row) {
#pragma unroll 1
    for (int n = 0; n < 32; ++n) {
        const int r = n >> 1, from = c + 32 * (n & 1);
        float mine = 0.f;
#pragma unroll
        for (int t = 0; t < 16; ++t) mine = t == r ? w[t] : mine;
        const float p = __shfl(mine, from);
        const bool on = (__shfl((int)seen, from) >> r) & 1;
        const float* x = row(acc_row(r, n & 1));
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const floatx4 y = load4(x, 32 * i + 8 * u + 4 * h, dim, vec);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][4 * u + e] += on ? p * y[e] : 0.f;
            }
    }
}

// S (32 x 32) = A B^T over DP dims on the fp32 matrix cores, A's row of lane column c and B's row
// both from memory.  The two k of a step are dims u and DP / 2 + u.
template <int DP>
__device__ __forceinline__ floatx16 rows_product(const float* a_row, const float* b_row, int dim, bool vec, int h) {
    floatx16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll 1
    for (int u = 0; u < DP / 2; u += 4) {
        const floatx4 x = load4(a_row, h * (DP / 2) + u, dim, vec), y = load4(b_row, h * (DP / 2) + u, dim, vec);
#pragma unroll
        for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], s, 0, 0, 0);
    }
    return s;
}

template <int N>
__device__ __forceinline__ void clear(floatx16 (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[i][r] = 0.f;
}

}  // namespace
}  // namespace fmlh
