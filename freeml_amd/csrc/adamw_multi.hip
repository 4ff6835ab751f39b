// One AdamW step over many tensors (fmlh_adamw_update_multi): fmlh_adamw_update's arithmetic,
// element by element and in its order, with the tensors of a launch in a table and states in 32 or in 8 bits.
//
// 8-bit states hold m and r = sqrt(v) (half the exponents v would need) as e4m3 codes, 256
// consecutive elements sharing a power-of-two scale 2^(E - 127): E is the exponent of the block's
// largest value less 7, so that it lands in [2^7, 2^8) and no code overflows (e4m3 ends at 448).
// A step changes r by less than half a code most of the time (v moves by 1 - beta2), which rounding
// to nearest would drop for good: codes are rounded up or down at random instead, up with the
// probability of m's (of v's, the square's) distance from below, so that m and v are kept on average.
// The 16 random bits of either come from a hash of the seed, the tensor's number and the element's.  A
// positive r keeps at least the smallest code: rounded to zero, its update would be divided by eps alone.
#include "fmlh_internal.h"

#include <algorithm>
#include <vector>

namespace fmlh {

namespace {

constexpr unsigned kThreads = 256;
constexpr uint32_t kBlock = 256;            // elements that share a scale: one wave, four per lane
constexpr uint32_t kChunk = 4 * kBlock;     // elements per work-group
constexpr uint32_t kTensors = 64;           // per launch: the table travels as a kernel argument (4 KB)

struct Tensor {
    float* p;
    const float* g;
    void *m, *v;
    uint8_t *me, *ve;
    uint64_t n;
};

struct Table {
    Tensor t[kTensors];
    uint32_t chunk0[kTensors];  // first work-group of each tensor
    uint32_t count, first;      // tensors here, and the number of the first of them in the call
};

struct Step {
    float lr, b1, b2, ib1, ib2, ib1p, ib2p, eps, decay;  // ib*: 1 - beta, 1 - beta^t; decay: lr wd
    uint32_t seed_lo, seed_hi;
};

typedef float floatx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t mix32(uint32_t h) {
    h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
    h = (h ^ (h >> 13)) * 0xC2B2AE35u;
    return h ^ (h >> 16);
}

// m, v and p of one element after the step (fmlh_adamw_update's order, no contraction).
__device__ __forceinline__ void adamw(const Step& s, float g, float& p, float& m, float& v) {
#pragma clang fp contract(off)
    m = s.b1 * m + s.ib1 * g;
    v = s.b2 * v + s.ib2 * g * g;
    const float update = s.lr * (m / s.ib1p) / (sqrtf(v / s.ib2p) + s.eps);
    p = p + update - s.decay * p;
}

// Code of x in units 1 / to_unit, sign on top: up from the code below where the random fraction is
// below x's share of the gap to the next one (SQUARE: its square's share of the squares' gap).
template <bool SQUARE>
__device__ __forceinline__ uint32_t encode(float x, float to_unit, uint32_t rnd) {
#pragma clang fp contract(off)
    const float y = fabsf(x) * to_unit;
    const uint32_t sign = x < 0.f ? 0x80u : 0u;
    if (!(y < 256.f)) return 0x7fu | sign;  // infinite or NaN (scales go by the finite values): NaN
    const bool normal = y >= 0x1p-6f;
    const uint32_t bits = __float_as_uint(y), cut = bits & 0xfff00000u;
    const float small = floorf(y * 512.f);
    const float low = normal ? __uint_as_float(cut) : small * 0x1p-9f;
    const float high = normal ? __uint_as_float(cut + 0x100000u) : low + 0x1p-9f;
    float gap = high - low, rest = y - low;
    if (SQUARE) {
        gap = gap * (high + low);
        rest = rest * (y + low);
    }
    const uint32_t code = normal ? (bits >> 20) - (120u << 3) : (uint32_t)small;
    return (code + ((float)rnd * 0x1p-16f * gap < rest ? 1u : 0u)) | sign;
}

__device__ __forceinline__ float decode(uint32_t code, float unit) {
    return __builtin_amdgcn_cvt_f32_fp8((int)code, 0) * unit;
}

// A block's E from its values: the exponent of the largest finite one less 7, at least 1.
__device__ __forceinline__ uint32_t block_exponent(const float (&x)[4]) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float a = fabsf(x[e]);
        top = fmaxf(top, a < INFINITY ? a : 0.f);
    }
    const uint32_t ex = __float_as_uint(wave_max(top)) >> 23;
    return ex > 8 ? ex - 7 : 1;
}

__device__ __forceinline__ float unit_of(uint32_t E) { return __uint_as_float(E << 23); }

template <int BITS>
__global__ __launch_bounds__(kThreads) void adamw_multi_kernel(Table tab, Step s) {
    uint32_t lo = 0, hi = tab.count;  // the tensor this work-group's chunk falls to
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (tab.chunk0[mid] <= blockIdx.x) lo = mid;
        else hi = mid;
    }
    const Tensor t = tab.t[lo];
    const uint32_t lane = threadIdx.x % kWave;
    const uint64_t block = (uint64_t)(blockIdx.x - tab.chunk0[lo]) * (kChunk / kBlock) + threadIdx.x / kWave;
    const uint64_t i0 = block * kBlock + 4 * lane;
    if (block * kBlock >= t.n) return;  // the whole wave
    const int n = (int)min((uint64_t)4, t.n > i0 ? t.n - i0 : 0);
    float p[4] = {}, g[4] = {}, m[4] = {}, v[4] = {};
    uint32_t me = 0, ve = 0;
    if (BITS == 8) {
        me = t.me[block];
        ve = t.ve[block];
    }
    for (int e = 0; e < n; ++e) {
        p[e] = t.p[i0 + e];
        g[e] = t.g[i0 + e];
        if (BITS == 32) {
            m[e] = ((const float*)t.m)[i0 + e];
            v[e] = ((const float*)t.v)[i0 + e];
        } else {
            m[e] = decode(((const uint8_t*)t.m)[i0 + e], unit_of(me));
            const float r = decode(((const uint8_t*)t.v)[i0 + e], unit_of(ve));
            v[e] = r * r;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) adamw(s, g[e], p[e], m[e], v[e]);
    if (BITS == 32) {
        for (int e = 0; e < n; ++e) {
            t.p[i0 + e] = p[e];
            ((float*)t.m)[i0 + e] = m[e];
            ((float*)t.v)[i0 + e] = v[e];
        }
        return;
    }
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (e >= n) m[e] = v[e] = 0.f;
        r[e] = sqrtf(v[e]);
    }
    me = block_exponent(m);
    ve = block_exponent(r);
    uint32_t key = mix32(s.seed_lo ^ 0x9E3779B9u);
    key = mix32(key ^ (tab.first + lo + s.seed_hi));
    key ^= (uint32_t)(i0 >> 32) * 0x9E3779B9u;
    for (int e = 0; e < n; ++e) {
        const uint32_t rnd = mix32((uint32_t)(i0 + e) ^ key);
        const uint32_t cr = encode<true>(r[e], unit_of(254 - ve), rnd >> 16);
        t.p[i0 + e] = p[e];
        ((uint8_t*)t.m)[i0 + e] = (uint8_t)encode<false>(m[e], unit_of(254 - me), rnd & 0xffffu);
        ((uint8_t*)t.v)[i0 + e] = (uint8_t)(r[e] > 0.f ? max(cr, 1u) : cr);
    }
    if (lane == 0) {
        t.me[block] = (uint8_t)me;
        t.ve[block] = (uint8_t)ve;
    }
}

// Written ranges must not meet one another or a gradient that another entry reads after: an
// element listed twice would be updated by two work-groups at once.
int check_overlap(const fmlh_adamw_tensor* t, uint32_t count, int bits) {
    struct Range {
        uintptr_t a, b;
        bool written;
    };
    std::vector<Range> r;
    r.reserve((size_t)count * 6);
    for (uint32_t i = 0; i < count; ++i) {
        const size_t n = t[i].n, state = bits == 32 ? 4 * n : n, blocks = (n + kBlock - 1) / kBlock;
        if (!n) continue;
        auto put = [&](const void* p, size_t bytes, bool w) { r.push_back({(uintptr_t)p, (uintptr_t)p + bytes, w}); };
        put(t[i].param, 4 * n, true);
        put(t[i].grad, 4 * n, false);
        put(t[i].m, state, true);
        put(t[i].v, state, true);
        if (bits == 8) {
            put(t[i].m_exp, blocks, true);
            put(t[i].v_exp, blocks, true);
        }
    }
    std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.a < y.a; });
    uintptr_t end_written = 0, end_any = 0;
    for (const Range& x : r) {
        FMLH_REQUIRE(x.a >= (x.written ? end_any : end_written),
                     "fmlh_adamw_update_multi: tensors or states share memory (an entry listed twice?)");
        end_any = std::max(end_any, x.b);
        if (x.written) end_written = std::max(end_written, x.b);
    }
    return FMLH_OK;
}

}  // namespace

}  // namespace fmlh

using namespace fmlh;

extern "C" int fmlh_adamw_update_multi(const fmlh_adamw_tensor* tensors, uint32_t count, int state_bits, float lr, float beta1,
                                       float beta2, float beta1_pow_t, float beta2_pow_t, float eps, float weight_decay,
                                       uint64_t seed) {
    const char* fn = "fmlh_adamw_update_multi";
    FMLH_REQUIRE(tensors || count == 0, "%s: null tensors", fn);
    FMLH_REQUIRE(state_bits == 32 || state_bits == 8, "%s: states of %d bits (32 or 8)", fn, state_bits);
    for (uint32_t i = 0; i < count; ++i) {
        const fmlh_adamw_tensor& t = tensors[i];
        if (t.n == 0) continue;
        FMLH_REQUIRE(t.param && t.grad && t.m && t.v, "%s: null pointer in tensor %u", fn, i);
        FMLH_REQUIRE(state_bits == 32 || (t.m_exp && t.v_exp), "%s: null scales in tensor %u", fn, i);
        FMLH_REQUIRE(t.n <= (size_t(1) << 33), "%s: tensor %u holds more than 2^33 elements", fn, i);
    }
    try {
        FMLH_TRY(check_overlap(tensors, count, state_bits));
    } catch (const std::bad_alloc&) {
        return set_error(FMLH_E_INVALID, "%s: no host memory for %u tensors", fn, count);
    }
    FMLH_TRY(ensure_init());
    Step s;
    s.lr = lr;
    s.b1 = beta1;
    s.b2 = beta2;
    s.ib1 = 1.0f - beta1;
    s.ib2 = 1.0f - beta2;
    s.ib1p = 1.0f - beta1_pow_t;
    s.ib2p = 1.0f - beta2_pow_t;
    s.eps = eps;
    s.decay = lr * weight_decay;
    s.seed_lo = (uint32_t)seed;
    s.seed_hi = (uint32_t)(seed >> 32);
    for (uint32_t i = 0; i < count;) {
        Table tab;
        tab.count = 0;
        tab.first = i;
        uint64_t chunks = 0;
        for (; i < count && tab.count < kTensors; ++i) {
            const fmlh_adamw_tensor& t = tensors[i];
            const uint64_t more = (t.n + kChunk - 1) / kChunk;
            if (chunks + more > (1u << 23)) break;  // a launch's threads stay inside 32 bits
            tab.t[tab.count] = Tensor{t.param, t.grad, t.m, t.v, t.m_exp, t.v_exp, t.n};
            tab.chunk0[tab.count++] = (uint32_t)chunks;
            chunks += more;
        }
        if (chunks == 0) continue;
        if (state_bits == 32)
            hipLaunchKernelGGL(adamw_multi_kernel<32>, dim3((unsigned)chunks), dim3(kThreads), 0, stream(), tab, s);
        else
            hipLaunchKernelGGL(adamw_multi_kernel<8>, dim3((unsigned)chunks), dim3(kThreads), 0, stream(), tab, s);
        FMLH_LAUNCHED("adamw_multi_kernel");
    }
    return FMLH_OK;
}
