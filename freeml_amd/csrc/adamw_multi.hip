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
//
// The bytes bound it: 10.7M elements with 32-bit states 63 us (301 MB, 4.75 TB/s), 124M with 8-bit ones 430 us (2.0 GB,
// 4.6 TB/s; a copy reaches 5.05).  With compiler divisions and roots, and one block per wave, 92 and 671.
#include "fmlh_internal.h"

#include <algorithm>
#include <vector>

namespace fmlh {

namespace {

constexpr unsigned kThreads = 256;
constexpr uint32_t kBlock = 256;                   // elements that share a scale: one wave, four per lane
constexpr int kPerWave = 4;                        // blocks that a wave requests before it works on the first
constexpr uint32_t kChunk = 4 * kPerWave * kBlock;  // elements per work-group
constexpr uint32_t kTensors = 64;                  // per launch: the table travels as a kernel argument (4 KB)

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
    float r1, r2;                                        // 1 / ib1p, 1 / ib2p
    uint32_t seed_lo, seed_hi;
    int fast;                                            // lr, eps, ib1p and ib2p lie where adamw_fast is exact
};

typedef float floatx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t mix32(uint32_t h) {
    h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
    h = (h ^ (h >> 13)) * 0xC2B2AE35u;
    return h ^ (h >> 16);
}

// m, v and p of one element after the step (fmlh_adamw_update's order, no contraction).
__device__ __forceinline__ void moments(const Step& s, float g, float& m, float& v) {
#pragma clang fp contract(off)
    m = s.b1 * m + s.ib1 * g;
    v = s.b2 * v + s.ib2 * g * g;
}
__device__ __forceinline__ float adamw_any(const Step& s, float p, float m, float v) {
#pragma clang fp contract(off)
    const float update = s.lr * (m / s.ib1p) / (sqrtf(v / s.ib2p) + s.eps);
    return p + update - s.decay * p;
}

// The same values in half the instructions, where no step leaves the normal numbers: correctly rounded
// quotients and roots by one exact residual each (P. Markstein, IBM J. Res. Dev. 34, 1990): with y the
// correctly rounded 1 / b and q near a / b, q + (a - b q) y rounds to a / b.
//   m: 0 or 2^-60 .. 2^96, v: 0 or 2^-96 .. 2^40, ib*: 2^-20 .. 1, lr: 2^-30 .. 2^20, eps: 2^-48 .. 2^20
// keep every residual a multiple of 2^-149 and every quotient above 2^-126.
__device__ __forceinline__ float divide(float a, float b, float y) {  // y: 1 / b
    const float q = a * y;
    return fmaf(fmaf(-b, q, a), y, q);
}
__device__ __forceinline__ float reciprocal(float b) {
    const float y = __builtin_amdgcn_rcpf(b);
    const float z = fmaf(fmaf(-b, y, 1.0f), y, y);
    return fmaf(fmaf(-b, z, 1.0f), z, z);
}
__device__ __forceinline__ float square_root(float x) {
    const float y = __builtin_amdgcn_rsqf(x);
    float g = x * y, h = 0.5f * y;
    const float e = fmaf(-h, g, 0.5f);
    g = fmaf(g, e, g);
    h = fmaf(h, e, h);
    return x == 0.f ? 0.f : fmaf(fmaf(-g, g, x), h, g);
}
__device__ __forceinline__ float adamw_fast(const Step& s, float p, float m, float v) {
#pragma clang fp contract(off)
    const float b = square_root(divide(v, s.ib2p, s.r2)) + s.eps;
    const float update = divide(s.lr * divide(m, s.ib1p, s.r1), b, reciprocal(b));
    return p + update - s.decay * p;
}

// Code of x in units 1 / to_unit, sign on top: up from the code below where the random fraction is
// below x's share of the gap to the next one.  In units of 2^-20 of a gap: up where 16 rnd < share.
__device__ __forceinline__ uint32_t encode(float x, float to_unit, uint32_t rnd) {
    const float y = fabsf(x) * to_unit;
    const uint32_t fine = (uint32_t)ceilf(y * 0x1p29f);  // below 2^-6, where the gap is 2^-9
    const uint32_t at = y >= 0x1p-6f ? __float_as_uint(y) - (960u << 20) : fine;
    return (at + (0xfffffu - (rnd << 4))) >> 20 | (x < 0.f ? 0x80u : 0u);
}
// Code of x >= 0, up where the fraction is below the square's share of the gap between the codes' squares.
__device__ __forceinline__ uint32_t encode_square(float x, float to_unit, uint32_t rnd) {
#pragma clang fp contract(off)
    const float y = x * to_unit;
    const bool normal = y >= 0x1p-6f;
    const uint32_t bits = __float_as_uint(y);
    const float small = floorf(y * 512.f);
    const float low = normal ? __uint_as_float(bits & 0xfff00000u) : small * 0x1p-9f;
    // 2^-3 of y's binade, at least 2^-9 (0x3b000000)
    const float gap = __int_as_float(max((int)(bits & 0x7f800000u) - (3 << 23), 0x3b000000));
    const float gap2 = gap * fmaf(2.0f, low, gap), rest = (y - low) * (y + low);
    uint32_t code = normal ? (bits >> 20) - 960u : (uint32_t)small;
    code += (float)rnd * 0x1p-16f * gap2 < rest ? 1u : 0u;
    return x > 0.f ? max(code, 1u) : code;
}

__device__ __forceinline__ float unit_of(uint32_t E) { return __uint_as_float(E << 23); }

// What a lane holds of a block: four consecutive elements.
template <int BITS>
struct Four {
    floatx4 p, g, m, v;  // v: 8-bit states' r until they are decoded
    uint32_t cm, cv;     // their codes
    uint32_t me, ve;
};

// `vec`: all 16-byte (codes: 4-byte) aligned and n >= 4; else n elements one by one, zeros behind.
template <int BITS>
__device__ __forceinline__ void load(Four<BITS>& f, const Tensor& t, uint64_t block, uint64_t i0, int n, bool vec) {
    f.p = f.g = f.m = f.v = floatx4{0.f, 0.f, 0.f, 0.f};
    f.cm = f.cv = f.me = f.ve = 0;
    const float *mf = (const float*)t.m, *vf = (const float*)t.v;
    const uint8_t *mc = (const uint8_t*)t.m, *vc = (const uint8_t*)t.v;
    if (BITS == 8) {
        f.me = t.me[block];
        f.ve = t.ve[block];
    }
    if (vec) {
        f.p = *reinterpret_cast<const floatx4*>(t.p + i0);
        f.g = *reinterpret_cast<const floatx4*>(t.g + i0);
        if (BITS == 32) {
            f.m = *reinterpret_cast<const floatx4*>(mf + i0);
            f.v = *reinterpret_cast<const floatx4*>(vf + i0);
        } else {
            f.cm = *reinterpret_cast<const uint32_t*>(mc + i0);
            f.cv = *reinterpret_cast<const uint32_t*>(vc + i0);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n) {
            f.p[e] = t.p[i0 + e];
            f.g[e] = t.g[i0 + e];
            if (BITS == 32) {
                f.m[e] = mf[i0 + e];
                f.v[e] = vf[i0 + e];
            } else {
                f.cm |= (uint32_t)mc[i0 + e] << (8 * e);
                f.cv |= (uint32_t)vc[i0 + e] << (8 * e);
            }
        }
}

template <int BITS>
__device__ __forceinline__ void store(const Four<BITS>& f, const Tensor& t, uint64_t i0, int n, bool vec) {
    float *mf = (float*)t.m, *vf = (float*)t.v;
    uint8_t *mc = (uint8_t*)t.m, *vc = (uint8_t*)t.v;
    if (vec) {
        *reinterpret_cast<floatx4*>(t.p + i0) = f.p;
        if (BITS == 32) {
            *reinterpret_cast<floatx4*>(mf + i0) = f.m;
            *reinterpret_cast<floatx4*>(vf + i0) = f.v;
        } else {
            *reinterpret_cast<uint32_t*>(mc + i0) = f.cm;
            *reinterpret_cast<uint32_t*>(vc + i0) = f.cv;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n) {
            t.p[i0 + e] = f.p[e];
            if (BITS == 32) {
                mf[i0 + e] = f.m[e];
                vf[i0 + e] = f.v[e];
            } else {
                mc[i0 + e] = (uint8_t)(f.cm >> (8 * e));
                vc[i0 + e] = (uint8_t)(f.cv >> (8 * e));
            }
        }
}

// A block's E: the exponent of its largest value less 7, at least 1.
__device__ __forceinline__ uint32_t block_exponent(floatx4 x) {
    const float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    const uint32_t ex = __float_as_uint(wave_max(top)) >> 23;
    return ex > 8 ? ex - 7 : 1;
}

// Whether every value is 0 or of 2^lo .. 2^hi (infinite and NaN are not).
__device__ __forceinline__ bool within(floatx4 x, int lo, int hi) {
    uint32_t least = 0xffffffffu, most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t twice = __float_as_uint(x[e]) << 1;  // without the sign
        least = min(least, twice - 1u);                     // 0 counts as the largest
        most = max(most, twice);
    }
    return least >= ((uint32_t)(lo + 127) << 24) - 1u && most < (uint32_t)(hi + 127) << 24;
}

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
    const bool aligned = (((uintptr_t)t.p | (uintptr_t)t.g) & 15) == 0 &&
                         (((uintptr_t)t.m | (uintptr_t)t.v) & (BITS == 32 ? 15 : 3)) == 0;
    const uint64_t first = (uint64_t)(blockIdx.x - tab.chunk0[lo]) * (kChunk / kBlock) + threadIdx.x / kWave;
    uint32_t key = mix32(s.seed_lo ^ 0x9E3779B9u);
    key = mix32(key ^ (tab.first + lo + s.seed_hi));
    Four<BITS> f[kPerWave];
#pragma unroll
    for (int b = 0; b < kPerWave; ++b) {
        const uint64_t block = first + 4 * b, i0 = block * kBlock + 4 * lane;
        if (block * kBlock >= t.n) break;  // the whole wave
        const int n = (int)min((uint64_t)4, t.n > i0 ? t.n - i0 : 0);
        load<BITS>(f[b], t, block, i0, n, aligned && (block + 1) * kBlock <= t.n);
    }
#pragma unroll
    for (int b = 0; b < kPerWave; ++b) {
        const uint64_t block = first + 4 * b, i0 = block * kBlock + 4 * lane;
        if (block * kBlock >= t.n) return;
        const int n = (int)min((uint64_t)4, t.n > i0 ? t.n - i0 : 0);
        Four<BITS>& x = f[b];
        if (BITS == 8) {
            typedef float floatx2 __attribute__((ext_vector_type(2)));
            const float mu = unit_of(x.me), vu = unit_of(x.ve);
            const floatx2 m0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)x.cm, false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)x.cm, true);
            const floatx2 r0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)x.cv, false), r1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)x.cv, true);
            x.m = floatx4{m0[0], m0[1], m1[0], m1[1]};
            const floatx4 r = floatx4{r0[0], r0[1], r1[0], r1[1]};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x.m[e] *= mu;
                const float root = r[e] * vu;
                x.v[e] = root * root;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float m = x.m[e], v = x.v[e];
            moments(s, x.g[e], m, v);
            x.m[e] = m;
            x.v[e] = v;
        }
        const bool ordinary = s.fast && !__ballot(!within(x.m, -60, 96) || !within(x.v, -96, 40));
        if (ordinary) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x.p[e] = adamw_fast(s, x.p[e], x.m[e], x.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x.p[e] = adamw_any(s, x.p[e], x.m[e], x.v[e]);
        }
        if (BITS == 8) {
            floatx4 r, m = x.m;
            uint32_t bad_m = 0, bad_r = 0;  // bytes of values that are not finite: NaN, and no part of the scales
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                r[e] = ordinary ? square_root(x.v[e]) : sqrtf(x.v[e]);
                if (!ordinary) {
                    if (!(fabsf(m[e]) < INFINITY)) bad_m |= (m[e] < 0.f ? 0xffu : 0x7fu) << (8 * e);
                    if (!(fabsf(r[e]) < INFINITY)) bad_r |= 0x7fu << (8 * e);
                    if (!(fabsf(m[e]) < INFINITY)) m[e] = 0.f;
                    if (!(fabsf(r[e]) < INFINITY)) r[e] = 0.f;
                }
                if (e >= n) m[e] = r[e] = 0.f;
            }
            const uint32_t me = block_exponent(m), ve = block_exponent(r);
            const uint32_t tkey = key ^ (uint32_t)(i0 >> 32) * 0x9E3779B9u;
            x.cm = bad_m;
            x.cv = bad_r;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t rnd = mix32((uint32_t)(i0 + e) ^ tkey);
                x.cm |= encode(m[e], unit_of(254 - me), rnd & 0xffffu) << (8 * e);
                x.cv |= encode_square(r[e], unit_of(254 - ve), rnd >> 16) << (8 * e);
            }
            if (lane == 0) {
                t.me[block] = (uint8_t)me;
                t.ve[block] = (uint8_t)ve;
            }
        }
        store<BITS>(x, t, i0, n, aligned && (block + 1) * kBlock <= t.n);
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
    s.r1 = 1.0f / s.ib1p;
    s.r2 = 1.0f / s.ib2p;
    auto in = [](float x, float lo, float hi) { return x >= lo && x <= hi; };
    s.fast = in(lr, 0x1p-30f, 0x1p20f) && in(eps, 0x1p-48f, 0x1p20f) && in(s.ib1p, 0x1p-20f, 1.0f) && in(s.ib2p, 0x1p-20f, 1.0f);
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
