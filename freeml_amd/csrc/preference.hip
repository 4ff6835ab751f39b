// Preference loss on the logits of packed pairs of sequences (fmlh_preference_logits) and the
// sequences' log-probabilities (fmlh_sequence_logprobs), beside cce_logits' cross entropy.
//
//   lp_s = sum over the rows of sequence s that have a target t of z[t] - log sum exp z
//   x_p = beta ((lp_2p - ref_2p) - (lp_2p+1 - ref_2p+1))         2p: chosen, 2p + 1: rejected
//   loss = mean over p of (1 - e) softplus(-x_p) + e softplus(x_p)
//   f_p = beta ((1 - e) sigmoid(-x_p) - e sigmoid(x_p)) / pairs  = -dloss/dlp_2p = dloss/dlp_2p+1
//   grad row = +f_p (onehot(t) - softmax z) for a chosen row, -f_p (...) for a rejected one
//
// Three launches: every row's log-probability (with its maximum and sum, kept for the gradient), each
// pair's x and f, and the gradient.  A row's factor needs both sequences of its pair, so the logits
// are read twice and the gradient written once: at 2841 rows of 50304, 1892 of them with a target, 98 us for the first
// pass (3.9 TB/s) and 165 for the gradient (952 MB, 5.8 TB/s, its first rows still in the memory-side cache).  Maxima and sums of exponentials are fp32; the
// log-probabilities and their sums over a sequence fp64 (a row adds about 10, a sequence 10^4).
#include "fmlh_internal.h"

namespace fmlh {

namespace {

constexpr unsigned kThreads = 256;

// What a row leaves in the workspace: log-probability (0 without a target), maximum, 1 / sum.
struct RowStat {
    double logp;
    float top, inv;
};

__device__ __forceinline__ uint32_t clamp_row(int32_t v, uint32_t rows) { return v < 0 ? 0u : min((uint32_t)v, rows); }

__device__ __forceinline__ int target_id(const float* target, uint32_t row, uint32_t vocab) {
    const float t = target[row];  // truncated, as cce_logits takes ids; -1 and what is outside: none
    return t > -1.0f && t < (float)vocab ? (int)t : -1;
}

// e^x for x <= 0 (below 2^-126: zero): x log2(e) rounds x twice, 2.3 |x| 2^-24 of the value where expf gives
// two units for twice the instructions (row_stat_kernel at 1900 rows of 50304: 115 us with expf, 98 so).
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// The running maximum and sum of exponentials of some values, joined over lanes and waves.
struct Running {
    float top = -INFINITY, sum = 0.f;
    __device__ __forceinline__ void add(const float (&x)[4]) {
        const float t = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), top);
        if (t != top) {  // a maximum moves a few times per thread
            sum *= top == -INFINITY ? 0.f : exp_neg(top - t);
            top = t;
        }
        const float base = top == -INFINITY ? 0.f : top;
        sum += (exp_neg(x[0] - base) + exp_neg(x[1] - base)) + (exp_neg(x[2] - base) + exp_neg(x[3] - base));
    }
    __device__ __forceinline__ void join_wave() {
        const float t = wave_max(top);
        sum = wave_sum(top == -INFINITY && !(sum != sum) ? 0.f : sum * expf(top - t));
        top = t;
    }
};

// Four floats at any 4-byte alignment (one load or store of 16 bytes).
typedef float floatx4 __attribute__((ext_vector_type(4), aligned(4)));

// Calls f(c, count, x) for the row's columns in fours (count 4 at c, the last ones alone, padded with
// -infinity), spread over `n` threads.  Which thread adds which columns does not go by the row's
// alignment: equal rows give equal bits wherever they lie.
template <int UNROLL, class F>
__device__ __forceinline__ void for_row(const float* z, uint32_t vocab, uint32_t tid, uint32_t n, F f) {
    const uint32_t body = vocab / 4, rest = vocab % 4;
    const floatx4* zb = reinterpret_cast<const floatx4*>(z);
    uint32_t i = tid;
    for (; i + (UNROLL - 1) * n < body; i += UNROLL * n) {
        floatx4 v[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) v[u] = zb[i + u * n];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const float x[4] = {v[u][0], v[u][1], v[u][2], v[u][3]};
            f(4 * (i + u * n), 4, x);
        }
    }
    for (; i < body; i += n) {
        const floatx4 v = zb[i];
        const float x[4] = {v[0], v[1], v[2], v[3]};
        f(4 * i, 4, x);
    }
    if (tid < rest) {
        const float x[4] = {z[4 * body + tid], -INFINITY, -INFINITY, -INFINITY};
        f(4 * body + tid, 1, x);
    }
}

// ROWS rows per work-group, a wave each (short rows), or one row for all its waves.
template <int ROWS>
__global__ __launch_bounds__(kThreads) void row_stat_kernel(RowStat* __restrict__ stats, const float* __restrict__ target,
                                                            const float* __restrict__ logits, uint32_t vocab, uint32_t rows) {
    __shared__ float sh[kThreads / kWave][2];
    const uint32_t wave = threadIdx.x / kWave;
    const uint32_t row = ROWS == 1 ? blockIdx.x : blockIdx.x * ROWS + wave;
    if (row >= rows) return;
    const int id = target_id(target, row, vocab);
    if (id < 0) {
        if (threadIdx.x % (ROWS == 1 ? kThreads : kWave) == 0) stats[row] = RowStat{0.0, 0.f, 0.f};
        return;
    }
    const float* z = logits + (size_t)row * vocab;
    const float zt = z[id];
    Running r;
    if (ROWS == 1) for_row<4>(z, vocab, threadIdx.x, kThreads, [&](uint32_t, int, const float(&x)[4]) { r.add(x); });
    else for_row<2>(z, vocab, threadIdx.x % kWave, kWave, [&](uint32_t, int, const float(&x)[4]) { r.add(x); });
    r.join_wave();
    float top = r.top, sum = r.sum;
    if (ROWS == 1) {
        if (threadIdx.x % kWave == 0) {
            sh[wave][0] = top;
            sh[wave][1] = sum;
        }
        __syncthreads();
        top = -INFINITY;
        for (int i = 0; i < (int)(kThreads / kWave); ++i) top = fmaxf(top, sh[i][0]);
        sum = 0.f;
        for (int i = 0; i < (int)(kThreads / kWave); ++i)
            sum += sh[i][0] == -INFINITY && sh[i][1] == 0.f ? 0.f : sh[i][1] * expf(sh[i][0] - top);
    }
    if (threadIdx.x % (ROWS == 1 ? kThreads : kWave) == 0) stats[row] = RowStat{(double)(zt - top) - log((double)sum), top, 1.0f / sum};
}

// The sum of a sequence's rows, by one wave: lanes take rows in turn, then a fixed tree.
__device__ __forceinline__ double sequence_sum(const RowStat* stats, const int32_t* off, uint32_t s, uint32_t rows) {
    const uint32_t a = clamp_row(off[s], rows), b = clamp_row(off[s + 1], rows);
    double t = 0.0;
    for (uint32_t r = a + threadIdx.x % kWave; r < b; r += kWave) t += stats[r].logp;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) t += __shfl_xor(t, d);
    return t;
}

__global__ void sequence_logp_kernel(float* __restrict__ logp, const RowStat* __restrict__ stats, const int32_t* __restrict__ off,
                                     uint32_t rows, uint32_t n_seq) {
    const uint32_t s = (blockIdx.x * blockDim.x + threadIdx.x) / kWave;
    if (s >= n_seq) return;
    const double t = sequence_sum(stats, off, s, rows);
    if (threadIdx.x % kWave == 0) logp[s] = (float)t;
}

__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

__global__ void pair_kernel(float* __restrict__ factor, double* __restrict__ pair_loss, float* __restrict__ logp,
                            const RowStat* __restrict__ stats, const int32_t* __restrict__ off, const float* __restrict__ ref,
                            uint32_t rows, uint32_t pairs, float beta, float smoothing) {
    const uint32_t p = (blockIdx.x * blockDim.x + threadIdx.x) / kWave;
    if (p >= pairs) return;
    const double c = sequence_sum(stats, off, 2 * p, rows), r = sequence_sum(stats, off, 2 * p + 1, rows);
    if (threadIdx.x % kWave != 0) return;
    const double e = smoothing;
    const double x = (double)beta * ((c - (double)ref[2 * p]) - (r - (double)ref[2 * p + 1]));
    pair_loss[p] = (1.0 - e) * softplus(-x) + (e > 0.0 ? e * softplus(x) : 0.0);  // softplus(inf) only where it counts
    factor[p] = (float)((double)beta * ((1.0 - e) / (1.0 + exp(x)) - e / (1.0 + exp(-x))) / (double)pairs);
    if (logp) {
        logp[2 * p] = (float)c;
        logp[2 * p + 1] = (float)r;
    }
}

// The mean of the pairs' losses: one wave, a fixed order.
__device__ __forceinline__ void pair_mean(float* loss, const double* pair_loss, uint32_t pairs) {
    double t = 0.0;
    for (uint32_t p = threadIdx.x % kWave; p < pairs; p += kWave) t += pair_loss[p];
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) t += __shfl_xor(t, d);
    if (threadIdx.x == 0) loss[0] = (float)(t / pairs);
}

__global__ void pair_mean_kernel(float* __restrict__ loss, const double* __restrict__ pair_loss, uint32_t pairs) {
    pair_mean(loss, pair_loss, pairs);
}

// The sequence that holds a row: the last offset at or below it (offsets do not fall), by 64 lanes.  -1: none.
__device__ __forceinline__ int row_sequence(const int32_t* off, uint32_t n_seq, uint32_t row) {
    if ((int64_t)row < off[0] || (int64_t)row >= off[n_seq]) return -1;
    uint32_t lo = 0, n = n_seq;  // among off[lo] .. off[lo + n - 1], off[lo] <= row
    while (n > 1) {
        const uint32_t step = (n + kWave - 1) / kWave, i = min((threadIdx.x % kWave) * step, n - 1);
        const uint64_t below = __ballot((int64_t)off[lo + i] <= row);
        const uint32_t last = below ? 63 - __builtin_clzll(below) : 0;  // the last lane at or below
        const uint32_t at = min(last * step, n - 1);
        n = min(step, n - at);
        lo += at;
        if (step == 1) break;
    }
    return (int)lo;
}

// grad may be logits: an element is read by the thread that writes it.  The last work-group but the
// rows' forms the loss.  Rows come in the reverse order of the first pass: what it read last may
// still lie in the memory-side cache.
template <int ROWS>
__global__ __launch_bounds__(kThreads) void pair_gradient_kernel(float* grad, const float* __restrict__ factor, const RowStat* __restrict__ stats,
                                                                 const float* __restrict__ target, const float* logits,
                                                                 const int32_t* __restrict__ off, uint32_t vocab, uint32_t rows,
                                                                 uint32_t n_seq, float* __restrict__ loss,
                                                                 const double* __restrict__ pair_loss) {
    if (blockIdx.x == gridDim.x - 1) {
        if (loss && threadIdx.x < kWave) pair_mean(loss, pair_loss, n_seq / 2);
        return;
    }
    const uint32_t at = ROWS == 1 ? blockIdx.x : blockIdx.x * ROWS + threadIdx.x / kWave;
    if (at >= rows) return;
    const uint32_t row = rows - 1 - at;
    const int id = target_id(target, row, vocab);
    const RowStat st = stats[row];
    const int s = row_sequence(off, n_seq, row);
    if (s < 0) return;
    float* g = grad + (size_t)row * vocab;
    const float* z = logits + (size_t)row * vocab;
    const uint32_t tid = ROWS == 1 ? threadIdx.x : threadIdx.x % kWave, n = ROWS == 1 ? kThreads : kWave;
    if (id < 0) {  // nothing to read
        for (uint32_t i = tid; i < vocab / 4; i += n) reinterpret_cast<floatx4*>(g)[i] = floatx4{0.f, 0.f, 0.f, 0.f};
        if (tid < vocab % 4) g[vocab / 4 * 4 + tid] = 0.f;
        return;
    }
    const float f = s & 1 ? -factor[s / 2] : factor[s / 2];
    auto value = [&](uint32_t c, int count, const float(&x)[4]) {
        floatx4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = f * (((int)(c + e) == id ? 1.0f : 0.0f) - exp_neg(x[e] - st.top) * st.inv);
        if (count == 4) *reinterpret_cast<floatx4*>(g + c) = y;
        else g[c] = y[0];
    };
    if (ROWS == 1) for_row<4>(z, vocab, tid, n, value);
    else for_row<2>(z, vocab, tid, n, value);
}

// Workspace: a RowStat per row, then a double and a float per pair.
size_t workspace_floats(uint32_t rows, uint32_t n_seq) { return (size_t)rows * 4 + ((size_t)n_seq + 1) / 2 * 3; }

int check(const char* fn, const void* ws, const float* target, const float* logits, const int32_t* off, uint32_t vocab,
          uint32_t rows, uint32_t n_seq) {
    FMLH_REQUIRE(off && ws && (rows == 0 || (target && logits)), "%s: null pointer", fn);
    FMLH_REQUIRE((uintptr_t)ws % 8 == 0, "%s: the workspace is not 8-byte aligned", fn);
    FMLH_REQUIRE(vocab >= 1 && vocab <= (1u << 24), "%s: vocab %u outside 1..2^24 (ids are floats)", fn, vocab);
    FMLH_REQUIRE(rows <= (1u << 23) && n_seq <= (1u << 24), "%s: more than 2^23 rows or 2^24 sequences", fn);
    return FMLH_OK;
}

// Rows of up to 1024 logits: a wave each.
bool short_rows(uint32_t vocab) { return vocab <= 1024; }

int launch_row_stats(RowStat* stats, const float* target, const float* logits, uint32_t vocab, uint32_t rows) {
    if (rows == 0) return FMLH_OK;
    if (short_rows(vocab))
        hipLaunchKernelGGL(row_stat_kernel<4>, dim3((rows + 3) / 4), dim3(kThreads), 0, stream(), stats, target, logits, vocab, rows);
    else
        hipLaunchKernelGGL(row_stat_kernel<1>, dim3(rows), dim3(kThreads), 0, stream(), stats, target, logits, vocab, rows);
    FMLH_LAUNCHED("row_stat_kernel");
    return FMLH_OK;
}

}  // namespace

}  // namespace fmlh

using namespace fmlh;

extern "C" {

int fmlh_preference_workspace(uint32_t rows, uint32_t n_seq, size_t* floats) {
    FMLH_REQUIRE(floats != nullptr, "fmlh_preference_workspace: null output pointer");
    *floats = workspace_floats(rows, n_seq);
    return FMLH_OK;
}

int fmlh_sequence_logprobs(float* logp, float* ws, const float* target, const float* logits, const int32_t* off, uint32_t vocab,
                           uint32_t rows, uint32_t n_seq) {
    const char* fn = "fmlh_sequence_logprobs";
    if (n_seq == 0) return FMLH_OK;
    FMLH_TRY(check(fn, ws, target, logits, off, vocab, rows, n_seq));
    FMLH_REQUIRE(logp != nullptr, "%s: null output pointer", fn);
    FMLH_TRY(ensure_init());
    RowStat* stats = reinterpret_cast<RowStat*>(ws);
    FMLH_TRY(launch_row_stats(stats, target, logits, vocab, rows));
    hipLaunchKernelGGL(sequence_logp_kernel, dim3((n_seq + 3) / 4), dim3(kThreads), 0, stream(), logp, stats, off, rows, n_seq);
    FMLH_LAUNCHED("sequence_logp_kernel");
    return FMLH_OK;
}

int fmlh_preference_logits(float* grad, float* loss, float* logp, float* ws, const float* target, const float* logits,
                           const int32_t* off, const float* ref_logp, uint32_t vocab, uint32_t rows, uint32_t pairs, float beta,
                           float smoothing) {
    const char* fn = "fmlh_preference_logits";
    FMLH_REQUIRE(pairs >= 1 && pairs <= (1u << 23), "%s: %u pairs (1..2^23)", fn, pairs);
    FMLH_TRY(check(fn, ws, target, logits, off, vocab, rows, 2 * pairs));
    FMLH_REQUIRE(ref_logp != nullptr, "%s: null reference log-probabilities", fn);
    FMLH_REQUIRE(grad || loss || logp, "%s: nothing to compute", fn);
    FMLH_REQUIRE(beta > 0.f && beta - beta == 0.f, "%s: beta %g is not positive and finite", fn, (double)beta);
    FMLH_REQUIRE(smoothing >= 0.f && smoothing <= 0.5f, "%s: smoothing %g outside 0..0.5", fn, (double)smoothing);
    FMLH_TRY(ensure_init());
    RowStat* stats = reinterpret_cast<RowStat*>(ws);
    double* pair_loss = reinterpret_cast<double*>(stats + rows);
    float* factor = reinterpret_cast<float*>(pair_loss + pairs);
    FMLH_TRY(launch_row_stats(stats, target, logits, vocab, rows));
    hipLaunchKernelGGL(pair_kernel, dim3((pairs + 3) / 4), dim3(kThreads), 0, stream(), factor, pair_loss, logp, stats, off,
                       ref_logp, rows, pairs, beta, smoothing);
    FMLH_LAUNCHED("pair_kernel");
    if (grad && rows) {
#define FMLH_GRADIENT(ROWS)                                                                                                     \
    hipLaunchKernelGGL(pair_gradient_kernel<ROWS>, dim3((rows + ROWS - 1) / ROWS + 1), dim3(kThreads), 0, stream(), grad, factor, \
                       stats, target, logits, off, vocab, rows, 2 * pairs, loss, pair_loss)
        if (short_rows(vocab)) FMLH_GRADIENT(4);
        else FMLH_GRADIENT(1);
#undef FMLH_GRADIENT
        FMLH_LAUNCHED("pair_gradient_kernel");
    } else if (loss) {
        hipLaunchKernelGGL(pair_mean_kernel, dim3(1), dim3(kWave), 0, stream(), loss, pair_loss, pairs);
        FMLH_LAUNCHED("pair_mean_kernel");
    }
    return FMLH_OK;
}

}  // extern "C"
