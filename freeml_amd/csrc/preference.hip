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
// are read twice and the gradient written once.  Maxima and sums of exponentials are fp32; the
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

template <class Op>
__device__ __forceinline__ float block_reduce(float v, float* sh, float identity, Op op) {
    v = wave_reduce(v, identity, op);
    __syncthreads();
    if (threadIdx.x % kWave == 0) sh[threadIdx.x / kWave] = v;
    __syncthreads();
    float r = sh[0];
    for (unsigned i = 1; i < blockDim.x / kWave; ++i) r = op(r, sh[i]);
    return r;
}

__global__ void row_stat_kernel(RowStat* __restrict__ stats, const float* __restrict__ target, const float* __restrict__ logits,
                                uint32_t vocab) {
    __shared__ float sh[kThreads / kWave];
    const uint32_t row = blockIdx.x;
    const int id = target_id(target, row, vocab);
    if (id < 0) {
        if (threadIdx.x == 0) stats[row] = RowStat{0.0, 0.f, 0.f};
        return;
    }
    const float* z = logits + (size_t)row * vocab;
    float top = -INFINITY;
    for (uint32_t c = threadIdx.x; c < vocab; c += kThreads) top = fmaxf(top, z[c]);
    top = block_reduce(top, sh, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
    float sum = 0.f;
    for (uint32_t c = threadIdx.x; c < vocab; c += kThreads) sum += expf(z[c] - top);
    sum = block_reduce(sum, sh, 0.f, [](float a, float b) { return a + b; });
    if (threadIdx.x == 0) stats[row] = RowStat{(double)(z[id] - top) - log((double)sum), top, 1.0f / sum};
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
__global__ void pair_mean_kernel(float* __restrict__ loss, const double* __restrict__ pair_loss, uint32_t pairs) {
    double t = 0.0;
    for (uint32_t p = threadIdx.x; p < pairs; p += kWave) t += pair_loss[p];
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) t += __shfl_xor(t, d);
    if (threadIdx.x == 0) loss[0] = (float)(t / pairs);
}

// The sequence that holds a row: the last offset at or below it (offsets do not fall).  -1: none.
__device__ __forceinline__ int row_sequence(const int32_t* off, uint32_t n_seq, uint32_t row) {
    if ((int64_t)row < off[0] || (int64_t)row >= off[n_seq]) return -1;
    uint32_t lo = 0, hi = n_seq;  // off[lo] <= row < off[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if ((int64_t)off[mid] <= row) lo = mid;
        else hi = mid;
    }
    return (int)lo;
}

// grad may be logits: an element is read by the thread that writes it.
__global__ void pair_gradient_kernel(float* grad, const float* __restrict__ factor, const RowStat* __restrict__ stats,
                                     const float* __restrict__ target, const float* logits,
                                     const int32_t* __restrict__ off, uint32_t vocab, uint32_t n_seq) {
    const uint32_t row = blockIdx.x;
    const int s = row_sequence(off, n_seq, row);
    if (s < 0) return;
    const int id = target_id(target, row, vocab);
    float* g = grad + (size_t)row * vocab;
    const float f = s & 1 ? -factor[s / 2] : factor[s / 2];
    const RowStat st = stats[row];
    const float* z = logits + (size_t)row * vocab;
    for (uint32_t c = threadIdx.x; c < vocab; c += kThreads)
        g[c] = id < 0 ? 0.f : f * (((int)c == id ? 1.0f : 0.0f) - expf(z[c] - st.top) * st.inv);
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

int launch_row_stats(RowStat* stats, const float* target, const float* logits, uint32_t vocab, uint32_t rows) {
    if (rows == 0) return FMLH_OK;
    hipLaunchKernelGGL(row_stat_kernel, dim3(rows), dim3(kThreads), 0, stream(), stats, target, logits, vocab);
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
    if (loss) {
        hipLaunchKernelGGL(pair_mean_kernel, dim3(1), dim3(kWave), 0, stream(), loss, pair_loss, pairs);
        FMLH_LAUNCHED("pair_mean_kernel");
    }
    if (grad && rows) {
        hipLaunchKernelGGL(pair_gradient_kernel, dim3(rows), dim3(kThreads), 0, stream(), grad, factor, stats, target, logits, off,
                           vocab, 2 * pairs);
        FMLH_LAUNCHED("pair_gradient_kernel");
    }
    return FMLH_OK;
}

}  // extern "C"
