// Drafted tokens against the target's probabilities (include/cbq_serve.h).
//
// Draft i is kept while u_i q_i(d_i) < p_i(d_i) and all before it are; one token more
// is drawn from w = max(p - q, 0) of the row behind them, or from p, by the inverse of
// its sums.  Two numbers a draft decide which row that is, so every block finds it for
// itself, and only that row of p (and of q) is read: HBM bounds a large batch, two
// launches a small one.  The first launch adds the row up in chunks, the second finds
// the chunk in which the sums pass u times the total and reads that chunk again.
//
// All of it in 64 bits: a vocabulary of 10^5 has borders every 10^-5 of the sum, and
// fp32 sums would move one in a hundred draws to another token.
#include "cbq_device.h"
#include "cbq_paged.h"
#include "../../include/cbq_serve.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / CBQ_WAVE, kPer = 8;
constexpr int kChunk = kThreads * kPer;     // tokens of a chunk

struct VerifyArgs {
    const void *p, *q;
    int64_t p_st[2], q_st[2];
    const int64_t *drafts;
    const int32_t *n_drafts;
    const float *uniforms;
    int64_t *tokens;
    int32_t *counts;
    double2 *sums;                          // [batch][chunk]: of w, of p
    int32_t n_max, chunks;
    int64_t vocab;
};

// The row that a sequence's last token is drawn from
template <typename T> struct Row {
    const T *p, *q;
    int kept, n;
    int64_t without;                        // token whose w is 0 (a certain draft's), or -1

    __device__ __forceinline__ double target(int64_t v) const
    {
        const double x = (double)(float)p[v];
        return x > 0 ? x : 0;
    }
    // w(v), given p(v)
    __device__ __forceinline__ double rest(int64_t v, double x) const
    {
        if (v == without) return 0;
        if (!q) return x;
        const double w = (double)(float)p[v] - (double)(float)q[v];
        return w > 0 ? w : 0;
    }
};

template <typename T> __device__ __forceinline__ Row<T> find_row(const VerifyArgs &a, int b)
{
    const int lane = threadIdx.x & 63;
    Row<T> r;
    const int n = a.n_drafts ? (int)cbq_clamp_length(a.n_drafts[b], a.n_max) : a.n_max;
    int kept = n;
    for (int i0 = 0; i0 < n; i0 += CBQ_WAVE) {
        const int i = i0 + lane;
        bool keep = true;
        if (i < n) {
            const int64_t d = a.drafts[(int64_t)b * a.n_max + i];
            const bool in = d >= 0 && d < a.vocab;
            double p = 0, q = a.q ? 0 : 1;
            if (in) {
                p = (double)(float)((const T *)a.p)[b * a.p_st[0] + i * a.p_st[1] + d];
                if (a.q) q = (double)(float)((const T *)a.q)[b * a.q_st[0] + i * a.q_st[1] + d];
            }
            keep = (double)a.uniforms[(int64_t)b * (a.n_max + 1) + i] * q < p;
        }
        const uint64_t refused = __ballot(!keep);
        if (refused) {
            kept = i0 + __builtin_ctzll(refused);
            break;
        }
    }
    r.kept = kept;
    r.n = n;
    r.p = (const T *)a.p + b * a.p_st[0] + kept * a.p_st[1];
    r.q = kept < n && a.q ? (const T *)a.q + b * a.q_st[0] + kept * a.q_st[1] : nullptr;
    r.without = kept < n && !a.q ? a.drafts[(int64_t)b * a.n_max + kept] : -1;
    return r;
}

__device__ __forceinline__ double wave_sum(double x)
{
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

template <typename T> __global__ __launch_bounds__(kThreads) void sums_kernel(VerifyArgs a)
{
    __shared__ double2 part[kWaves];
    const int b = blockIdx.y, chunk = blockIdx.x;
    const Row<T> r = find_row<T>(a, b);
    const int64_t v0 = (int64_t)chunk * kChunk + threadIdx.x;
    double w = 0, p = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const int64_t v = v0 + i * kThreads;
        if (v < a.vocab) {
            const double x = r.target(v);
            p += x;
            w += r.rest(v, x);
        }
    }
    w = wave_sum(w);
    p = wave_sum(p);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / CBQ_WAVE] = make_double2(w, p);
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kWaves; i++) {
            w += part[i].x;
            p += part[i].y;
        }
        a.sums[(int64_t)b * a.chunks + chunk] = make_double2(w, p);
    }
}

// One wave a sequence.  Sums of lanes before this one, and of all.
__device__ __forceinline__ double lanes_before(double x, double &all)
{
    const int lane = threadIdx.x & 63;
    double s = x;
    for (int o = 1; o < CBQ_WAVE; o <<= 1) {
        const double y = __shfl_up(s, o);
        if (lane >= o) s += y;
    }
    all = __shfl(s, CBQ_WAVE - 1);
    const double before = __shfl_up(s, 1);
    return lane ? before : 0;
}

template <typename T> __global__ __launch_bounds__(CBQ_WAVE) void pick_kernel(VerifyArgs a)
{
    const int b = blockIdx.x, lane = threadIdx.x;
    const Row<T> r = find_row<T>(a, b);
    const double2 *sums = a.sums + (int64_t)b * a.chunks;
    double w = 0, p = 0;
    for (int c = lane; c < a.chunks; c += CBQ_WAVE) {
        w += sums[c].x;
        p += sums[c].y;
    }
    w = wave_sum(w);
    p = wave_sum(p);
    const bool all = !(w > 0);              // nothing left: p itself
    const double goal = (double)a.uniforms[(int64_t)b * (a.n_max + 1) + a.n_max] * (all ? p : w);
    // the first chunk whose sum passes the goal, or the last that adds to it
    double before = 0, start = 0;
    int at = -1;
    bool passed = false;
    for (int c0 = 0; c0 < a.chunks && !passed; c0 += CBQ_WAVE) {
        const int c = c0 + lane;
        const double x = c < a.chunks ? (all ? sums[c].y : sums[c].x) : 0;
        double total;
        const double mine = before + lanes_before(x, total);
        const uint64_t over = __ballot(x > 0 && mine + x > goal), some = __ballot(x > 0);
        passed = over != 0;
        const int from = passed ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
        if (from >= 0) {
            at = c0 + from;
            start = __shfl(mine, from);
        }
        before += total;
    }
    int64_t token = -1;
    if (at >= 0) {
        // the same inside the chunk, 64 lanes by 8 tokens in order
        const int64_t base = (int64_t)at * kChunk;
        bool found = false;
        for (int i0 = 0; i0 < kChunk && !found; i0 += CBQ_WAVE * kPer) {
            const int64_t v0 = base + i0 + lane * kPer;
            double x[kPer], sum = 0;
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                x[i] = 0;
                if (v0 + i < a.vocab) {
                    x[i] = r.target(v0 + i);
                    if (!all) x[i] = r.rest(v0 + i, x[i]);
                }
                sum += x[i];
            }
            double total;
            double run = start + lanes_before(sum, total);
            int64_t mine = -1, last = -1;
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                run += x[i];
                if (x[i] > 0) {
                    last = v0 + i;
                    if (mine < 0 && run > goal) mine = v0 + i;
                }
            }
            const uint64_t over = __ballot(mine >= 0), some = __ballot(last >= 0);
            found = over != 0;
            if (found) token = __shfl(mine, __builtin_ctzll(over));
            else if (some) token = __shfl(last, 63 - __builtin_clzll(some));
            start += total;
        }
    }
    for (int i = lane; i <= a.n_max; i += CBQ_WAVE)
        a.tokens[(int64_t)b * (a.n_max + 1) + i] =
            i < r.kept ? a.drafts[(int64_t)b * a.n_max + i] : i == r.kept ? token : -1;
    if (lane == 0) a.counts[b] = r.kept + 1;
}

template <typename T> int launch(const VerifyArgs &a, int batch, hipStream_t stream)
{
    for (int b = 0; b < batch; b += 65535) {        // a launch's second dimension
        VerifyArgs x = a;
        const int n = batch - b < 65535 ? batch - b : 65535;
        x.p = (const T *)a.p + b * a.p_st[0];
        if (a.q) x.q = (const T *)a.q + b * a.q_st[0];
        x.drafts += (int64_t)b * a.n_max;
        if (a.n_drafts) x.n_drafts += b;
        x.uniforms += (int64_t)b * (a.n_max + 1);
        x.tokens += (int64_t)b * (a.n_max + 1);
        x.counts += b;
        x.sums += (int64_t)b * a.chunks;
        sums_kernel<T><<<dim3(a.chunks, n), kThreads, 0, stream>>>(x);
        pick_kernel<T><<<n, CBQ_WAVE, 0, stream>>>(x);
        const int rc = cbq_launch_status("cbq_verify_drafts");
        if (rc != CK_SUCCESS) return rc;
    }
    return CK_SUCCESS;
}

bool sizes_ok(int64_t batch, int64_t vocab)
{
    return batch >= 0 && batch < (1 << 24) && vocab >= 1 && vocab < (1ll << 31);
}

int64_t chunks_of(int64_t vocab) { return cbq_ceil(vocab, kChunk); }

}  // namespace

extern "C" size_t cbq_verify_drafts_workspace(int batch, int64_t vocab)
{
    return sizes_ok(batch, vocab) ? (size_t)batch * chunks_of(vocab) * sizeof(double2) : 0;
}

extern "C" int cbq_verify_drafts(const void *probs, const int64_t *p_stride, const int64_t *drafts,
                                 const void *draft_probs, const int64_t *q_stride, int dtype,
                                 const int32_t *n_drafts, const float *uniforms, int batch,
                                 int n_max, int64_t vocab, int64_t *tokens, int32_t *counts,
                                 void *workspace, size_t workspace_bytes, hipStream_t stream)
{
    if (!sizes_ok(batch, vocab) || n_max < 0 || n_max >= (1 << 20) ||
        (int64_t)batch * n_max >= (1ll << 30) || dtype < CBQ_F32 || dtype > CBQ_F16)
        return CK_ERR_ARG;
    if (batch == 0) return CK_SUCCESS;
    if (!probs || !p_stride || (n_max > 0 && !drafts) || (draft_probs && !q_stride) || !uniforms ||
        !tokens || !counts || !workspace || ((uintptr_t)workspace & 15) != 0 ||
        workspace_bytes < cbq_verify_drafts_workspace(batch, vocab))
        return CK_ERR_ARG;
    VerifyArgs a;
    a.p = probs;
    a.q = n_max > 0 ? draft_probs : nullptr;
    for (int i = 0; i < 2; i++) {
        a.p_st[i] = p_stride[i];
        a.q_st[i] = a.q ? q_stride[i] : 0;
    }
    a.drafts = drafts;
    a.n_drafts = n_drafts;
    a.uniforms = uniforms;
    a.tokens = tokens;
    a.counts = counts;
    a.sums = (double2 *)workspace;
    a.n_max = n_max;
    a.chunks = (int32_t)chunks_of(vocab);
    a.vocab = vocab;
    if (dtype == CBQ_F32) return launch<float>(a, batch, stream);
    if (dtype == CBQ_BF16) return launch<__bf16>(a, batch, stream);
    return launch<_Float16>(a, batch, stream);
}
