// Drafted tokens against the target's probabilities (include/cbq_serve.h).
//
// Draft i is kept while u_i q_i(d_i) < p_i(d_i) and all before it are; one token more
// is drawn from w = max(p - q, 0) of the row behind them, or from p, by the inverse of
// its sums.  Two numbers a draft decide which row that is, so every wave finds it for
// itself, and only that row of p (and of q) is read: HBM bounds a large batch, two
// launches and their chains of dependent loads a small one.  The first launch adds the
// row up, a wave 512 tokens, the second finds the sum in which they pass u times the
// total and reads its tokens again.
//
// 64 sequences of seven drafts, 151936 tokens, fp32: 21 us, of which the sums take 16 (78
// MB, 4.9 TB/s where a copy of 1 GiB reaches 5.3); one of four drafts 10, the host and two
// launches of 4.
//
// All of it in 64 bits: a vocabulary of 10^5 has borders every 10^-5 of the sum, and
// fp32 sums would move one in a hundred draws to another token.
#include "cbq_device.h"
#include "cbq_paged.h"
#include "../../include/cbq_serve.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / CBQ_WAVE;
constexpr int kPer = 8, kUnit = CBQ_WAVE * kPer;        // tokens of a sum

struct VerifyArgs {
    const void *p, *q;
    int64_t p_st[2], q_st[2];
    const int64_t *drafts;
    const int32_t *n_drafts;
    const float *uniforms;
    int64_t *tokens;
    int32_t *counts;
    double2 *sums;                          // [batch][unit]: of w, of p
    int32_t *kept;                          // [batch]
    int32_t n_max, units;
    int64_t vocab;
};

template <typename T> struct alignas(sizeof(T)) Four {  // rows begin anywhere
    T e[4];
};

// The row that a sequence's last token is drawn from
template <typename T> struct Row {
    const T *p, *q;
    int64_t without;                        // token whose w is 0 (a certain draft's), or -1

    // p and w of n tokens from v on (n < 4: the row's last ones)
    __device__ __forceinline__ void four(int64_t v, int64_t n, double (&x)[4], double (&w)[4]) const
    {
        Four<T> a = {}, b = {};
        if (n >= 4) {
            a = *(const Four<T> *)(p + v);
            if (q) b = *(const Four<T> *)(q + v);
        } else {
#pragma unroll
            for (int i = 0; i < 3; i++)
                if (i < n) {
                    a.e[i] = p[v + i];
                    if (q) b.e[i] = q[v + i];
                }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double y = (double)(float)a.e[i], z = y - (double)(float)b.e[i];
            x[i] = y > 0 ? y : 0;
            w[i] = z > 0 && v + i != without ? z : 0;
        }
    }
};

// The first of a sequence's drafts that is refused, or their count
template <typename T> __device__ __forceinline__ int find_kept(const VerifyArgs &a, int b)
{
    const int lane = threadIdx.x & 63;
    const int n = a.n_drafts ? (int)cbq_clamp_length(a.n_drafts[b], a.n_max) : a.n_max;
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
        if (refused) return i0 + __builtin_ctzll(refused);
    }
    return n;
}

template <typename T> __device__ __forceinline__ Row<T> row_of(const VerifyArgs &a, int b, int kept)
{
    const int n = a.n_drafts ? (int)cbq_clamp_length(a.n_drafts[b], a.n_max) : a.n_max;
    Row<T> r;
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
    const int b = blockIdx.y, lane = threadIdx.x & 63;
    const int64_t u = (int64_t)blockIdx.x * kWaves + threadIdx.x / CBQ_WAVE;
    if (u >= a.units) return;
    const int kept = find_kept<T>(a, b);
    if (u == 0 && lane == 0) a.kept[b] = kept;
    const Row<T> r = row_of<T>(a, b, kept);
    double w = 0, p = 0;
#pragma unroll
    for (int i = 0; i < kPer / 4; i++) {
        const int64_t v = u * kUnit + i * 4 * CBQ_WAVE + lane * 4;
        double x[4], y[4];
        r.four(v, a.vocab - v, x, y);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            p += x[k];
            w += y[k];
        }
    }
    w = wave_sum(w);
    p = wave_sum(p);
    if (lane == 0) a.sums[(int64_t)b * a.units + u] = make_double2(w, p);
}

// The sum of the lanes before this one, and of all
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

// A block a sequence: its waves add up the sums, the first one finds the token
template <typename T> __global__ __launch_bounds__(kThreads) void pick_kernel(VerifyArgs a)
{
    __shared__ double2 part[kWaves];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const double2 *sums = a.sums + (int64_t)b * a.units;
    const int kept = a.kept[b];
    double w = 0, p = 0;
    for (int u = tid; u < a.units; u += kThreads) {
        w += sums[u].x;
        p += sums[u].y;
    }
    w = wave_sum(w);
    p = wave_sum(p);
    if (lane == 0) part[tid / CBQ_WAVE] = make_double2(w, p);
    __syncthreads();
    if (tid >= CBQ_WAVE) return;
    const Row<T> r = row_of<T>(a, b, kept);
    w = p = 0;
    for (int i = 0; i < kWaves; i++) {
        w += part[i].x;
        p += part[i].y;
    }
    const bool all = !(w > 0);              // nothing left: p itself
    const double goal = (double)a.uniforms[(int64_t)b * (a.n_max + 1) + a.n_max] * (all ? p : w);
    // the first unit whose sum passes the goal, or the last that adds to it; eight a lane
    double before = 0, start = 0;
    int64_t at = -1;
    bool passed = false;
    for (int64_t u0 = 0; u0 < a.units && !passed; u0 += kUnit) {
        double x[kPer], sum = 0, total;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int64_t u = u0 + lane * kPer + i;
            const double2 s = u < a.units ? sums[u] : make_double2(0, 0);
            x[i] = all ? s.y : s.x;
            sum += x[i];
        }
        double run = before + lanes_before(sum, total);
        double here = 0;
        int mine = -1, last = -1;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            if (x[i] > 0 && mine < 0) {
                last = i;
                here = run;
                if (run + x[i] > goal) mine = i;
            }
            run += x[i];
        }
        const uint64_t over = __ballot(mine >= 0), some = __ballot(last >= 0);
        passed = over != 0;
        const int from = passed ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
        if (from >= 0) {
            at = u0 + from * kPer + __shfl(last, from);     // mine, where it is one
            start = __shfl(here, from);
        }
        before += total;
    }
    int64_t token = -1;
    if (at >= 0) {
        // the same inside the unit, eight tokens a lane in order
        double x[kPer], sum = 0, total;
        const int64_t v0 = at * kUnit + lane * kPer;
#pragma unroll
        for (int i = 0; i < kPer / 4; i++) {
            double y[4], z[4];
            r.four(v0 + 4 * i, a.vocab - v0 - 4 * i, y, z);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                x[4 * i + k] = all ? y[k] : z[k];
                sum += x[4 * i + k];
            }
        }
        double run = start + lanes_before(sum, total);
        int mine = -1, last = -1;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            run += x[i];
            if (x[i] > 0) {
                last = i;
                if (mine < 0 && run > goal) mine = i;
            }
        }
        const uint64_t over = __ballot(mine >= 0), some = __ballot(last >= 0);
        const int from = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some | 1);
        const int in = __shfl(over ? mine : last, from);
        if (in >= 0) token = at * kUnit + from * kPer + in;
    }
    for (int i = lane; i <= a.n_max; i += CBQ_WAVE)
        a.tokens[(int64_t)b * (a.n_max + 1) + i] =
            i < kept ? a.drafts[(int64_t)b * a.n_max + i] : i == kept ? token : -1;
    if (lane == 0) a.counts[b] = kept + 1;
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
        x.sums += (int64_t)b * a.units;
        x.kept += b;
        sums_kernel<T><<<dim3((uint32_t)cbq_ceil(a.units, kWaves), n), kThreads, 0, stream>>>(x);
        pick_kernel<T><<<n, kThreads, 0, stream>>>(x);
        const int rc = cbq_launch_status("cbq_verify_drafts");
        if (rc != CK_SUCCESS) return rc;
    }
    return CK_SUCCESS;
}

bool sizes_ok(int64_t batch, int64_t vocab)
{
    return batch >= 0 && batch < (1 << 24) && vocab >= 1 && vocab < (1ll << 31);
}

int64_t units_of(int64_t vocab) { return cbq_ceil(vocab, kUnit); }

size_t sums_bytes(int64_t batch, int64_t vocab) { return (size_t)batch * units_of(vocab) * sizeof(double2); }

}  // namespace

extern "C" size_t cbq_verify_drafts_workspace(int batch, int64_t vocab)
{
    return sizes_ok(batch, vocab) ? sums_bytes(batch, vocab) + (size_t)batch * sizeof(int32_t) : 0;
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
    a.kept = (int32_t *)((char *)workspace + sums_bytes(batch, vocab));
    a.units = (int32_t)units_of(vocab);
    a.vocab = vocab;
    if (dtype == CBQ_F32) return launch<float>(a, batch, stream);
    if (dtype == CBQ_BF16) return launch<__bf16>(a, batch, stream);
    return launch<_Float16>(a, batch, stream);
}
