// rlgpu_ops.hip — the operators of include/rlgpu.h for a policy network of the caller's own: log-probabilities and entropy of given actions, the clipped
// policy loss with a KL term, both with their gradients, and the gradient norm over many tensors with the clip.
//
// The mathematics of a row of logits x (temperature T, k = log2(e) / T, all exponentials in base 2):
//   t_i = k (x_i - max x) <= 0, e_i = 2^t_i, S = sum e_i, W = sum e_i t_i, L = log2 S
//   log s_i = ln2 (t_i - L), entropy H = -sum s_i log s_i = ln2 (L - W / S)
//   d(c logp + h H) / dx_i = (1/T) [c (1{i = a} - s_i) - h s_i (log s_i + H)]
// so one reading of the row gives everything a row needs (S and W), and a second one, from wherever the row still is, the gradient.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <utility>
#include <vector>

#include "../../include/rlgpu.h"

namespace {

constexpr float LN2 = 0.69314718055994530942f, LOG2E = 1.44269504088896340736f;
constexpr int STATS = RLGPU_POLICY_STATS;

__device__ __forceinline__ float wave_sum(float v) { for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64); return v; }
__device__ __forceinline__ float wave_max(float v) { for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64)); return v; }

template <typename T> struct Lowest;
template <> struct Lowest<float> { static constexpr float value = -3.4028234663852886e38f; };
template <> struct Lowest<__bf16> { static constexpr float value = -3.3895313892515355e38f; };
template <> struct Lowest<_Float16> { static constexpr float value = -65504.f; };

// what a launch over rows takes; mode decides which of the outputs are there
struct RowArgs {
    RlgpuPolicyRows p;
    float k, inv_t, log_floor;            // log2(e) / T, 1 / T, log(min_prob)
    float *logp, *entropy;                // optional
    const float *d_logp, *d_entropy;      // backward
    RlgpuPolicyLoss loss;                 // loss
    void* dlogits; int64_t ldd;           // optional
    float* row_stats;                     // [rows][STATS]
};
enum Mode { LOGP, BACKWARD, LOSS };

// exp(x) - 1 - x: near 0 by its series (the terms left out are under 2^-26 of the first), since the subtraction would cancel there
__device__ __forceinline__ float exp_minus_1_minus(float x) {
    if (fabsf(x) < 0.25f)
        return x * x * (0.5f + x * (1.f / 6 + x * (1.f / 24 + x * (1.f / 120 + x * (1.f / 720 + x * (1.f / 5040 + x * (1.f / 40320)))))));
    return expf(x) - 1.f - x;
}

// one row of the loss: d loss / d logp and d loss / d entropy, and the row's part of the statistics
__device__ void loss_row(const RowArgs& g, int row, float w, float logp, float H, bool floored, float& c, float& h, float (&st)[STATS]) {
    const RlgpuPolicyLoss& l = g.loss;
    const float x = logp - l.old_logp[row], adv = l.adv[row];
    const float r = expf(x);
    const float surr = r * adv, clipped = fminf(fmaxf(r, 1.f - l.clip_low), 1.f + l.clip_high) * adv;
    float value = -(clipped < surr ? clipped : surr);     // (a NaN in either stays: surr holds it)
    c = clipped < surr ? 0.f : -surr;
    float ref = 0.f;
    if (l.ref_logp) {
        const float d = l.ref_logp[row] - logp;
        ref = exp_minus_1_minus(d);
        value += l.kl_coef * ref;
        c -= l.kl_coef * expm1f(d);
    }
    value -= l.ent_coef * H;
    c = floored ? 0.f : c * w * l.scale;
    h = -l.ent_coef * w * l.scale;
    st[0] = H; st[1] = exp_minus_1_minus(x); st[2] = (r < 1.f - l.clip_low || r > 1.f + l.clip_high) ? 1.f : 0.f; st[3] = r;
    st[4] = ref; st[5] = 1.f; st[6] = value * w * l.scale; st[7] = w;
}

// One workgroup of 256 threads a row, three readings of it.
template <typename T, Mode MODE>
__global__ void __launch_bounds__(256) k_rows(RowArgs g) {
    __shared__ float red[3][4];
    const int row = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, A = g.p.n_actions;
    const T* x = (const T*)g.p.logits + (int64_t)row * g.p.ld;
    const uint8_t* mask = g.p.mask ? g.p.mask + (int64_t)row * g.p.ld_mask : nullptr;
    T* dx = (T*)g.dlogits + (int64_t)row * g.ldd;
    auto at = [&](int i) -> float { return mask && !mask[i] ? -INFINITY : (float)x[i]; };
    const int a = g.p.actions[row];
    const float w = MODE == LOSS && g.loss.weights ? g.loss.weights[row] : 1.f;
    bool on = a >= 0 && a < A && w != 0.f;
    float logp = 0.f, H = 0.f, c = 0.f, h = 0.f, mc = 0.f, L = 0.f, lpa = 0.f;
    float st[STATS] = {};
    if (on) {
        const float xa = at(a);
        float m = -INFINITY;
        for (int i = tid; i < A; i += 256) m = fmaxf(m, at(i));
        m = wave_max(m);
        if ((tid & 63) == 0) red[0][wave] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        // a row without an allowed action (or one of NaN alone: fmaxf passes over NaN) is summed against 0: it gives 0 or NaN
        const bool live = m > Lowest<T>::value && fabsf(m * g.k) < 3e38f;
        mc = live ? m * g.k : 0.f;
        float S = 0.f, W = 0.f;
        for (int i = tid; i < A; i += 256) {
            const float t = fmaf(at(i), g.k, -mc), e = exp2f(t);
            S += e; W += e * fmaxf(t, -1e30f);
        }
        S = wave_sum(S); W = wave_sum(W);
        if ((tid & 63) == 0) { red[1][wave] = S; red[2][wave] = W; }
        __syncthreads();
        S = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]); W = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
        if (!live) { on = S != 0.f; S = NAN; }
        if (on) {
            L = log2f(S);
            H = LN2 * (L - W / S);
            lpa = LN2 * (fmaf(xa, g.k, -mc) - L);
            H = H < 0.f ? 0.f : H; lpa = lpa > 0.f ? 0.f : lpa;          // (the rounding of mc can leave either an ulp of t off; a NaN stays)
            const bool floored = lpa < g.log_floor;
            logp = floored ? g.log_floor : lpa;
            if (MODE == BACKWARD) { c = floored ? 0.f : g.d_logp[row]; h = g.d_entropy ? g.d_entropy[row] : 0.f; }
            if (MODE == LOSS) loss_row(g, row, w, logp, H, floored, c, h, st);
        }
    }
    if (tid == 0) {
        if (g.logp) g.logp[row] = logp;
        if (g.entropy) g.entropy[row] = H;
    }
    if (MODE == LOSS && tid < STATS) g.row_stats[(int64_t)row * STATS + tid] = st[tid];
    if (MODE == LOGP || !g.dlogits) return;
    for (int i = tid; i < A; i += 256) {
        float d = 0.f;
        if (on) {
            const float t = fmaxf(fmaf(at(i), g.k, -mc), -1e30f), s = exp2f(t - L);
            d = -s * (c + h * (LN2 * (t - L) + H)) + (i == a ? c : 0.f);
        }
        dx[i] = (T)(d * g.inv_t);
    }
}

// the rows' statistics in a fixed order: 64 slices of rows, then the slices, in 64 bits
__global__ void __launch_bounds__(512) k_row_stats(const float* part, int64_t n, float* stats) {
    __shared__ double red[512];
    const int k = threadIdx.x & 7;
    double s = 0;
    for (int64_t i = threadIdx.x >> 3; i < n; i += 64) s += (double)part[i * STATS + k];
    red[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < STATS) {
        for (int j = 1; j < 64; j++) s += red[j * STATS + k];
        stats[k] = (float)s;
    }
}

// ---- gradient norm and clip ----------------------------------------------------------------------------------------------------------------------------
// A launch takes up to TENSORS tensors by value, cut into pieces of PIECE elements; workgroup b takes the pieces b, b + gridDim.x, ...
constexpr int TENSORS = 160, PIECE = 16384, CLIP_BLOCKS = 1024;
struct ClipBatch {
    int n;
    int first[TENSORS + 1];               // the first piece of each tensor; [n] = how many there are
    uint8_t dtype[TENSORS];
    void* g[TENSORS]; int64_t count[TENSORS];
};
static_assert(sizeof(ClipBatch) < 3900, "kernel arguments by value");

template <typename F> __device__ __forceinline__ void for_pieces(const ClipBatch& b, F&& f) {
    for (int piece = blockIdx.x; piece < b.first[b.n]; piece += gridDim.x) {
        int lo = 0, hi = b.n;                                          // the last tensor whose first piece is <= piece (empty tensors share their successor's)
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (b.first[mid] <= piece) lo = mid; else hi = mid; }
        const int64_t at = (int64_t)(piece - b.first[lo]) * PIECE;
        f(lo, at, (int)min((int64_t)PIECE, b.count[lo] - at));
    }
}
template <typename T> __device__ __forceinline__ double square_sum(const T* g, int n) {
    double s = 0;
    for (int i = threadIdx.x; i < n; i += 256) { const double v = (double)(float)g[i]; s += v * v; }
    return s;
}
__device__ __forceinline__ double block_sum(double s, double* red) {
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}
__global__ void __launch_bounds__(256) k_grad_squares(ClipBatch b, double* part) {
    __shared__ double red[4];
    double s = 0;
    for_pieces(b, [&](int t, int64_t at, int n) {
        if (b.dtype[t] == RLGPU_F32) s += square_sum((const float*)b.g[t] + at, n);
        else if (b.dtype[t] == RLGPU_BF16) s += square_sum((const __bf16*)b.g[t] + at, n);
        else s += square_sum((const _Float16*)b.g[t] + at, n);
    });
    s = block_sum(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}
template <typename T> __device__ __forceinline__ void scale_piece(T* g, int n, float f) {
    for (int i = threadIdx.x; i < n; i += 256) g[i] = (T)((float)g[i] * f);
}
// every workgroup adds the partial sums up itself, all in the same order: no launch in between
__global__ void __launch_bounds__(256) k_grad_scale(ClipBatch b, const double* part, int n_part, float max_norm, float grad_scale, float* norm_out) {
    __shared__ double red[4];
    double s = 0;
    for (int i = threadIdx.x; i < n_part; i += 256) s += part[i];
    s = block_sum(s, red);
    const double norm = (double)grad_scale * sqrt(s);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float f = (float)((double)grad_scale * fmin(1.0, (double)max_norm / (norm + 1e-6)));
    if (!(norm < INFINITY) || f == 1.f) return;
    for_pieces(b, [&](int t, int64_t at, int n) {
        if (b.dtype[t] == RLGPU_F32) scale_piece((float*)b.g[t] + at, n, f);
        else if (b.dtype[t] == RLGPU_BF16) scale_piece((__bf16*)b.g[t] + at, n, f);
        else scale_piece((_Float16*)b.g[t] + at, n, f);
    });
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------------------
thread_local char g_error[256] = "";
int fail(int code, const char* fmt, ...) {
    va_list v; va_start(v, fmt);
    vsnprintf(g_error, sizeof g_error, fmt, v);
    va_end(v);
    return code;
}
#define OCHK(call)                                                                                              \
    do {                                                                                                        \
        const hipError_t _s = (call);                                                                           \
        if (_s != hipSuccess) return fail(RLGPU_ERR_HIP, "%s: %s", #call, hipGetErrorString(_s));               \
    } while (0)

// the caller's current device is its own again when the call returns
struct OnDevice {
    int before = -1; hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device); else before = -1;
    }
    ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};

int64_t size_of(int dtype) { return dtype == RLGPU_F32 ? 4 : (dtype == RLGPU_BF16 || dtype == RLGPU_F16 ? 2 : 0); }
bool misaligned(const void* p, int64_t to) { return (uintptr_t)p % (uintptr_t)to != 0; }

int64_t workspace_bytes_for(int rows) { return std::max<int64_t>(16, (int64_t)rows * STATS * 4); }

int check_rows(const char* who, const RlgpuPolicyRows* p, const void* workspace, int64_t bytes) {
    if (!p) return fail(RLGPU_ERR_ARG, "%s: no rows", who);
    const int64_t size = size_of(p->dtype);
    if (!size) return fail(RLGPU_ERR_ARG, "%s: dtype %d is none of RLGPU_F32, RLGPU_BF16, RLGPU_F16", who, p->dtype);
    if (p->rows < 0 || p->n_actions < 1 || p->n_actions > (1 << 28)) return fail(RLGPU_ERR_ARG, "%s: %d rows of %d actions", who, p->rows, p->n_actions);
    if (!(p->temperature > 0.f) || !(p->temperature < INFINITY) || !(1.f / p->temperature < INFINITY)) return fail(RLGPU_ERR_ARG, "%s: temperature %g", who, (double)p->temperature);
    if (!(p->min_prob > 0.f && p->min_prob < 1.f)) return fail(RLGPU_ERR_ARG, "%s: min_prob %g is not between 0 and 1", who, (double)p->min_prob);
    if (p->rows == 0) return RLGPU_OK;
    if (!p->logits || !p->actions) return fail(RLGPU_ERR_ARG, "%s: logits and actions are needed", who);
    if (p->rows > 1 && p->ld < p->n_actions) return fail(RLGPU_ERR_ARG, "%s: logits' row stride %lld is under %d actions", who, (long long)p->ld, p->n_actions);
    if (p->mask && p->rows > 1 && p->ld_mask != 0 && p->ld_mask < p->n_actions) return fail(RLGPU_ERR_ARG, "%s: mask's row stride %lld", who, (long long)p->ld_mask);
    if (misaligned(p->logits, size) || misaligned(p->actions, 4)) return fail(RLGPU_ERR_ARG, "%s: logits or actions are not aligned to their type", who);
    if (!workspace || misaligned(workspace, 16) || bytes < workspace_bytes_for(p->rows))
        return fail(RLGPU_ERR_ARG, "%s: a workspace of %lld bytes, aligned to 16, is needed", who, (long long)workspace_bytes_for(p->rows));
    return RLGPU_OK;
}
// dlogits is the logits' own buffer, or shares no element with it: apart, or the other columns of the same rows
int check_gradient(const char* who, const RlgpuPolicyRows* p, const void* dlogits, int64_t ldd) {
    if (!dlogits) return fail(RLGPU_ERR_ARG, "%s: dlogits is needed", who);
    const int64_t size = size_of(p->dtype), A = p->n_actions, R = p->rows;
    if (R > 1 && ldd < A) return fail(RLGPU_ERR_ARG, "%s: dlogits' row stride %lld is under %lld actions", who, (long long)ldd, (long long)A);
    if (misaligned(dlogits, size)) return fail(RLGPU_ERR_ARG, "%s: dlogits is not aligned to its type", who);
    const int64_t ld = R > 1 ? p->ld : A;
    if (R <= 1) ldd = A;
    if (dlogits == p->logits && ldd == ld) return RLGPU_OK;
    const int64_t gap = (int64_t)((intptr_t)dlogits - (intptr_t)p->logits);      // bytes
    if (gap >= ((R - 1) * ld + A) * size || -gap >= ((R - 1) * ldd + A) * size) return RLGPU_OK;
    if (ld == ldd) { const int64_t d = ((gap % (ld * size)) + ld * size) % (ld * size); if (d >= A * size && d + A * size <= ld * size) return RLGPU_OK; }
    return fail(RLGPU_ERR_ARG, "%s: dlogits overlaps logits", who);
}

RowArgs row_args(const RlgpuPolicyRows* p) {
    RowArgs g{};
    g.p = *p;
    g.inv_t = 1.f / p->temperature; g.k = (float)(1.4426950408889634 / (double)p->temperature); g.log_floor = (float)std::log((double)p->min_prob);
    return g;
}
template <Mode MODE> int launch_rows(const RowArgs& g, hipStream_t s) {
    if (g.p.rows == 0) return RLGPU_OK;
    const dim3 grid(g.p.rows), block(256);
    if (g.p.dtype == RLGPU_F32) hipLaunchKernelGGL((k_rows<float, MODE>), grid, block, 0, s, g);
    else if (g.p.dtype == RLGPU_BF16) hipLaunchKernelGGL((k_rows<__bf16, MODE>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((k_rows<_Float16, MODE>), grid, block, 0, s, g);
    OCHK(hipGetLastError());
    return RLGPU_OK;
}

int clip_batches(int n) { return std::max(1, (n + TENSORS - 1) / TENSORS); }
int clip_share(int n_batches) { return std::max(256, 2 * CLIP_BLOCKS / n_batches); }   // workgroups of a launch, so that the partial sums stay few

}  // namespace

extern "C" {

const char* rlgpu_ops_last_error(void) { return g_error; }

int64_t rlgpu_policy_workspace(int32_t dtype, int32_t rows, int32_t n_actions) {
    if (!size_of(dtype) || rows < 0 || n_actions < 1) return fail(RLGPU_ERR_ARG, "rlgpu_policy_workspace: bad argument");
    return workspace_bytes_for(rows);
}

int rlgpu_action_logp(int device, const RlgpuPolicyRows* p, float* logp, float* entropy, void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_rows("rlgpu_action_logp", p, workspace, workspace_bytes)) return rc;
    if (p->rows == 0) return RLGPU_OK;
    if (!logp || misaligned(logp, 4) || misaligned(entropy, 4)) return fail(RLGPU_ERR_ARG, "rlgpu_action_logp: logp is needed, aligned to its type as entropy is");
    const OnDevice on(device); OCHK(on.err);
    RowArgs g = row_args(p);
    g.logp = logp; g.entropy = entropy;
    return launch_rows<LOGP>(g, (hipStream_t)stream);
}

int rlgpu_action_logp_backward(int device, const RlgpuPolicyRows* p, const float* d_logp, const float* d_entropy, void* dlogits, int64_t ld_dlogits,
                               void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "rlgpu_action_logp_backward";
    if (int rc = check_rows(who, p, workspace, workspace_bytes)) return rc;
    if (p->rows == 0) return RLGPU_OK;
    if (!d_logp || misaligned(d_logp, 4) || misaligned(d_entropy, 4)) return fail(RLGPU_ERR_ARG, "%s: d_logp is needed, aligned to its type as d_entropy is", who);
    if (int rc = check_gradient(who, p, dlogits, ld_dlogits)) return rc;
    const OnDevice on(device); OCHK(on.err);
    RowArgs g = row_args(p);
    g.d_logp = d_logp; g.d_entropy = d_entropy; g.dlogits = dlogits; g.ldd = ld_dlogits;
    return launch_rows<BACKWARD>(g, (hipStream_t)stream);
}

int rlgpu_policy_loss(int device, const RlgpuPolicyRows* p, const RlgpuPolicyLoss* l, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "rlgpu_policy_loss";
    if (int rc = check_rows(who, p, workspace, workspace_bytes)) return rc;
    if (!l || !l->stats || misaligned(l->stats, 4)) return fail(RLGPU_ERR_ARG, "%s: the loss and its stats are needed", who);
    if (!(l->clip_low >= 0.f && l->clip_low < 1.f && l->clip_high >= 0.f && l->clip_high < INFINITY))
        return fail(RLGPU_ERR_ARG, "%s: clip range %g below and %g above 1", who, (double)l->clip_low, (double)l->clip_high);
    if (!std::isfinite(l->ent_coef) || !std::isfinite(l->kl_coef) || !std::isfinite(l->scale)) return fail(RLGPU_ERR_ARG, "%s: a coefficient or the scale is not finite", who);
    if (l->kl_coef != 0.f && !l->ref_logp && p->rows) return fail(RLGPU_ERR_ARG, "%s: kl_coef without ref_logp", who);
    if (p->rows) {
        if (!l->old_logp || !l->adv) return fail(RLGPU_ERR_ARG, "%s: old_logp and adv are needed", who);
        for (const void* v : {(const void*)l->old_logp, (const void*)l->adv, (const void*)l->ref_logp, (const void*)l->weights, (const void*)l->logp})
            if (misaligned(v, 4)) return fail(RLGPU_ERR_ARG, "%s: a row vector is not aligned to its type", who);
        if (l->dlogits) if (int rc = check_gradient(who, p, l->dlogits, l->ld_dlogits)) return rc;
    }
    const OnDevice on(device); OCHK(on.err);
    RowArgs g = row_args(p);
    g.loss = *l; g.logp = l->logp; g.dlogits = l->dlogits; g.ldd = l->ld_dlogits; g.row_stats = (float*)workspace;
    if (int rc = launch_rows<LOSS>(g, (hipStream_t)stream)) return rc;
    hipLaunchKernelGGL(k_row_stats, dim3(1), dim3(512), 0, (hipStream_t)stream, (const float*)workspace, (int64_t)p->rows, l->stats);
    OCHK(hipGetLastError());
    return RLGPU_OK;
}

int64_t rlgpu_clip_grad_workspace(int32_t n) {
    if (n < 0) return fail(RLGPU_ERR_ARG, "rlgpu_clip_grad_workspace: %d tensors", n);
    return (int64_t)clip_batches(n) * clip_share(clip_batches(n)) * 8;
}

int rlgpu_clip_grad_norm(int device, int32_t n, void* const* grads, const int64_t* counts, const int32_t* dtypes, float max_norm, float grad_scale,
                         float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "rlgpu_clip_grad_norm";
    if (n < 0 || (n && (!grads || !counts || !dtypes))) return fail(RLGPU_ERR_ARG, "%s: %d tensors", who, n);
    if (!(max_norm >= 0.f)) return fail(RLGPU_ERR_ARG, "%s: max_norm %g", who, (double)max_norm);
    if (!(grad_scale > 0.f && grad_scale < INFINITY)) return fail(RLGPU_ERR_ARG, "%s: grad_scale %g", who, (double)grad_scale);
    if (!norm || misaligned(norm, 4)) return fail(RLGPU_ERR_ARG, "%s: norm is needed", who);
    if (!workspace || misaligned(workspace, 16) || workspace_bytes < rlgpu_clip_grad_workspace(n))
        return fail(RLGPU_ERR_ARG, "%s: a workspace of %lld bytes, aligned to 16, is needed", who, (long long)rlgpu_clip_grad_workspace(n));
    const bool writes = max_norm < INFINITY || grad_scale != 1.f;
    try {
        std::vector<std::pair<uintptr_t, uintptr_t>> spans;            // [begin, end) of every tensor with elements
        spans.reserve((size_t)n);
        for (int i = 0; i < n; i++) {
            const int64_t size = size_of(dtypes[i]);
            if (!size) return fail(RLGPU_ERR_ARG, "%s: tensor %d: dtype %d is none of RLGPU_F32, RLGPU_BF16, RLGPU_F16", who, i, dtypes[i]);
            if (counts[i] < 0 || counts[i] > (1ll << 40)) return fail(RLGPU_ERR_ARG, "%s: tensor %d: %lld elements", who, i, (long long)counts[i]);
            if (counts[i] == 0) continue;
            if (!grads[i] || misaligned(grads[i], size)) return fail(RLGPU_ERR_ARG, "%s: tensor %d is null or not aligned to its type", who, i);
            spans.emplace_back((uintptr_t)grads[i], (uintptr_t)grads[i] + (uintptr_t)(counts[i] * size));
        }
        if (writes) {
            std::sort(spans.begin(), spans.end());
            for (size_t i = 1; i < spans.size(); i++)
                if (spans[i].first < spans[i - 1].second) return fail(RLGPU_ERR_ARG, "%s: two of the tensors overlap: they would be scaled twice", who);
        }
    } catch (...) { return fail(RLGPU_ERR_NOMEM, "%s: out of host memory", who); }
    const OnDevice on(device); OCHK(on.err);
    const hipStream_t s = (hipStream_t)stream;
    double* const part = (double*)workspace;
    const int n_batches = clip_batches(n), share = clip_share(n_batches);
    auto batch = [&](int k, ClipBatch& b) {                            // -> workgroups for it
        int64_t pieces = 0;
        b.n = std::min(TENSORS, n - k * TENSORS);
        for (int i = 0; i < b.n; i++) {
            const int j = k * TENSORS + i;
            b.g[i] = grads[j]; b.count[i] = counts[j]; b.dtype[i] = (uint8_t)dtypes[j]; b.first[i] = (int)pieces;
            pieces += (counts[j] + PIECE - 1) / PIECE;
        }
        b.first[b.n] = (int)pieces;
        return pieces > INT32_MAX ? -1 : (int)std::min<int64_t>(pieces, share);
    };
    ClipBatch b;
    int n_part = 0;
    for (int k = 0; k < n_batches; k++) {
        const int blocks = batch(k, b);
        if (blocks < 0) return fail(RLGPU_ERR_ARG, "%s: too many elements", who);
        if (blocks == 0) continue;
        hipLaunchKernelGGL(k_grad_squares, dim3(blocks), dim3(256), 0, s, b, part + n_part);
        OCHK(hipGetLastError());
        n_part += blocks;
    }
    for (int k = 0; k < n_batches; k++) {
        int blocks = batch(k, b);
        if (!writes) { if (k) break; b.n = 0; b.first[0] = 0; blocks = 1; }   // the norm alone
        if (k && blocks == 0) continue;
        hipLaunchKernelGGL(k_grad_scale, dim3(std::max(1, blocks)), dim3(256), 0, s, b, (const double*)part, n_part, max_norm, grad_scale, k == 0 ? norm : (float*)nullptr);
        OCHK(hipGetLastError());
    }
    return RLGPU_OK;
}

}  // extern "C"
