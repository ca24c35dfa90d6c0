// rlgpu_ops.hip — the operators of include/rlgpu.h for a policy network of the caller's own: log-probabilities and entropy of given actions, the clipped
// policy loss with a KL term, both with their gradients, and the gradient norm over many tensors with the clip.
//
// The mathematics of a row of logits x (temperature T, k = log2(e) / T, all exponentials in base 2):
//   t_i = k x_i - m for an m near k max x, e_i = 2^t_i, S = sum e_i, W = sum e_i t_i, L = log2 S
//   log s_i = ln2 (t_i - L), entropy H = -sum s_i log s_i = ln2 (L - W / S)
//   d(c logp + h H) / dx_i = (1/T) [c (1{i = a} - s_i) - h s_i (log s_i + H)]
// so one reading of the row gives everything a row needs (S and W), and a second one, from wherever the row still is, the gradient.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <type_traits>
#include <utility>
#include <vector>

#include "../../include/rlgpu.h"

namespace {

constexpr float LN2 = 0.69314718055994530942f, LOG2E = 1.44269504088896340736f;
constexpr int STATS = RLGPU_POLICY_STATS, ROW_BLOCKS = 2048, SPLIT_ROWS = 128;
constexpr int64_t CACHE_BYTES = 256ll << 20, STREAM_BYTES = 2 * CACHE_BYTES;   // the last-level cache

// what a launch over rows takes; mode decides which of the outputs are there
struct RowArgs {
    RlgpuPolicyRows p;
    float k, inv_t, log_floor;            // log2(e) / T, 1 / T, log(min_prob)
    float near;                           // the least m that is neither far nor within CLEAR of Pack::LIMIT k
    unsigned turn;
    float *logp, *entropy;                // optional
    const float *d_logp, *d_entropy;      // backward
    RlgpuPolicyLoss loss;                 // loss
    void* dlogits; int64_t ldd;           // optional
    float* row_stats;                     // the workspace: of the loss [workgroups][STATS], each workgroup's sums over its rows; or a split call's parts
};
enum Mode { LOGP, BACKWARD, LOSS };
__device__ __forceinline__ int64_t row_offset(int row, int64_t ld) { return (int64_t)((uint64_t)(uint32_t)row * (uint32_t)ld); }   // (a stride has 32 bits, or there is one row)

// e^x by the hardware's 2^x: off by an ulp and by the rounding of x log2(e), |x| 2^-24, which is what a difference of log-probabilities is off by already
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }
// exp(x) - 1 - x: near 0 by its series (the terms left out are under 2^-26 of the first), since the subtraction would cancel there
__device__ __forceinline__ float exp_minus_1_minus(float x) {
    const float near = x * x * (0.5f + x * (1.f / 6 + x * (1.f / 24 + x * (1.f / 120 + x * (1.f / 720 + x * (1.f / 5040 + x * (1.f / 40320)))))));
    return fabsf(x) < 0.25f ? near : exp_of(x) - 1.f - x;
}
// exp(x) - 1, from that sum only where it is small against x: behind a reference that rules an action out, x is far below 0 or -inf
__device__ __forceinline__ float exp_minus_1(float x, float minus_x) { return fabsf(x) < 0.25f ? minus_x + x : exp_of(x) - 1.f; }

// what a row's numbers need besides its logits, asked for before the sums over them
struct RowInputs { float w, u, v, ref; };                 // weight; d_logp and d_entropy, or old_logp and adv; ref_logp
template <Mode MODE> __device__ __forceinline__ RowInputs row_inputs(const RowArgs& g, int row, float w) {
    RowInputs r{w, 0.f, 0.f, 0.f};
    if (MODE == BACKWARD) { r.u = g.d_logp[row]; r.v = g.d_entropy ? g.d_entropy[row] : 0.f; }
    if (MODE == LOSS) { r.u = g.loss.old_logp[row]; r.v = g.loss.adv[row]; if (g.loss.ref_logp) r.ref = g.loss.ref_logp[row]; }
    return r;
}
// one row of the loss: d loss / d logp and d loss / d entropy, and the row's part of the statistics.  In 32 bits, as logp itself is, whose error of a few 2^-24 is
// the larger one: a ratio that is nearer than that to a border of the clip can fall on either side of it, and counts there in the statistics too.
__device__ __forceinline__ void loss_row(const RowArgs& g, const RowInputs& in, float logp, float H, bool floored, float& c, float& h, float (&st)[STATS]) {
    const RlgpuPolicyLoss& l = g.loss;
    const float x = logp - in.u, adv = in.v, w = in.w;
    const float r = exp_of(x);
    const float surr = adv == 0.f && r == INFINITY ? 0.f : r * adv;       // (a ratio past float32's range)
    const float clipped = fminf(fmaxf(r, 1.f - l.clip_low), 1.f + l.clip_high) * adv;
    float value = -(clipped < surr ? clipped : surr);     // (a NaN in either stays: surr holds it)
    c = clipped < surr ? 0.f : -surr;
    float ref = 0.f;
    if (l.ref_logp) {
        const float d = in.ref - logp;
        ref = exp_minus_1_minus(d);
        if (l.kl_coef != 0.f) { value += l.kl_coef * ref; c -= l.kl_coef * exp_minus_1(d, ref); }
    }
    value -= l.ent_coef * H;
    c = floored ? 0.f : c * w * l.scale;
    h = -l.ent_coef * w * l.scale;
    st[0] = H; st[1] = exp_minus_1_minus(x); st[2] = (r < 1.f - l.clip_low || r > 1.f + l.clip_high) ? 1.f : 0.f; st[3] = r;
    st[4] = ref; st[5] = 1.f; st[6] = value * w * l.scale; st[7] = w;
}

// ---- 16 bytes of a row --------------------------------------------------------------------------------------------------------------------------------
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
typedef u32x4 __attribute__((aligned(2))) u32x4_any;      // a row starts wherever its stride puts it: global memory takes 16-byte accesses at any address
typedef uint64_t __attribute__((aligned(1))) u64_any;
typedef uint32_t __attribute__((aligned(1))) u32_any;
using f32x2 = __attribute__((ext_vector_type(2))) float;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;

// N values of T in 16 bytes.  An action that is not allowed and places behind a row's end hold FILL (as a number LIMIT: -9.97e36; float16: its lowest value, -65504):
// finite (an e t of 0 times -inf would be NaN), and 0 in any sum as long as its exponent is CLEAR of the row's.  Where it is not (a row's logits are next to it, or
// the temperature makes it an ordinary exponent: float16 from T of about 590 on) CAREFUL and EXACT sums leave it out by its value.  A caller's own logits of LIMIT or less
// are so left out too: they are masks.
template <typename T> struct Pack;
template <> struct Pack<float> {
    static constexpr int N = 4; static constexpr uint32_t FILL = 0xfcf00000u; static constexpr float LIMIT = -0x1.ep122f;
    static __device__ __forceinline__ float get(u32x4 v, int j) { const uint32_t w = v[j]; return __builtin_bit_cast(float, w); }   // (of v[j] itself the builtin takes element 0)
    static __device__ __forceinline__ u32x4 put(const float (&d)[4]) { u32x4 v; for (int j = 0; j < 4; j++) v[j] = __builtin_bit_cast(uint32_t, d[j]); return v; }
    using Bytes = uint32_t;                               // the mask of N values
    static __device__ __forceinline__ Bytes bytes(const uint8_t* m) { return *(const u32_any*)m; }
    static __device__ __forceinline__ u32x4 forbid(u32x4 v, Bytes b) {
        for (int j = 0; j < 4; j++) v[j] = (b >> (8 * j)) & 0xff ? v[j] : FILL;
        return v;
    }
};
template <typename T, typename T2> struct Pack16 {
    static constexpr int N = 8;
    using Bytes = uint64_t;
    static __device__ __forceinline__ Bytes bytes(const uint8_t* m) { return *(const u64_any*)m; }
    static __device__ __forceinline__ u32x4 put(const float (&d)[8]) {
        u32x4 v;
        for (int j = 0; j < 4; j++) v[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{d[2 * j], d[2 * j + 1]}), T2));
        return v;
    }
    static __device__ __forceinline__ u32x4 forbid16(u32x4 v, Bytes b, uint32_t fill) {
        for (int j = 0; j < 4; j++) {
            const uint32_t w = (uint32_t)(b >> (16 * j));
            v[j] = ((w & 0xff) ? v[j] & 0xffffu : fill) | ((w & 0xff00) ? v[j] & 0xffff0000u : fill << 16);
        }
        return v;
    }
};
template <> struct Pack<__bf16> : Pack16<__bf16, bf16x2> {
    static constexpr uint32_t FILL = 0xfcf0fcf0u; static constexpr float LIMIT = -0x1.ep122f;
    static __device__ __forceinline__ float get(u32x4 v, int j) { const uint32_t w = v[j >> 1]; return __builtin_bit_cast(float, j & 1 ? w & 0xffff0000u : w << 16); }
    static __device__ __forceinline__ u32x4 forbid(u32x4 v, Bytes b) { return forbid16(v, b, 0xfcf0u); }
};
template <> struct Pack<_Float16> : Pack16<_Float16, f16x2> {
    static constexpr uint32_t FILL = 0xfbfffbffu; static constexpr float LIMIT = -65504.f;
    static __device__ __forceinline__ float get(u32x4 v, int j) { return (float)__builtin_bit_cast(f16x2, (uint32_t)v[j >> 1])[j & 1]; }
    static __device__ __forceinline__ u32x4 forbid(u32x4 v, Bytes b) { return forbid16(v, b, 0xfbffu); }
};

// STREAM: past the caches.  Data of more than twice the last-level cache is gone from it before anybody asks again, and leaves there what others could use.
template <bool STREAM> __device__ __forceinline__ u32x4 load(const void* p) { return STREAM ? __builtin_nontemporal_load((const u32x4_any*)p) : *(const u32x4_any*)p; }
template <bool STREAM> __device__ __forceinline__ void store(void* p, u32x4 v) { if (STREAM) __builtin_nontemporal_store(v, (u32x4_any*)p); else *(u32x4_any*)p = v; }

// The larger of three.  (fmaxf would first quiet each operand, an instruction a value; a NaN that is dropped here still makes the row's sum NaN.)
__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c)); return r; }

// Between two pieces of a row.  Left alone, the scheduler unpacks every piece first and adds later, as the sums are one long chain, or keeps the 32-bit values of
// one pass for the next (219 registers where 32 hold a row in 16 bits).  The sets of 16 pieces a lane are at the limit of 128 registers all the same: their gradient
// spills 4 to 6 in 16 bits, the loss 4 to 10 in float32 and 20 to 23 in 16 bits, once a row.
__device__ __forceinline__ void piece_done() { __builtin_amdgcn_sched_barrier(0); }

// What a lane has of S and W.  `m` is the exponent (k x0) that its sums are taken against: not the maximum, but within SLACK of it, so that it hardly ever moves
// after the first piece and a row is summed in one pass, piece by piece as it arrives.
//
// A quick sum can fail where logits are far from what a policy has: e t is NaN where t is -inf, and where k x passes FAR (the mask's FILL, a caller's -1e30) the
// rounding of m would be an exponent itself.  W is then not finite, and the lane sums again with CAREFUL: against the exact maximum, with (x - x0) k for
// k x - m where m is far, no t below LOW, and without what is not allowed.
//
// A row whose m passes ROW_FAR, or in which FILL shows, is summed again as a whole, with EXACT: all t are (x - x0) k then.  The two kinds of t differ by the rounding of
// m, up to 2^2 at ROW_FAR, and must not be added up as one; a lane's own choice of them, at twice ROW_FAR, is of no account in a row that is not far.
enum Care { QUICK, CAREFUL, EXACT };
constexpr float SLACK = 8.f, ROW_FAR = 5e7f, FAR = 2 * ROW_FAR, LOWEST = -3.4028234663852886e38f;
constexpr float CLEAR = 160.f;            // so far under m FILL's e is 0 (float32 ends at 2^-149)
constexpr float LOW = -1e4f;              // 2^LOW is 0, and LOW times anything that occurs is finite: an exponent below is as good as LOW
// k x0, rounded: left to itself the compiler joins the product with the difference that it is used in, and m would have another value in every place
__device__ __forceinline__ float times_k(float x0, float k) {
#pragma clang fp contract(off)
    return x0 * k;
}
__device__ __forceinline__ bool is_far(float m) { return !(fabsf(m) < FAR); }
template <Care C> __device__ __forceinline__ float exponent(float x, float k, float x0, float m) { return C == EXACT || (C == CAREFUL && is_far(m)) ? (x - x0) * k : fmaf(x, k, -m); }
__device__ __forceinline__ float allowed(float x, float limit) { return x <= limit ? -INFINITY : x; }                 // (a NaN stays)
__device__ __forceinline__ bool needs_exact(const RowArgs& g, float m) { return !(m >= g.near && m < ROW_FAR); }   // far, or FILL shows
template <Care C> __device__ __forceinline__ float step_to(float x0, float m, float new_x0, float new_m, float k) {
    return fmaxf(C == EXACT || (C == CAREFUL && (is_far(m) || is_far(new_m))) ? (x0 - new_x0) * k : m - new_m, LOW);
}
// what a row's exponents are taken against: t = (x - a) k - b with a = x0 and b = 0, or a = 0 and b = m
struct Base {
    float a, b;
    __device__ __forceinline__ Base(bool exact, float x0, float m) : a(exact ? x0 : 0.f), b(exact ? 0.f : m) {}
    __device__ __forceinline__ float t(float x, float k) const { return fmaf(x - a, k, -b); }
};
template <Care C> using care = std::integral_constant<Care, C>;
struct RowSum {
    float x0, m, s[2], w[2];
    __device__ __forceinline__ void clear() { x0 = LOWEST; m = -INFINITY; s[0] = s[1] = w[0] = w[1] = 0.f; }
    // `top`: the largest x of what comes next
    template <Care C> __device__ __forceinline__ void reach(float top, float k) {
        const float to = times_k(top, k);
        if (C != QUICK ? top > x0 : to > m + SLACK) {
            const float by = step_to<C>(x0, m, top, to, k), f = __builtin_amdgcn_exp2f(by);
            for (int j = 0; j < 2; j++) { w[j] = f * fmaf(s[j], by, w[j]); s[j] *= f; }
            x0 = top; m = to;
        }
    }
    template <Care C, typename P> __device__ __forceinline__ void add(float x, float k, int j) {
        if (C != QUICK) x = allowed(x, P::LIMIT);
        const float t = exponent<C>(x, k, x0, m), e = __builtin_amdgcn_exp2f(t);
        s[j] += e; w[j] = fmaf(e, C != QUICK ? fmaxf(t, LOW) : t, w[j]);
    }
    template <Care C, typename P> __device__ __forceinline__ void piece(u32x4& v, float k) {
        float top = max3(P::get(v, 0), P::get(v, 1), P::get(v, 2));
#pragma unroll
        for (int j = 3; j + 1 < P::N; j += 2) top = max3(top, P::get(v, j), P::get(v, j + 1));
        reach<C>(max3(top, P::get(v, P::N - 1), P::get(v, P::N - 1)), k);
#pragma unroll
        for (int j = 0; j < P::N; j++) add<C, P>(P::get(v, j), k, j & 1);
        asm("" : "+v"(v), "+v"(s[0]), "+v"(s[1]), "+v"(w[0]), "+v"(w[1]));
        piece_done();
    }
    __device__ __forceinline__ float S() const { return s[0] + s[1]; }
    __device__ __forceinline__ float W() const { return w[0] + w[1]; }
};

// ---- sums and maxima over the G lanes of a row; G <= 16 stays in a DPP row, more than 64 goes through LDS (`red`: one float a wavefront) ----------------------
// (a bound-checked move of a lane that is always there: the compiler folds it into the operation)
template <int CTRL> __device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }
struct Sum { static __device__ __forceinline__ int of(int a, int b) { return __builtin_bit_cast(int, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b)); } };
struct Max { static __device__ __forceinline__ int of(int a, int b) { return max(a, b); } };        // of in_order()
template <int N, typename OP> __device__ __forceinline__ int lanes_of(int v) {        // over aligned groups of N lanes, every lane gets the result
    v = OP::of(v, dpp<0xB1>(v));                          // quad_perm 1 0 3 2
    if (N > 2) v = OP::of(v, dpp<0x4E>(v));               // quad_perm 2 3 0 1
    if (N > 4) v = OP::of(v, dpp<0x141>(v));              // row_half_mirror
    if (N > 8) v = OP::of(v, dpp<0x140>(v));              // row_mirror
    if (N > 16) v = OP::of(v, __shfl_xor(v, 16, 64));
    if (N > 32) v = OP::of(v, __shfl_xor(v, 32, 64));
    return v;
}
// floats as integers of the same order (their own inverse): maxima of integers need no quieting of NaN, which none of these is
__device__ __forceinline__ int in_order(int i) { return i ^ ((i >> 31) & 0x7fffffff); }
template <int N, typename OP> __device__ __forceinline__ float lanes(float f) {
    const int v = __builtin_bit_cast(int, f);
    if constexpr (std::is_same_v<OP, Max>) return __builtin_bit_cast(float, in_order(lanes_of<N, Max>(in_order(v))));
    else return __builtin_bit_cast(float, lanes_of<N, Sum>(v));
}
template <int G, typename OP> __device__ __forceinline__ void put_wave(float v, float* red) { v = lanes<64, OP>(v); if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v; }
template <int G, typename OP> __device__ __forceinline__ float get_waves(const float* red) { constexpr int W = G / 64; return lanes<W, OP>(red[threadIdx.x & (W - 1)]); }

// What follows from a row's x0, S and W and its action's logit: whether it counts, its outputs, and what its gradient needs.
struct RowNumbers { float logp, H, lpa, L, c, h; bool on; };
template <Mode MODE, typename P> __device__ __forceinline__ RowNumbers row_numbers(const RowArgs& g, const RowInputs& in, float x0, Base base, float S, float W, float xa, float (&st)[STATS]) {
    RowNumbers n{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, true};
    if (!(x0 > P::LIMIT)) n.on = S != S;                    // nothing is allowed, but a NaN shows
    if (!n.on) return n;
    n.L = __builtin_amdgcn_logf(S);                       // (log2; S is about 1 at least)
    const float H = LN2 * (n.L - W * __builtin_amdgcn_rcpf(S)), lpa = LN2 * (base.t(xa, g.k) - n.L);
    n.H = H < 0.f ? 0.f : H;                              // (the rounding of m can leave either an ulp of t off; a NaN stays)
    n.lpa = xa <= P::LIMIT ? LOW : lpa > 0.f ? 0.f : (lpa < LOW ? LOW : lpa);    // (below every floor)
    const bool floored = n.lpa < g.log_floor;
    n.logp = floored ? g.log_floor : n.lpa;
    if (MODE == BACKWARD) { n.c = floored ? 0.f : in.u; n.h = in.v; }
    if (MODE == LOSS) loss_row(g, in, n.logp, n.H, floored, n.c, n.h, st);
    return n;
}
// The gradient of a piece: e_i / S [ -c - h (H + ln2 (t_i - L)) ] / T as e_i (p0 + p1 t_i).  The action's own c / T comes in a store of its own, of the lane that
// wrote the 16 bytes around it.
struct RowGradient {
    float k, p0, p1; Base base; bool careful;
    __device__ __forceinline__ RowGradient(const RowArgs& g, const RowNumbers& n, Base base, bool careful) : k(g.k), base(base) {
        const float inv = g.inv_t * __builtin_amdgcn_exp2f(-n.L);
        p1 = -n.h * LN2 * inv; p0 = -(n.c + n.h * (n.H - LN2 * n.L)) * inv;
        // an e_i of 0 times p0 + p1 t_i is 0 while that is finite: any t_i may be -3e38
        this->careful = careful || !(fmaf(fabsf(p0), 0x1p-126f, fabsf(p1)) < 0.5f);
    }
    __device__ __forceinline__ float quick(float x) const { const float t = fmaf(x, k, -base.b); return __builtin_amdgcn_exp2f(t) * fmaf(p1, t, p0); }
    template <typename P> __device__ __forceinline__ float of(float x) const {
        // (e first: an e of 0 leaves nothing of a p1 t that is not finite)
        const float t = fmaxf(base.t(x, k), LOW), e = __builtin_amdgcn_exp2f(t);
        return x <= P::LIMIT ? 0.f : fmaf(e * p1, t, e * p0);
    }
    template <typename P> __device__ __forceinline__ u32x4 piece(u32x4 q) const {
        float d[P::N];
        if (careful) {
#pragma unroll
            for (int j = 0; j < P::N; j++) d[j] = of<P>(P::get(q, j));
        } else {
#pragma unroll
            for (int j = 0; j < P::N; j++) d[j] = quick(P::get(q, j));
        }
        return P::put(d);
    }
    // (a forbidden action has c = 0 and an lpa of LOW: no gradient, also where h is infinite)
    static __device__ __forceinline__ float action(const RowArgs& g, const RowNumbers& n) { return n.lpa <= LOW ? 0.f : (n.c - exp_of(n.lpa) * (n.c + n.h * (n.lpa + n.H))) * g.inv_t; }
};

// G lanes take a row and hold it in registers, NV times 16 bytes each, from its one reading to the writing of the gradient.  What is over after the whole
// 16-byte pieces (fewer than G values) goes to the first lanes, one value each.  MORE: the row may be longer than the registers; the pieces beyond are read in
// batches, and for the gradient once more.  Workgroups stay for row after row; the rows of a pass over the grid are turned by `turn`, so that sequences padded at
// the same places do not leave some workgroups all the padding.  With 1024 lanes only one workgroup fits a CU, and it asks for its next row's pieces as it
// writes the last's gradient: otherwise memory would wait for the sums and the sums for memory.
//
// Wavefronts a SIMD are asked for where they pay: 8 for the gradient of short rows (in 16 bits 2 to 6 registers spill for it: 1.5 M rows of 90 float16 actions 166 us
// against 190 without, 1 M of 128 116 and 128, but 335 544 of 400 124 and 119), 6 for the loss of up to 3 pieces a lane (one register fewer: 191 739 rows of 700
// bfloat16 actions 124 and 128 us).
template <typename T, int G, int NV, Mode MODE, bool MORE, bool STREAM>
__global__ void __launch_bounds__(G <= 64 ? 256 : G, G == 512 ? 4 : MODE == BACKWARD && G <= 16 ? 8 : MODE == LOSS && G <= 64 && NV <= 3 ? 6 : 1) k_rows(RowArgs g) {
    using P = Pack<T>;
    constexpr int N = P::N, RPB = G <= 64 ? 256 / G : 1, W = G <= 64 ? 1 : G / 64, BATCH = MODE == LOGP ? 4 : 2;
    constexpr bool AHEAD = G == 1024;
    __shared__ float red[3][W];
    __shared__ double sums[RPB][STATS];                   // the loss's statistics: a workgroup may have 2^19 rows
    const int lane = G <= 64 ? threadIdx.x % G : threadIdx.x, sub = G <= 64 ? threadIdx.x / G : 0;
    const int A = g.p.n_actions, whole = A / N, rest = A - whole * N, groups = (g.p.rows + RPB - 1) / RPB;
    const float k = g.k;
    const bool masked = g.p.mask != nullptr;
    u32x4 v[NV];
    if (MODE == LOSS && lane < STATS) sums[sub][lane] = 0;
    auto row_at = [&](int pass) { return (pass * (int)gridDim.x + (int)((blockIdx.x + (unsigned)pass * g.turn) % gridDim.x)) * RPB + sub; };
    auto logits = [&](int row) { return (const T*)g.p.logits + row_offset(row, g.p.ld); };
    int row = row_at(0), a = -1; float w = 0.f;
    auto look = [&](int row, int& a, float& w) {          // a row beyond the last is left out
        a = -1; w = 0.f;
        if (row < g.p.rows) { a = g.p.actions[row]; w = MODE == LOSS && g.loss.weights ? g.loss.weights[row] : 1.f; }
    };
    auto counts = [&](int a, float w) { return a >= 0 && a < A && w != 0.f; };
    // piece i of the lane: a base that all lanes share (scalar registers) and one offset for all i
    const uint32_t at = (uint32_t)lane * 16u;
    auto fetch = [&](const T* x, int i) { if (lane < whole - i * G) v[i] = load<STREAM>((const char*)x + i * G * 16 + at); };
    look(row, a, w);
    for (int pass = 0; pass * (int)gridDim.x < groups; pass++) {
        const T* x = logits(row);
        const int next = row_at(pass + 1);
        int next_a; float next_w;
        const bool last = (pass + 1) * (int)gridDim.x >= groups;
        if (last) { next_a = -1; next_w = 0.f; } else look(next, next_a, next_w);
        const uint8_t* mask = g.p.mask + row_offset(row, g.p.ld_mask);
        T* dx = (T*)g.dlogits + row_offset(row, g.ldd);
        bool on = counts(a, w);
        const bool here = row < g.p.rows;
        auto one = [&](int i) -> float { return masked && !mask[i] ? P::get(u32x4{P::FILL, P::FILL, P::FILL, P::FILL}, 0) : (float)x[i]; };
        auto piece = [&](int c) -> u32x4 { u32x4 q = load<STREAM>(x + c * N); if (masked) q = P::forbid(q, P::bytes(mask + c * N)); return q; };
        Base base(false, 0.f, 0.f);
        RowNumbers n{};
        float xt = P::get(u32x4{P::FILL, P::FILL, P::FILL, P::FILL}, 0);
        bool careful = false;
        // (a short row is asked for before its action is known: two trips to memory would take longer than reading what is left out)
        if ((!AHEAD || pass == 0) && (G <= 16 ? here : on)) {
#pragma unroll
            for (int i = 0; i < NV; i++) { v[i] = u32x4{P::FILL, P::FILL, P::FILL, P::FILL}; fetch(x, i); }
        }
        if (on) {
            const RowInputs in = row_inputs<MODE>(g, row, w);
            if (lane < rest) xt = one(whole * N + lane);
            const float xa = one(a);
            if (masked) {
                typename P::Bytes b[NV];
#pragma unroll
                for (int i = 0; i < NV; i++) { b[i] = ~(typename P::Bytes)0; if (lane < whole - i * G) b[i] = P::bytes(mask + i * G * N + at / (16 / N)); }
#pragma unroll
                for (int i = 0; i < NV; i++) { v[i] = P::forbid(v[i], b[i]); piece_done(); }
            }
            RowSum r;
            auto sum = [&](auto care) {
                constexpr Care C = decltype(care)::value;
#pragma unroll
                for (int i = 0; i < NV; i++) r.template piece<C, P>(v[i], k);
                if (MORE)
                    for (int p = lane + NV * G; p < whole; p += BATCH * G) {
                        u32x4 q[BATCH];
#pragma unroll
                        for (int i = 0; i < BATCH; i++) { q[i] = u32x4{P::FILL, P::FILL, P::FILL, P::FILL}; if (p + i * G < whole) q[i] = piece(p + i * G); }
#pragma unroll
                        for (int i = 0; i < BATCH; i++) r.template piece<C, P>(q[i], k);
                    }
                r.template reach<C>(xt, k);
                r.template add<C, P>(xt, k, 1);
            };
            r.clear();
            sum(care<QUICK>{});
            careful = !(fabsf(r.W()) < INFINITY);
            if (careful) { r.clear(); sum(care<CAREFUL>{}); }
            // the lanes' sums against the row's x0
            auto largest = [&]() {
                if (G <= 64) return lanes<G, Max>(r.x0);
                put_wave<G, Max>(r.x0, red[0]);
                __syncthreads();
                return get_waves<G, Max>(red[0]);
            };
            float x0 = largest(), by;
            const float m = times_k(x0, k);
            const bool exact = needs_exact(g, m);
            if (exact) {
                careful = true;
                // (two of a far row's largest may be one exponent once rounded: the x0 of the quick sums need not be the larger)
                r.clear();
                sum(care<EXACT>{});
                if (G > 64) __syncthreads();
                x0 = largest();
                by = step_to<EXACT>(r.x0, r.m, x0, m, k);
            } else by = step_to<QUICK>(r.x0, r.m, x0, m, k);
            base = Base(exact, x0, m);
            const float f = __builtin_amdgcn_exp2f(by);
            // (scaled first: a lane that has nothing but a caller's -1e9 can hold an S of up to 2^127, whose product with `by` is not finite)
            float S = f * r.S(), Wt = fmaf(S, by, f * r.W());
            if (G <= 64) { S = lanes<G, Sum>(S); Wt = lanes<G, Sum>(Wt); }
            else {
                put_wave<G, Sum>(S, red[1]); put_wave<G, Sum>(Wt, red[2]);
                __syncthreads();
                S = get_waves<G, Sum>(red[1]); Wt = get_waves<G, Sum>(red[2]);
            }
            float st[STATS];
            n = row_numbers<MODE, P>(g, in, x0, base, S, Wt, xa, st);
            on = n.on;
            // (a lane for each statistic; added in LDS, so that no sum is in a register: nobody else adds to it)
            if (MODE == LOSS && on && lane < STATS) {
                const float a0 = lane & 1 ? st[1] : st[0], a1 = lane & 1 ? st[3] : st[2], a2 = lane & 1 ? st[5] : st[4], a3 = lane & 1 ? st[7] : st[6];
                const float b0 = lane & 2 ? a1 : a0, b1 = lane & 2 ? a3 : a2;
                __hip_atomic_fetch_add(&sums[sub][lane], (double)(lane & 4 ? b1 : b0), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
        }
        const bool ahead = AHEAD && counts(next_a, next_w);
        const T* next_x = logits(ahead ? next : 0);
        if (here && lane == 0) {
            if (g.logp) g.logp[row] = n.logp;
            if (g.entropy) g.entropy[row] = n.H;
        }
        if (MODE == LOGP || !g.dlogits || !here || !on) {
            if (ahead) {
#pragma unroll
                for (int i = 0; i < NV; i++) { v[i] = u32x4{P::FILL, P::FILL, P::FILL, P::FILL}; fetch(next_x, i); }
            }
            if (MODE != LOGP && g.dlogits && here) {
                for (int p = lane; p < whole; p += G) store<STREAM>(dx + p * N, u32x4{0, 0, 0, 0});
                if (lane < rest) dx[whole * N + lane] = (T)0.f;
            }
        } else {
            const RowGradient d(g, n, base, careful);
#pragma unroll
            for (int i = 0; i < NV; i++) {
                if (lane < whole - i * G) store<STREAM>((char*)dx + i * G * 16 + at, d.template piece<P>(v[i]));
                if (ahead) fetch(next_x, i);
                piece_done();
            }
            if (MORE)
                for (int p = lane + NV * G; p < whole; p += BATCH * G) {
                    u32x4 q[BATCH];
#pragma unroll
                    for (int i = 0; i < BATCH; i++) if (p + i * G < whole) q[i] = piece(p + i * G);
#pragma unroll
                    for (int i = 0; i < BATCH; i++) { if (p + i * G < whole) store<STREAM>(dx + (p + i * G) * N, d.template piece<P>(q[i])); piece_done(); }
                }
            if (lane < rest) dx[whole * N + lane] = (T)d.template of<P>(xt);
            const int pa = a / N;
            if (lane == (pa < whole ? pa % G : a - whole * N)) dx[a] = (T)RowGradient::action(g, n);
        }
        row = next; a = next_a; w = next_w;
    }
    if (MODE != LOSS) return;
    __syncthreads();
    if (threadIdx.x < STATS) {
        double s = sums[0][threadIdx.x];
        for (int j = 1; j < RPB; j++) s += sums[j][threadIdx.x];
        g.row_stats[(int64_t)blockIdx.x * STATS + threadIdx.x] = (float)s;
    }
}

// ---- few rows of many actions: a row over `splits` workgroups, `per` pieces each ---------------------------------------------------------------------------
// k_parts leaves x0, S (negative where the sums are EXACT) and W of its part in part[row][split] and the action's logit behind the row's parts (the gradient may overwrite it before another part of
// the row is done); k_join adds a row's parts up in every workgroup that needs them and writes the outputs and its part of the gradient.  (Those workgroups join in
// the same order; the one of the loss's statistics has fewer lanes for a row and another order, and its last bits may not be those of logp and the gradient.)
struct SplitArgs { int splits, per; float* part; };      // part: [rows][3 * splits + 1]
template <typename T, Mode MODE> __device__ __forceinline__ bool row_counts(const RowArgs& g, int row, int& a, float& w) {
    a = g.p.actions[row]; w = MODE == LOSS && g.loss.weights ? g.loss.weights[row] : 1.f;
    return a >= 0 && a < g.p.n_actions && w != 0.f;
}
template <typename T> struct SplitRow {
    using P = Pack<T>;
    const T* x; const uint8_t* mask; bool masked; int whole, rest, from, to;
    __device__ __forceinline__ SplitRow(const RowArgs& g, const SplitArgs& sp, int row, int split)
        : x((const T*)g.p.logits + row_offset(row, g.p.ld)), mask(g.p.mask + row_offset(row, g.p.ld_mask)), masked(g.p.mask != nullptr), whole(g.p.n_actions / P::N),
          rest(split == sp.splits - 1 ? g.p.n_actions - whole * P::N : 0), from(split * sp.per), to(min(whole, from + sp.per)) {}
    __device__ __forceinline__ u32x4 piece(int c) const { u32x4 q = *(const u32x4_any*)(x + c * P::N); if (masked) q = P::forbid(q, P::bytes(mask + c * P::N)); return q; }
    __device__ __forceinline__ float one(int i) const { return masked && !mask[i] ? P::get(u32x4{P::FILL, P::FILL, P::FILL, P::FILL}, 0) : (float)x[i]; }
};
template <typename T, Mode MODE> __global__ void __launch_bounds__(256) k_parts(RowArgs g, SplitArgs sp) {
    using P = Pack<T>;
    __shared__ float red[3][4];
    const int split = blockIdx.x, row = blockIdx.y, lane = threadIdx.x;
    int a; float w;
    if (!row_counts<T, MODE>(g, row, a, w)) return;       // (k_join does not look at it then)
    const SplitRow<T> r(g, sp, row, split);
    float* const part = sp.part + (int64_t)row * (3 * sp.splits + 1);
    if (split == 0 && lane == 0) part[3 * sp.splits] = r.one(a);
    const float xt = lane < r.rest ? r.one(r.whole * P::N + lane) : P::get(u32x4{P::FILL, P::FILL, P::FILL, P::FILL}, 0);
    RowSum s;
    auto sum = [&](auto care) {
        constexpr Care C = decltype(care)::value;
        for (int p = r.from + lane; p < r.to; p += 4 * 256) {
            u32x4 q[4];
#pragma unroll
            for (int i = 0; i < 4; i++) { q[i] = u32x4{P::FILL, P::FILL, P::FILL, P::FILL}; if (p + i * 256 < r.to) q[i] = r.piece(p + i * 256); }
#pragma unroll
            for (int i = 0; i < 4; i++) s.template piece<C, P>(q[i], g.k);
        }
        s.template reach<C>(xt, g.k);
        s.template add<C, P>(xt, g.k, 1);
    };
    s.clear();
    sum(care<QUICK>{});
    if (!(fabsf(s.W()) < INFINITY)) { s.clear(); sum(care<CAREFUL>{}); }
    auto largest = [&]() { put_wave<256, Max>(s.x0, red[0]); __syncthreads(); return get_waves<256, Max>(red[0]); };
    float x0 = largest(), by;
    const float m = times_k(x0, g.k);
    const bool exact = needs_exact(g, m);
    if (exact) {                                          // (as in k_rows)
        s.clear();
        sum(care<EXACT>{});
        __syncthreads();
        x0 = largest();
        by = step_to<EXACT>(s.x0, s.m, x0, m, g.k);
    } else by = step_to<QUICK>(s.x0, s.m, x0, m, g.k);
    const float f = __builtin_amdgcn_exp2f(by);
    put_wave<256, Sum>(f * s.S(), red[1]); put_wave<256, Sum>(fmaf(f * s.S(), by, f * s.W()), red[2]);
    __syncthreads();
    const float S = get_waves<256, Sum>(red[1]), W = get_waves<256, Sum>(red[2]);
    if (lane == 0) { part[split] = x0; part[sp.splits + split] = exact ? -S : S; part[2 * sp.splits + split] = W; }
}
// the parts of a row joined by `n` lanes, of which this is `at`
__device__ __forceinline__ Base join(const RowArgs& g, const SplitArgs& sp, const float* part, int at, int n, float& x0, float& S, float& W) {
    x0 = LOWEST; S = W = 0.f;
    for (int i = at; i < sp.splits; i += n) x0 = fmaxf(x0, part[i]);
    for (int o = n >> 1; o > 0; o >>= 1) x0 = fmaxf(x0, __shfl_xor(x0, o, 64));
    const float m = times_k(x0, g.k);
    const Base base(needs_exact(g, m), x0, m);
    for (int i = at; i < sp.splits; i += n) {
        const float at_x0 = part[i], Si = part[sp.splits + i];
        const Base of(signbit(Si), at_x0, times_k(at_x0, g.k));
        // the step between two bases, of either kind, without the rounding of any m
        const float by = fmaxf(fmaf(of.a - base.a, g.k, of.b - base.b), LOW), f = __builtin_amdgcn_exp2f(by), size = fabsf(Si);
        S += f * size; W += f * fmaf(size, by, part[2 * sp.splits + i]);
    }
    for (int o = n >> 1; o > 0; o >>= 1) { S += __shfl_xor(S, o, 64); W += __shfl_xor(W, o, 64); }
    return base;
}
// The loss's statistics, by one workgroup beside those that write the gradient: 2 to 64 lanes a row, so that all rows are joined at once, then a sum over them in
// 64 bits.  (A launch behind this one takes 3 us more, and 4 us more of the call.)
template <typename T> __device__ __forceinline__ void split_stats(const RowArgs& g, const SplitArgs& sp) {
    __shared__ float st[SPLIT_ROWS][STATS];
    int n = 64;
    while (n * g.p.rows > 256) n >>= 1;
    const int row = threadIdx.x / n, at = threadIdx.x % n;
    if (row < g.p.rows) {
        float mine[STATS] = {}; bool on = false;
        int a; float w;
        if (row_counts<T, LOSS>(g, row, a, w)) {
            const float* const part = sp.part + (int64_t)row * (3 * sp.splits + 1);
            float x0, S, W;
            const Base base = join(g, sp, part, at, n, x0, S, W);
            on = row_numbers<LOSS, Pack<T>>(g, row_inputs<LOSS>(g, row, w), x0, base, S, W, part[3 * sp.splits], mine).on;
        }
        if (at == 0) for (int j = 0; j < STATS; j++) st[row][j] = on ? mine[j] : 0.f;
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    double sum = 0;
    for (int i = threadIdx.x / STATS; i < g.p.rows; i += 64 / STATS) sum += st[i][threadIdx.x % STATS];
    for (int o = 32; o >= STATS; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (threadIdx.x < STATS) g.loss.stats[threadIdx.x] = (float)sum;
}
template <typename T, Mode MODE> __global__ void __launch_bounds__(256) k_join(RowArgs g, SplitArgs sp) {
    using P = Pack<T>;
    const int split = blockIdx.x, row = blockIdx.y, lane = threadIdx.x;
    if (MODE == LOSS && split == (int)gridDim.x - 1) {    // (the loss has one workgroup more a row)
        if (row == 0) split_stats<T>(g, sp);
        return;
    }
    const SplitRow<T> r(g, sp, row, split);
    int a; float w;
    Base base(false, 0.f, 0.f);
    RowNumbers n{};
    // (the first pieces are asked for before the parts are joined)
    constexpr int BATCH = 4;
    const bool grad = MODE != LOGP && g.dlogits;
    u32x4 q[BATCH];
    auto fetch = [&](int p) {
#pragma unroll
        for (int i = 0; i < BATCH; i++) if (p + i * 256 < r.to) q[i] = r.piece(p + i * 256);
    };
    if (grad) fetch(r.from + lane);
    if (row_counts<T, MODE>(g, row, a, w)) {
        const float* const part = sp.part + (int64_t)row * (3 * sp.splits + 1);
        float x0, S, W, st[STATS];
        base = join(g, sp, part, lane & 63, 64, x0, S, W);
        n = row_numbers<MODE, P>(g, row_inputs<MODE>(g, row, w), x0, base, S, W, part[3 * sp.splits], st);
    }
    if (split == 0 && lane == 0) {
        if (g.logp) g.logp[row] = n.logp;
        if (g.entropy) g.entropy[row] = n.H;
    }
    if (!grad) return;
    T* const dx = (T*)g.dlogits + row_offset(row, g.ldd);
    const RowGradient d(g, n, base, true);
    for (int p = r.from + lane; p < r.to; p += BATCH * 256) {
        if (p != r.from + lane) fetch(p);
#pragma unroll
        for (int i = 0; i < BATCH; i++) if (p + i * 256 < r.to) store<false>(dx + (p + i * 256) * P::N, n.on ? d.template piece<P>(q[i]) : u32x4{0, 0, 0, 0});
    }
    if (lane < r.rest) dx[r.whole * P::N + lane] = (T)(n.on ? d.template of<P>(r.one(r.whole * P::N + lane)) : 0.f);
    if (!n.on) return;
    const int pa = a / P::N;
    if (pa < r.whole ? pa >= r.from && pa < r.to && lane == (pa - r.from) % 256 : lane == a - r.whole * P::N && lane < r.rest) dx[a] = (T)RowGradient::action(g, n);
}

// The workgroups' statistics in a fixed order, in 64 bits: thread t adds the float4 t, t + 1024, ... (its four statistics of every 512th workgroup), the lanes of
// like statistics are joined by xor, and the wavefronts in order.
__global__ void __launch_bounds__(1024) k_row_stats(const float4* part, int n, float* stats) {
    __shared__ double red[16][STATS];
    const int tid = threadIdx.x;
    double s[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 2 * ROW_BLOCKS / 1024; i++) {
        const int at = tid + i * 1024;
        const float4 v = at < 2 * n ? part[at] : float4{0.f, 0.f, 0.f, 0.f};
        s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
    }
#pragma unroll
    for (int o = 32; o > 1; o >>= 1) for (int j = 0; j < 4; j++) s[j] += __shfl_xor(s[j], o, 64);
    if ((tid & 63) < 2) for (int j = 0; j < 4; j++) red[tid >> 6][(tid & 1) * 4 + j] = s[j];
    __syncthreads();
    if (tid < STATS) {
        double sum = red[0][tid];
#pragma unroll
        for (int j = 1; j < 16; j++) sum += red[j][tid];
        stats[tid] = (float)sum;
    }
}

// ---- gradient norm and clip ----------------------------------------------------------------------------------------------------------------------------
// A launch takes up to TENSORS tensors by value, cut into pieces; workgroup b takes the pieces b, b + gridDim.x, ...  A piece is PIECE elements where they fill the
// device, SMALL_PIECE (two 16-byte loads a lane in float32) where they would not: the time is then one trip to memory.  A small network goes in a small batch:
// 16 tensors take 28 us from the call to the end of the work with 0.6 KB of kernel arguments and 43 us with 3.8 KB (16.1 and 16.8 us a call in a row of calls).
constexpr int TENSORS = 160, FEW_TENSORS = 24, PIECE = 16384, SMALL_PIECE = 2048, CLIP_BLOCKS = 1024;
template <int TENSORS> struct ClipBatch {
    int n, piece;                         // tensors, elements of a piece
    int first[TENSORS + 1];               // the first piece of each tensor; [n] = how many there are
    uint8_t dtype[TENSORS];
    void* g[TENSORS]; int64_t count[TENSORS];
};
static_assert(sizeof(ClipBatch<TENSORS>) < 3900, "kernel arguments by value");

// `from_end`: the pieces in the opposite order.  The second reading of the gradients begins with what the first read last and the caches still hold.
template <typename B, typename F> __device__ __forceinline__ void for_pieces(const B& b, bool from_end, F&& f) {
    const int n = b.first[b.n];
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int piece = from_end ? n - 1 - i : i;
        int lo = 0, hi = b.n;                                          // the last tensor whose first piece is <= piece (empty tensors share their successor's)
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (b.first[mid] <= piece) lo = mid; else hi = mid; }
        const int64_t at = (int64_t)(piece - b.first[lo]) * b.piece;
        f(piece, lo, at, (int)min((int64_t)b.piece, b.count[lo] - at));
    }
}
constexpr int IN_FLIGHT = 2;              // 16-byte loads of a lane
template <bool STREAM, typename T> __device__ __forceinline__ double square_sum(const T* g, int n) {
    using P = Pack<T>;
    const int whole = n / P::N;
    double s[2] = {0, 0};
    for (int i = threadIdx.x; i < whole; i += IN_FLIGHT * 256) {
        u32x4 v[IN_FLIGHT];
#pragma unroll
        for (int j = 0; j < IN_FLIGHT; j++) { v[j] = u32x4{0, 0, 0, 0}; if (i + j * 256 < whole) v[j] = load<STREAM>(g + (i + j * 256) * P::N); }
#pragma unroll
        for (int j = 0; j < IN_FLIGHT; j++)
#pragma unroll
            for (int e = 0; e < P::N; e++) { const double x = P::get(v[j], e); s[e & 1] = fma(x, x, s[e & 1]); }
    }
    const int i = whole * P::N + threadIdx.x;
    if (i < n) { const double x = (float)g[i]; s[0] = fma(x, x, s[0]); }
    return s[0] + s[1];
}
__device__ __forceinline__ double block_sum(double s, double* red) {
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}
template <bool STREAM, typename B> __device__ __forceinline__ double squares_of(const B& b, int t, int64_t at, int n) {
    if (b.dtype[t] == RLGPU_F32) return square_sum<STREAM>((const float*)b.g[t] + at, n);
    if (b.dtype[t] == RLGPU_BF16) return square_sum<STREAM>((const __bf16*)b.g[t] + at, n);
    return square_sum<STREAM>((const _Float16*)b.g[t] + at, n);
}
// `stream`: so many of the first pieces are read past the caches, which is left to the last ones: the clip begins with those
template <typename B> __global__ void __launch_bounds__(256) k_grad_squares(B b, double* part, int stream) {
    __shared__ double red[4];
    double s = 0;
    for_pieces(b, false, [&](int piece, int t, int64_t at, int n) { s += piece < stream ? squares_of<true>(b, t, at, n) : squares_of<false>(b, t, at, n); });
    s = block_sum(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}
template <typename T> __device__ __forceinline__ void scale_piece(T* g, int n, float f0, float f) {
    using P = Pack<T>;
    const int whole = n / P::N;
    for (int i = threadIdx.x; i < whole; i += IN_FLIGHT * 256) {
        u32x4 v[IN_FLIGHT];
#pragma unroll
        for (int j = 0; j < IN_FLIGHT; j++) if (i + j * 256 < whole) v[j] = *(const u32x4_any*)(g + (i + j * 256) * P::N);
#pragma unroll
        for (int j = 0; j < IN_FLIGHT; j++) {
            float d[P::N];
#pragma unroll
            for (int e = 0; e < P::N; e++) d[e] = P::get(v[j], e) * f0 * f;
            if (i + j * 256 < whole) *(u32x4_any*)(g + (i + j * 256) * P::N) = P::put(d);
        }
    }
    const int i = whole * P::N + threadIdx.x;
    if (i < n) g[i] = (T)((float)g[i] * f0 * f);
}
// every workgroup adds the partial sums up itself, all in the same order: no launch in between
template <typename B> __global__ void __launch_bounds__(256) k_grad_scale(B b, const double* part, int n_part, float max_norm, float grad_scale, float* norm_out) {
    __shared__ double red[4];
    double s = 0;
    for (int i = threadIdx.x; i < n_part; i += 8 * 256) {
        double v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = i + j * 256 < n_part ? part[i + j * 256] : 0.0;
#pragma unroll
        for (int j = 0; j < 8; j++) s += v[j];
    }
    s = block_sum(s, red);
    const double norm = (double)grad_scale * sqrt(s);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const double scale = (double)grad_scale * fmin(1.0, (double)max_norm / (norm + 1e-6));
    // in two factors: gradients near float32's largest value are scaled by less than its smallest normal one.  f0 is a power of two, 1 elsewhere, and small enough
    // for f to be a normal number wherever a product can be one (scale >= 2^-252), with g f0 still normal there
    const float f0 = scale < 0x1p-180 ? 0x1p-126f : scale < 0x1p-100 ? 0x1p-64f : 1.f, f = (float)(scale / (double)f0);
    // not a norm to clip by (as the caller sees it, in 32 bits), or nothing to clip
    if (!((float)norm < INFINITY) || (grad_scale == 1.f && norm + 1e-6 <= (double)max_norm)) return;
    for_pieces(b, true, [&](int, int t, int64_t at, int n) {
        if (b.dtype[t] == RLGPU_F32) scale_piece((float*)b.g[t] + at, n, f0, f);
        else if (b.dtype[t] == RLGPU_BF16) scale_piece((__bf16*)b.g[t] + at, n, f0, f);
        else scale_piece((_Float16*)b.g[t] + at, n, f0, f);
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

float exponents(float temperature) { return (float)(1.4426950408889634 / (double)temperature); }     // k
int64_t policy_bytes(int dtype, int rows, int n_actions, bool loss);

int check_rows(const char* who, const RlgpuPolicyRows* p, const void* workspace, int64_t bytes, bool loss = false) {
    if (!p) return fail(RLGPU_ERR_ARG, "%s: no rows", who);
    const int64_t size = size_of(p->dtype);
    if (!size) return fail(RLGPU_ERR_ARG, "%s: dtype %d is none of RLGPU_F32, RLGPU_BF16, RLGPU_F16", who, p->dtype);
    if (p->rows < 0 || p->rows > (1 << 30) || p->n_actions < 1 || p->n_actions > (1 << 28)) return fail(RLGPU_ERR_ARG, "%s: %d rows of %d actions", who, p->rows, p->n_actions);
    if (!(p->temperature > 0.f) || !(p->temperature < INFINITY) || !(exponents(p->temperature) < INFINITY)) return fail(RLGPU_ERR_ARG, "%s: temperature %g", who, (double)p->temperature);
    if (!(p->min_prob > 0.f && p->min_prob < 1.f)) return fail(RLGPU_ERR_ARG, "%s: min_prob %g is not between 0 and 1", who, (double)p->min_prob);
    if (p->rows == 0) return RLGPU_OK;
    if (!p->logits || !p->actions) return fail(RLGPU_ERR_ARG, "%s: logits and actions are needed", who);
    if (p->rows > 1 && (p->ld < p->n_actions || p->ld > INT32_MAX)) return fail(RLGPU_ERR_ARG, "%s: logits' row stride %lld of %d actions", who, (long long)p->ld, p->n_actions);
    if (p->mask && p->rows > 1 && p->ld_mask != 0 && (p->ld_mask < p->n_actions || p->ld_mask > INT32_MAX)) return fail(RLGPU_ERR_ARG, "%s: mask's row stride %lld", who, (long long)p->ld_mask);
    if (misaligned(p->logits, size) || misaligned(p->actions, 4)) return fail(RLGPU_ERR_ARG, "%s: logits or actions are not aligned to their type", who);
    const int64_t need = policy_bytes(p->dtype, p->rows, p->n_actions, loss);
    if (need && (!workspace || misaligned(workspace, 16) || bytes < need)) return fail(RLGPU_ERR_ARG, "%s: a workspace of %lld bytes, aligned to 16, is needed", who, (long long)need);
    return RLGPU_OK;
}
// dlogits is the logits' own buffer, or shares no element with it: apart, or the other columns of the same rows
int check_gradient(const char* who, const RlgpuPolicyRows* p, const void* dlogits, int64_t ldd) {
    if (!dlogits) return fail(RLGPU_ERR_ARG, "%s: dlogits is needed", who);
    const int64_t size = size_of(p->dtype), A = p->n_actions, R = p->rows;
    if (R > 1 && (ldd < A || ldd > INT32_MAX)) return fail(RLGPU_ERR_ARG, "%s: dlogits' row stride %lld of %lld actions", who, (long long)ldd, (long long)A);
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
    g.inv_t = 1.f / p->temperature; g.k = exponents(p->temperature); g.log_floor = (float)std::log((double)p->min_prob);
    return g;
}
// Workgroups of a kernel that the device keeps at once (a second, partly filled round would leave most of it idle).  `waves`: of a SIMD as its 800 scalar registers
// have room for them, which the query does not count: 8 with up to 80 each, 7 with up to 96, 6 with the 112 that most of the kernels have that write a gradient
// (loss of 33 554 rows of 4 000 float32 actions on a grid for 7 wavefronts, where 6 fit: 249 us, on one for 6: 215).
template <typename K> int resident(K kernel, int threads, int waves) {
    int device = 0, cus = 256, per_cu = 1;
    (void)hipGetDevice(&device);
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device);
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, threads, 0) != hipSuccess) { (void)hipGetLastError(); per_cu = 1; }
    return std::max(1, std::min(ROW_BLOCKS, cus * std::min(per_cu, waves * 4 * 64 / threads)));
}
// Few rows of many actions: a workgroup a row would leave the device idle.  Parts of at least a piece a lane, as many as give every CU two.  Measured in parts
// and as a workgroup a row, us for the backward pass in bfloat16: 131 072 actions 6.6 and 17.1 for 1 row, 8.9 and 18.2 for 32, 20.0 and 21.9 for 128, 34.4 and
// 27.8 for 256; 20 000 actions (2 500 pieces) 6.2 and 5.7 for 1 row, 8.1 and 6.6 for 128.
constexpr int SPLIT_PIECES = 4096, SPLIT_BLOCKS = 512;
int splits_for(int dtype, int rows, int n_actions) {
    const int whole = n_actions / (dtype == RLGPU_F32 ? 4 : 8);
    if (rows == 0 || rows > SPLIT_ROWS || whole <= SPLIT_PIECES) return 1;
    return std::max(1, std::min((whole + 255) / 256, SPLIT_BLOCKS / rows));
}
constexpr int STATS_DONE = -1;            // (for `blocks`) there are no sums of workgroups to join
int64_t stats_bytes(int rows) { return (int64_t)std::min(rows, ROW_BLOCKS) * STATS * 4; }
template <typename T, Mode MODE> int launch_split(RowArgs& g, hipStream_t s, int splits, int& blocks) {
    SplitArgs sp;
    const int whole = g.p.n_actions / Pack<T>::N;
    sp.per = (whole + splits - 1) / splits; sp.splits = (whole + sp.per - 1) / sp.per;
    sp.part = g.row_stats;
    blocks = STATS_DONE;
    hipLaunchKernelGGL((k_parts<T, MODE>), dim3(sp.splits, g.p.rows), dim3(256), 0, s, g, sp);
    OCHK(hipGetLastError());
    const bool sums = MODE == LOGP || !g.dlogits;
    hipLaunchKernelGGL((k_join<T, MODE>), dim3((sums ? 1 : sp.splits) + (MODE == LOSS ? 1 : 0), g.p.rows), dim3(sums && MODE != LOSS ? 64 : 256), 0, s, g, sp);
    OCHK(hipGetLastError());
    return RLGPU_OK;
}
template <typename T, int G, int NV, Mode MODE, bool MORE, bool STREAM = false> int launch_rows_as(RowArgs& g, hipStream_t s, int& blocks) {
    constexpr int threads = G <= 64 ? 256 : G, rpb = threads / G;
    // (512 lanes of a loss: two workgroups a CU and not three, 201 and 212 us for 12 201 rows of 11 000 float32 actions)
    constexpr int waves = MODE == LOGP || (MODE == BACKWARD && G <= 16) ? 8 : MODE == BACKWARD && G <= 64 && NV < 6 ? 7 : MODE == LOSS && G == 512 ? 4 : 6;
    static const int most = resident(&k_rows<T, G, NV, MODE, MORE, STREAM>, threads, waves);
    const int groups = (g.p.rows + rpb - 1) / rpb, passes = (groups + most - 1) / most;
    blocks = (groups + passes - 1) / passes;              // as many rows for each (2 048 groups: 1 024 workgroups twice, 12.1 us, not 1 536 and then 512, 12.5)
    g.turn = blocks * 5u / 13u;
    const bool alone = MODE == LOSS && blocks == 1;       // its sums are the statistics
    if (alone) g.row_stats = g.loss.stats;
    hipLaunchKernelGGL((k_rows<T, G, NV, MODE, MORE, STREAM>), dim3(blocks), dim3(threads), 0, s, g);
    OCHK(hipGetLastError());
    if (alone) blocks = STATS_DONE;
    return RLGPU_OK;
}
// Lanes and 16-byte pieces a row: the smallest set of registers that holds it.  Sums alone need no more of a row than what is in flight: 256 lanes take any.
template <typename T, Mode MODE> int launch_rows_of(RowArgs g, hipStream_t s, int& blocks) {
    const int whole = g.p.n_actions / Pack<T>::N;
    g.near = std::max(Pack<T>::LIMIT * g.k + CLEAR, -ROW_FAR);
    const int splits = splits_for(g.p.dtype, g.p.rows, g.p.n_actions);
    if (splits > 1) return launch_split<T, MODE>(g, s, splits, blocks);
    if (whole <= 8) return launch_rows_as<T, 8, 1, MODE, false>(g, s, blocks);
    if (whole <= 8 * 2) return launch_rows_as<T, 8, 2, MODE, false>(g, s, blocks);
    if (whole <= 8 * 3) return launch_rows_as<T, 8, 3, MODE, false>(g, s, blocks);
    if (whole <= 8 * 4) return launch_rows_as<T, 8, 4, MODE, false>(g, s, blocks);
    if (whole <= 16 * 4) return launch_rows_as<T, 16, 4, MODE, false>(g, s, blocks);
    if (whole <= 32 * 3) return launch_rows_as<T, 32, 3, MODE, false>(g, s, blocks);
    if (whole <= 32 * 4) return launch_rows_as<T, 32, 4, MODE, false>(g, s, blocks);
    if (whole <= 64 * 3) return launch_rows_as<T, 64, 3, MODE, false>(g, s, blocks);
    if (whole <= 64 * 4) return launch_rows_as<T, 64, 4, MODE, false>(g, s, blocks);
    if (whole <= 64 * 6) return launch_rows_as<T, 64, 6, MODE, false>(g, s, blocks);
    if (whole <= 64 * 8) return launch_rows_as<T, 64, 8, MODE, false>(g, s, blocks);
    if (whole <= 64 * 12) return launch_rows_as<T, 64, 12, MODE, false>(g, s, blocks);
    if (whole <= 256 * 4) return launch_rows_as<T, 256, 4, MODE, false>(g, s, blocks);
    const bool stream = (int64_t)g.p.rows * g.p.n_actions * (int64_t)sizeof(T) * (MODE != LOGP && g.dlogits ? 2 : 1) > STREAM_BYTES;
    if constexpr (MODE == LOGP) return stream ? launch_rows_as<T, 256, 2, LOGP, true, true>(g, s, blocks) : launch_rows_as<T, 256, 2, LOGP, true>(g, s, blocks);
    else {
        if (whole <= 256 * 6) return launch_rows_as<T, 256, 6, MODE, false>(g, s, blocks);
        if (whole <= 256 * 8) return launch_rows_as<T, 256, 8, MODE, false>(g, s, blocks);
        if (whole <= 512 * 5) return launch_rows_as<T, 512, 5, MODE, false>(g, s, blocks);
        if (whole <= 512 * 6) return launch_rows_as<T, 512, 6, MODE, false>(g, s, blocks);
        if (whole <= 512 * 8) return launch_rows_as<T, 512, 8, MODE, false>(g, s, blocks);
        if (whole <= 512 * 12) return stream ? launch_rows_as<T, 512, 12, MODE, false, true>(g, s, blocks) : launch_rows_as<T, 512, 12, MODE, false>(g, s, blocks);
        if (whole <= 512 * 26) return stream ? launch_rows_as<T, 512, 16, MODE, true, true>(g, s, blocks) : launch_rows_as<T, 512, 16, MODE, true>(g, s, blocks);
        return stream ? launch_rows_as<T, 1024, 16, MODE, true, true>(g, s, blocks) : launch_rows_as<T, 1024, 16, MODE, true>(g, s, blocks);
    }
}
template <Mode MODE> int launch_rows(const RowArgs& g, hipStream_t s, int& blocks) {
    blocks = 0;
    if (g.p.rows == 0) return RLGPU_OK;
    if (g.p.dtype == RLGPU_F32) return launch_rows_of<float, MODE>(g, s, blocks);
    if (g.p.dtype == RLGPU_BF16) return launch_rows_of<__bf16, MODE>(g, s, blocks);
    return launch_rows_of<_Float16, MODE>(g, s, blocks);
}

int64_t policy_bytes(int dtype, int rows, int n_actions, bool loss) {
    const int splits = splits_for(dtype, rows, n_actions);
    return splits > 1 ? (int64_t)rows * (3 * splits + 1) * 4 : (loss ? stats_bytes(rows) : 0);
}

constexpr int MOST_TENSORS = 1 << 24;     // (their partial sums are counted in 32 bits)
int clip_batches(int n) { return std::max(1, (n + TENSORS - 1) / TENSORS); }
int clip_share(int n_batches) { return std::max(256, 2 * CLIP_BLOCKS / n_batches); }   // workgroups of a launch, so that the partial sums stay few

template <int TENSORS> int launch_clip(const char* who, int n, void* const* grads, const int64_t* counts, const int32_t* dtypes, bool writes, float max_norm, float grad_scale,
                                       float* norm, double* part, hipStream_t s) {
    const int n_batches = std::max(1, (n + TENSORS - 1) / TENSORS), share = clip_share(n_batches);
    using Batch = ClipBatch<TENSORS>;
    int64_t elements = 0, to_stream = -CACHE_BYTES * 3 / 4;            // (bytes before those that shall be in the cache at the end)
    for (int i = 0; i < n; i++) { elements += counts[i]; to_stream += counts[i] * size_of(dtypes[i]); }
    const int piece = elements < (int64_t)CLIP_BLOCKS * SMALL_PIECE ? SMALL_PIECE : PIECE;
    auto batch = [&](int k, Batch& b) {                                // -> workgroups for it
        int64_t pieces = 0;
        b.piece = piece;
        b.n = std::min(TENSORS, n - k * TENSORS);
        for (int i = 0; i < b.n; i++) {
            const int j = k * TENSORS + i;
            b.g[i] = grads[j]; b.count[i] = counts[j]; b.dtype[i] = (uint8_t)dtypes[j]; b.first[i] = (int)pieces;
            pieces += (counts[j] + piece - 1) / piece;
        }
        b.first[b.n] = (int)pieces;
        return pieces > INT32_MAX ? -1 : (int)std::min<int64_t>(pieces, share);
    };
    Batch b;
    int n_part = 0;
    for (int k = 0; k < n_batches; k++) {
        const int blocks = batch(k, b);
        if (blocks < 0) return fail(RLGPU_ERR_ARG, "%s: too many elements", who);
        if (blocks == 0) continue;
        int64_t bytes = 0;
        for (int i = 0; i < b.n; i++) bytes += b.count[i] * size_of(b.dtype[i]);
        const int stream = to_stream <= 0 ? 0 : (int)std::min<double>(b.first[b.n], (double)to_stream / (double)bytes * b.first[b.n]);
        to_stream -= bytes;
        hipLaunchKernelGGL(k_grad_squares<Batch>, dim3(blocks), dim3(256), 0, s, b, part + n_part, stream);
        OCHK(hipGetLastError());
        n_part += blocks;
    }
    for (int k = n_batches - 1; k >= 0; k--) {
        int blocks = writes ? (k == n_batches - 1 && k == 0 ? std::min(b.first[b.n], share) : batch(k, b)) : 0;
        if (blocks == 0) { if (k) continue; b.n = 0; b.first[0] = 0; blocks = 1; }   // the last launch writes the norm, whatever there is to scale
        hipLaunchKernelGGL(k_grad_scale<Batch>, dim3(blocks), dim3(256), 0, s, b, (const double*)part, n_part, max_norm, grad_scale, k == 0 ? norm : (float*)nullptr);
        OCHK(hipGetLastError());
    }
    return RLGPU_OK;
}

}  // namespace

extern "C" {

const char* rlgpu_ops_last_error(void) { return g_error; }

int64_t rlgpu_policy_workspace(int32_t dtype, int32_t rows, int32_t n_actions, int32_t loss) {
    if (!size_of(dtype) || rows < 0 || rows > (1 << 30) || n_actions < 1 || n_actions > (1 << 28)) return fail(RLGPU_ERR_ARG, "rlgpu_policy_workspace: bad argument");
    return policy_bytes(dtype, rows, n_actions, loss != 0);
}

int rlgpu_action_logp(int device, const RlgpuPolicyRows* p, float* logp, float* entropy, void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_rows("rlgpu_action_logp", p, workspace, workspace_bytes)) return rc;
    if (p->rows == 0) return RLGPU_OK;
    if (!logp || misaligned(logp, 4) || misaligned(entropy, 4)) return fail(RLGPU_ERR_ARG, "rlgpu_action_logp: logp is needed, aligned to its type as entropy is");
    const OnDevice on(device); OCHK(on.err);
    RowArgs g = row_args(p);
    g.logp = logp; g.entropy = entropy; g.row_stats = (float*)workspace;
    int blocks;
    return launch_rows<LOGP>(g, (hipStream_t)stream, blocks);
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
    g.d_logp = d_logp; g.d_entropy = d_entropy; g.dlogits = dlogits; g.ldd = ld_dlogits; g.row_stats = (float*)workspace;
    int blocks;
    return launch_rows<BACKWARD>(g, (hipStream_t)stream, blocks);
}

int rlgpu_policy_loss(int device, const RlgpuPolicyRows* p, const RlgpuPolicyLoss* l, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "rlgpu_policy_loss";
    if (int rc = check_rows(who, p, workspace, workspace_bytes, true)) return rc;
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
    int blocks;
    if (int rc = launch_rows<LOSS>(g, (hipStream_t)stream, blocks)) return rc;
    if (blocks == STATS_DONE) return RLGPU_OK;
    hipLaunchKernelGGL(k_row_stats, dim3(1), dim3(1024), 0, (hipStream_t)stream, (const float4*)workspace, blocks, l->stats);
    OCHK(hipGetLastError());
    return RLGPU_OK;
}

int64_t rlgpu_clip_grad_workspace(int32_t n) {
    if (n < 0 || n > MOST_TENSORS) return fail(RLGPU_ERR_ARG, "rlgpu_clip_grad_workspace: %d tensors", n);
    return (int64_t)clip_batches(n) * clip_share(clip_batches(n)) * 8;
}

int rlgpu_clip_grad_norm(int device, int32_t n, void* const* grads, const int64_t* counts, const int32_t* dtypes, float max_norm, float grad_scale,
                         float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "rlgpu_clip_grad_norm";
    if (n < 0 || n > MOST_TENSORS || (n && (!grads || !counts || !dtypes))) return fail(RLGPU_ERR_ARG, "%s: %d tensors", who, n);
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
    const auto launch = n <= FEW_TENSORS ? launch_clip<FEW_TENSORS> : launch_clip<TENSORS>;
    return launch(who, n, grads, counts, dtypes, writes, max_norm, grad_scale, norm, (double*)workspace, (hipStream_t)stream);
}

}  // extern "C"
