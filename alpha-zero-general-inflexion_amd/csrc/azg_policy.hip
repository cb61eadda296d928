// azg_policy.hip -- operators over rows of policy logits (azg_amd.policy):
//
//   log-probabilities of given actions with the policy's entropy and its top alternatives, and their gradient:
//     m = max x, s = sum 2^((x - m) c), c = log2(e) / T;  lse = m / T + ln s
//     logp(a) = (x_a - m) / T - ln s,   H = ln s - sum p (x - m) / T
//     dx_v = (g_logp ([v = a] - p_v) + g_lse p_v - g_H p_v (logp_v + H)) / T
//   distillation from a teacher's top alternatives (id_j, t_j), its loss and gradient:
//     q = softmax(t) over the entries:          KL = sum q_j (ln q_j - ln p_j),  dx = w (p - q) / T
//     rest: q_j = exp t_j, q_R = 1 - sum q_j, p_R = the student's mass outside the entries:
//       KL += q_R (ln q_R - ln p_R),  dx = w (p S - q) / T on the entries, w p' (S p_R - q_R) / T elsewhere
//       (S = sum q_j + q_R, p' = p / p_R by the outside's own maximum and sum: p_R may be far below the
//       smallest f32 where the entries hold nearly everything)
//
// Sums are over the legal actions (a byte mask, or all).  Logits are f32, bf16 or f16; a row's statistics are f32,
// those of a KL (a difference of near values) and its few terms f64.
//
// All of it is bound by HBM from some thousand rows x columns on, by chains of dependent steps and the call below.
// On an MI355X (a 1 GiB copy reaches 5.2 TB/s, reading alone 6.4):
//   scores, 8192 x 32768 bf16, top 8             94 us   5.7 TB/s of reads
//   scores and gradient, 4092 x 50001 bf16       78 + 132 us (the second from the caches in part)
//   loss alone, 4096 x 65536 f16, 16 entries     86 us   6.2 TB/s of reads
//   loss with gradient, 8192 x 32768 bf16, 32   203 us   5.3 TB/s read and written once
//   loss, then gradient, 2048 x 100003 f32, 128 138 + 299 us, 5.5 TB/s over both
//   1 x 131072 bf16, top 20                      7.1 + 5.7 us (32 parts, joined)
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "../../include/azg.h"

int azg_host_fail(int code, const std::string& msg);  // azg_capi.cpp: the thread-local message

namespace {

constexpr int TOP_MAX = AZG_POLICY_TOP_MAX;
constexpr float LN2 = 0.69314718055994530942f;
constexpr float LOWEST = -3.402823466e38f;
constexpr float FAR = 1.2676506e30f;  // 2^100: beyond any log2 of a ratio that a sum can hold
constexpr int GROUP = 4;              // 16-byte loads that a thread has in flight together

using bf16_t = __bf16;
using f16_t = _Float16;

// one row's place, and the mask's
struct Rows {
    const void* x;
    const uint8_t* mask;
    long long rows, inner, so, si, mo, mi;
    int V;
    float c;     // log2(e) / T
    float invT;  // 1 / T
};

// (rows at one stride, the usual case, are spared the 64-bit division)
__device__ __forceinline__ long long row_at(const Rows& R, long long r, long long so, long long si) {
    if (R.inner >= R.rows) return r * si;
    const long long o = r / R.inner;
    return o * so + (r - o * R.inner) * si;
}
template <class T>
__device__ __forceinline__ const T* row_ptr(const Rows& R, long long r) {
    return (const T*)R.x + row_at(R, r, R.so, R.si);
}
__device__ __forceinline__ const uint8_t* mask_ptr(const Rows& R, long long r) {
    return R.mask ? R.mask + row_at(R, r, R.mo, R.mi) : nullptr;
}

// rows over the grid's x and y (a dimension holds fewer than 2^32 threads)
__device__ __forceinline__ long long block_row() { return blockIdx.x + (long long)gridDim.x * blockIdx.y; }
dim3 row_grid(long long rows) {
    const long long x = rows < (1 << 20) ? rows : 1 << 20;
    return dim3((unsigned)x, (unsigned)((rows + x - 1) / x));
}


// max that keeps a NaN (fmaxf drops it, and costs a canonicalisation of what was loaded)
__device__ __forceinline__ float nmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float lg2(float x) { return __builtin_amdgcn_logf(x); }

// ---- wave and team reductions -------------------------------------------------------------------
// Within rows of 16 lanes by DPP (the partner's value arrives with the instruction, no LDS round trip), the four
// rows by readlane.  Every lane gets the result; the order is fixed.
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned x) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) { return __uint_as_float(dpp<CTRL>(__float_as_uint(x))); }
template <int CTRL>
__device__ __forceinline__ unsigned long long dpp(unsigned long long x) {
    return ((unsigned long long)dpp<CTRL>((unsigned)(x >> 32)) << 32) | dpp<CTRL>((unsigned)x);
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
    return __longlong_as_double((long long)dpp<CTRL>((unsigned long long)__double_as_longlong(x)));
}
__device__ __forceinline__ unsigned lane_of(unsigned x, int l) { return (unsigned)__builtin_amdgcn_readlane((int)x, l); }
__device__ __forceinline__ float lane_of(float x, int l) { return __uint_as_float(lane_of(__float_as_uint(x), l)); }
__device__ __forceinline__ unsigned long long lane_of(unsigned long long x, int l) {
    return ((unsigned long long)lane_of((unsigned)(x >> 32), l) << 32) | lane_of((unsigned)x, l);
}
__device__ __forceinline__ double lane_of(double x, int l) {
    return __longlong_as_double((long long)lane_of((unsigned long long)__double_as_longlong(x), l));
}
constexpr int QUAD_XOR1 = 0xB1, QUAD_XOR2 = 0x4E, HALF_MIRROR = 0x141, MIRROR = 0x140;
template <class V, class F>
__device__ __forceinline__ V wave_reduce(V x, F f) {
    x = f(x, dpp<QUAD_XOR1>(x));
    x = f(x, dpp<QUAD_XOR2>(x));
    x = f(x, dpp<HALF_MIRROR>(x));
    x = f(x, dpp<MIRROR>(x));
    return f(f(lane_of(x, 0), lane_of(x, 16)), f(lane_of(x, 32), lane_of(x, 48)));
}
template <class V>
__device__ __forceinline__ V wave_sum(V x) { return wave_reduce(x, [](V a, V b) { return a + b; }); }
__device__ __forceinline__ float wave_max(float x) {
    return wave_reduce(x, [](float a, float b) { return nmax(a, b); });
}

// A team is the threads that share a row: a wave (64; four teams in a block) or a block.
template <int TEAM>
__device__ __forceinline__ void team_sync() {
    if constexpr (TEAM == 64) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // the wave's own LDS and global accesses, in order
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}
template <int TEAM>
constexpr int block_of = TEAM == 64 ? 256 : TEAM;
template <int TEAM>
__device__ __forceinline__ int team_tid() { return TEAM == 64 ? threadIdx.x & 63 : threadIdx.x; }
template <int TEAM>
__device__ __forceinline__ int team_in_block() {  // by readfirstlane: the same for a wave, so its row is scalar work
    return TEAM == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
}
template <int TEAM>
__device__ __forceinline__ long long team_row() {
    return TEAM == 64 ? block_row() * 4 + team_in_block<TEAM>() : block_row();
}

// ---- vectors of 16 bytes ------------------------------------------------------------------------------
// A row may start at any element and so may its vectors (the loads need no more than the element's alignment; vectors
// from the first 16-byte boundary on measured no faster: 76.8 us against 76.2, 4092 x 50001 bf16); the elements
// behind the last whole one are taken one a thread.
template <class T>
constexpr int VN = 16 / (int)sizeof(T);
template <class T>
constexpr unsigned MINF_BITS = sizeof(T) == 4 ? 0xFF800000u : std::is_same_v<T, f16_t> ? 0xFC00FC00u : 0xFF80FF80u;

// NT: without a place in the caches, for what is not read again (6.4 TB/s against 5.6, 4096 x 65536 f16)
template <bool NT, class T>
__device__ __forceinline__ uint4 load16(const T* p) {
    using W = unsigned __attribute__((ext_vector_type(4), aligned(sizeof(T)), may_alias));
    W w;
    if constexpr (NT)
        w = __builtin_nontemporal_load((const W*)p);
    else
        w = *(const W*)p;
    return make_uint4(w.x, w.y, w.z, w.w);
}
template <class T>
__device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            f[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same_v<T, bf16_t>) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            f[2 * i] = (float)__builtin_bit_cast(f16_t, (unsigned short)w[i]);
            f[2 * i + 1] = (float)__builtin_bit_cast(f16_t, (unsigned short)(w[i] >> 16));
        }
    }
}
template <bool NT, class T>
__device__ __forceinline__ void store16(T* p, const float* f) {
    using W = unsigned __attribute__((ext_vector_type(4), aligned(sizeof(T)), may_alias));
    T t[VN<T>];
#pragma unroll
    for (int i = 0; i < VN<T>; ++i) t[i] = (T)f[i];  // round to nearest even
    W w;
    __builtin_memcpy(&w, t, 16);
    if constexpr (NT)
        __builtin_nontemporal_store(w, (W*)p);
    else
        *(W*)p = w;
}
// illegal actions of a vector -> none
template <class T>
__device__ __forceinline__ void apply_mask(const uint8_t* mk, float* f, float none = -INFINITY) {
    uint8_t b[VN<T>];
    __builtin_memcpy(b, mk, VN<T>);
#pragma unroll
    for (int i = 0; i < VN<T>; ++i) f[i] = b[i] ? f[i] : none;
}

// 1 / x for x in the normal range: the instruction's estimate (2^-24 or better) and two Newton steps, which square its
// error; a quarter of the division's instructions, correct to a few 2^-53
__device__ __forceinline__ double rcp_f64(double x) {
    double y = __builtin_amdgcn_rcp(x);
    y = __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
    return __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
}
// ln s in f64, s >= 0: s = 2^e f, f in [0.75, 1.5), ln f = 2 atanh(v), v = (f - 1) / (f + 1), |v| <= 0.2, by its power
// series to v^15 (what is left is under 2e-13)
__device__ __forceinline__ double ln_f64(double s) {
    if (!(s > 0.0 && s < INFINITY)) return s == 0.0 ? -INFINITY : s == INFINITY ? INFINITY : NAN;
    int e = __builtin_amdgcn_frexp_exp(s);
    double f = __builtin_amdgcn_frexp_mant(s);
    if (f < 0.75) {
        f *= 2.0;
        --e;
    }
    const double v = (f - 1.0) * rcp_f64(f + 1.0), w = v * v;
    double t = 1.0 / 15;
    t = t * w + 1.0 / 13;
    t = t * w + 1.0 / 11;
    t = t * w + 1.0 / 9;
    t = t * w + 1.0 / 7;
    t = t * w + 1.0 / 5;
    t = t * w + 1.0 / 3;
    t = t * w + 1.0;
    return 0.69314718055994530942 * e + 2.0 * v * t;
}
// e^t in f64: t = n ln 2 + z, |z| <= 0.35, its power series to z^9 (what is left is under 1e-11 of it).  0 below
// -800 (f64 ends at -745): an entry at the type's lowest value would leave a z whose powers pass f64.  A NaN stays.
__device__ __forceinline__ double exp_f64(double t) {
    t = t < -800.0 ? -800.0 : t;
    const double n = fmin(rint(t * 1.4426950408889634074), 2000.0);
    const double z = __builtin_fma(n, -0.69314718055994530942, t);
    double p = 1.0 / 362880;
    p = p * z + 1.0 / 40320;
    p = p * z + 1.0 / 5040;
    p = p * z + 1.0 / 720;
    p = p * z + 1.0 / 120;
    p = p * z + 1.0 / 24;
    p = p * z + 1.0 / 6;
    p = p * z + 0.5;
    p = p * z + 1.0;
    p = p * z + 1.0;
    return __builtin_amdgcn_ldexp(p, (int)n);
}

// ---- softmax statistics -------------------------------------------------------------------------
// s = sum 2^u, w = sum u 2^u with u = x c - r and r a whole number near max x c: moving a sum to another r is exact
// (a power of two), and x c - r is one rounding.  r follows the maximum lazily (u <= 8.5), and starts at -2^100 with
// an empty sum.  From 2^24 on r is f32's number next to max x c and off by more than a half: by up to 8 below 2^28, by more
// than f32's exponents reach soon after.  A row whose sum is out of proportion for that (its largest logit a mask's fill,
// or one far above the others) or that holds no number is done again with u = (x - m) c (far_stat).
// ENT: f32 sums with the entropy's; else s alone, in f64 beyond a thread's 16 or 32 terms (a KL is a difference of
// near values: what s is off by comes to twenty times that of it).
template <bool ENT>
struct Sum {
    float r;
    std::conditional_t<ENT, float, double> s;
    float w;
};
__device__ __forceinline__ float scale2(float x, int k) { return __builtin_amdgcn_ldexpf(x, k); }
__device__ __forceinline__ double scale2(double x, int k) { return __builtin_amdgcn_ldexp(x, k); }
// to a reference r >= a.r.  By more than 300, which nothing of a finite sum outlasts, it is set to 0: d s would pass
// f32 for a sum of fills (-1e9 and the like) although 2^d leaves nothing of it, and so may s.  A NaN stays.
template <bool ENT>
__device__ __forceinline__ Sum<ENT> move_sum(Sum<ENT> a, float r) {
    const float d = a.r - r;
    const int k = (int)fmaxf(d, -4096.f);
    const bool gone = d < -300.f && a.s > 0;
    if constexpr (ENT) a.w = gone ? 0.f : scale2(__builtin_fmaf(d, a.s, a.w), k);
    a.s = gone ? 0 : scale2(a.s, k);
    a.r = r;
    return a;
}
template <bool ENT, int N>
__device__ __forceinline__ void sum_group(Sum<ENT>& a, const float* x, float gm, float c) {
    if (__builtin_fmaf(gm, c, -a.r) > 8.f) a = move_sum(a, rintf(gm * c));
    float s0 = 0.f, s1 = 0.f, w0 = 0.f, w1 = 0.f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float u0 = __builtin_fmaf(x[i], c, -a.r), u1 = __builtin_fmaf(x[i + 1], c, -a.r);
        const float e0 = ex2(u0), e1 = ex2(u1);
        s0 += e0;
        s1 += e1;
        if constexpr (ENT) {
            w0 = __builtin_fmaf(e0, nmax(u0, -1000.f), w0);
            w1 = __builtin_fmaf(e1, nmax(u1, -1000.f), w1);
        }
    }
    a.s += s0 + s1;
    if constexpr (ENT) a.w += w0 + w1;
}
template <int TEAM, bool ENT>
__device__ __forceinline__ Sum<ENT> team_sum(Sum<ENT> a, Sum<ENT>* sh) {
    a = move_sum(a, wave_max(a.r));
    a.s = wave_sum(a.s);
    if constexpr (ENT) a.w = wave_sum(a.w);
    if constexpr (TEAM > 64) {
        constexpr int W = TEAM / 64;
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
        __syncthreads();
        float r = sh[0].r;
#pragma unroll
        for (int i = 1; i < W; ++i) r = fmaxf(r, sh[i].r);
        a = Sum<ENT>{r, 0, 0.f};
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const Sum<ENT> b = move_sum(sh[i], r);
            a.s += b.s;
            a.w += b.w;
        }
    }
    return a;
}

// A row's statistics as the gradients use them: u = x c - ref, or (x - ref) c on a wide row; p = 2^(u - l2)
template <bool ENT>
struct Stat {
    float ref;
    std::conditional_t<ENT, float, double> s;
    float w;
    bool wide;
};
__device__ __forceinline__ float u_of(float x, float ref, bool wide, float c) {
    return wide ? (x - ref) * c : __builtin_fmaf(x, c, -ref);
}
// the reference in units of x c (48 bits of a product: exact)
__device__ __forceinline__ double place(float ref, bool wide, float c) { return wide ? (double)ref * (double)c : ref; }
// the log-probability of a logit, l2 = log2 of the row's sum: a difference of near values for a nearly sure policy,
// which rounding leaves above 0 now and then.  A NaN stays.
__device__ __forceinline__ float logp_of(float x, const Stat<true>& st, float l2, float c, float invT) {
    float p;
    if (st.wide)
        p = (x - st.ref) * invT - LN2 * l2;
    else if (fabsf(x) > 1e30f)
        p = x * invT - LN2 * (st.ref + l2);  // x c may pass f32 where x / T does not
    else
        p = LN2 * (__builtin_fmaf(x, c, -st.ref) - l2);
    return p > 0.f ? 0.f : p;
}
// is this sum one of up to V logits at a reference near their maximum?  Empty ones are not, nor what holds a NaN.  Off by
// 16 and more, log2 s would cost the f32 results their last bits; a KL's logarithms are f64, and its gradient's factors
// fit f32 up to 64 (a fill of -1e9 at temperature 1: 202 us as without, 326 done again, 8192 x 32768 bf16).
template <bool ENT>
__device__ __forceinline__ bool plain_sum(const Sum<ENT>& a, int V) {
    constexpr float most = ENT ? 0x1p16f : 0x1p64f;
    return a.s >= 1.f / most && a.s <= most * (float)V && fabsf(a.w) < INFINITY;
}

// a and p of disjoint parts of a row -> a of both, at the larger reference.  A part without probability counts for
// nothing, one that holds a NaN makes the sum one.
template <bool ENT>
__device__ __forceinline__ void stat_add(Stat<ENT>& a, Stat<ENT> p, float c) {
    if (p.s == 0) return;
    if (a.s == 0) {
        a = p;
        return;
    }
    const double d = place(p.ref, p.wide, c) - place(a.ref, a.wide, c);
    if (d > 0.0) {
        const Stat<ENT> t = a;
        a = p;
        p = t;
    }
    const float t = -fabsf((float)d);
    const float k = a.wide || p.wide ? ex2(t) : __builtin_amdgcn_ldexpf(1.f, (int)fmaxf(t, -4096.f));  // whole: exact
    a.s += p.s * k;
    if constexpr (ENT) a.w += k == 0.f ? 0.f : (p.w + t * p.s) * k;
}

// order of the alternatives: larger logit first (NaN before all), then the lower index.  0: not an alternative.
__device__ __forceinline__ unsigned long long order_key(float x, unsigned idx) {
    const unsigned b = __float_as_uint(x + 0.f);  // -0 -> +0
    const unsigned k = x != x ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((unsigned long long)k << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float key_value(unsigned long long key) {
    const unsigned k = (unsigned)(key >> 32);
    return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ unsigned key_index(unsigned long long key) { return 0xFFFFFFFFu - (unsigned)key; }

// ---- one pass over a row --------------------------------------------------------------------------
// GROUP vectors of a thread at once: loads first, then the group's maximum, then its exponentials.
// bound by HBM: 8 operations and one exponential for a 2-byte logit are half of what the chip can do while it
// loads it.
template <class T, int U>
struct Loaded {
    uint4 v[U];
};
// Hides from the compiler what these registers hold: it would unpack all groups at once, and keep the unpacked
// logits (twice the registers) from one use to the next.
template <class T, int U>
__device__ __forceinline__ void opaque(Loaded<T, U>& L) {
#pragma unroll
    for (int u = 0; u < U; ++u) asm volatile("" : "+v"(L.v[u].x), "+v"(L.v[u].y), "+v"(L.v[u].z), "+v"(L.v[u].w));
}

// what the top alternatives need of a pass: each thread's best vector and the maximum of each of its groups (LDS)
struct Best {
    float v;
    int last;  // the last index of the first vector that holds v
};

// `edit` may take elements out of a vector (set them to -inf): edit(vector, its elements), edit.one(index).
struct NoEdit {
    template <class F>
    __device__ __forceinline__ void operator()(int, F*) const {}
    __device__ __forceinline__ bool one(int) const { return false; }
};

template <class T, int TEAM, bool MASK, bool ENT, bool TOP, bool NT, class Edit>
__device__ __forceinline__ void row_pass(const T* x, const uint8_t* mk, int V, float c, Sum<ENT>& a, float& mx,
                                         Best& best, float* gmax, const Edit& edit) {
    constexpr int N = VN<T>;
    const int tid = team_tid<TEAM>(), nvec = V / N, step = TEAM * GROUP;
    // a vector's elements and maximum
    auto take = [&](const uint4& v, int vi, float* f) {
        unpack<T>(v, f);
        if constexpr (MASK)
            if (vi < nvec) apply_mask<T>(mk + vi * N, f);
        edit(vi, f);
        float m = f[0];
#pragma unroll
        for (int i = 1; i < N; ++i) m = nmax(m, f[i]);
        if constexpr (TOP) {
            const bool up = m > best.v;
            best.v = up ? m : best.v;
            best.last = up ? vi * N + N - 1 : best.last;
        }
        return m;
    };
    int g = 0, vi = tid;
    for (; vi - tid + step <= nvec; vi += step, ++g) {
        uint4 v[GROUP];
#pragma unroll
        for (int u = 0; u < GROUP; ++u) v[u] = load16<NT>(x + (long long)(vi + u * TEAM) * N);
        float f[GROUP * N], gm = -INFINITY;
#pragma unroll
        for (int u = 0; u < GROUP; ++u) gm = nmax(gm, take(v[u], vi + u * TEAM, f + u * N));
        mx = nmax(mx, gm);
        if constexpr (TOP) gmax[g * TEAM + tid] = gm;
        sum_group<ENT, GROUP * N>(a, f, gm, c);
    }
    const int left = nvec - (vi - tid);  // the last group: only as many vectors as it has
    if (left > 0) {
        uint4 v[GROUP];
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
            v[u] = make_uint4(MINF_BITS<T>, MINF_BITS<T>, MINF_BITS<T>, MINF_BITS<T>);
            if (vi + u * TEAM < nvec) v[u] = load16<NT>(x + (long long)(vi + u * TEAM) * N);
        }
        float gm = -INFINITY;
#pragma unroll
        for (int u = 0; u < GROUP; ++u)
            if (u * TEAM < left) {
                float f[N];
                const float m = take(v[u], vi + u * TEAM, f);
                gm = nmax(gm, m);
                sum_group<ENT, N>(a, f, m, c);
            }
        mx = nmax(mx, gm);
        if constexpr (TOP) gmax[g * TEAM + tid] = gm;
        ++g;
    }
    float f[2] = {-INFINITY, -INFINITY};  // what is behind the last vector, an element a thread
    const int i = nvec * N + tid;
    if (i < V && (!MASK || mk[i]) && !edit.one(i)) f[0] = (float)x[i];
    if constexpr (TOP) {
        gmax[g * TEAM + tid] = f[0];
        if (f[0] > best.v) best = Best{f[0], i};
    }
    mx = nmax(mx, f[0]);
    if (nvec * N < V) sum_group<ENT, 2>(a, f, f[0], c);
}
template <class T, int TEAM, bool MASK, bool ENT, bool TOP, class Edit>
__device__ __forceinline__ void row_pass(const T* x, const uint8_t* mk, int V, float c, Sum<ENT>& a, float& mx,
                                         Best& best, float* gmax, const Edit& edit, bool nt) {
    if (nt)  // the same for the whole team
        row_pass<T, TEAM, MASK, ENT, TOP, true>(x, mk, V, c, a, mx, best, gmax, edit);
    else
        row_pass<T, TEAM, MASK, ENT, TOP, false>(x, mk, V, c, a, mx, best, gmax, edit);
}

template <int TEAM>
__device__ __forceinline__ float team_max(float x, float* sh) {
    x = wave_max(x);
    if constexpr (TEAM > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
        __syncthreads();
        x = sh[0];
        for (int i = 1; i < TEAM / 64; ++i) x = nmax(x, sh[i]);
        __syncthreads();
    }
    return x;
}

template <bool ENT>
union Shared {  // one reduction at a time
    Sum<ENT> sum[16];
    Stat<ENT> stat[16];
    float f[16];
};

// what Sum does not hold, from the logits' maximum m: a pass more.  An infinite m or a NaN makes s a NaN.
template <class T, int TEAM, bool ENT, class Edit>
__device__ __forceinline__ Stat<ENT> far_stat(float m, const T* x, const uint8_t* mk, int V, float c, Shared<ENT>& sh,
                                              const Edit& edit) {
    constexpr int N = VN<T>;
    const int tid = team_tid<TEAM>(), nvec = V / N;
    Sum<ENT> a{0.f, 0, 0.f};
    auto add = [&](float y) {
        const float u = (y - m) * c, e = ex2(u);
        a.s += e;
        if constexpr (ENT) a.w = __builtin_fmaf(e, nmax(u, -1000.f), a.w);
    };
    for (int vi = tid; vi < nvec; vi += TEAM) {
        float f[N];
        unpack<T>(load16<false>(x + (long long)vi * N), f);
        if (mk) apply_mask<T>(mk + vi * N, f);
        edit(vi, f);
#pragma unroll
        for (int i = 0; i < N; ++i) add(f[i]);
    }
    const int i = nvec * N + tid;
    if (i < V && (!mk || mk[i]) && !edit.one(i)) add((float)x[i]);
    a = team_sum<TEAM, ENT>(a, sh.sum);
    return Stat<ENT>{m, a.s, a.w, true};
}

// the statistics of a row, or of a part of it, from its pass; without a legal action s = 0
template <class T, int TEAM, bool ENT, class Edit>
__device__ __forceinline__ Stat<ENT> row_stat(Sum<ENT> a, float mx, const T* x, const uint8_t* mk, int V, float c,
                                              Shared<ENT>& sh, const Edit& edit) {
    a = team_sum<TEAM, ENT>(a, sh.sum);
    if (plain_sum(a, V)) return Stat<ENT>{a.r, a.s, a.w, false};
    mx = team_max<TEAM>(mx, sh.f);
    if (mx == -INFINITY) return Stat<ENT>{0.f, 0, 0.f, false};
    return far_stat<T, TEAM, ENT>(mx, x, mk, V, c, sh, edit);
}

// the statistics of a row from those of its parts, of which each thread has joined some
template <int TEAM, bool ENT>
__device__ __forceinline__ Stat<ENT> team_join(Stat<ENT> v, float c, Shared<ENT>& sh) {
    const bool wide = TEAM == 64 ? __ballot(v.wide) != 0 : __syncthreads_or(v.wide);
    if (!wide) {
        const Sum<ENT> a = team_sum<TEAM, ENT>(Sum<ENT>{v.s == 0 ? -FAR : v.ref, v.s, v.w}, sh.sum);
        return Stat<ENT>{a.s == 0 ? 0.f : a.r, a.s, a.w, false};
    }
    for (int o = 32; o > 0; o >>= 1)
        stat_add(v, Stat<ENT>{__shfl_xor(v.ref, o), __shfl_xor(v.s, o), __shfl_xor(v.w, o), (bool)__shfl_xor((int)v.wide, o)}, c);
    if constexpr (TEAM > 64) {
        if ((threadIdx.x & 63) == 0) sh.stat[threadIdx.x >> 6] = v;
        __syncthreads();
        v = sh.stat[0];
        for (int i = 1; i < TEAM / 64; ++i) stat_add(v, sh.stat[i], c);
        return v;
    }
    // the first lane's for all: at one place two lanes may hold references of either kind
    return Stat<ENT>{lane_of(v.ref, 0), lane_of(v.s, 0), lane_of(v.w, 0), lane_of((unsigned)v.wide, 0) != 0};
}

// ---- the k largest of a row -----------------------------------------------------------------------
// A lower bound of the k-th largest: the k-th largest of the threads' (or of 64 groups of threads') own best is one,
// for each of those k has an element at least as large.  In the order (value, index) it stays sharp where values
// are equal: k threads of a constant row bound it by the index.  Only the groups whose maximum reaches the bound are
// read again (cached, some k of them), what of them reaches it are the candidates, and a candidate's rank is the
// number of those before it.  Where the list overflows (the largest crowd into few threads) or a logit is no
// number, the bound is found by radix selection over the whole order, eight digits of 256.
template <int TEAM>
struct TopShare {
    static constexpr int CANDS = TEAM == 64 ? 512 : 1024, HITS = TEAM == 64 ? 256 : 512;
    unsigned long long cand[CANDS];  // before: the threads' best; in the radix selection: the histogram
    int hits[HITS];
    int nh, nc;
    unsigned long long bound;
};

// The k-th largest of a wave's words, or less where that needs fewer steps (in any case k words are at least as
// large): a binary digit a step, counted by ballot.  *wanted: how many of the words equal to it are among the k,
// 0 if all are.
__device__ __forceinline__ unsigned kth_word(unsigned w, int k, int* wanted) {
    unsigned t = 0;
    int above = 0;
    *wanted = 0;
    for (int d = 31; d >= 0; --d) {
        const unsigned u = t | (1u << d);
        const int n = __popcll(__ballot(w >= u));
        if (n == k) return u;
        if (n > k)
            t = u;
        else
            above = n;
    }
    *wanted = k - above;
    return t;
}
__device__ __forceinline__ unsigned long long kth_pair(unsigned long long key, int k) {
    const unsigned w = (unsigned)(key >> 32);
    if (__popcll(__ballot(w != 0)) < k) return 0;
    int wanted;
    const unsigned t = kth_word(w, k, &wanted);
    if (wanted == 0) return (unsigned long long)t << 32;
    const unsigned low = kth_word(w == t ? (unsigned)key : 0u, wanted, &wanted);  // equal values: by index
    return ((unsigned long long)t << 32) | low;
}

template <int G>
__device__ __forceinline__ int rank_in(const unsigned long long* arr, unsigned long long me) {
    int rank = 0;
#pragma unroll 16
    for (int i = 0; i < G; ++i) rank += arr[i] > me;
    return rank;
}

// a bound of the k-th largest of a row from its threads' best.  A wave by ballots (75 us against 82 with ranks, 65536 x
// 343 f32, top 16: the fewest instructions).  A block by ranks in LDS, each wave for itself over 64 groups of
// threads where these are enough (the shorter chain: 91 us against 98, 8192 x 32768 bf16, top 8), else over 128 pairs
// (35 us against 39 over all, 2000 x 32768 bf16, top 50) or over all.
template <int TEAM>
__device__ __forceinline__ unsigned long long kth_best(unsigned long long best, int k, TopShare<TEAM>& S) {
    const int tid = team_tid<TEAM>(), lane = threadIdx.x & 63;
    if (tid == 0) S.nh = 0, S.nc = 0, S.bound = 0;
    if constexpr (TEAM == 64) {
        team_sync<64>();
        return k > 64 ? 0 : kth_pair(best, k);
    } else {
        static_assert(TEAM == 256, "groups of a quad");
        unsigned long long* arr = S.cand;
        if (k <= 32) {
            auto mx = [](unsigned long long a, unsigned long long b) { return a > b ? a : b; };
            best = mx(best, dpp<QUAD_XOR1>(best));
            best = mx(best, dpp<QUAD_XOR2>(best));
            if ((tid & 3) == 0) arr[tid / 4] = best;
            __syncthreads();
            const unsigned long long me = arr[lane];
            const unsigned long long at = __ballot(me != 0 && rank_in<64>(arr, me) == k - 1);
            __syncthreads();  // arr becomes the candidates
            return at ? lane_of(me, __builtin_ctzll(at)) : 0;
        }
        if (k <= 64) {  // 128 pairs of threads, by two waves
            const unsigned long long b = dpp<QUAD_XOR1>(best);
            best = best > b ? best : b;
            if ((tid & 1) == 0) arr[tid / 2] = best;
            __syncthreads();
            if (tid < 128) {
                const unsigned long long me = arr[tid];
                if (me != 0 && rank_in<128>(arr, me) == k - 1) S.bound = me;
            }
        } else {
            arr[tid] = best;
            __syncthreads();
            if (best != 0 && rank_in<TEAM>(arr, best) == k - 1) S.bound = best;
        }
        __syncthreads();  // and arr becomes the candidates
        return S.bound;
    }
}

template <class T, int TEAM>
__device__ unsigned long long radix_kth(const T* x, const uint8_t* mk, int V, int k, unsigned* hist) {
    unsigned long long prefix = 0;
    int need = k;
    for (int d = 7; d >= 0; --d) {
        for (int i = team_tid<TEAM>(); i < 256; i += TEAM) hist[i] = 0;
        team_sync<TEAM>();
        for (int i = team_tid<TEAM>(); i < V; i += TEAM) {
            const float v = (float)x[i];
            if ((mk && !mk[i]) || v == -INFINITY) continue;
            const unsigned long long key = order_key(v, i);
            if (d < 7 && (key >> (8 * d + 8)) != (prefix >> (8 * d + 8))) continue;
            atomicAdd(&hist[(key >> (8 * d)) & 255], 1u);
        }
        team_sync<TEAM>();
        int bin = 255, above = 0;
        for (; bin >= 0; --bin) {  // every thread walks the same counts
            const int n = hist[bin];
            if (above + n >= need) break;
            above += n;
        }
        team_sync<TEAM>();
        if (bin < 0) return 0;  // fewer than k: all of them (only possible at the first digit)
        prefix |= (unsigned long long)bin << (8 * d);
        need -= above;
    }
    return prefix;
}

// the candidates by radix selection: exactly min(k, alternatives) of them
template <class T, int TEAM>
__device__ int radix_select(const T* x, const uint8_t* mk, int V, int k, TopShare<TEAM>& S) {
    const int tid = team_tid<TEAM>();
    team_sync<TEAM>();
    const unsigned long long lo = radix_kth<T, TEAM>(x, mk, V, k, (unsigned*)S.cand);
    if (tid == 0) S.nc = 0;
    team_sync<TEAM>();
    for (int i = tid; i < V; i += TEAM) {
        const float f = (float)x[i];
        if ((mk && !mk[i]) || f == -INFINITY) continue;
        const unsigned long long key = order_key(f, i);
        if (key >= lo) S.cand[atomicAdd(&S.nc, 1)] = key;
    }
    team_sync<TEAM>();
    return S.nc;
}

template <class T, int TEAM, bool MASK>
__device__ int top_select(const T* x, const uint8_t* mk, int V, int k, bool plain, Best b, const float* gmax,
                          TopShare<TEAM>& S) {
    constexpr int N = VN<T>;
    const int tid = team_tid<TEAM>(), nvec = V / N, ng = (nvec + TEAM * GROUP - 1) / (TEAM * GROUP);
    if (plain) {  // uniform over the team
        const unsigned long long bound = kth_best<TEAM>(b.v > -INFINITY ? order_key(b.v, b.last) : 0, k, S);
        const float bv = bound ? key_value(bound) : LOWEST;
        for (int g = 0; g <= ng; ++g) {
            const float gm = gmax[g * TEAM + tid];
            if (gm >= bv) {
                const int h = atomicAdd(&S.nh, 1);
                if (h < S.HITS) S.hits[h] = g * TEAM + tid;
            }
        }
        team_sync<TEAM>();
        const int nh = S.nh;
        if (nh <= S.HITS) {
            const int sh = nvec > 2 * TEAM ? 2 : nvec > TEAM ? 1 : 0;  // 2^sh vectors a group has
            static_assert(GROUP == 4, "sh");
            for (int i = tid; i < nh << sh; i += TEAM) {
                const int h = S.hits[i >> sh], u = i & ((1 << sh) - 1), g = h / TEAM, t = h % TEAM;
                float f[N];
                int i0, n = 0;
                if (g == ng) {
                    i0 = nvec * N + t;
                    if (u == 0) {
                        f[0] = (float)x[i0];
                        n = 1;
                    }
                } else {
                    const int vi = (g * GROUP + u) * TEAM + t;
                    i0 = vi * N;
                    if (vi < nvec) {
                        unpack<T>(load16<false>(x + i0), f);
                        if constexpr (MASK) apply_mask<T>(mk + i0, f);
                        n = N;
                    }
                }
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    if (j >= n || !(f[j] >= bv)) continue;
                    const int b = (int)__float_as_uint(f[j] + 0.f);  // order_key without its NaN
                    const unsigned long long key =
                        ((unsigned long long)((unsigned)b ^ (unsigned)((b >> 31) | 0x80000000)) << 32) |
                        (0xFFFFFFFFu - (unsigned)(i0 + j));
                    if (key < bound) continue;
                    const int at = atomicAdd(&S.nc, 1);
                    if (at < S.CANDS) S.cand[at] = key;
                }
            }
            team_sync<TEAM>();
            const int n = S.nc;
            if (n <= S.CANDS) return n;
        }
    }
    return radix_select<T, TEAM>(x, mk, V, k, S);
}

// out(rank, key) of the first k candidates, out(rank, 0) where there are fewer
template <int TEAM, class Out>
__device__ __forceinline__ void top_out(const TopShare<TEAM>& S, int n, int k, Out out) {
    const int tid = team_tid<TEAM>();
    for (int i = tid; i < n; i += TEAM) {
        const unsigned long long me = S.cand[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += S.cand[j] > me;
        if (rank < k) out(rank, me);
    }
    for (int j = n + tid; j < k; j += TEAM) out(j, 0ull);
}

// ---- log-probabilities ------------------------------------------------------------------------------
struct LogprobsOut {
    const void* actions;
    int act64, k;
    float *stats, *logp, *entropy, *lse, *top_logp;
    long long* top_ids;
    long long keep;  // rows from here on are left in the caches for the backward pass
};

// a row's given action: its index is read ahead of the pass, its logit (by then cached) after it
__device__ __forceinline__ long long action_of(const LogprobsOut& O, long long r) {
    if (!O.logp) return -1;
    return O.act64 ? ((const long long*)O.actions)[r] : ((const int*)O.actions)[r];
}

template <class T>
__device__ __forceinline__ void write_row(const Rows& R, const LogprobsOut& O, long long r, const Stat<true>& st,
                                          float l2, long long act, const T* x, const uint8_t* mk) {
    const bool empty = st.s == 0.f;
    float H = empty ? 0.f : LN2 * (l2 - st.w / st.s);
    if (H < 0.f) H = 0.f;  // a difference of near values, as logp_of's; a NaN stays
    if (O.stats) ((float4*)O.stats)[r] = make_float4(st.ref, st.s, H, st.wide ? 1.f : 0.f);
    O.entropy[r] = H;
    O.lse[r] = empty ? -INFINITY : st.wide ? st.ref * R.invT + LN2 * l2 : LN2 * (st.ref + l2);
    if (O.logp) {
        float p = 0.f;
        if (act >= 0 && act < R.V) {
            p = empty || (mk && !mk[act]) ? -INFINITY : logp_of((float)x[act], st, l2, R.c, R.invT);
            if (st.s != st.s) p = st.s;
        }
        O.logp[r] = p;
    }
}

// rows split over blocks
struct Split {
    float4* part;               // [rows][n]: a part's Stat (ref, s and w, or s in two words, wide)
    unsigned long long* keys;   // [rows][n][k], by rank, 0: none
    int n, len;                 // parts, elements in each but the last
};

template <class T, int TEAM, bool MASK, bool TOP, bool PART>
__global__ __launch_bounds__(block_of<TEAM>) void logprobs_rows_kernel(Rows R, LogprobsOut O, Split P) {
    extern __shared__ float gmax_all[];
    constexpr int TEAMS = block_of<TEAM> / TEAM;
    __shared__ Shared<true> sh;
    __shared__ TopShare<TEAM> tops[TOP ? TEAMS : 1];
    const long long r = team_row<TEAM>();
    if (r >= R.rows) return;
    const T* x = row_ptr<T>(R, r);
    const uint8_t* mk = MASK ? mask_ptr(R, r) : nullptr;
    const int tid = team_tid<TEAM>();
    int V = R.V, from = 0;
    if constexpr (PART) {
        from = blockIdx.z * P.len;
        V = V - from < P.len ? V - from : P.len;
        x += from;
        if constexpr (MASK) mk += from;
    }
    float* gmax = gmax_all + team_in_block<TEAM>() * ((V / VN<T> + TEAM * GROUP - 1) / (TEAM * GROUP) + 1) * TEAM;
    long long act = -1;
    if constexpr (!PART) act = action_of(O, r);
    Sum<true> a{-FAR, 0.f, 0.f};
    float mx = -INFINITY;
    Best best{-INFINITY, 0};
    row_pass<T, TEAM, MASK, true, TOP>(x, mk, V, R.c, a, mx, best, gmax, NoEdit{}, r < O.keep);
    const Stat<true> st = row_stat<T, TEAM, true>(a, mx, x, mk, V, R.c, sh, NoEdit{});
    const bool numbers = st.s == st.s;  // no NaN, no +inf: the alternatives by their bound
    float l2 = 0.f;
    if constexpr (PART) {
        if (tid == 0) P.part[r * P.n + blockIdx.z] = make_float4(st.ref, st.s, st.w, st.wide);
    } else {
        l2 = lg2(st.s);
        if (tid == 0) write_row<T>(R, O, r, st, l2, act, x, mk);
    }
    if constexpr (TOP) {
        TopShare<TEAM>& S = tops[team_in_block<TEAM>()];
        const int n = top_select<T, TEAM, MASK>(x, mk, V, O.k, numbers, best, gmax, S);
        top_out<TEAM>(S, n, O.k, [&](int rank, unsigned long long key) {
            if constexpr (PART) {
                // the index within the row: the key holds its complement
                P.keys[((long long)r * P.n + blockIdx.z) * O.k + rank] = key ? key - from : 0;
            } else {
                O.top_ids[r * O.k + rank] = key ? (long long)key_index(key) : -1;
                O.top_logp[r * O.k + rank] =
                    key ? logp_of(key_value(key), st, l2, R.c, R.invT) : -INFINITY;
            }
        });
    }
}

// rows split over blocks: the parts' statistics and alternatives joined
template <class T, bool TOP>
__global__ __launch_bounds__(256) void logprobs_join_kernel(Rows R, LogprobsOut O, Split P) {
    __shared__ Shared<true> sh;
    __shared__ TopShare<256> S;
    const long long r = block_row();
    if (r >= R.rows) return;
    const T* x = row_ptr<T>(R, r);
    const uint8_t* mk = mask_ptr(R, r);
    const int tid = threadIdx.x;
    const long long act = action_of(O, r);
    Stat<true> st{0.f, 0.f, 0.f, false};
    for (int i = tid; i < P.n; i += 256) {
        const float4 p = P.part[r * P.n + i];
        stat_add(st, Stat<true>{p.x, p.y, p.z, p.w != 0.f}, R.c);
    }
    unsigned long long best = 0;
    const unsigned long long* keys = nullptr;
    const int nk = P.n * O.k;
    if constexpr (TOP) {
        keys = P.keys + r * nk;
        for (int i = tid; i < nk; i += 256) best = best > keys[i] ? best : keys[i];
    }
    st = team_join<256, true>(st, R.c, sh);
    const float l2 = lg2(st.s);
    if (tid == 0) write_row<T>(R, O, r, st, l2, act, x, mk);
    if constexpr (TOP) {
        const unsigned long long bound = kth_best<256>(best, O.k, S);
        for (int i = tid; i < nk; i += 256) {
            const unsigned long long key = keys[i];
            if (key == 0 || key < bound) continue;
            const int at = atomicAdd(&S.nc, 1);
            if (at < S.CANDS) S.cand[at] = key;
        }
        __syncthreads();
        int n = S.nc;
        if (n > S.CANDS) n = radix_select<T, 256>(x, mk, R.V, O.k, S);
        top_out<256>(S, n, O.k, [&](int rank, unsigned long long key) {
            O.top_ids[r * O.k + rank] = key ? (long long)key_index(key) : -1;
            O.top_logp[r * O.k + rank] = key ? logp_of(key_value(key), st, l2, R.c, R.invT) : -INFINITY;
        });
    }
}

// A gradient kernel's row, or its part of one: rows from the last to the first, a row's parts next to each other
// (across rows first, the blocks at work touch memory all over: 354 us against 300, 2048 x 100003 f32).
struct Part {
    long long r;
    int from;
};
template <int TEAM>
__device__ __forceinline__ Part part_of(const Rows& R, int len) {
    const unsigned n = ((unsigned)R.V + (unsigned)len - 1) / (unsigned)len;
    const long long id = team_row<TEAM>(), q = n == 1 ? id : id / n;
    return Part{R.rows - 1 - q, (int)(id - q * n) * len};
}

// Elementwise over a row or a part of it: f(x, legal) for each element, vectors of 16 bytes.  Rows are taken from
// the last to the first: what a forward pass read last may still be in the Infinity Cache.
template <class T, int TEAM, bool MASK, bool NT, class F>
__device__ __forceinline__ void map_row(const T* x, const uint8_t* mk, T* d, int V, F f) {
    constexpr int N = VN<T>;
    const int tid = team_tid<TEAM>(), nvec = V / N, step = TEAM * GROUP;
    auto put = [&](const uint4& v, int vi) {
        float y[N];
        unpack<T>(v, y);
        if constexpr (MASK) {
            uint8_t b[N];
            __builtin_memcpy(b, mk + vi * N, N);
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = b[i] ? f(y[i], vi * N + i) : 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = f(y[i], vi * N + i);
        }
        store16<NT>(d + (long long)vi * N, y);
    };
    int vi = tid;
    for (; vi - tid + step <= nvec; vi += step) {
        uint4 v[GROUP];
#pragma unroll
        for (int u = 0; u < GROUP; ++u) v[u] = load16<true>(x + (long long)(vi + u * TEAM) * N);
#pragma unroll
        for (int u = 0; u < GROUP; ++u) put(v[u], vi + u * TEAM);
    }
    if (vi - tid < nvec) {
        uint4 v[GROUP];
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
            v[u] = make_uint4(0u, 0u, 0u, 0u);
            if (vi + u * TEAM < nvec) v[u] = load16<true>(x + (long long)(vi + u * TEAM) * N);
        }
#pragma unroll
        for (int u = 0; u < GROUP; ++u)
            if (vi + u * TEAM < nvec) put(v[u], vi + u * TEAM);
    }
    const int i = nvec * N + tid;
    if (i < V) d[i] = (T)(!MASK || mk[i] ? f((float)x[i], i) : 0.f);
}

template <class T, int TEAM, bool MASK, class F>
__device__ __forceinline__ void map_row(const T* x, const uint8_t* mk, T* d, int V, bool nt, F f) {
    // one loop or the other: within one the compiler joins the two kinds of store, and loses the hint
    if (nt)
        map_row<T, TEAM, MASK, true>(x, mk, d, V, f);
    else
        map_row<T, TEAM, MASK, false>(x, mk, d, V, f);
}

template <class T, int TEAM, bool MASK>
__global__ __launch_bounds__(block_of<TEAM>) void logprobs_bwd_kernel(Rows R, const void* actions, int act64,
                                                           const float* __restrict__ stats, const float* gl,
                                                           long long gl_s, const float* ge, long long ge_s,
                                                           const float* gz, long long gz_s, T* __restrict__ dx,
                                                           int len, bool nt) {
    const Part at = part_of<TEAM>(R, len);
    const long long r = at.r;
    if (r < 0) return;
    const int from = at.from, V = R.V - from < len ? R.V - from : len;
    const T* x = row_ptr<T>(R, r) + from;
    const uint8_t* mk = MASK ? mask_ptr(R, r) + from : nullptr;
    const float4 st = ((const float4*)stats)[r];
    const float ref = st.x, s = st.y, H = st.z;
    long long a = -1;
    if (actions) a = act64 ? ((const long long*)actions)[r] : ((const int*)actions)[r];
    const bool given = a >= 0 && a < R.V;
    const float g1 = gl && given ? gl[r * gl_s] : 0.f, g2 = ge ? ge[r * ge_s] : 0.f, g3 = gz ? gz[r * gz_s] : 0.f;
    // p = 2^u / s and ln p = ln2 (u - log2 s): dx = 2^u (c0 - c1 u)
    const float c1 = g2 * R.invT * LN2 / s, ga = g1 * R.invT;
    const float c0 = (g3 - g1 - g2 * H) * R.invT / s + c1 * lg2(s);
    T* d = dx + r * (long long)R.V + from;
    const int mine = given ? (int)(a - from) : -1;  // outside this part: no element's index
    if (s == 0.f || (!given && !ge && !gz)) {  // no legal action, or nothing that reaches the row
        map_row<T, TEAM, false>(x, mk, d, V, nt, [](float, int) { return 0.f; });
    } else if (st.w != 0.f) {
        map_row<T, TEAM, MASK>(x, mk, d, V, nt, [&](float y, int i) {
            const float u = nmax((y - ref) * R.c, -1000.f);
            return ex2(u) * (c0 - c1 * u) + (i == mine ? ga : 0.f);
        });
    } else {
        map_row<T, TEAM, MASK>(x, mk, d, V, nt, [&](float y, int i) {
            const float u = nmax(__builtin_fmaf(y, R.c, -ref), -1000.f);
            const float g = ex2(u) * __builtin_fmaf(-c1, u, c0);
            return i == mine ? g + ga : g;
        });
    }
}

// ---- distillation ---------------------------------------------------------------------------------------
struct Teacher {
    const void* logp;
    const void* ids;
    int dtype, ids64, k, rest;
};

// a row's teacher entries: ids (-1: none), the student's logits there (illegal: -inf), t, q = exp(t - tm) / qs (rest:
// exp t); first: no earlier entry has the same id
struct Entries {
    double q[TOP_MAX];
    int id[TOP_MAX];
    float x[TOP_MAX], t[TOP_MAX];
    bool first[TOP_MAX];
};
struct EntryHead {
    double qs;  // the entries' sum (rest: of q)
    float tm;
    bool any;
};
struct EntryRegs {  // as loaded, an entry or two a lane
    int id[2];
    float t[2], x[2];
    bool legal[2];
};

// by one wave, with the logits of the entries in [lo, hi) alone; nothing here waits for the last loads, so that what a
// team loads of the row comes right behind them
template <class T>
__device__ __forceinline__ EntryRegs fetch_entries(const Teacher& Te, long long r, int V, const T* x, const uint8_t* mk,
                                                   int lo, int hi) {
    const int lane = threadIdx.x & 63;
    EntryRegs e;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int j = lane + 64 * u;
        e.t[u] = -INFINITY;
        e.id[u] = -1;
        e.x[u] = 0.f;
        e.legal[u] = false;
        if (j < Te.k) {
            const long long o = r * Te.k + j;
            const long long i = Te.ids64 ? ((const long long*)Te.ids)[o] : ((const int*)Te.ids)[o];
            e.id[u] = i >= 0 && i < V ? (int)i : -1;
            e.t[u] = Te.dtype == AZG_F32 ? ((const float*)Te.logp)[o]
                     : Te.dtype == AZG_BF16 ? (float)((const bf16_t*)Te.logp)[o]
                                            : (float)((const f16_t*)Te.logp)[o];
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (64 * u >= Te.k) continue;
        const int i = e.id[u];
        if (i < lo || i >= hi) continue;  // -1 as well
        e.x[u] = (float)x[i];
        e.legal[u] = !mk || mk[i];
    }
    return e;
}

__device__ __forceinline__ EntryHead load_entries(Entries& E, const EntryRegs& e, const Teacher& Te) {
    const int lane = threadIdx.x & 63;
    EntryHead h;
    int id[2];
    h.tm = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        id[u] = e.t[u] == -INFINITY ? -1 : e.id[u];
        if (id[u] >= 0) h.tm = nmax(h.tm, e.t[u]);
    }
    h.tm = wave_max(h.tm);
    h.any = h.tm != -INFINITY;
    if (Te.rest || !h.any) h.tm = 0.f;
    double q[2] = {0.0, 0.0};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (64 * u >= Te.k) continue;
        if (id[u] >= 0) q[u] = exp_f64((double)e.t[u] - (double)h.tm);
    }
    h.qs = wave_sum(q[0] + q[1]);
    const double iq = Te.rest || !h.any ? 1.0 : rcp_f64(h.qs);  // qs >= 1: the largest entry is e^0
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int j = lane + 64 * u;
        if (64 * u >= Te.k) continue;
        if (j < Te.k) {
            E.id[j] = id[u];
            E.t[j] = e.t[u];
            E.x[j] = id[u] >= 0 && e.legal[u] ? e.x[u] : -INFINITY;
            E.q[j] = q[u] * iq;
            E.first[j] = true;
        }
    }
    team_sync<64>();
    return h;
}

// which entries repeat an earlier one's id; true if any does
__device__ __forceinline__ bool find_repeats(Entries& E, int k) {
    const int lane = threadIdx.x & 63;
    const int id0 = lane < k ? E.id[lane] : -1, id1 = lane + 64 < k ? E.id[lane + 64] : -1;
    bool d0 = false, d1 = false;
#pragma unroll 8
    for (int i = 0; i + 1 < k; ++i) {
        const int e = E.id[i];
        d0 |= i < lane && e == id0;
        d1 |= i < lane + 64 && e == id1;
    }
    d0 &= id0 >= 0;
    d1 &= id1 >= 0;
    if (d0) E.first[lane] = false;
    if (d1) E.first[lane + 64] = false;
    team_sync<64>();
    return __ballot(d0 || d1) != 0;
}

struct Row {  // what the gradient needs of a row: p(x, ref, s) = 2^u(x, ref) / s
    float ro, so, b;  // dx = b p(x, ro, so) w / T (so = 0: 0, whatever the logits are), but
    float ra, sa, a;  // dx = (a p(x, ra, sa) - q) w / T at the entries
    int flags;
    float unused;
};
// flags: ro is a logit, ra is (each as Stat's `wide`: entries far from all else have a reference of their own
// kind); an action is given twice
constexpr int WIDE_OUT = 1, WIDE_ALL = 2, REPEATS = 4;
struct RowSums {  // so, sa as summed, for the loss
    double so, sa;
};

// a row's coefficients, by one wave, from the student's statistics v over all legal actions outside the entries
// (rest) or over all (else)
__device__ __forceinline__ Row row_coefficients(const Rows& R, const Teacher& Te, const Entries& E, const EntryHead& h,
                                                const Stat<false>& v, bool repeats, RowSums* sums) {
    const int lane = threadIdx.x & 63;
    Stat<false> all = v;
    double po = 1.0;  // the student's mass outside the entries
    if (Te.rest) {
        float xj[2], mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int j = lane + 64 * u;
            xj[u] = -INFINITY;
            if (j < Te.k && E.first[j]) xj[u] = E.x[j];
            mx = nmax(mx, xj[u]);
        }
        mx = wave_max(mx);
        Stat<false> e{0.f, 0.0, 0.f, false};
        if (mx != -INFINITY) {
            // near 0 the whole number next to max x c; from 2^24 on (a mask's fill, a low temperature) f32 may not hold that,
            // and what it is off by passes the exponential's range: there the maximum itself
            e.wide = v.wide || !(fabsf(mx * R.c) < 16777216.f);
            e.ref = e.wide ? mx : rintf(mx * R.c);
            e.s = wave_sum((double)ex2(u_of(xj[0], e.ref, e.wide, R.c)) + (double)ex2(u_of(xj[1], e.ref, e.wide, R.c)));
        }
        po = v.s != 0.0 ? 1.0 : 0.0;
        if (e.s != 0.0 && v.s != 0.0) {  // the sum of both at the larger reference
            const double d = place(v.ref, v.wide, R.c) - place(e.ref, e.wide, R.c);
            const double se = d > 0.0 ? e.s * (double)ex2((float)-d) : e.s;
            const double sv = d > 0.0 ? v.s : v.s * (double)ex2((float)d);
            if (!(d > 0.0)) all = e;
            all.s = se + sv;
            po = sv / all.s;
        } else if (e.s != 0.0) {
            all = e;
        }
    }
    double S = Te.rest ? h.qs : 1.0, qr = 0.0;
    if (Te.rest && v.s != 0.0) {
        qr = 1.0 - h.qs;
        if (qr < 0.0) qr = 0.0;
        S += qr;
    }
    *sums = RowSums{v.s, all.s};
    if (!h.any || all.s == 0.0) return Row{0.f, 0.f, 0.f, 0.f, 1.f, 0.f, 0, 0.f};  // no entry or no legal action
    return Row{v.ref, (float)v.s, (float)(S * po - qr), all.ref, (float)all.s, (float)S,
               (v.wide ? WIDE_OUT : 0) | (all.wide ? WIDE_ALL : 0) | (repeats ? REPEATS : 0), 0.f};
}

// the row's loss, by one wave, its terms in f64
__device__ __forceinline__ float row_kl(const Rows& R, const Teacher& Te, const Entries& E, const EntryHead& h,
                                        const Row& o, const RowSums& sums) {
    if (!h.any || sums.sa == 0.0) return 0.f;
    const int lane = threadIdx.x & 63;
    const bool wide = o.flags & WIDE_ALL;
    const double cd = R.c, ln2 = 0.69314718055994530942;
    // the row's logarithms at once, one a lane: of the sums over all and outside, of the entries' sum, of what is left
    const double qr = 1.0 - h.qs;
    const double ln = ln_f64(lane == 0 ? sums.sa : lane == 1 ? sums.so : lane == 2 ? h.qs : qr);
    const double lns = lane_of(ln, 0), lnq = Te.rest ? 0.0 : lane_of(ln, 2);
    double loss = 0.0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int j = lane + 64 * u;
        if (64 * u >= Te.k || j >= Te.k || E.id[j] < 0) continue;
        const double q = E.q[j];
        const double lq = ((double)E.t[j] - (double)h.tm) - lnq;
        const double uj = wide ? ((double)E.x[j] - (double)o.ra) * cd : (double)E.x[j] * cd - (double)o.ra;
        if (q > 0.0 || q != q) loss += q * (lq - (uj * ln2 - lns));
    }
    loss = wave_sum(loss);
    if (Te.rest && sums.so != 0.0) {
        const double d = place(o.ro, o.flags & WIDE_OUT, R.c) - place(o.ra, wide, R.c);
        if (!(qr <= 0.0)) loss += qr * (lane_of(ln, 3) - (d * ln2 + lane_of(ln, 1) - lns));
    }
    return (float)loss;
}

// the entries of a row as bits, an element each: what a pass leaves out
template <class T>
struct SkipBits {
    const unsigned* bits;
    bool on;
    __device__ __forceinline__ void operator()(int vi, float* f) const {
        if (!on) return;
        constexpr int N = VN<T>;
        unsigned b = ((const uint8_t*)bits)[N == 8 ? vi : vi >> 1];
        if (N == 4) b = (b >> (4 * (vi & 1))) & 15;
        if (b) {
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = (b >> i) & 1 ? -INFINITY : f[i];
        }
    }
    __device__ __forceinline__ bool one(int i) const { return on && (bits[i >> 5] >> (i & 31) & 1); }
};
// words of the bitmap: whole groups of vectors (NV of them) are looked up, also past the row's end
template <class T, int TEAM, int NV = 0>
__host__ __device__ constexpr int bit_words(int V) {
    return (NV > 0 ? TEAM * NV : (V / VN<T> / (TEAM * GROUP) + 1) * TEAM * GROUP) * VN<T> / 32 + 1;
}
__device__ __forceinline__ bool set_bit(unsigned* bits, int id, int from, int V) {  // was it set?
    const int i = id - from;
    return id >= 0 && i >= 0 && i < V && (atomicOr(&bits[i >> 5], 1u << (i & 31)) >> (i & 31) & 1);
}

// the entries' elements of a row (or a part of it), after all its elements
template <class T, int TEAM>
__device__ __forceinline__ void write_entries(const Rows& R, const Teacher& Te, const Entries& E, const Row& o, float g,
                                              const uint8_t* mk, T* d, int from, int V) {
    for (int j = team_tid<TEAM>(); j < Te.k; j += TEAM) {
        const int id = E.id[j], i = id - from;
        if (id < 0 || i < 0 || i >= V || (mk && !mk[i])) continue;
        float q = (float)E.q[j];
        if (o.flags & REPEATS) {  // the same index twice: its entries' probabilities add
            double all = 0.0;
            for (int e = 0; e < Te.k; ++e) all += E.id[e] == id ? E.q[e] : 0.0;
            q = (float)all;
        }
        const float p = ex2(u_of(E.x[j], o.ra, o.flags & WIDE_ALL, R.c)) * (o.a / o.sa);
        d[i] = (T)(o.a == 0.f ? 0.f : (p - q) * g);  // a = 0: a row without a legal action
    }
}

template <class T, int TEAM, bool MASK>
__device__ __forceinline__ void write_outside(const Rows& R, const Row& o, float g, const T* x, const uint8_t* mk, T* d,
                                              int V, bool nt) {
    const float b = o.so == 0.f ? 0.f : o.b * g / o.so;
    if (o.so == 0.f)
        map_row<T, TEAM, false>(x, mk, d, V, nt, [](float, int) { return 0.f; });
    else if (o.flags & WIDE_OUT)
        map_row<T, TEAM, MASK>(x, mk, d, V, nt, [&](float y, int) { return ex2((y - o.ro) * R.c) * b; });
    else
        map_row<T, TEAM, MASK>(x, mk, d, V, nt, [&](float y, int) { return ex2(__builtin_fmaf(y, R.c, -o.ro)) * b; });
}

struct DistillOut {
    float *stats, *row_loss;
    const float* w;
    long long w_s;
    float scale;
    void* dx;
    long long keep;  // rows from here on are left in the caches for the backward pass
    bool nt;         // the gradient is not
};
__device__ __forceinline__ float row_weight(const Rows& R, const DistillOut& O, long long r) {
    return (O.w ? O.w[r * O.w_s] : 1.f) * O.scale * R.invT;
}

// A team a row: statistics, loss and (dx) the gradient.  NV > 0: the row stays in registers (NV vectors a thread)
// between its two uses, and HBM sees it once; NV = 0: it is read again from the cache.
// Waves that a SIMD has to hold (the compiler keeps to the registers that leaves): all eight for a wave's short rows
// (86 us against 97 with the 5 it took by itself, step 65536 x 343 f32); 6 for up to 8 vectors a thread (203 us
// with 512 threads against 230 with 256 threads of 16 vectors and 4 waves, step 8192 x 32768 bf16: three rows of
// 64 KB a CU against four, each with half the serial work); 4 for 16 vectors.
template <int TEAM, int NV>
constexpr int waves_of = NV > 8 ? 4 : TEAM == 64 && NV <= 2 ? 8 : 6;

template <class T, int TEAM, bool MASK, int NV>
__global__ __launch_bounds__(block_of<TEAM>) __attribute__((amdgpu_waves_per_eu(waves_of<TEAM, NV>)))
void distill_rows_kernel(Rows R, Teacher Te, DistillOut O) {
    extern __shared__ unsigned bits_all[];
    constexpr int TEAMS = block_of<TEAM> / TEAM, N = VN<T>;
    __shared__ Shared<false> sh;
    __shared__ Entries Es[TEAMS];
    __shared__ Row rows[TEAMS];
    __shared__ RowSums sums[TEAMS];
    const long long r = team_row<TEAM>();
    if (r >= R.rows) return;
    const T* x = row_ptr<T>(R, r);
    const uint8_t* mk = MASK ? mask_ptr(R, r) : nullptr;
    const int tid = team_tid<TEAM>(), V = R.V, nvec = V / N, mine = team_in_block<TEAM>();
    const int words = bit_words<T, TEAM, NV>(V);
    unsigned* bits = bits_all + mine * words;
    Entries& E = Es[mine];
    // the entries' loads first: they are few, and the row's come behind them
    EntryRegs er;
    if (tid < 64) er = fetch_entries<T>(Te, r, V, x, mk, 0, V);
    constexpr int U = NV * N >= 16 ? 16 / N : 1, Q = NV > 0 ? NV / U : 1;  // 16 logits unpacked at a time
    Loaded<T, U> L[Q];
    if constexpr (NV > 0) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int u = 0; u < U; ++u) {  // past the end: the last vector again, made -inf when it is used
                const int vi = tid + (q * U + u) * TEAM;
                L[q].v[u] = make_uint4(0u, 0u, 0u, 0u);
                if ((q * U + u) * TEAM < nvec) L[q].v[u] = load16<true>(x + (long long)(vi < nvec ? vi : nvec - 1) * N);
            }
    }
    const bool marked = Te.rest || O.dx || O.stats;  // only the loss without rest needs no bits
    if (marked)
        for (int i = tid; i < words; i += TEAM) bits[i] = 0;
    EntryHead h;
    if (tid < 64) h = load_entries(E, er, Te);
    bool repeats = false;
    team_sync<TEAM>();
    if (marked) {
        if (tid < 64) {
            for (int j = tid; j < Te.k; j += 64) repeats |= set_bit(bits, E.id[j], 0, V);
            repeats = __ballot(repeats) != 0;
            if (repeats) find_repeats(E, Te.k);
        }
        team_sync<TEAM>();
    }
    const SkipBits<T> skip{bits, Te.rest != 0};
    Sum<false> a{-FAR, 0.0, 0.f};
    float mx = -INFINITY;
    if constexpr (NV > 0) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if (q * U * TEAM >= nvec) continue;  // the same for the whole team
            float f[U * N], gm = -INFINITY;
            opaque(L[q]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int vi = tid + (q * U + u) * TEAM;
                const uint4 w = L[q].v[u];
                constexpr unsigned none = MINF_BITS<T>;
                unpack<T>(vi < nvec ? w : make_uint4(none, none, none, none), f + u * N);
                if constexpr (MASK)
                    if (vi < nvec) apply_mask<T>(mk + vi * N, f + u * N);
                skip(vi, f + u * N);
#pragma unroll
                for (int i = 0; i < N; ++i) gm = nmax(gm, f[u * N + i]);
            }
            mx = nmax(mx, gm);
            sum_group<false, U * N>(a, f, gm, R.c);
            __builtin_amdgcn_sched_barrier(0);  // one group unpacked at a time
        }
        if (nvec * N < V) {
            const int i = nvec * N + tid;
            float f[2] = {-INFINITY, -INFINITY};
            if (i < V && (!MASK || mk[i]) && !skip.one(i)) f[0] = (float)x[i];
            mx = nmax(mx, f[0]);
            sum_group<false, 2>(a, f, f[0], R.c);
        }
    } else {
        Best none{-INFINITY, 0};
        row_pass<T, TEAM, MASK, false, false>(x, mk, V, R.c, a, mx, none, nullptr, skip, r < O.keep);
    }
    const Stat<false> v =
        row_stat<T, TEAM, false>(a, mx, x, mk, V, R.c, sh, skip);
    if (tid < 64) {
        RowSums both;
        const Row o = row_coefficients(R, Te, E, h, v, repeats, &both);
        if (tid == 0) {
            rows[mine] = o;
            sums[mine] = both;
            if (O.stats) ((Row*)O.stats)[r] = o;
        }
    }
    team_sync<TEAM>();
    auto loss = [&] {
        if (tid < 64) {
            const float kl = row_kl(R, Te, E, h, rows[mine], sums[mine]);
            if (tid == 0) O.row_loss[r] = kl;
        }
    };
    if (!O.dx) {
        loss();
        return;
    }
    if constexpr (NV > 0)
        for (int q = 0; q < Q; ++q) opaque(L[q]);
    const Row o = rows[mine];
    const float g = row_weight(R, O, r);
    T* d = (T*)O.dx + r * (long long)V;
    if (NV > 0 && !(o.flags & WIDE_OUT) && o.so != 0.f) {
        const float b = o.b * g / o.so;
        auto write = [&](auto nt) {
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int vi = tid + (q * U + u) * TEAM;
                    if ((q * U + u) * TEAM >= nvec || vi >= nvec) continue;
                    float y[N];
                    unpack<T>(L[q].v[u], y);
#pragma unroll
                    for (int i = 0; i < N; ++i) y[i] = ex2(__builtin_fmaf(y[i], R.c, -o.ro)) * b;
                    if constexpr (MASK) apply_mask<T>(mk + vi * N, y, 0.f);  // not before: b may be no number
                    store16<decltype(nt)::value>(d + (long long)vi * N, y);
                    __builtin_amdgcn_sched_barrier(0);
                }
        };
        if (O.nt)
            write(std::true_type{});
        else
            write(std::false_type{});
        const int i = nvec * N + tid;
        if (i < V) d[i] = (T)(!MASK || mk[i] ? ex2(__builtin_fmaf((float)x[i], R.c, -o.ro)) * b : 0.f);
    } else {
        write_outside<T, TEAM, MASK>(R, o, g, x, mk, d, V, O.nt);
    }
    team_sync<TEAM>();
    write_entries<T, TEAM>(R, Te, E, o, g, mk, d, 0, V);
    loss();  // last: the other waves do not wait for it
}

// a part of a row of few rows: its statistics outside the entries
__device__ __forceinline__ Stat<false> part_stat(float4 p) {
    const unsigned long long s = ((unsigned long long)__float_as_uint(p.z) << 32) | __float_as_uint(p.y);
    return Stat<false>{p.x, __longlong_as_double((long long)s), 0.f, p.w != 0.f};
}
template <class T, bool MASK>
__global__ __launch_bounds__(256) void distill_part_kernel(Rows R, Teacher Te, DistillOut O, Split P) {
    extern __shared__ unsigned bits[];
    __shared__ Shared<false> sh;
    const long long r = block_row();
    if (r >= R.rows) return;
    const int tid = threadIdx.x, from = blockIdx.z * P.len, V = R.V - from < P.len ? R.V - from : P.len;
    const T* x = row_ptr<T>(R, r) + from;
    const uint8_t* mk = MASK ? mask_ptr(R, r) + from : nullptr;
    if (Te.rest) {
        for (int i = tid; i < bit_words<T, 256>(V); i += 256) bits[i] = 0;
        int id = -1;
        if (tid < Te.k) {
            const long long o = r * Te.k + tid;
            const long long i = Te.ids64 ? ((const long long*)Te.ids)[o] : ((const int*)Te.ids)[o];
            const float f = Te.dtype == AZG_F32 ? ((const float*)Te.logp)[o]
                            : Te.dtype == AZG_BF16 ? (float)((const bf16_t*)Te.logp)[o]
                                                   : (float)((const f16_t*)Te.logp)[o];
            if (i >= 0 && i < R.V && f != -INFINITY) id = (int)i;
        }
        __syncthreads();
        set_bit(bits, id, from, V);
        __syncthreads();
    }
    Sum<false> a{-FAR, 0.0, 0.f};
    float mx = -INFINITY;
    Best none{-INFINITY, 0};
    const SkipBits<T> skip{bits, Te.rest != 0};
    row_pass<T, 256, MASK, false, false>(x, mk, V, R.c, a, mx, none, nullptr, skip, r < O.keep);
    const Stat<false> st = row_stat<T, 256, false>(a, mx, x, mk, V, R.c, sh, skip);
    if (tid == 0) {
        const unsigned long long s = (unsigned long long)__double_as_longlong(st.s);
        P.part[r * P.n + blockIdx.z] =
            make_float4(st.ref, __uint_as_float((unsigned)s), __uint_as_float((unsigned)(s >> 32)), st.wide);
    }
}

// a row or a part of it of the gradient, from the row's statistics (stats) or from its parts (JOIN: then the first
// part's block writes the row's loss and statistics as well)
template <class T, int TEAM, bool MASK, bool JOIN>
__global__ __launch_bounds__(block_of<TEAM>) void distill_bwd_kernel(Rows R, Teacher Te, DistillOut O, Split P,
                                                                     int len) {
    constexpr int TEAMS = block_of<TEAM> / TEAM;
    __shared__ Shared<false> sh;
    __shared__ Entries Es[TEAMS];
    __shared__ Row row;
    // from parts: few rows, or long ones whose many coefficients a block should not work out for little of it
    const Part at = JOIN ? Part{R.rows - 1 - team_row<TEAM>(), (int)blockIdx.z * len} : part_of<TEAM>(R, len);
    const long long r = at.r;
    if (r < 0) return;
    const int tid = team_tid<TEAM>(), from = at.from, V = R.V - from < len ? R.V - from : len;
    const T* x = row_ptr<T>(R, r);
    const uint8_t* mk = MASK ? mask_ptr(R, r) : nullptr;
    Entries& E = Es[team_in_block<TEAM>()];
    EntryHead h;
    bool repeats = false;
    float4 part{0.f, 0.f, 0.f, 0.f};  // ahead of the entries: their loads wait for each other
    if constexpr (JOIN)
        if (tid < P.n) part = P.part[r * P.n + tid];
    if (tid < 64) {
        h = load_entries(E, fetch_entries<T>(Te, r, R.V, x, mk, JOIN ? 0 : from, JOIN ? R.V : from + V), Te);
        if constexpr (JOIN) repeats = find_repeats(E, Te.k);
    }
    Row o;
    RowSums sums;
    if constexpr (JOIN) {
        if (tid < 64) {
            Stat<false> v = part_stat(part);
            for (int i = tid + 64; i < P.n; i += 64) stat_add(v, part_stat(P.part[r * P.n + i]), R.c);
            v = team_join<64, false>(v, R.c, sh);
            o = row_coefficients(R, Te, E, h, v, repeats, &sums);
            if (tid == 0) row = o;
        }
        __syncthreads();
        o = row;
    } else {
        o = ((const Row*)O.stats)[r];
    }
    if (!JOIN || O.dx) {
        const float g = row_weight(R, O, r);
        T* d = (T*)O.dx + r * (long long)R.V + from;
        write_outside<T, TEAM, MASK>(R, o, g, x + from, MASK ? mk + from : nullptr, d, V, O.nt);
        team_sync<TEAM>();
        write_entries<T, TEAM>(R, Te, E, o, g, MASK ? mk + from : nullptr, d, from, V);
    }
    if constexpr (JOIN)
        if (blockIdx.z == 0 && tid < 64) {
            const float kl = row_kl(R, Te, E, h, o, sums);
            if (tid == 0) {
                O.row_loss[r] = kl;
                if (O.stats) ((Row*)O.stats)[r] = o;
            }
        }
}

// out = scale sum_r w_r loss_r in a fixed order, f64: one block, eight loads a thread in flight
__global__ __launch_bounds__(1024) void loss_total_kernel(const float* __restrict__ loss, const float* w,
                                                          long long w_s, float scale, long long n,
                                                          float* __restrict__ out) {
    __shared__ double sh[16];
    double a = 0.0;
    long long i = threadIdx.x;
    for (; i + 7 * 1024 < n; i += 8 * 1024) {
        float l[8], g[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            l[u] = loss[i + u * 1024];
            g[u] = w ? w[(i + u * 1024) * w_s] : 1.f;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) a += (double)l[u] * (double)g[u];
    }
    for (; i < n; i += 1024) a += (double)loss[i] * (w ? (double)w[i * w_s] : 1.0);
    a = wave_sum(a);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) a += sh[i];
        out[0] = (float)(a * (double)scale);
    }
}

// ---- the C entries ----------------------------------------------------------------------------

bool rows_of(const azg_logits* L, Rows* R) {
    if (!L || !L->x || L->rows < 1 || L->vocab < 1 || L->vocab > AZG_POLICY_VOCAB_MAX ||
        L->rows > AZG_POLICY_ROWS_MAX) return false;
    if (L->inner < 1 || L->dtype < AZG_F32 || L->dtype > AZG_F16 || L->rows > (1LL << 60) / L->vocab) return false;
    if (L->stride_outer < 0 || L->stride_inner < 0 || L->mask_outer < 0 || L->mask_inner < 0) return false;
    if (!(L->temperature > 0.f) || !std::isfinite(L->temperature)) return false;
    const double c = 1.4426950408889634074 / (double)L->temperature;
    *R = Rows{L->x, L->mask, L->rows, L->inner, L->stride_outer, L->stride_inner, L->mask_outer, L->mask_inner,
              (int)L->vocab, (float)c, (float)(1.0 / (double)L->temperature)};
    return std::isfinite(R->c) && R->c > 0.f;
}

int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : azg_host_fail(AZG_ERR_HIP, std::string("azg_policy: ") + hipGetErrorString(e));
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int bad(const char* what) { return azg_host_fail(AZG_ERR_ARG, what); }

template <class F>
auto by_type(int dtype, F f) {
    if (dtype == AZG_F32) return f(float{});
    if (dtype == AZG_BF16) return f(bf16_t{});
    return f(f16_t{});
}

template <class F>
int by_mask(const Rows& R, F f) {
    if (R.mask) return f(std::true_type{});
    return f(std::false_type{});
}

bool teacher_of(const azg_teacher* t, Teacher* Te) {
    if (!t || !t->logp || !t->ids || t->k < 1 || t->k > TOP_MAX || t->dtype < AZG_F32 || t->dtype > AZG_F16)
        return false;
    *Te = Teacher{t->logp, t->ids, t->dtype, t->ids64 != 0, t->k, t->rest != 0};
    return true;
}

// What is read again is worth a place in the Infinity Cache (256 MB): of a forward pass whose backward pass follows the
// last rows, which that takes first, and of a gradient what fits, for the products that read it next.  All else
// goes past the caches.
constexpr long long CACHE_BYTES = 256LL << 20;
template <class T>
long long keep_from(const Rows& R, bool backward) {
    const long long fit = CACHE_BYTES / ((long long)R.V * (int)sizeof(T));
    return !backward ? R.rows : fit < R.rows ? R.rows - fit : 0;
}
template <class T>
bool too_large(const Rows& R) { return R.rows * R.V * (int)sizeof(T) > CACHE_BYTES / 2; }

// Which team takes a row.  A wave: rows of up to 4 KB, and of up to 16 KB where there are waves enough (94 us against
// 242, 38364 x 1135 f32, top 35; 58 against 89, 20000 x 4096 bf16: a block leaves most of its threads idle and pays for
// its reductions).  A block: longer ones.  Parts: rows longer than a block holds the maxima or bits (LDS) or the logits
// (registers) of; and rows of more than 8192 elements where there are fewer than 128, in parts of 4096 or more (with
// 128 to 1024 rows parts were slower: 58 us against 44, 802 x 89386 f16, top 87).
constexpr int WAVE_BYTES = 4096, WAVE_ROWS = 2048, PART_MIN = 4096;
template <class T>
int logprobs_most(bool top) { return top ? 1024 * 16 * VN<T> : 1 << 30; }
// With the gradient, rows for which one block would fill a CU's registers alone are taken in parts also where all of
// the logits fit the Infinity Cache, from which the second kernel reads them (102 us against 116, 1055 x 83523 bf16;
// beyond it the registers are the better: 255 us, 2048 x 131072 bf16, 1.05 of three passes' time at 5.2 TB/s).
template <class T>
long long distill_most(const Rows& R, bool grad) {
    if (!grad) return 1 << 18;
    const bool alone = R.V > 512 * 16 * VN<T> && R.rows * R.V * (int)sizeof(T) <= CACHE_BYTES;
    return (alone ? 512 : 1024) * 16 * VN<T>;
}

Split parts_of(const Rows& R, long long most) {
    Split P{nullptr, nullptr, 1, R.V};
    long long n = (R.V - 1) / most + 1;
    if (R.rows < 128 && R.V > 2 * PART_MIN) {
        long long want = 512 / R.rows;
        if (want > R.V / PART_MIN) want = R.V / PART_MIN;
        if (want > n) n = want;
    }
    if (n > 1) {
        P.len = (int)(((R.V + n - 1) / n + 1023) / 1024 * 1024);
        P.n = (R.V + P.len - 1) / P.len;
    }
    return P;
}
template <class T>
bool by_wave(const Rows& R) {
    return (long long)R.V * (int)sizeof(T) <= (R.rows >= WAVE_ROWS ? 4 * WAVE_BYTES : WAVE_BYTES);
}

template <int TEAM>
dim3 team_grid(long long rows, int z = 1) {
    dim3 g = row_grid(TEAM == 64 ? (rows + 3) / 4 : rows);
    g.z = (unsigned)z;
    return g;
}
template <class T, int TEAM>
unsigned gmax_bytes(int V) {
    const int ng = (V / VN<T> + TEAM * GROUP - 1) / (TEAM * GROUP);
    return (unsigned)((ng + 1) * block_of<TEAM> * 4);
}
template <class T, int TEAM, int NV = 0>
unsigned bits_bytes(int V) {
    return (unsigned)(bit_words<T, TEAM, NV>(V) * 4 * (block_of<TEAM> / TEAM));
}
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

// a block of a gradient kernel takes 16 KB of a row, four vectors a thread and no loop
template <class T>
constexpr int bwd_len = 16384 / (int)sizeof(T);

template <class T, bool MASK>
void distill_bwd(const Rows& R, const Teacher& Te, const DistillOut& O, hipStream_t st) {
    const Split none{nullptr, nullptr, 0, 0};
    if (by_wave<T>(R))
        hipLaunchKernelGGL((distill_bwd_kernel<T, 64, MASK, false>), team_grid<64>(R.rows), dim3(256), 0, st, R, Te, O,
                           none, R.V);
    else
        hipLaunchKernelGGL((distill_bwd_kernel<T, 256, MASK, false>),
                           team_grid<256>(R.rows * ((R.V + bwd_len<T> - 1) / bwd_len<T>)), dim3(256), 0, st, R, Te, O, none,
                           bwd_len<T>);
}

template <class T, int TEAM, bool MASK, int NV>
void distill_rows(const Rows& R, const Teacher& Te, const DistillOut& O, hipStream_t st) {
    hipLaunchKernelGGL((distill_rows_kernel<T, TEAM, MASK, NV>), team_grid<TEAM>(R.rows), dim3(block_of<TEAM>),
                       (bits_bytes<T, TEAM, NV>(R.V)), st, R, Te, O);
}

template <class T, bool MASK>
void distill_fwd(const Rows& R, const Teacher& Te, const DistillOut& O, Split P, float4* work, hipStream_t st) {
    constexpr int N = VN<T>;
    const int V = R.V;
    if (P.n > 1) {
        P.part = work;
        hipLaunchKernelGGL((distill_part_kernel<T, MASK>), team_grid<256>(R.rows, P.n), dim3(256),
                           (bits_bytes<T, 256>(P.len)), st, R, Te, O, P);
        hipLaunchKernelGGL((distill_bwd_kernel<T, 256, MASK, true>), team_grid<256>(R.rows, O.dx ? P.n : 1), dim3(256),
                           0, st, R, Te, O, P, P.len);
    } else if (!O.dx) {
        if (by_wave<T>(R))
            distill_rows<T, 64, MASK, 0>(R, Te, O, st);
        else
            distill_rows<T, 256, MASK, 0>(R, Te, O, st);
    } else if (V <= 64 * N * 2) {
        distill_rows<T, 64, MASK, 2>(R, Te, O, st);
    } else if (V <= 64 * N * 8) {
        distill_rows<T, 64, MASK, 8>(R, Te, O, st);
    } else if (V <= 256 * N * 8) {
        distill_rows<T, 256, MASK, 8>(R, Te, O, st);
    } else if (V <= 512 * N * 8) {
        distill_rows<T, 512, MASK, 8>(R, Te, O, st);
    } else if (V <= 512 * N * 16) {
        distill_rows<T, 512, MASK, 16>(R, Te, O, st);
    } else {
        distill_rows<T, 1024, MASK, 16>(R, Te, O, st);
    }
}

template <class T, bool MASK, bool TOP>
void logprobs_fwd(const Rows& R, const LogprobsOut& O, Split P, char* work, hipStream_t st) {
    if (P.n > 1) {
        P.part = (float4*)work;
        P.keys = (unsigned long long*)(work + up16(R.rows * P.n * 16));
        hipLaunchKernelGGL((logprobs_rows_kernel<T, 256, MASK, TOP, true>), team_grid<256>(R.rows, P.n), dim3(256),
                           TOP ? (gmax_bytes<T, 256>(P.len)) : 0, st, R, O, P);
        hipLaunchKernelGGL((logprobs_join_kernel<T, TOP>), team_grid<256>(R.rows), dim3(256), 0, st, R, O, P);
    } else if (by_wave<T>(R) && (O.k <= 64 || R.V <= TopShare<64>::CANDS)) {
        hipLaunchKernelGGL((logprobs_rows_kernel<T, 64, MASK, TOP, false>), team_grid<64>(R.rows), dim3(256),
                           TOP ? (gmax_bytes<T, 64>(R.V)) : 0, st, R, O, P);
    } else {
        hipLaunchKernelGGL((logprobs_rows_kernel<T, 256, MASK, TOP, false>), team_grid<256>(R.rows), dim3(256),
                           TOP ? (gmax_bytes<T, 256>(R.V)) : 0, st, R, O, P);
    }
}

}  // namespace

extern "C" int64_t azg_logprobs_work(const azg_logits* L, int32_t top) {
    Rows R;
    if (!rows_of(L, &R) || top < 0 || top > TOP_MAX) return bad("azg_logprobs_work: bad argument");
    return by_type(L->dtype, [&](auto z) -> int64_t {
        const Split P = parts_of(R, logprobs_most<decltype(z)>(top > 0));
        return P.n > 1 ? up16(R.rows * P.n * 16) + R.rows * P.n * top * 8 : 0;
    });
}
extern "C" int64_t azg_distill_work(const azg_logits* L, int32_t grad) {
    Rows R;
    if (!rows_of(L, &R)) return bad("azg_distill_work: bad argument");
    return by_type(L->dtype, [&](auto z) -> int64_t {
        const Split P = parts_of(R, distill_most<decltype(z)>(R, grad));
        return P.n > 1 ? R.rows * P.n * 16 : 0;
    });
}

extern "C" int azg_logprobs_fwd(const azg_logits* L, const void* actions, int32_t actions64, int32_t top, float* stats,
                                float* logp, float* entropy, float* lse, float* top_logp, int64_t* top_ids, void* work,
                                int64_t work_bytes, void* stream) {
    Rows R;
    if (!rows_of(L, &R) || !entropy || !lse || (actions != nullptr) != (logp != nullptr) || top < 0 || top > TOP_MAX ||
        (top > 0 && (!top_logp || !top_ids)) || !aligned16(stats) || !aligned16(work))
        return bad("azg_logprobs_fwd: bad argument");
    const int64_t need = azg_logprobs_work(L, top);
    if (need > 0 && (!work || work_bytes < need)) return bad("azg_logprobs_fwd: work is too small");
    LogprobsOut O{actions, actions64 != 0, top, stats, logp, entropy, lse, top_logp, (long long*)top_ids, 0};
    by_type(L->dtype, [&](auto z) {
        using T = decltype(z);
        return by_mask(R, [&](auto m) {
            constexpr bool MASK = decltype(m)::value;
            O.keep = keep_from<T>(R, stats != nullptr);
            if (top)
                logprobs_fwd<T, MASK, true>(R, O, parts_of(R, logprobs_most<T>(true)), (char*)work, (hipStream_t)stream);
            else
                logprobs_fwd<T, MASK, false>(R, O, parts_of(R, logprobs_most<T>(false)), (char*)work, (hipStream_t)stream);
            return 0;
        });
    });
    return launched();
}

extern "C" int azg_logprobs_bwd(const azg_logits* L, const void* actions, int32_t actions64, const float* stats,
                                const float* g_logp, int64_t g_logp_stride, const float* g_entropy,
                                int64_t g_entropy_stride, const float* g_lse, int64_t g_lse_stride, void* dx,
                                void* stream) {
    Rows R;
    if (!rows_of(L, &R) || !stats || !dx || (g_logp && !actions) || !aligned16(stats))
        return bad("azg_logprobs_bwd: bad argument");
    by_type(L->dtype, [&](auto z) {
        using T = decltype(z);
        return by_mask(R, [&](auto m) {
            constexpr bool MASK = decltype(m)::value;
            if (by_wave<T>(R))
                hipLaunchKernelGGL((logprobs_bwd_kernel<T, 64, MASK>), team_grid<64>(R.rows), dim3(256), 0,
                                   (hipStream_t)stream, R, actions, actions64, stats, g_logp, (long long)g_logp_stride,
                                   g_entropy, (long long)g_entropy_stride, g_lse, (long long)g_lse_stride, (T*)dx, R.V,
                                   too_large<T>(R));
            else
                hipLaunchKernelGGL((logprobs_bwd_kernel<T, 256, MASK>),
                                   team_grid<256>(R.rows * ((R.V + bwd_len<T> - 1) / bwd_len<T>)), dim3(256), 0,
                                   (hipStream_t)stream, R, actions, actions64, stats, g_logp, (long long)g_logp_stride,
                                   g_entropy, (long long)g_entropy_stride, g_lse, (long long)g_lse_stride, (T*)dx,
                                   bwd_len<T>, too_large<T>(R));
            return 0;
        });
    });
    return launched();
}

extern "C" int azg_distill_fwd(const azg_logits* L, const azg_teacher* t, float* stats, float* row_loss,
                               const float* weight, int64_t weight_stride, float scale, float* total, void* dx,
                               void* work, int64_t work_bytes, void* stream) {
    Rows R;
    Teacher Te;
    if (!rows_of(L, &R) || !teacher_of(t, &Te) || !row_loss || !aligned16(stats) || !aligned16(work))
        return bad("azg_distill_fwd: bad argument");
    const int64_t need = azg_distill_work(L, dx != nullptr);
    if (need > 0 && (!work || work_bytes < need)) return bad("azg_distill_fwd: work is too small");
    hipStream_t st = (hipStream_t)stream;
    DistillOut O{stats, row_loss, weight, (long long)weight_stride, scale, dx, 0, false};
    by_type(L->dtype, [&](auto z) {
        using T = decltype(z);
        O.keep = keep_from<T>(R, stats != nullptr || dx != nullptr);
        O.nt = too_large<T>(R);
        return by_mask(R, [&](auto m) {
            distill_fwd<T, decltype(m)::value>(R, Te, O, parts_of(R, distill_most<T>(R, dx != nullptr)), (float4*)work, st);
            return 0;
        });
    });
    if (total)
        hipLaunchKernelGGL(loss_total_kernel, dim3(1), dim3(1024), 0, st, row_loss, weight, (long long)weight_stride,
                           scale, (long long)L->rows, total);
    return launched();
}

extern "C" int azg_distill_bwd(const azg_logits* L, const azg_teacher* t, const float* stats, const float* weight,
                               int64_t weight_stride, float scale, void* dx, void* stream) {
    Rows R;
    Teacher Te;
    if (!rows_of(L, &R) || !teacher_of(t, &Te) || !stats || !dx || !aligned16(stats)) return bad("azg_distill_bwd: bad argument");
    DistillOut O{const_cast<float*>(stats), nullptr, weight, (long long)weight_stride, scale, dx, 0, false};
    by_type(L->dtype, [&](auto z) {
        using T = decltype(z);
        O.nt = too_large<T>(R);
        return by_mask(R, [&](auto m) {
            distill_bwd<T, decltype(m)::value>(R, Te, O, (hipStream_t)stream);
            return 0;
        });
    });
    return launched();
}
