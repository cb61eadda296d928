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
// Sums are over the legal actions (a byte mask, or all).  Logits are f32, bf16 or f16; statistics are f32, the
// few terms of a row's KL (a difference of near values) f64.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/azg.h"

int azg_host_fail(int code, const std::string& msg);  // azg_capi.cpp: the thread-local message

namespace {

constexpr int TOP_MAX = AZG_POLICY_TOP_MAX;
constexpr float LN2 = 0.69314718055994530942f;
constexpr float LOWEST = -3.402823466e38f;

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

template <class T>
__device__ __forceinline__ const T* row_ptr(const Rows& R, long long r) {
    const long long o = r / R.inner, i = r - o * R.inner;
    return (const T*)R.x + o * R.so + i * R.si;
}
__device__ __forceinline__ const uint8_t* mask_ptr(const Rows& R, long long r) {
    const long long o = r / R.inner, i = r - o * R.inner;
    return R.mask ? R.mask + o * R.mo + i * R.mi : nullptr;
}

// rows over the grid's x and y (a dimension holds fewer than 2^32 threads)
__device__ __forceinline__ long long block_row() { return blockIdx.x + (long long)gridDim.x * blockIdx.y; }
dim3 row_grid(long long rows) {
    const long long x = rows < (1 << 20) ? rows : 1 << 20;
    return dim3((unsigned)x, (unsigned)((rows + x - 1) / x));
}

// max that keeps a NaN (fmaxf drops it): a NaN logit makes its row's statistics NaN
__device__ __forceinline__ float nmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = nmax(x, __shfl_xor(x, o));
    return x;
}
template <class F>
__device__ __forceinline__ F wave_sum(F x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// ln s in f64 for f32 s > 0: s = 2^e f, f in [0.75, 1.5), ln f = 2 atanh(u), u = (f - 1) / (f + 1), |u| <= 0.2,
// by its power series to u^15 (what is left is under 2e-13)
__device__ __forceinline__ double ln_f64(float s) {
    if (!(s > 0.f) || s == INFINITY) return s == 0.f ? -INFINITY : (double)s;
    int e;
    float f = frexpf(s, &e);
    if (f < 0.75f) {
        f *= 2.f;
        --e;
    }
    const double u = ((double)f - 1.0) / ((double)f + 1.0), w = u * u;
    double t = 1.0 / 15;
    t = t * w + 1.0 / 13;
    t = t * w + 1.0 / 11;
    t = t * w + 1.0 / 9;
    t = t * w + 1.0 / 7;
    t = t * w + 1.0 / 5;
    t = t * w + 1.0 / 3;
    t = t * w + 1.0;
    return 0.69314718055994530942 * e + 2.0 * u * t;
}

// (m, s, w): max, sum 2^u and sum u 2^u with u = (x - m) c.  An empty set is (LOWEST, 0, 0): a finite start,
// so that a -inf logit (u = -inf) and a row of the type's lowest value (u = 0) both come out as they should.
struct Soft {
    float m, s, w;
};
__device__ __forceinline__ void soft_add(Soft& a, float x, float c) {
    const float m = nmax(a.m, x);
    const float d = nmax((a.m - m) * c, -1e30f), k = ex2(d);  // an earlier sum moved to the new maximum: u' = u + d
    const float u = (x - m) * c, uc = nmax(u, -1000.f);
    const float e = ex2(u);
    a.w = (k == 0.f ? 0.f : (a.w + d * a.s) * k) + e * uc;
    a.s = a.s * k + e;
    a.m = m;
}
__device__ __forceinline__ Soft soft_join(Soft a, Soft b, float c) {
    const float m = nmax(a.m, b.m);
    const float da = nmax((a.m - m) * c, -1e30f), db = nmax((b.m - m) * c, -1e30f);
    const float ka = ex2(da), kb = ex2(db);
    Soft r;
    r.m = m;
    r.s = a.s * ka + b.s * kb;
    r.w = (ka == 0.f ? 0.f : (a.w + da * a.s) * ka) + (kb == 0.f ? 0.f : (b.w + db * b.s) * kb);
    return r;
}

// order of the alternatives: larger logit first (NaN before all), then the lower index.  0: not an alternative.
__device__ __forceinline__ unsigned long long order_key(float x, unsigned idx) {
    unsigned b = __float_as_uint(x + 0.f);  // -0 -> +0
    unsigned k = x != x ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((unsigned long long)k << 32) | (0xFFFFFFFFu - idx);
}

template <int TEAM>
__device__ Soft block_soft(Soft v, float c, Soft* sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = soft_join(v, Soft{__shfl_xor(v.m, o), __shfl_xor(v.s, o), __shfl_xor(v.w, o)}, c);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int i = 1; i < TEAM / 64; ++i) v = soft_join(v, sh[i], c);
    __syncthreads();
    return v;
}

// the k-th key of a row by radix selection over the 64-bit order (value, then index: no two are equal), a
// histogram of 256 digits at a time; returns the smallest key among the top k (0 if fewer are alternatives)
template <class T, int TEAM>
__device__ unsigned long long radix_kth(const T* x, const uint8_t* mk, int V, int k, unsigned* hist) {
    unsigned long long prefix = 0;
    int need = k;
    for (int d = 7; d >= 0; --d) {
        for (int i = threadIdx.x; i < 256; i += TEAM) hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < V; i += TEAM) {
            const float v = (float)x[i];
            if ((mk && !mk[i]) || v == -INFINITY) continue;
            const unsigned long long key = order_key(v, i);
            if (d < 7 && (key >> (8 * d + 8)) != (prefix >> (8 * d + 8))) continue;
            atomicAdd(&hist[(key >> (8 * d)) & 255], 1u);
        }
        __syncthreads();
        int bin = 255, above = 0;
        for (; bin >= 0; --bin) {  // every thread walks the same counts
            const int n = hist[bin];
            if (above + n >= need) break;
            above += n;
        }
        __syncthreads();
        if (bin < 0) return prefix;  // fewer than k: all of them (only possible at the first digit)
        prefix |= (unsigned long long)bin << (8 * d);
        need -= above;
    }
    return prefix;
}

template <class T, bool TOP>
__global__ __launch_bounds__(256) void logprobs_rows_kernel(Rows R, const void* actions, int act64, int k,
                                                            float* __restrict__ stats, float* __restrict__ logp,
                                                            float* __restrict__ entropy, float* __restrict__ lse,
                                                            float* __restrict__ top_logp,
                                                            long long* __restrict__ top_ids) {
    __shared__ Soft sh[4];
    __shared__ unsigned hist[256];
    __shared__ unsigned long long cand[TOP_MAX];
    __shared__ unsigned ncand;
    const long long r = block_row();
    if (r >= R.rows) return;
    const T* x = row_ptr<T>(R, r);
    const uint8_t* mk = mask_ptr(R, r);
    const int tid = threadIdx.x;
    Soft v{LOWEST, 0.f, 0.f};
    for (int i = tid; i < R.V; i += 256)
        if (!mk || mk[i]) soft_add(v, (float)x[i], R.c);
    v = block_soft<256>(v, R.c, sh);
    const float l2 = __builtin_amdgcn_logf(v.s);
    if (tid == 0) {
        const bool empty = v.s == 0.f;
        const float H = empty ? 0.f : LN2 * (l2 - v.w / v.s);
        if (stats) {
            stats[4 * r] = v.m;
            stats[4 * r + 1] = l2;
            stats[4 * r + 2] = H;
        }
        entropy[r] = H;
        lse[r] = empty ? -INFINITY : v.m * R.invT + LN2 * l2;
        if (logp) {
            const long long a = act64 ? ((const long long*)actions)[r] : ((const int*)actions)[r];
            float p = 0.f;
            if (a >= 0 && a < R.V) {
                p = empty || (mk && !mk[a]) ? -INFINITY : ((float)x[a] - v.m) * R.invT - LN2 * l2;
                if (v.s != v.s) p = v.s;
            }
            logp[r] = p;
        }
    }
    if constexpr (TOP) {
        const unsigned long long lo = radix_kth<T, 256>(x, mk, R.V, k, hist);
        if (tid == 0) ncand = 0;
        __syncthreads();
        for (int i = tid; i < R.V; i += 256) {
            const float f = (float)x[i];
            if ((mk && !mk[i]) || f == -INFINITY) continue;
            const unsigned long long key = order_key(f, i);
            if (key >= lo) cand[atomicAdd(&ncand, 1u)] = key;
        }
        __syncthreads();
        const int n = ncand;
        for (int j = tid; j < k; j += 256) {
            if (j < n) {
                const unsigned long long me = cand[j];
                int rank = 0;
                for (int i = 0; i < n; ++i) rank += cand[i] > me;
                const unsigned id = 0xFFFFFFFFu - (unsigned)me;
                top_ids[r * k + rank] = id;
                top_logp[r * k + rank] = ((float)x[id] - v.m) * R.invT - LN2 * l2;
            } else {
                top_ids[r * k + j] = -1;
                top_logp[r * k + j] = -INFINITY;
            }
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(Rows R, const void* actions, int act64,
                                                           const float* __restrict__ stats, const float* gl,
                                                           long long gl_s, const float* ge, long long ge_s,
                                                           const float* gz, long long gz_s, T* __restrict__ dx) {
    const long long r = block_row();
    if (r >= R.rows) return;
    const T* x = row_ptr<T>(R, r);
    const uint8_t* mk = mask_ptr(R, r);
    const float m = stats[4 * r], l2 = stats[4 * r + 1], H = stats[4 * r + 2];
    long long a = -1;
    if (actions) a = act64 ? ((const long long*)actions)[r] : ((const int*)actions)[r];
    const bool given = a >= 0 && a < R.V;
    const float g1 = gl && given ? gl[r * gl_s] : 0.f, g2 = ge ? ge[r * ge_s] : 0.f, g3 = gz ? gz[r * gz_s] : 0.f;
    const float c0 = (g3 - g1 - g2 * H) * R.invT, c1 = g2 * R.invT * LN2, ga = g1 * R.invT;
    T* d = dx + r * (long long)R.V;
    const bool empty = l2 == -INFINITY;
    for (int i = threadIdx.x; i < R.V; i += 256) {
        float g = 0.f;
        if (!empty && (!mk || mk[i])) {
            const float z = nmax(((float)x[i] - m) * R.c - l2, -1000.f);
            g = ex2(z) * (c0 - c1 * z);
            if (i == a) g += ga;
        }
        d[i] = (T)g;
    }
}

// ---- distillation ---------------------------------------------------------------------------

struct Teacher {
    const void* logp;
    const void* ids;
    int dtype, ids64, k, rest;
};

// a row's teacher entries, by its first wave: ids (-1: none), t, q, and tm, qs with q = exp(t - tm) / qs (rest: exp t)
struct Entries {
    int id[TOP_MAX];
    float t[TOP_MAX], q[TOP_MAX];
    float tm, qs;
    int any;
};

__device__ void load_entries(Entries& E, const Teacher& Te, long long r, int V) {
    const int lane = threadIdx.x & 63;
    float tm = -INFINITY;
    float t[2];
    int id[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int j = lane + 64 * u;
        t[u] = -INFINITY;
        id[u] = -1;
        if (j < Te.k) {
            const long long o = r * Te.k + j;
            const long long i = Te.ids64 ? ((const long long*)Te.ids)[o] : ((const int*)Te.ids)[o];
            const float f = Te.dtype == AZG_F32 ? ((const float*)Te.logp)[o]
                            : Te.dtype == AZG_BF16 ? (float)((const bf16_t*)Te.logp)[o]
                                                   : (float)((const f16_t*)Te.logp)[o];
            if (i >= 0 && i < V && f != -INFINITY) {
                id[u] = (int)i;
                t[u] = f;
            }
        }
        tm = nmax(tm, t[u]);
    }
    tm = wave_max(tm);
    const bool any = tm != -INFINITY;
    if (Te.rest || !any) tm = 0.f;
    float q[2], qs = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        q[u] = id[u] >= 0 ? expf(t[u] - tm) : 0.f;
        qs += q[u];
    }
    qs = wave_sum(qs);
    const float iq = Te.rest || !any ? 1.f : 1.f / qs;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int j = lane + 64 * u;
        if (j < Te.k) {
            E.id[j] = id[u];
            E.t[j] = t[u];
            E.q[j] = q[u] * iq;
        }
    }
    if (lane == 0) {
        E.tm = tm;
        E.qs = qs;
        E.any = any;
    }
}

// is an earlier entry of the row this one's id as well
__device__ __forceinline__ bool earlier(const Entries& E, int j) {
    for (int i = 0; i < j; ++i)
        if (E.id[i] == E.id[j]) return true;
    return false;
}

struct Row {  // what the gradient needs of a row: with e(x, m, l) = 2^((x - m) c - l)
    float mo, lo, b;  // dx = b e(x, mo, lo) w / T, but
    float m, l, a;    // dx = (a e(x, m, l) - q) w / T at the entries
    float pad[2];
};

// one row's loss and coefficients by the first wave, from the student's statistics over all legal actions outside
// the entries (rest) or over all (else)
template <class T>
__device__ float finish_row(const Rows& R, const Teacher& Te, const Entries& E, Soft v, const T* x,
                            const uint8_t* mk, Row* out) {
    const int lane = threadIdx.x & 63;
    float xj[2];
    bool ok[2];
    Soft e{LOWEST, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int j = lane + 64 * u;
        ok[u] = j < Te.k && E.id[j] >= 0;
        xj[u] = ok[u] && (!mk || mk[E.id[j]]) ? (float)x[E.id[j]] : -INFINITY;
        if (Te.rest && ok[u] && !earlier(E, j)) soft_add(e, xj[u], R.c);
    }
    Soft all = v;
    if (Te.rest) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            e = soft_join(e, Soft{__shfl_xor(e.m, o), __shfl_xor(e.s, o), __shfl_xor(e.w, o)}, R.c);
        all = soft_join(v, e, R.c);
    }
    const double invT = (double)R.c * 0.69314718055994530942;
    const double lns = ln_f64(all.s), lnq = Te.rest ? 0.0 : ln_f64(E.qs);
    double loss = 0.0, Q = 0.0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (!ok[u]) continue;
        const int j = lane + 64 * u;
        const double q = E.q[j];
        Q += q;
        const double lq = ((double)E.t[j] - (double)E.tm) - lnq;
        const double lp = ((double)xj[u] - (double)all.m) * invT - lns;
        if (q > 0.0 || q != q) loss += q * (lq - lp);
    }
    loss = wave_sum(loss);
    Q = wave_sum(Q);
    double S = Q, pr = 1.0, qr = 0.0;
    if (Te.rest) {
        pr = 0.0;
        if (v.s != 0.f) {
            const double lpr = ((double)v.m - (double)all.m) * invT + ln_f64(v.s) - lns;
            pr = exp(lpr);
            qr = 1.0 - Q;
            if (qr < 0.0) qr = 0.0;
            if (qr != 0.0) loss += qr * (ln_f64((float)qr) - lpr);
            S += qr;
        }
    }
    const bool none = !E.any || all.s == 0.f;
    if (none) loss = 0.0, S = 0.0, qr = 0.0;
    if (lane == 0) {
        out->mo = v.m;
        out->lo = v.s == 0.f ? 0.f : __builtin_amdgcn_logf(v.s);
        out->b = (float)(S * pr - qr);
        out->m = all.m;
        out->l = all.s == 0.f ? 0.f : __builtin_amdgcn_logf(all.s);
        out->a = (float)S;
    }
    return (float)loss;
}

template <class T>
__global__ __launch_bounds__(256) void distill_rows_kernel(Rows R, Teacher Te, float* __restrict__ stats,
                                                           float* __restrict__ row_loss) {
    constexpr int CH = 65536;  // elements between two settings of the bitmap of entries
    __shared__ Soft sh[4];
    __shared__ Entries E;
    __shared__ unsigned bits[CH / 32];
    const long long r = block_row();
    if (r >= R.rows) return;
    const T* x = row_ptr<T>(R, r);
    const uint8_t* mk = mask_ptr(R, r);
    const int tid = threadIdx.x;
    if (tid < 64) load_entries(E, Te, r, R.V);
    Soft v{LOWEST, 0.f, 0.f};
    for (int c0 = 0; c0 < R.V; c0 += CH) {
        const int n = R.V - c0 < CH ? R.V - c0 : CH;
        if (Te.rest) {
            __syncthreads();
            for (int i = tid; i < (n + 31) / 32; i += 256) bits[i] = 0;
            __syncthreads();
            for (int j = tid; j < Te.k; j += 256) {
                const int i = E.id[j] - c0;
                if (E.id[j] >= 0 && i >= 0 && i < n) atomicOr(&bits[i >> 5], 1u << (i & 31));
            }
            __syncthreads();
        }
        for (int i = tid; i < n; i += 256)
            if ((!mk || mk[c0 + i]) && !(Te.rest && (bits[i >> 5] >> (i & 31) & 1))) soft_add(v, (float)x[c0 + i], R.c);
    }
    v = block_soft<256>(v, R.c, sh);
    if (tid < 64) {
        Row o;
        const float loss = finish_row<T>(R, Te, E, v, x, mk, &o);
        if (tid == 0) {
            row_loss[r] = loss;
            if (stats) ((Row*)stats)[r] = o;
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void distill_bwd_kernel(Rows R, Teacher Te, const float* __restrict__ stats,
                                                          const float* w, long long w_s, float w0,
                                                          T* __restrict__ dx) {
    __shared__ Entries E;
    const long long r = block_row();
    if (r >= R.rows) return;
    const T* x = row_ptr<T>(R, r);
    const uint8_t* mk = mask_ptr(R, r);
    const int tid = threadIdx.x;
    const Row st = ((const Row*)stats)[r];
    const float g = (w ? w[r * w_s] : 1.f) * w0 * R.invT;
    T* d = dx + r * (long long)R.V;
    if (tid < 64) load_entries(E, Te, r, R.V);
    for (int i = tid; i < R.V; i += 256) {
        float f = 0.f;
        if (!mk || mk[i]) f = ex2(((float)x[i] - st.mo) * R.c - st.lo) * st.b * g;
        d[i] = (T)f;
    }
    __syncthreads();
    for (int j = tid; j < Te.k; j += 256) {
        const int id = E.id[j];
        if (id < 0 || (mk && !mk[id])) continue;
        float q = 0.f;  // the same index twice: its entries' probabilities add
        for (int i = 0; i < Te.k; ++i) q += E.id[i] == id ? E.q[i] : 0.f;
        if (st.a == 0.f) q = 0.f;  // a row without a legal action
        d[id] = (T)((ex2(((float)x[id] - st.m) * R.c - st.l) * st.a - q) * g);
    }
}

// out = scale sum_r w_r loss_r in a fixed order, f64
__global__ __launch_bounds__(1024) void loss_total_kernel(const float* __restrict__ loss, const float* w,
                                                          long long w_s, float scale, long long n,
                                                          float* __restrict__ out) {
    __shared__ double sh[16];
    double a = 0.0;
    for (long long i = threadIdx.x; i < n; i += 1024) a += (double)loss[i] * (w ? (double)w[i * w_s] : 1.0);
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
    if (L->inner < 1 || L->dtype < AZG_F32 || L->dtype > AZG_F16) return false;
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
int bad(const char* what) { return azg_host_fail(AZG_ERR_ARG, what); }

template <class F>
int by_type(int dtype, F f) {
    if (dtype == AZG_F32) return f(float{});
    if (dtype == AZG_BF16) return f(bf16_t{});
    return f(f16_t{});
}

bool teacher_of(const azg_teacher* t, Teacher* Te) {
    if (!t || !t->logp || !t->ids || t->k < 1 || t->k > TOP_MAX || t->dtype < AZG_F32 || t->dtype > AZG_F16)
        return false;
    *Te = Teacher{t->logp, t->ids, t->dtype, t->ids64 != 0, t->k, t->rest != 0};
    return true;
}

}  // namespace

extern "C" int64_t azg_logprobs_work(const azg_logits* L, int32_t top) {
    Rows R;
    if (!rows_of(L, &R) || top < 0 || top > TOP_MAX) return bad("azg_logprobs_work: bad argument");
    return 0;
}
extern "C" int64_t azg_distill_work(const azg_logits* L, int32_t) {
    Rows R;
    if (!rows_of(L, &R)) return bad("azg_distill_work: bad argument");
    return 0;
}

extern "C" int azg_logprobs_fwd(const azg_logits* L, const void* actions, int32_t actions64, int32_t top, float* stats,
                                float* logp, float* entropy, float* lse, float* top_logp, int64_t* top_ids, void* work,
                                int64_t work_bytes, void* stream) {
    Rows R;
    if (!rows_of(L, &R) || !entropy || !lse || (actions != nullptr) != (logp != nullptr) || top < 0 || top > TOP_MAX ||
        (top > 0 && (!top_logp || !top_ids)) || work_bytes < azg_logprobs_work(L, top))
        return bad("azg_logprobs_fwd: bad argument");
    hipStream_t st = (hipStream_t)stream;
    return by_type(L->dtype, [&](auto z) {
        using T = decltype(z);
        if (top)
            hipLaunchKernelGGL((logprobs_rows_kernel<T, true>), row_grid(L->rows), dim3(256), 0, st, R, actions,
                               actions64, top, stats, logp, entropy, lse, top_logp, (long long*)top_ids);
        else
            hipLaunchKernelGGL((logprobs_rows_kernel<T, false>), row_grid(L->rows), dim3(256), 0, st, R, actions,
                               actions64, top, stats, logp, entropy, lse, top_logp, (long long*)top_ids);
        return launched();
    });
}

extern "C" int azg_logprobs_bwd(const azg_logits* L, const void* actions, int32_t actions64, const float* stats,
                                const float* g_logp, int64_t g_logp_stride, const float* g_entropy,
                                int64_t g_entropy_stride, const float* g_lse, int64_t g_lse_stride, void* dx,
                                void* stream) {
    Rows R;
    if (!rows_of(L, &R) || !stats || !dx || (g_logp && !actions)) return bad("azg_logprobs_bwd: bad argument");
    return by_type(L->dtype, [&](auto z) {
        using T = decltype(z);
        hipLaunchKernelGGL((logprobs_bwd_kernel<T>), row_grid(L->rows), dim3(256), 0, (hipStream_t)stream, R,
                           actions, actions64, stats, g_logp, (long long)g_logp_stride, g_entropy,
                           (long long)g_entropy_stride, g_lse, (long long)g_lse_stride, (T*)dx);
        return launched();
    });
}

extern "C" int azg_distill_fwd(const azg_logits* L, const azg_teacher* t, float* stats, float* row_loss,
                               const float* weight, int64_t weight_stride, float scale, float* total, void* dx,
                               void* work, int64_t work_bytes, void* stream) {
    Rows R;
    Teacher Te;
    if (!rows_of(L, &R) || !teacher_of(t, &Te) || !row_loss || (dx && !stats) ||
        work_bytes < azg_distill_work(L, dx != nullptr))
        return bad("azg_distill_fwd: bad argument");
    hipStream_t st = (hipStream_t)stream;
    return by_type(L->dtype, [&](auto z) {
        using T = decltype(z);
        hipLaunchKernelGGL((distill_rows_kernel<T>), row_grid(L->rows), dim3(256), 0, st, R, Te, stats, row_loss);
        if (dx)
            hipLaunchKernelGGL((distill_bwd_kernel<T>), row_grid(L->rows), dim3(256), 0, st, R, Te, stats, weight,
                               (long long)weight_stride, scale, (T*)dx);
        if (total)
            hipLaunchKernelGGL(loss_total_kernel, dim3(1), dim3(1024), 0, st, row_loss, weight,
                               (long long)weight_stride, scale, (long long)L->rows, total);
        return launched();
    });
}

extern "C" int azg_distill_bwd(const azg_logits* L, const azg_teacher* t, const float* stats, const float* weight,
                               int64_t weight_stride, float scale, void* dx, void* stream) {
    Rows R;
    Teacher Te;
    if (!rows_of(L, &R) || !teacher_of(t, &Te) || !stats || !dx) return bad("azg_distill_bwd: bad argument");
    return by_type(L->dtype, [&](auto z) {
        using T = decltype(z);
        hipLaunchKernelGGL((distill_bwd_kernel<T>), row_grid(L->rows), dim3(256), 0, (hipStream_t)stream, R, Te,
                           stats, weight, (long long)weight_stride, scale, (T*)dx);
        return launched();
    });
}
