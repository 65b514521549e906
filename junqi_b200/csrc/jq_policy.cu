// jq_policy.cu -- a policy's action distribution under a legal mask: the
// log-probability of an action and the entropy with their gradient, and the
// verification of drafted actions (with no drafts: sampling).
//
// Over a row's legal places L = {j : mask_j != 0 and x_j > -inf}:
//
//   m = max x, Z = sum exp(x - m), p_j = exp(x_j - m) / Z, c_j = x_j - m
//   log p_a = c_a - log Z,  H = log Z - sum p_j c_j
//   d/dx_j (u log p_a + v H) = u ([j = a] - p_j) - v p_j (log p_j + H)
//
// Bound: memory.  What has to be read is the mask (a byte per place) and the
// logits at legal places only: a position has some tens of legal moves among
// 16,641, so the mask is packed to bits first and a thread touches the
// logits of the bits it found.  The packed mask (an eighth of the mask) is
// also what the backward pass keeps: the masks that the environment and the
// rollout history hand out are buffers that their next call overwrites.
#include <limits.h>
#include <math.h>

#include "jq_ops.cuh"

namespace jq {

constexpr float LOWEST = -3.402823466e38f;  // start of a running maximum: every finite logit is at least this
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Bits of 32 mask bytes, byte 32 w first, from 16-byte loads of the aligned
// blocks around them; at the row's ends, where those would leave the row,
// byte by byte.
__device__ __forceinline__ uint32_t legal_word(const uint8_t *row, int n, int w) {
    const int j0 = 32 * w;
    const uint8_t *p = row + j0;
    const int a = (int)((uintptr_t)p & 15);
    if (j0 >= a && (int64_t)j0 - a + (a ? 48 : 32) <= n) {
        const uint4 *q = (const uint4 *)(p - a);
        const uint4 u0 = q[0], u1 = q[1], u2 = a ? q[2] : make_uint4(0, 0, 0, 0);
        uint32_t v[13] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w, u2.x, u2.y, u2.z, u2.w, 0};
        const int s = a >> 2, f = (a & 3) * 8;
        if (s & 2)
#pragma unroll
            for (int i = 0; i < 11; ++i) v[i] = v[i + 2];
        if (s & 1)
#pragma unroll
            for (int i = 0; i < 10; ++i) v[i] = v[i + 1];
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = __vminu4(__funnelshift_r(v[i], v[i + 1], f), 0x01010101u);
            bits |= ((b * 0x01020408u) >> 24) << (4 * i);  // byte k's bit 8 k lands at 24 + k
        }
        return bits;
    }
    uint32_t bits = 0;
    const int end = n - j0 < 32 ? n - j0 : 32;
#pragma unroll 8
    for (int i = 0; i < end; ++i) bits |= (uint32_t)(p[i] != 0) << i;
    return bits;
}

// Running maximum, sum of exp(x - m) and sum of exp(x - m)(x - m).
struct Soft {
    float m, s, t;
    template <int N>
    __device__ __forceinline__ void add(const float (&x)[N]) {
        float c = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) c = fmaxf(c, x[i]);
        if (c > m) {
            const float d = m - c, k = ex2(d * LOG2E);
            t = k > 0.f ? k * (t + s * d) : 0.f;  // k = 0: d may be far, or infinite
            s *= k;
            m = c;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float d = x[i] - m, e = ex2(d * LOG2E);
            s += e;
            if (e > 0.f) t += e * d;
        }
    }
    __device__ __forceinline__ void join(float m2, float s2, float t2) {
        const float M = fmaxf(m, m2), d1 = m - M, d2 = m2 - M;
        const float k1 = ex2(d1 * LOG2E), k2 = ex2(d2 * LOG2E);
        const float a = k1 > 0.f ? k1 * (t + s * d1) : 0.f, b = k2 > 0.f ? k2 * (t2 + s2 * d2) : 0.f;
        // NaN sums (a NaN or +inf at a legal place) stay NaN
        s = (s == 0.f ? 0.f : s * k1) + (s2 == 0.f ? 0.f : s2 * k2);
        t = a + b;
        m = M;
    }
};

// A thread's legal logits, four loads in flight.
template <typename T>
__device__ __forceinline__ void add_bits(Soft &a, const T *x, uint32_t bits) {
    while (bits) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = -INFINITY;
            if (bits) {
                v[i] = to_f(x[__ffs(bits) - 1]);
                bits &= bits - 1;
            }
        }
        a.add(v);
    }
}

constexpr int LOGP_THREADS = 256;

struct LogpArgs {
    const void *x;
    const uint8_t *mask;
    uint32_t *bits;        // (rows, words): the packed mask; written by the forward pass (may be NULL there)
    const int32_t *act;
    float *lp, *ent;       // forward outputs
    float4 *stats;         // (rows): m, 1 / Z, log Z, H
    const float *glp, *gent;
    void *dx;
    int64_t x_stride, mask_stride, glp_stride, gent_stride;
    int32_t n, words;
};

__device__ __forceinline__ bool is_legal(const uint8_t *mask, const uint32_t *bits, int j) {
    return bits ? (bits[j >> 5] >> (j & 31)) & 1 : !mask || mask[j] != 0;
}

template <typename T, bool MASK>
__global__ void __launch_bounds__(LOGP_THREADS) logp_fwd_kernel(const LogpArgs a) {
    __shared__ float red[LOGP_THREADS / 32][3];
    pdl_enter();
    const int64_t row = blockIdx.x;
    const T *x = (const T *)a.x + row * a.x_stride;
    const int tid = threadIdx.x, lane = tid & 31;
    Soft acc{LOWEST, 0.f, 0.f};
    if (MASK) {
        const uint8_t *mask = a.mask + row * a.mask_stride;
        for (int w0 = tid - lane; w0 < a.words; w0 += LOGP_THREADS) {
            const int w = w0 + lane;
            const uint32_t bits = w < a.words ? legal_word(mask, a.n, w) : 0;
            if (a.bits && w < a.words) a.bits[row * a.words + w] = bits;
            // few legal places: each lane its own; many: the warp's words one after another, a lane per place
            if (__reduce_add_sync(ALL, __popc(bits)) <= 256) {
                add_bits(acc, x + 32 * w, bits);
            } else {
                for (int k = 0; k < 32; ++k) {
                    const uint32_t b = __shfl_sync(ALL, bits, k);
                    if (!b) continue;
                    float v[1] = {(b >> lane) & 1 ? to_f(x[32 * (w0 + k) + lane]) : -INFINITY};
                    acc.add(v);
                }
            }
        }
    } else {
        constexpr int VEC = 16 / sizeof(T);
        const int head = min(a.n, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
        const int packs = (a.n - head) / VEC;
        const Pack<T, VEC> *px = (const Pack<T, VEC> *)(x + head);
        for (int k = tid; k < packs; k += LOGP_THREADS) {
            const Pack<T, VEC> p = px[k];
            float v[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = to_f(p.v[i]);
            acc.add(v);
        }
        const int rest = a.n - packs * VEC;  // before the first pack and behind the last: at most 2 VEC - 2
        if (tid < rest) {
            float v[1] = {to_f(x[tid < head ? tid : tid + packs * VEC])};
            acc.add(v);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        acc.join(__shfl_xor_sync(ALL, acc.m, o), __shfl_xor_sync(ALL, acc.s, o), __shfl_xor_sync(ALL, acc.t, o));
    if (lane == 0) red[tid >> 5][0] = acc.m, red[tid >> 5][1] = acc.s, red[tid >> 5][2] = acc.t;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int i = 1; i < LOGP_THREADS / 32; ++i) acc.join(red[i][0], red[i][1], red[i][2]);
        const bool empty = acc.s == 0.f;
        const float logz = empty ? 0.f : logf(acc.s), inv = empty ? 0.f : 1.f / acc.s;
        const float h = empty ? 0.f : logz - acc.t * inv;
        const int act = a.act[row];
        float lp = 0.f;
        if (act >= 0 && act < a.n) {
            const bool legal = !MASK || a.mask[row * a.mask_stride + act] != 0;
            // -inf at the action's place gives -inf, NaN anywhere legal NaN
            lp = legal && !empty ? (to_f(x[act]) - acc.m) - logz : -INFINITY;
            if (acc.s != acc.s) lp = acc.s;
        }
        a.lp[row] = lp;
        a.ent[row] = h;
        if (a.stats) a.stats[row] = make_float4(acc.m, inv, logz, h);
    }
}

// Gradient: zeros over the row, then the legal places.
template <typename T, bool MASK>
__global__ void __launch_bounds__(LOGP_THREADS) logp_bwd_kernel(const LogpArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    pdl_enter();
    const int64_t row = blockIdx.x;
    const T *x = (const T *)a.x + row * a.x_stride;
    T *dx = (T *)a.dx + row * a.n;
    const int tid = threadIdx.x, lane = tid & 31;
    const float4 st = a.stats[row];  // m, 1 / Z, log Z, H
    const int act = a.act[row];
    const uint32_t *bits = MASK ? a.bits + row * a.words : nullptr;
    // the action's gradient: none without an action, or with one whose log-probability is -inf
    const bool taken = act >= 0 && act < a.n && (!MASK || is_legal(nullptr, bits, act)) && to_f(x[act]) != -INFINITY;
    const float u = taken && a.glp ? a.glp[row * a.glp_stride] : 0.f;
    const float v = a.gent ? a.gent[row * a.gent_stride] : 0.f;
    auto grad = [&](int j, float xj) {
        const float c = xj - st.x, p = ex2(c * LOG2E) * st.y;
        const float g = -p * (u + v * (c - st.z + st.w));
        return (p == 0.f ? 0.f : g) + (j == act ? u : 0.f);
    };
    const int head = min(a.n, (int)((16 - ((uintptr_t)dx & 15)) & 15) / (int)sizeof(T));
    const int packs = (a.n - head) / VEC, rest = a.n - packs * VEC;
    Pack<T, VEC> *pd = (Pack<T, VEC> *)(dx + head);
    if (MASK) {
        Pack<T, VEC> zero;
#pragma unroll
        for (int i = 0; i < VEC; ++i) zero.v[i] = from_f<T>(0.f);
        for (int k = tid; k < packs; k += LOGP_THREADS) pd[k] = zero;
        if (tid < rest) dx[tid < head ? tid : tid + packs * VEC] = zero.v[0];
        __syncthreads();
        for (int w0 = tid - lane; w0 < a.words; w0 += LOGP_THREADS) {
            const int w = w0 + lane;
            uint32_t b = w < a.words ? bits[w] : 0;
            if (__reduce_add_sync(ALL, __popc(b)) <= 256) {
                while (b) {
                    float g[4];
                    int at[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        at[i] = -1;
                        if (b) {
                            at[i] = 32 * w + __ffs(b) - 1;
                            b &= b - 1;
                            g[i] = to_f(x[at[i]]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (at[i] >= 0) dx[at[i]] = from_f<T>(grad(at[i], g[i]));
                }
            } else {
                for (int k = 0; k < 32; ++k) {
                    const uint32_t c = __shfl_sync(ALL, b, k);
                    const int j = 32 * (w0 + k) + lane;
                    if ((c >> lane) & 1) dx[j] = from_f<T>(grad(j, to_f(x[j])));
                }
            }
        }
    } else {
        const bool same = (((uintptr_t)x ^ (uintptr_t)dx) & 15) == 0;  // x's packs start where dx's do
        const Pack<T, VEC> *px = (const Pack<T, VEC> *)(x + head);
        for (int k = tid; k < packs; k += LOGP_THREADS) {
            const int j = head + k * VEC;
            Pack<T, VEC> p;
            if (same)
                p = px[k];
            else
#pragma unroll
                for (int i = 0; i < VEC; ++i) p.v[i] = x[j + i];
#pragma unroll
            for (int i = 0; i < VEC; ++i) p.v[i] = from_f<T>(grad(j + i, to_f(p.v[i])));
            pd[k] = p;
        }
        if (tid < rest) {
            const int j = tid < head ? tid : tid + packs * VEC;
            dx[j] = from_f<T>(grad(j, to_f(x[j])));
        }
    }
}

// ---------------------------------------------------------------------------
// Verification of drafted actions
// ---------------------------------------------------------------------------
// Place i of a game is kept while u_i q_i(a_i) < p_i(a_i), p the target's and
// q the draft's probabilities; at the first place that is not, the action is
// drawn from max(p - q, 0), after the last from p: the least j whose running
// sum exceeds r times the total.  The result is a whole number and borders
// have to fall the same way for everybody, so everything is in 64 bits.

constexpr int VERIFY_THREADS = 256, VERIFY_WARPS = VERIFY_THREADS / 32;
constexpr double RESIDUAL_MIN = 1.0 / (double)(1ull << 40);  // less left after a rejection counts as none

struct VerifyArgs {
    jq_drafts d;
    int32_t words;
};

struct VerifySmem {
    double red[2][2][VERIFY_WARPS];
    float redf[2][2][VERIFY_WARPS];
    double level[VERIFY_WARPS + 1];
    int last[VERIFY_WARPS];
    int pick;
};

// One row of logits and what its probabilities need.
struct Dist {
    float m;
    double z;
    bool any;   // a legal place above -inf
};

__device__ __forceinline__ double weight(float x, const Dist &d) {
    return d.any ? exp((double)x - (double)d.m) : x != x ? (double)x : 0.0;
}

template <typename T, bool MASK>
__global__ void __launch_bounds__(VERIFY_THREADS) verify_kernel(const VerifyArgs a) {
    extern __shared__ uint32_t bits[];  // MASK: the place's packed mask
    __shared__ VerifySmem sm;
    pdl_enter();
    const jq_drafts &d = a.d;
    const int game = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = d.actions, words = a.words;
    int len = d.lengths ? d.lengths[game] : d.drafts;
    len = len < 0 ? 0 : len > d.drafts ? d.drafts : len;
    int32_t *out = d.out_actions + (int64_t)game * (d.drafts + 1);
    float *out_lp = d.log_probs + (int64_t)game * (d.drafts + 1);
    int buf = 0;
    for (int i = 0;; ++i) {
        const T *x = (const T *)d.logits + game * d.logits_game + i * d.logits_place;
        const T *y = d.draft_logits && i < len
                         ? (const T *)d.draft_logits + game * d.draft_game + i * d.draft_place : nullptr;
        const uint8_t *mask = MASK ? d.mask + game * d.mask_game + i * d.mask_place : nullptr;
        __syncthreads();  // the last place's bits have been read
        if (MASK) {
            for (int w = tid; w < words; w += VERIFY_THREADS) bits[w] = legal_word(mask, n, w);
        }
        // every legal place of this thread: words tid, tid + 256, ..., or with no mask places tid, tid + 256, ...
        auto each = [&](auto &&f) {
            if (MASK) {
                for (int w = tid; w < words; w += VERIFY_THREADS)
                    for (uint32_t b = bits[w]; b; b &= b - 1) f(32 * w + __ffs(b) - 1);
            } else {
#pragma unroll 4
                for (int j = tid; j < n; j += VERIFY_THREADS) f(j);
            }
        };
        float mx = -INFINITY, my = -INFINITY;
        each([&](int j) {
            mx = fmaxf(mx, to_f(x[j]));
            if (y) my = fmaxf(my, to_f(y[j]));
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(ALL, mx, o));
            my = fmaxf(my, __shfl_xor_sync(ALL, my, o));
        }
        if (lane == 0) sm.redf[buf][0][warp] = mx, sm.redf[buf][1][warp] = my;
        __syncthreads();
        Dist p{sm.redf[buf][0][0], 0, false}, q{sm.redf[buf][1][0], 0, false};
        for (int k = 1; k < VERIFY_WARPS; ++k) p.m = fmaxf(p.m, sm.redf[buf][0][k]), q.m = fmaxf(q.m, sm.redf[buf][1][k]);
        p.any = p.m > -INFINITY, q.any = y && q.m > -INFINITY;
        double zx = 0, zy = 0;
        each([&](int j) {
            zx += weight(to_f(x[j]), p);
            if (y) zy += weight(to_f(y[j]), q);
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            zx += __shfl_xor_sync(ALL, zx, o);
            zy += __shfl_xor_sync(ALL, zy, o);
        }
        if (lane == 0) sm.red[buf][0][warp] = zx, sm.red[buf][1][warp] = zy;
        __syncthreads();
        for (int k = 0; k < VERIFY_WARPS; ++k) p.z += sm.red[buf][0][k], q.z += sm.red[buf][1][k];
        buf ^= 1;
        const bool broken = p.z != p.z || q.z != q.z;  // NaN or +inf at a legal place: no distribution
        const double logz = log(p.z);
        const int act = i < len ? d.drafted[(int64_t)game * d.drafts + i] : -1;
        if (act >= 0 && act < n && !broken && is_legal(nullptr, MASK ? bits : nullptr, act) && p.any) {
            const float xa = to_f(x[act]);
            const double pa = weight(xa, p) / p.z;
            const double qa = !d.draft_logits ? 1.0 : q.any ? weight(to_f(y[act]), q) / q.z : 0.0;
            if ((double)d.accept_u[(int64_t)game * d.drafts + i] * qa < pa) {
                if (tid == 0) out[i] = act, out_lp[i] = (float)(((double)xa - (double)p.m) - logz);
                continue;
            }
        }
        // place i is not kept (or i == len): draw here, and be done
        const bool bare = !d.draft_logits && i < len;  // q is one-hot at the drafted action
        const bool use_q = i < len && (bare ? act >= 0 && act < n : q.any);
        auto w_of = [&](int j, bool residual) {
            const double pj = weight(to_f(x[j]), p) / p.z;
            if (!residual) return pj;
            const double qj = bare ? (j == act ? 1.0 : 0.0) : weight(to_f(y[j]), q) / q.z;
            return pj > qj ? pj - qj : 0.0;
        };
        int next = -1;
        if (p.any && !broken) {
            float rf = d.sample_u[game];
            const double r = rf > 0.f ? (double)rf : 0.0;
            // a thread's share is consecutive, so that running sums follow the order of the actions
            const int units = MASK ? words : n, share = (units + VERIFY_THREADS - 1) / VERIFY_THREADS;
            const int u0 = min(units, tid * share), u1 = min(units, u0 + share);
            for (int pass = use_q ? 0 : 1; pass < 2; ++pass) {
                const bool residual = pass == 0;
                auto walk = [&](auto &&f) {
                    for (int u = u0; u < u1; ++u) {
                        if (MASK) {
                            for (uint32_t b = bits[u]; b; b &= b - 1) f(32 * u + __ffs(b) - 1);
                        } else {
                            f(u);
                        }
                    }
                };
                double part = 0;
                walk([&](int j) { part += w_of(j, residual); });
                double inc = part;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double v = __shfl_up_sync(ALL, inc, o);
                    if (lane >= o) inc += v;
                }
                __syncthreads();
                if (lane == 31) sm.level[warp] = inc;
                if (tid == 0) sm.pick = INT_MAX;
                __syncthreads();
                double before = 0, total = 0;
                for (int k = 0; k < VERIFY_WARPS; ++k) {
                    if (k < warp) before += sm.level[k];
                    total += sm.level[k];
                }
                if (residual && !(total > RESIDUAL_MIN)) continue;
                double lo = __shfl_up_sync(ALL, inc, 1);
                lo = before + (lane ? lo : 0.0);
                const double hi = before + inc, target = r * total;
                int last = -1;
                if (part > 0) {
                    double run = lo;
                    bool crossed = false;
                    walk([&](int j) {
                        const double w = w_of(j, residual);
                        run += w;
                        if (w > 0) {
                            if (!crossed) last = j;
                            if (run > target) crossed = true;
                        }
                    });
                    if (lo <= target && hi > target) atomicMin(&sm.pick, last);
                }
                __syncthreads();
                next = sm.pick;
                if (next == INT_MAX) {  // the point is at the total or beyond: the last place with weight
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(ALL, last, o));
                    if (lane == 0) sm.last[warp] = last;
                    __syncthreads();
                    next = -1;
                    for (int k = 0; k < VERIFY_WARPS; ++k) next = max(next, sm.last[k]);
                }
                break;
            }
        }
        if (tid == 0) {
            d.accepted[game] = i;
            out[i] = next;
            out_lp[i] = next >= 0 ? (float)(((double)to_f(x[next]) - (double)p.m) - logz)
                                  : broken ? __int_as_float(0x7fc00000) : 0.f;
        }
        for (int k = i + 1 + tid; k <= d.drafts; k += VERIFY_THREADS) out[k] = -1, out_lp[k] = 0.f;
        return;
    }
}

}  // namespace jq

using namespace jq;

extern "C" {

static int logp_check(const void *x, int64_t stride, int32_t dtype, int64_t rows, int32_t n) {
    if (!x || rows <= 0 || n <= 0) return fail(JQ_ERR_ARG, "action scores: at least one row of at least one action");
    if (!known_dtype(dtype)) return fail(JQ_ERR_ARG, "action scores: unknown dtype");
    if (rows > INT32_MAX) return fail(JQ_ERR_CAPACITY, "action scores: more than 2^31 - 1 rows");
    if (n > JQ_POLICY_MAX_ACTIONS) return fail(JQ_ERR_CAPACITY, "more actions than JQ_POLICY_MAX_ACTIONS");
    if (stride < 0) return fail(JQ_ERR_ARG, "action scores: negative row stride");
    if ((uintptr_t)x & (elem_size(dtype) - 1)) return fail(JQ_ERR_ARG, "action scores: logits are misaligned");
    return JQ_OK;
}

#define LOGP_LAUNCH(KERNEL, MASKED)                                                                             \
    do {                                                                                                        \
        cudaStream_t s = (cudaStream_t)stream;                                                                  \
        const unsigned g = (unsigned)rows;                                                                      \
        if (dtype == JQ_F32)                                                                                    \
            CU((MASKED) ? launch_pdl(KERNEL<float, true>, g, LOGP_THREADS, 0, s, a)                             \
                        : launch_pdl(KERNEL<float, false>, g, LOGP_THREADS, 0, s, a));                          \
        else if (dtype == JQ_F16)                                                                               \
            CU((MASKED) ? launch_pdl(KERNEL<__half, true>, g, LOGP_THREADS, 0, s, a)                            \
                        : launch_pdl(KERNEL<__half, false>, g, LOGP_THREADS, 0, s, a));                         \
        else                                                                                                    \
            CU((MASKED) ? launch_pdl(KERNEL<__nv_bfloat16, true>, g, LOGP_THREADS, 0, s, a)                     \
                        : launch_pdl(KERNEL<__nv_bfloat16, false>, g, LOGP_THREADS, 0, s, a));                  \
    } while (0)

int jq_action_log_prob(const void *d_logits, int64_t row_stride, int32_t dtype, const uint8_t *d_mask,
                       int64_t mask_stride, const int32_t *d_actions, int64_t rows, int32_t actions,
                       float *d_log_prob, float *d_entropy, float *d_stats, uint32_t *d_bits, void *stream) {
    int rc = logp_check(d_logits, row_stride, dtype, rows, actions);
    if (rc) return rc;
    if (!d_actions || !d_log_prob || !d_entropy) return fail(JQ_ERR_ARG, "action scores: actions or outputs missing");
    if (mask_stride < 0) return fail(JQ_ERR_ARG, "action scores: negative mask stride");
    if (((uintptr_t)d_actions | (uintptr_t)d_log_prob | (uintptr_t)d_entropy | (uintptr_t)d_bits) & 3 ||
        (uintptr_t)d_stats & 15)
        return fail(JQ_ERR_ARG, "action scores: an array is not aligned to its elements");
    LogpArgs a{};
    a.x = d_logits, a.mask = d_mask, a.bits = d_mask ? d_bits : nullptr, a.act = d_actions;
    a.lp = d_log_prob, a.ent = d_entropy, a.stats = (float4 *)d_stats;
    a.x_stride = row_stride, a.mask_stride = mask_stride, a.n = actions, a.words = (actions + 31) / 32;
    LOGP_LAUNCH(logp_fwd_kernel, d_mask);
    return JQ_OK;
}

int jq_action_log_prob_backward(const void *d_logits, int64_t row_stride, int32_t dtype, const uint32_t *d_bits,
                                const int32_t *d_actions, const float *d_stats, const float *d_grad_log_prob,
                                int64_t grad_log_prob_stride, const float *d_grad_entropy,
                                int64_t grad_entropy_stride, int64_t rows, int32_t actions, void *d_dlogits,
                                void *stream) {
    int rc = logp_check(d_logits, row_stride, dtype, rows, actions);
    if (rc) return rc;
    if (!d_actions || !d_stats || !d_dlogits) return fail(JQ_ERR_ARG, "action scores: actions, statistics or output missing");
    if (grad_log_prob_stride < 0 || grad_entropy_stride < 0) return fail(JQ_ERR_ARG, "action scores: negative stride");
    if (((uintptr_t)d_actions | (uintptr_t)d_bits | (uintptr_t)d_grad_log_prob | (uintptr_t)d_grad_entropy) & 3 ||
        (uintptr_t)d_stats & 15 || (uintptr_t)d_dlogits & (elem_size(dtype) - 1))
        return fail(JQ_ERR_ARG, "action scores: an array is not aligned to its elements");
    LogpArgs a{};
    a.x = d_logits, a.bits = const_cast<uint32_t *>(d_bits), a.act = d_actions;
    a.stats = (float4 *)const_cast<float *>(d_stats), a.glp = d_grad_log_prob, a.gent = d_grad_entropy;
    a.glp_stride = grad_log_prob_stride, a.gent_stride = grad_entropy_stride, a.dx = d_dlogits;
    a.x_stride = row_stride, a.n = actions, a.words = (actions + 31) / 32;
    LOGP_LAUNCH(logp_bwd_kernel, d_bits);
    return JQ_OK;
}

int jq_verify_drafts(const jq_drafts *d, void *stream) {
    if (!d || d->games <= 0 || d->drafts < 0) return fail(JQ_ERR_ARG, "drafts: at least one game");
    int rc = logp_check(d->logits, 0, d->dtype, d->games, d->actions);
    if (rc) return rc;
    if (d->drafts > JQ_POLICY_MAX_DRAFTS) return fail(JQ_ERR_CAPACITY, "more drafts than JQ_POLICY_MAX_DRAFTS");
    if (!d->sample_u || !d->accepted || !d->out_actions || !d->log_probs ||
        (d->drafts > 0 && (!d->drafted || !d->accept_u)))
        return fail(JQ_ERR_ARG, "drafts: inputs or outputs missing");
    if (d->logits_game < 0 || d->logits_place < 0 || d->draft_game < 0 || d->draft_place < 0 || d->mask_game < 0 ||
        d->mask_place < 0)
        return fail(JQ_ERR_ARG, "drafts: negative stride");
    if (((uintptr_t)d->drafted | (uintptr_t)d->lengths | (uintptr_t)d->accept_u | (uintptr_t)d->sample_u |
         (uintptr_t)d->accepted | (uintptr_t)d->out_actions | (uintptr_t)d->log_probs) & 3 ||
        (uintptr_t)d->draft_logits & (elem_size(d->dtype) - 1))
        return fail(JQ_ERR_ARG, "drafts: an array is not aligned to its elements");
    VerifyArgs a{*d, (d->actions + 31) / 32};
    const bool masked = d->mask != nullptr;
    const size_t smem = masked ? 4 * (size_t)a.words : 0;
    const unsigned g = (unsigned)d->games;
    cudaStream_t s = (cudaStream_t)stream;
    if (d->dtype == JQ_F32)
        CU(masked ? launch_pdl(verify_kernel<float, true>, g, VERIFY_THREADS, smem, s, a)
                  : launch_pdl(verify_kernel<float, false>, g, VERIFY_THREADS, smem, s, a));
    else if (d->dtype == JQ_F16)
        CU(masked ? launch_pdl(verify_kernel<__half, true>, g, VERIFY_THREADS, smem, s, a)
                  : launch_pdl(verify_kernel<__half, false>, g, VERIFY_THREADS, smem, s, a));
    else
        CU(masked ? launch_pdl(verify_kernel<__nv_bfloat16, true>, g, VERIFY_THREADS, smem, s, a)
                  : launch_pdl(verify_kernel<__nv_bfloat16, false>, g, VERIFY_THREADS, smem, s, a));
    return JQ_OK;
}

}  // extern "C"
