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
#include <math.h>

#include <atomic>

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
//
// The places of a game are worked on at the same time, up to 8 of them, and
// the first that is not kept then draws: a game's chain is one place and one
// draw, whatever its drafts.  That reads places behind the first rejection in
// vain, but a game that goes place by place takes as long as its longest
// chain, and the others wait for it.
//
// That is with a mask, where a place is one warp's: it packs the mask, lists
// the legal actions in order, and does the rest on the list without a barrier;
// what bounds it is the mask's bytes (with many games) or the chain of some
// thousand cycles (with few).  Without a mask the bound is the exponentials in
// 64 bits (verify_dense_kernel).

constexpr double RESIDUAL_MIN = 1.0 / (double)(1ull << 40);  // less left after a rejection counts as none
constexpr int PLACES = 8;      // of a game at the same time
constexpr int LIST = 320;      // legal actions of a place's list; with more, the packed mask is walked instead

struct VerifyArgs {
    jq_drafts d;
    int32_t games_per_cta;  // masked: a game per warp, with no drafts; else 1
    int32_t share;          // masked: bytes of shared memory of a warp
};

// e^d for d <= 0 in 64 bits: d = k ln 2 / 16 + r, e^d = 2^(k / 16) e^r, from a
// table of 16 and five terms of the series (Tang's table-driven exponential,
// ACM TOMS 1989); |r| <= 0.0217, so the sixth is below 1.5e-13.  Below -700: 0.
// Ten operations, where the library's function has about three times that:
// without a mask they are the kernel's bound.  16 entries, because they lie in
// banks of their own.
constexpr int EXP_STEPS = 16;
__device__ __forceinline__ double exp_table(int i) { return exp2((double)i / EXP_STEPS); }
__device__ __forceinline__ double exp_neg(double d, const double *table) {
    constexpr double MAGIC = 1.5 * 4503599627370496.0;  // 1.5 * 2^52: a sum's last bit is 1
    constexpr double PER = EXP_STEPS * 1.4426950408889634, LN = 0.69314718055994531 / EXP_STEPS;
    const double near = fma(d, PER, MAGIC);
    const int k = __double2loint(near);
    const double r = fma(near - MAGIC, -LN, d);
    const double e = r * fma(r, fma(r, fma(r, fma(r, 1.0 / 120, 1.0 / 24), 1.0 / 6), 0.5), 1.0);
    const double at = table[k & (EXP_STEPS - 1)];
    const double v = fma(at, e, at);
    static_assert(EXP_STEPS == 16, "k >> 4");
    const double scaled = __hiloint2double(__double2hiint(v) + ((k >> 4) << 20), __double2loint(v));
    return d < -700.0 ? 0.0 : d == d ? scaled : d;
}

// One row of logits and what its probabilities need.
struct Dist {
    double m, z, iz; // the largest logit, Z and its reciprocal
    bool any;        // a legal place above -inf
    __device__ __forceinline__ double weight(float x, const double *table) const {  // exp(x - m)
        return any ? exp_neg((double)x - m, table) : x != x ? (double)x : 0.0;
    }
    __device__ __forceinline__ void start(float top, bool there) {
        any = there && top > -INFINITY;
        m = top, z = iz = 0;
    }
    __device__ __forceinline__ bool broken() const { return z != z; }  // NaN or +inf at a legal place
};

// What a place is, and whether its draft is kept.
template <typename T>
struct Place {
    const T *x, *y;       // logits; of the draft, or NULL
    const uint8_t *mask;
    int act;              // the drafted action; -1 behind the last
    bool drafted;         // i < len
    float u;
    Dist p, q;
    __device__ __forceinline__ Place(const jq_drafts &d, int game, int i, int len)
        : x((const T *)d.logits + game * d.logits_game + i * d.logits_place), y(nullptr),
          mask(d.mask ? d.mask + game * d.mask_game + i * d.mask_place : nullptr), act(-1), drafted(i < len), u(0.f) {
        if (drafted) {
            act = d.drafted[(int64_t)game * d.drafts + i];
            u = d.accept_u[(int64_t)game * d.drafts + i];
            if (d.draft_logits) y = (const T *)d.draft_logits + game * d.draft_game + i * d.draft_place;
        }
        if (act >= d.actions) act = -1;
    }
    __device__ __forceinline__ bool broken() const { return p.broken() || q.broken(); }
    __device__ __forceinline__ bool kept(bool legal, const double *table) const {
        if (act < 0 || !legal || broken() || !p.any) return false;
        const double pa = p.weight(to_f(x[act]), table) * p.iz;
        const double qa = !y ? 1.0 : q.any ? q.weight(to_f(y[act]), table) * q.iz : 0.0;
        return (double)u * qa < pa;
    }
    // the distribution that is drawn from: max(p - q, 0) while `residual`, else p
    __device__ __forceinline__ bool has_residual() const { return drafted && (y ? q.any : act >= 0); }
    __device__ __forceinline__ double draw_weight(int j, float xj, float yj, bool residual, const double *table) const {
        const double pj = p.weight(xj, table) * p.iz;
        if (!residual) return pj;
        const double qj = y ? q.weight(yj, table) * q.iz : j == act ? 1.0 : 0.0;
        return pj > qj ? pj - qj : 0.0;
    }
    __device__ __forceinline__ double draw_weight(int j, bool residual, const double *table) const {
        return draw_weight(j, to_f(x[j]), y && residual ? to_f(y[j]) : 0.f, residual, table);
    }
    __device__ __forceinline__ float log_prob(int j) const {  // in 64 bits, rounded once
        return (float)(((double)to_f(x[j]) - p.m) - log(p.z));
    }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(ALL, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(ALL, v, o));
    return v;
}
__device__ __forceinline__ double warp_scan(double v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_up_sync(ALL, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Bits of 16 mask bytes: bytes of 0 and 1 are dot products with powers of two.
__device__ __forceinline__ uint32_t pack_block(uint4 v) {
    if ((v.x | v.y | v.z | v.w) & 0xfefefefeu)  // other truth values
        v = make_uint4(__vminu4(v.x, 0x01010101u), __vminu4(v.y, 0x01010101u), __vminu4(v.z, 0x01010101u), __vminu4(v.w, 0x01010101u));
    const uint32_t lo = __dp4a(v.y, 0x80402010u, __dp4a(v.x, 0x08040201u, 0u));
    const uint32_t hi = __dp4a(v.w, 0x80402010u, __dp4a(v.z, 0x08040201u, 0u));
    return lo | hi << 8;
}

// A row's mask in bits, in blocks of 16 bytes as they lie in memory: bit
// (row & 15) + j for place j; by a warp, eight loads in flight a lane.  Blocks
// with legal places go to `found` too, in order, as block << 16 | bits, as
// long as there are at most `most`; their number is returned.
__device__ __forceinline__ int pack_mask(uint16_t *bits, uint32_t *found, int most, const uint8_t *row, int places, int lane) {
    constexpr int AHEAD = 8;
    const int skip = (int)((uintptr_t)row & 15), blocks = (skip + places + 15) >> 4;
    const uint8_t *first = row - skip;
    const int k0 = skip ? 1 : 0, k1 = (skip + places) >> 4;  // whole blocks of the row
    // the row's ends, a byte per lane, and the last word's upper half
    const int ke = lane < 16 ? 0 : blocks - 1, je = 16 * ke + (lane & 15) - skip;
    const bool end = lane < 16 ? k0 > 0 || k1 == 0 : k1 < blocks && blocks > 1;
    const uint32_t ends = __ballot_sync(ALL, end && je >= 0 && je < places && row[je] != 0);
    if ((lane & 15) == 0 && end) bits[ke] = (uint16_t)(lane ? ends >> 16 : ends);
    if (lane == 0 && (blocks & 1)) bits[blocks] = 0;
    int n = 0;
    if (ends & 0xffff) {
        if (lane == 0) found[0] = ends & 0xffff;
        n = 1;
    }
    for (int b0 = k0; b0 < k1; b0 += 32 * AHEAD) {
        uint4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int k = b0 + 32 * i + lane;
            v[i] = make_uint4(0, 0, 0, 0);
            if (k < k1) v[i] = *(const uint4 *)(first + 16 * k);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int k = b0 + 32 * i + lane;
            const uint32_t b = pack_block(v[i]);
            if (k < k1) bits[k] = (uint16_t)b;
            const uint32_t some = __ballot_sync(ALL, b != 0);
            if (b) {
                const int at = n + __popc(some & ((1u << lane) - 1));
                if (at < most) found[at] = (uint32_t)k << 16 | b;
            }
            n += __popc(some);
        }
    }
    if (ends >> 16) {
        if (lane == 0 && n < most) found[n] = (uint32_t)(blocks - 1) << 16 | ends >> 16;
        ++n;
    }
    return n;
}

template <typename T>
__global__ void __launch_bounds__(32 * PLACES, 4) verify_masked_kernel(const VerifyArgs a) {
    extern __shared__ __align__(16) char verify_smem[];
    __shared__ double table[EXP_STEPS];
    __shared__ int keeps[2][PLACES];
    const jq_drafts &d = a.d;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, n = d.actions;
    for (int i = threadIdx.x; i < EXP_STEPS; i += blockDim.x) table[i] = exp_table(i);
    pdl_enter();
    __syncthreads();
    int *list = (int *)(verify_smem + warp * a.share);     // the legal actions in order, their logits, the draft's
    float *lx = (float *)(list + LIST), *ly = lx + LIST;
    uint32_t *bits = (uint32_t *)(ly + LIST);
    const bool alone = a.games_per_cta > 1;  // a game is this warp's, and has one place
    const int game = alone ? blockIdx.x * a.games_per_cta + warp : blockIdx.x;
    if (game >= d.games) return;             // (alone: no barrier follows)
    int len = d.lengths ? d.lengths[game] : d.drafts;
    len = len < 0 ? 0 : len > d.drafts ? d.drafts : len;
    int32_t *out = d.out_actions + (int64_t)game * (d.drafts + 1);
    float *out_lp = d.log_probs + (int64_t)game * (d.drafts + 1);
    for (int base = 0, round = 0;; base += warps, round ^= 1) {
        const int i = alone ? 0 : base + warp;
        const bool active = i <= len;
        bool kept = false;
        Place<T> at(d, game, active ? i : len, len);
        int count = 0, lo = 0, hi = 0;
        const int skip = (int)((uintptr_t)at.mask & 15), words = (skip + n + 31) >> 5;
        const int share = (words + 31) >> 5, w0 = min(words, lane * share), w1 = min(words, w0 + share);
        // this lane's legal actions, consecutive ones, with their logits: of the list, or of the packed mask
        auto each = [&](auto &&f) {
            if (count <= LIST) {
                for (int k = lo; k < hi; ++k) f(list[k], lx[k], ly[k]);
            } else {
                for (int w = w0; w < w1; ++w)
                    for (uint32_t b = bits[w]; b; b &= b - 1) {
                        const int j = 32 * w + __ffs(b) - 1 - skip;
                        f(j, to_f(at.x[j]), at.y ? to_f(at.y[j]) : 0.f);
                    }
            }
        };
        if (active) {
            __syncwarp();
            uint32_t *found = (uint32_t *)lx;
            const int blocks = pack_mask((uint16_t *)bits, found, LIST, at.mask, n, lane);
            __syncwarp();
            // this lane's legal places: of its share of the blocks that have some, or of the words
            const bool few = blocks <= LIST;
            const int per_lane = (blocks + 31) >> 5, e0 = min(blocks, lane * per_lane), e1 = min(blocks, e0 + per_lane);
            int before = 0;
            if (few)
                for (int e = e0; e < e1; ++e) before += __popc(found[e] & 0xffff);
            else
                for (int w = w0; w < w1; ++w) before += __popc(bits[w]);
            const int own = before;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(ALL, before, o);
                if (lane >= o) before += u;
            }
            count = __shfl_sync(ALL, before, 31);
            before -= own;
            if (count <= LIST) {
                for (int e = e0; e < e1; ++e) {
                    const int j0 = (int)(found[e] >> 16) * 16 - skip;
                    for (uint32_t b = found[e] & 0xffff; b; b &= b - 1) list[before++] = j0 + __ffs(b) - 1;
                }
                const int per = (count + 31) >> 5;
                lo = min(count, lane * per), hi = min(count, lo + per);
                __syncwarp();
                for (int k0 = 0; k0 < count; k0 += 128) {  // four scattered logits of each in flight
                    float vx[4], vy[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k = k0 + 32 * i + lane;
                        if (k < count) {
                            vx[i] = to_f(at.x[list[k]]);
                            if (at.y) vy[i] = to_f(at.y[list[k]]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k = k0 + 32 * i + lane;
                        if (k < count) lx[k] = vx[i], ly[k] = at.y ? vy[i] : 0.f;
                    }
                }
                __syncwarp();
            }
            float mx = -INFINITY, my = -INFINITY;
            each([&](int, float x, float y) { mx = fmaxf(mx, x), my = fmaxf(my, y); });
            at.p.start(warp_max(mx), true);
            at.q.start(warp_max(my), at.y != nullptr);
            double zx = 0, zy = 0;
            each([&](int, float x, float y) {
                zx += at.p.weight(x, table);
                if (at.y) zy += at.q.weight(y, table);
            });
            at.p.z = warp_sum(zx), at.q.z = warp_sum(zy);
            at.p.iz = 1.0 / at.p.z, at.q.iz = 1.0 / at.q.z;
            const int b = at.act + skip;
            kept = at.kept(at.act >= 0 && ((bits[b >> 5] >> (b & 31)) & 1), table);
        }
        int first = alone ? 0 : warps;  // the first place of this round that is not kept
        if (!alone) {
            if (lane == 0) keeps[round][warp] = kept;
            __syncthreads();
            for (int k = warps - 1; k >= 0; --k)
                if (!keeps[round][k]) first = k;
            if (kept && warp < first && lane == 0) out[i] = at.act, out_lp[i] = at.log_prob(at.act);
            if (first == warps) continue;
            if (warp != first) return;
        }
        int next = -1;
        if (at.p.any && !at.broken()) {
            const float rf = d.sample_u[game];
            const double r = rf > 0.f ? (double)rf : 0.0;
            for (int pass = at.has_residual() ? 0 : 1; pass < 2; ++pass) {
                const bool residual = pass == 0;
                double part = 0;
                each([&](int j, float x, float y) { part += at.draw_weight(j, x, y, residual, table); });
                const double above = warp_scan(part, lane), total = __shfl_sync(ALL, above, 31);
                if (residual && !(total > RESIDUAL_MIN)) continue;
                const double up = __shfl_up_sync(ALL, above, 1), below = lane ? up : 0.0, target = r * total;
                // the first lane whose running sum is above the point; with none, the last that has weight
                const unsigned cross = __ballot_sync(ALL, part > 0 && above > target), some = __ballot_sync(ALL, part > 0);
                const int who = cross ? __ffs(cross) - 1 : 31 - __clz(some);
                if (lane == who) {
                    double run = below;
                    bool crossed = false;
                    each([&](int j, float x, float y) {
                        const double w = at.draw_weight(j, x, y, residual, table);
                        run += w;
                        if (w > 0 && !crossed) next = j, crossed = run > target;
                    });
                }
                next = __shfl_sync(ALL, next, who);
                break;
            }
        }
        if (lane == 0) {
            d.accepted[game] = i;
            out[i] = next;
            out_lp[i] = next >= 0 ? at.log_prob(next) : at.broken() ? __int_as_float(0x7fc00000) : 0.f;
        }
        for (int k = i + 1 + lane; k <= d.drafts; k += 32) out[k] = -1, out_lp[k] = 0.f;
        return;
    }
}

// Without a mask: a cluster per game, each CTA a consecutive share of every
// row.  Place by place, since a place is enough work for the whole cluster:
// no row behind the first rejection is read.
constexpr int DENSE_THREADS = 256, DENSE_WARPS = DENSE_THREADS / 32, DENSE_CTAS = 8;

// Every logit of x[0, n), by the CTA: 8 bytes a load, the ends one by one.
template <typename T, typename F>
__device__ __forceinline__ void dense_each(const T *x, int n, int tid, F &&f) {
    constexpr int VEC = 8 / sizeof(T);
    const int head = min(n, (int)((8 - ((uintptr_t)x & 7)) & 7) / (int)sizeof(T)), packs = (n - head) / VEC;
    const Pack<T, VEC> *px = (const Pack<T, VEC> *)(x + head);
    int k = tid;
    for (; k + 3 * DENSE_THREADS < packs; k += 4 * DENSE_THREADS) {
        Pack<T, VEC> p[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) p[u] = px[k + u * DENSE_THREADS];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) f(to_f(p[u].v[i]));
    }
    for (; k < packs; k += DENSE_THREADS) {
        const Pack<T, VEC> p = px[k];
#pragma unroll
        for (int i = 0; i < VEC; ++i) f(to_f(p.v[i]));
    }
    const int rest = n - packs * VEC;  // before the first pack and behind the last
    if (tid < rest) f(to_f(x[tid < head ? tid : tid + packs * VEC]));
}

// Sum of exp(x - m) over this thread's logits of x[0, n).
template <typename T>
__device__ __forceinline__ double dense_sum(const T *x, int n, int tid, const Dist &d, const double *table) {
    double z = 0;
    if (d.any)
        dense_each(x, n, tid, [&](float v) { z += exp_neg((double)v - d.m, table); });
    else
        dense_each(x, n, tid, [&](float v) { z += v != v ? (double)v : 0.0; });
    return z;
}

struct DenseSmem {
    double table[EXP_STEPS];
    double sums[2][DENSE_WARPS], level[DENSE_WARPS];
    float tops[2][DENSE_WARPS];
    double told[2][DENSE_CTAS][4];  // what the game's CTAs tell each other: two rounds' m, Z of the target, m, Z of the draft
    int pick;
};

template <typename T>
__global__ void __launch_bounds__(DENSE_THREADS, 4) verify_dense_kernel(const VerifyArgs a) {
    __shared__ DenseSmem sm;
    const jq_drafts &d = a.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = d.actions;
    const int rank = (int)cluster_rank(), ranks = (int)cluster_size(), game = blockIdx.x / ranks;
    if (tid < EXP_STEPS) sm.table[tid] = exp_table(tid);
    const double *table = sm.table;
    pdl_enter();
    cluster_sync();  // the game's CTAs have all started: their shared memory may be written
    int len = d.lengths ? d.lengths[game] : d.drafts;
    len = len < 0 ? 0 : len > d.drafts ? d.drafts : len;
    int32_t *out = d.out_actions + (int64_t)game * (d.drafts + 1);
    float *out_lp = d.log_probs + (int64_t)game * (d.drafts + 1);
    const int all = ((n + ranks - 1) / ranks + 31) & ~31, s0 = min(n, rank * all), s1 = min(n, s0 + all);
    int round = 0;
    // `v` (of thread 0) of every CTA to every CTA, as told[round][rank][at]
    auto tell = [&](int at, double v) {
        for (int k = 0; k < ranks; ++k) cluster_store(&sm.told[round][rank][at], k, v);
    };
    for (int i = 0;; ++i) {
        Place<T> at(d, game, i, len);
        {
            float mx = -INFINITY, my = -INFINITY;
            dense_each(at.x + s0, s1 - s0, tid, [&](float v) { mx = fmaxf(mx, v); });
            if (at.y) dense_each(at.y + s0, s1 - s0, tid, [&](float v) { my = fmaxf(my, v); });
            mx = warp_max(mx), my = warp_max(my);
            __syncthreads();
            if (lane == 0) sm.tops[0][warp] = mx, sm.tops[1][warp] = my;
            __syncthreads();
            for (int k = 0; k < DENSE_WARPS; ++k) mx = fmaxf(mx, sm.tops[0][k]), my = fmaxf(my, sm.tops[1][k]);
            at.p.start(mx, true), at.q.start(my, at.y != nullptr);
            double zx = dense_sum(at.x + s0, s1 - s0, tid, at.p, table);
            double zy = at.y ? dense_sum(at.y + s0, s1 - s0, tid, at.q, table) : 0.0;
            zx = warp_sum(zx), zy = warp_sum(zy);
            if (lane == 0) sm.sums[0][warp] = zx, sm.sums[1][warp] = zy;
            __syncthreads();
            for (int k = 0; k < DENSE_WARPS; ++k) at.p.z += sm.sums[0][k], at.q.z += sm.sums[1][k];
            if (ranks > 1) {
                if (tid == 0) tell(0, at.p.m), tell(1, at.p.z), tell(2, at.q.m), tell(3, at.q.z);
                cluster_sync();
                double m[2] = {-INFINITY, -INFINITY}, z[2] = {0, 0};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    for (int k = 0; k < ranks; ++k) m[h] = fmax(m[h], sm.told[round][k][2 * h]);
                    for (int k = 0; k < ranks; ++k) {
                        const double mk = sm.told[round][k][2 * h], zk = sm.told[round][k][2 * h + 1];
                        z[h] += mk > -INFINITY ? zk * exp_neg(mk - m[h], table) : zk;  // (a share of -inf has Z = 0 or NaN)
                    }
                }
                round ^= 1;
                at.p.start((float)m[0], true), at.q.start((float)m[1], at.y != nullptr);
                at.p.z = z[0], at.q.z = z[1];
            }
            at.p.iz = 1.0 / at.p.z, at.q.iz = 1.0 / at.q.z;
        }
        if (at.kept(true, table)) {  // the same for the whole game: all its CTAs have the same numbers
            if (rank == 0 && tid == 0) out[i] = at.act, out_lp[i] = at.log_prob(at.act);
            continue;
        }
        int next = -1;
        bool mine = rank == 0;  // whose share holds the point
        if (at.p.any && !at.broken()) {
            const float rf = d.sample_u[game];
            const double r = rf > 0.f ? (double)rf : 0.0;
            // the first of `count` whose running sum exceeds the point, or the last that has weight; `below`: the sum before it
            auto find = [&](int count, auto &&weight, double &below, double target) {
                double run = below, before = below;
                int last = 0;
                for (int k = 0; k < count; ++k) {
                    const double w = weight(k);
                    if (w > 0) {
                        last = k, before = run;
                        if (run + w > target) break;
                    }
                    run += w;
                }
                below = before;
                return last;
            };
            // weights of [from, from + share), [from + share, ...): a warp's each
            auto shares = [&](int from, int to, int share, bool residual) {
                const int w0 = min(to, from + warp * share), w1 = min(to, w0 + share);
                double part = 0;
                if (residual && at.y) {
#pragma unroll 4
                    for (int j = w0 + lane; j < w1; j += 32) {
                        const double pj = exp_neg((double)to_f(at.x[j]) - at.p.m, table) * at.p.iz;
                        const double qj = exp_neg((double)to_f(at.y[j]) - at.q.m, table) * at.q.iz;
                        part += fmax(pj - qj, 0.0);
                    }
                } else {
#pragma unroll 4
                    for (int j = w0 + lane; j < w1; j += 32) part += at.draw_weight(j, residual, table);
                }
                part = warp_sum(part);
                __syncthreads();
                if (lane == 0) sm.level[warp] = part;
                __syncthreads();
            };
            for (int pass = at.has_residual() ? 0 : 1; pass < 2; ++pass) {
                const bool residual = pass == 0;
                int from = s0, to = s1, share = ((to - from + DENSE_WARPS - 1) / DENSE_WARPS + 31) & ~31;
                shares(from, to, share, residual);
                double total = 0, below = 0;
                for (int k = 0; k < DENSE_WARPS; ++k) total += sm.level[k];
                if (ranks > 1) {
                    if (tid == 0) tell(0, total);
                    cluster_sync();
                    total = 0;
                    for (int k = 0; k < ranks; ++k) total += sm.told[round][k][0];
                }
                const double target = r * total;
                if (residual && !(total > RESIDUAL_MIN)) {
                    round ^= 1;
                    continue;
                }
                if (ranks > 1) mine = find(ranks, [&](int k) { return sm.told[round][k][0]; }, below, target) == rank;
                if (!mine) break;
                // an eighth of the share, of that an eighth, and so on
                for (;;) {
                    const int who = find(DENSE_WARPS, [&](int k) { return sm.level[k]; }, below, target);
                    from = min(to, from + who * share), to = min(to, from + share);
                    if (to - from <= 32) break;
                    share = ((to - from + DENSE_WARPS - 1) / DENSE_WARPS + 31) & ~31;
                    shares(from, to, share, residual);
                }
                if (warp == 0) {
                    const int j = from + lane;
                    const double w = j < to ? at.draw_weight(j, residual, table) : 0.0;
                    const double above = warp_scan(w, lane);
                    const unsigned cross = __ballot_sync(ALL, w > 0 && below + above > target), some = __ballot_sync(ALL, w > 0);
                    if (lane == 0) sm.pick = from + (cross ? __ffs(cross) - 1 : some ? 31 - __clz(some) : 0);
                }
                __syncthreads();
                next = sm.pick;
                break;
            }
        }
        if (!mine) return;
        if (tid == 0) {
            d.accepted[game] = i;
            out[i] = next;
            out_lp[i] = next >= 0 ? at.log_prob(next) : at.broken() ? __int_as_float(0x7fc00000) : 0.f;
        }
        for (int k = i + 1 + tid; k <= d.drafts; k += DENSE_THREADS) out[k] = -1, out_lp[k] = 0.f;
        return;
    }
}

template <typename T>
static int verify_launch(const jq_drafts &d, cudaStream_t s) {
    VerifyArgs a{d, 1, 0};
    if (!d.mask) {
        int sms, rc = device_sms(sms);
        if (rc) return rc;
        // enough CTAs for all SMs, several of which wait for one another's answers meanwhile, of a thousand places or more
        int ctas = 1;
        while (ctas < DENSE_CTAS && (int64_t)d.games * ctas < 6 * (int64_t)sms && d.actions > 1024 * ctas) ctas *= 2;
        if ((int64_t)d.games * ctas > INT32_MAX) return fail(JQ_ERR_CAPACITY, "drafts: too many games for one call");
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)d.games * ctas);
        cfg.blockDim = dim3(DENSE_THREADS);
        cfg.stream = s;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr, cfg.numAttrs = 2;
        CU(cudaLaunchKernelEx(&cfg, verify_dense_kernel<T>, a));
        return JQ_OK;
    }
    a.share = 4 * (3 * LIST + (d.actions + 15 + 31) / 32 + 1);
    a.share = (a.share + 15) & ~15;
    int warps = d.drafts + 1 < PLACES ? d.drafts + 1 : PLACES;
    if (d.drafts == 0) warps = a.games_per_cta = 4;
    while (warps > 1 && (size_t)warps * a.share > 200 * 1024) --warps;
    if (d.drafts == 0) a.games_per_cta = warps;
    const size_t smem = (size_t)warps * a.share;
    if (smem > 40 * 1024) {
        static std::atomic<uint64_t> raised{0};
        int dev = 0;
        CU(cudaGetDevice(&dev));
        const uint64_t bit = 1ull << (dev & 63);
        if (!(raised.load(std::memory_order_relaxed) & bit)) {
            CU(cudaFuncSetAttribute(verify_masked_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 210 * 1024));
            raised.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    const unsigned g = (unsigned)((d.games + a.games_per_cta - 1) / a.games_per_cta);
    CU(launch_pdl(verify_masked_kernel<T>, g, 32 * warps, smem, s, a));
    return JQ_OK;
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
    cudaStream_t s = (cudaStream_t)stream;
    if (d->dtype == JQ_F32) return verify_launch<float>(*d, s);
    if (d->dtype == JQ_F16) return verify_launch<__half>(*d, s);
    return verify_launch<__nv_bfloat16>(*d, s);
}

}  // extern "C"
