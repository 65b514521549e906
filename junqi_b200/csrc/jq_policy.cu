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

// Bits of 16 mask bytes, each 0 or 1: dot products with powers of two.
__device__ __forceinline__ uint32_t pack_block(uint4 v) {
    const uint32_t lo = __dp4a(v.y, 0x80402010u, __dp4a(v.x, 0x08040201u, 0u));
    const uint32_t hi = __dp4a(v.w, 0x80402010u, __dp4a(v.z, 0x08040201u, 0u));
    return lo + hi * 256;
}
__device__ __forceinline__ uint4 ones(uint4 v) {  // other truth values
    return make_uint4(__vminu4(v.x, 0x01010101u), __vminu4(v.y, 0x01010101u), __vminu4(v.z, 0x01010101u), __vminu4(v.w, 0x01010101u));
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
    const uint32_t lower = (1u << lane) - 1;
    for (int b0 = k0; b0 < k1; b0 += 32 * AHEAD) {
        const uint8_t *from = first + 16 * (b0 + lane);
        const int left = k1 - b0 - lane;
        uint4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            v[i] = make_uint4(0, 0, 0, 0);
            if (32 * i < left) v[i] = *(const uint4 *)(from + 512 * i);
        }
        uint32_t odd = 0;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) odd |= v[i].x | v[i].y | v[i].z | v[i].w;
        if (__any_sync(ALL, odd & 0xfefefefeu))
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) v[i] = ones(v[i]);
        uint16_t *to = bits + b0 + lane;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const uint32_t b = pack_block(v[i]);
            if (32 * i < left) to[32 * i] = (uint16_t)b;
            const uint32_t some = __ballot_sync(ALL, b != 0);
            const int at = n + __popc(some & lower);
            if (b && at < most) found[at] = (uint32_t)(b0 + 32 * i + lane) << 16 | b;
            n += __popc(some);
        }
    }
    if (ends >> 16) {
        if (lane == 0 && n < most) found[n] = (uint32_t)(blocks - 1) << 16 | ends >> 16;
        ++n;
    }
    return n;
}

// A row's legal places, by a warp in its shared memory: the packed mask, and
// the blocks of 16 that have some, as block << 16 | bits, as long as there are
// at most `most` (with more, only the packed mask counts).
constexpr int BLOCKS = 512;  // of the log-probability: 36 warps on an SM
constexpr int LIST = 320;    // of the verification, and the places of its list: 24 warps, as by registers
struct Legal {
    uint32_t *found, *bits;
    int most, blocks, skip, words;
    __device__ __forceinline__ Legal(char *bits, void *found, int most) : found((uint32_t *)found), bits((uint32_t *)bits), most(most) {}
    static size_t bytes(int places) { return (4 * ((places + 15 + 31) / 32 + 1) + 15) & ~(size_t)15; }  // of `bits`
    __device__ __forceinline__ void read(const uint8_t *mask, int places, int lane) {
        skip = (int)((uintptr_t)mask & 15), words = (skip + places + 31) >> 5;
        __syncwarp();  // the last row's has been read
        blocks = pack_mask((uint16_t *)bits, found, most, mask, places, lane);
        __syncwarp();
    }
    // The places in order, as far as there are at most LIST, and their number.
    __device__ __forceinline__ int list(int *to, int lane) const {
        // this lane's: of its share of the blocks that have some, or of the words
        const bool few = blocks <= most;
        const int share = ((few ? blocks : words) + 31) >> 5, e0 = lane * share, e1 = min(few ? blocks : words, e0 + share);
        int before = 0;
        for (int e = e0; e < e1; ++e) before += __popc(few ? found[e] & 0xffff : bits[e]);
        const int own = before;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(ALL, before, o);
            if (lane >= o) before += u;
        }
        const int count = __shfl_sync(ALL, before, 31);  // (`most` is LIST: more blocks than that have more places, too)
        before -= own;
        if (count <= LIST)
            for (int e = e0; e < e1; ++e) {
                const int j0 = (int)(found[e] >> 16) * 16 - skip;
                for (uint32_t b = found[e] & 0xffff; b; b &= b - 1) to[before++] = j0 + __ffs(b) - 1;
            }
        __syncwarp();
        return count;
    }
    // The next ones in order from word w on, whole words of them, at most LIST places, and their number; w: behind them.
    // (With more than LIST legal actions the list holds a part of them at a time, for the maximum, the sum and the draw
    // again: 1,000 games of up to 8 drafts of 16,641 bfloat16 with up to 512 take 150 us; a lane per place of every word of
    // the mask, which kept no list, took 1,040.)
    __device__ __forceinline__ int part(int *to, int lane, int &w) const {
        __syncwarp();  // the last part has been read
        int count = 0, took = 32;
        while (took == 32) {
            uint32_t b = w + lane < words ? bits[w + lane] : 0;
            int upto = __popc(b);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(ALL, upto, o);
                if (lane >= o) upto += u;
            }
            const bool fits = w + lane < words && count + upto <= LIST;
            took = __popc(__ballot_sync(ALL, fits));  // (ten words or more, as far as there are any)
            if (fits)
                for (int k = count + upto - __popc(b); b; b &= b - 1) to[k++] = 32 * (w + lane) + __ffs(b) - 1 - skip;
            if (took) count += __shfl_sync(ALL, upto, took - 1);
            w += took;
        }
        __syncwarp();
        return count;
    }
    __device__ __forceinline__ bool has(int j) const { return (bits[(j + skip) >> 5] >> ((j + skip) & 31)) & 1; }
    // bits of places [32 w, 32 w + 32)
    __device__ __forceinline__ uint32_t word(int w, int places) const {
        const uint32_t hi = skip && w + 1 < words ? bits[w + 1] : 0, v = __funnelshift_r(bits[w], hi, skip);
        return places - 32 * w >= 32 ? v : v & ((1u << (places - 32 * w)) - 1);
    }
};

// The larger of two, or NaN where one is: so a maximum tells of every NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr float FAR = -3000.f;  // exp of it is 0, and so is its product with it: keeps -inf out of the sums

// Running maximum, sum of exp(x - m) and sum of exp(x - m)(x - m).
struct Soft {
    float m, s, t;
    __device__ __forceinline__ void raise(float c) {
        if (c > m) {
            const float d = m - c, k = ex2(d * LOG2E);
            t = k > 0.f ? k * (t + s * d) : 0.f;  // k = 0: d may be far, or infinite
            s *= k;
            m = c;
        }
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&x)[N]) {
        float c = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) c = fmaxf(c, x[i]);
        raise(c);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float d = max_nan(x[i] - m, FAR), e = ex2(d * LOG2E);
            s += e;
            t += e * d;
        }
    }
    template <int N>
    __device__ __forceinline__ void add_pairs(const f2 (&x)[N]) {
        float c = m;
#pragma unroll
        for (int i = 0; i < N; ++i) c = fmaxf(c, fmaxf(parts(x[i]).x, parts(x[i]).y));
        raise(c);
        const f2 nm = both(-m), l = both(LOG2E);
        f2 ss = both(0.f), tt = both(0.f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float2 q = parts(x[i] + nm);
            q.x = max_nan(q.x, FAR), q.y = max_nan(q.y, FAR);
            const f2 d = make_f2(q.x, q.y);
            const float2 w = parts(d * l);
            const f2 e = make_f2(ex2(w.x), ex2(w.y));
            ss = ss + e;
            tt = fma2(e, d, tt);
        }
        s += parts(ss).x + parts(ss).y;
        t += parts(tt).x + parts(tt).y;
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

constexpr int LOGP_THREADS = 256;

struct LogpArgs {
    const void *x;
    const uint8_t *mask;
    uint32_t *bits;        // (rows, words): the packed mask; written by the forward pass (may be NULL there)
    const int32_t *act;
    float *lp, *ent;       // forward outputs
    float4 *stats;         // (rows): m, 1 / Z, H - log Z, and the action's bits
    const float *glp, *gent;
    void *dx;
    int64_t rows, x_stride, mask_stride, glp_stride, gent_stride;
    int32_t n, words, share;  // share: bytes of shared memory of a warp
};

// A row's scores from its sums, by one thread.
template <typename T>
__device__ __forceinline__ void logp_finish(const LogpArgs &a, int64_t row, const Soft &acc, const T *x, int act, bool legal) {
    const bool empty = acc.s == 0.f;
    const float logz = empty ? 0.f : logf(acc.s), inv = empty ? 0.f : 1.f / acc.s;
    const float h = empty ? 0.f : logz - acc.t * inv;
    float lp = 0.f;
    if (act >= 0 && act < a.n) {
        // -inf at the action's place gives -inf, NaN anywhere legal NaN
        lp = legal && !empty ? (to_f(x[act]) - acc.m) - logz : -INFINITY;
        if (acc.s != acc.s) lp = acc.s;
    }
    a.lp[row] = lp;
    a.ent[row] = h;
    if (a.stats) a.stats[row] = make_float4(acc.m, inv, h - logz, __int_as_float(act));
}

__device__ __forceinline__ void warp_join(Soft &acc) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        acc.join(__shfl_xor_sync(ALL, acc.m, o), __shfl_xor_sync(ALL, acc.s, o), __shfl_xor_sync(ALL, acc.t, o));
}

// With a mask: a warp per row, whose chain (mask, blocks, scattered logits, sum)
// needs no barrier; 36 warps an SM hide it.  A CTA per row, each thread with
// the bits of its own 32 places, took 38 us where this takes 22 (4,096 rows of
// 16,641 bfloat16 with up to 80 legal places: 68 MB of mask, 3.1 TB/s).  With
// many legal places a row it is DRAM's: a scattered logit costs 64 bytes or
// more there (8,192 rows of float32 with up to 400: 61 us for 337 MB, 5.5 TB/s).
constexpr int LOGP_WARPS = 4;

template <typename T>
__global__ void __launch_bounds__(32 * LOGP_WARPS, 9) logp_masked_kernel(const LogpArgs a) {
    extern __shared__ __align__(16) char logp_smem[];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * LOGP_WARPS + warp;
    if (row >= a.rows) return;
    const T *x = (const T *)a.x + row * a.x_stride;
    const int act = a.act[row];
    Legal legal(logp_smem + warp * a.share, logp_smem + (warp + 1) * a.share - 4 * BLOCKS, BLOCKS);
    legal.read(a.mask + row * a.mask_stride, a.n, lane);
    Soft acc{LOWEST, 0.f, 0.f};
    if (legal.blocks <= BLOCKS) {
        // a lane's blocks, four scattered logits in flight
        uint32_t block = 0;
        for (int e = lane; e < legal.blocks || (block & 0xffff);) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!(block & 0xffff) && e < legal.blocks) block = legal.found[e], e += 32;
                v[i] = -INFINITY;
                if (block & 0xffff) {
                    v[i] = to_f(x[(int)(block >> 16) * 16 - legal.skip + __ffs(block) - 1]);
                    block &= block - 1;
                }
            }
            acc.add(v);
        }
    } else {
        for (int w = 0; w < legal.words; w += 8) {  // many: a lane per place, eight words at a time
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = 32 * (w + i) + lane - legal.skip;
                v[i] = -INFINITY;
                if (w + i < legal.words && (legal.bits[w + i] >> lane) & 1) v[i] = to_f(x[j]);
            }
            acc.add(v);
        }
    }
    warp_join(acc);
    if (lane == 0) logp_finish(a, row, acc, x, act, act >= 0 && act < a.n && legal.has(act));
    if (a.bits)
        for (int w = lane; w < a.words; w += 32) a.bits[row * a.words + w] = legal.word(w, a.n);
}

// Without: a CTA per row, 16 bytes a load, the ends one by one.  31 us for 2,048
// rows of 30,001 float16 (4.0 TB/s, 0.61 of a plain copy's rate; two thirds of
// the issue slots, and the exponentials alone need 14 us of the special function
// units: nothing of these is full).
template <typename T>
__global__ void __launch_bounds__(LOGP_THREADS, 6) logp_dense_kernel(const LogpArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ float red[LOGP_THREADS / 32][3];
    pdl_enter();
    const int64_t row = blockIdx.x;
    const T *x = (const T *)a.x + row * a.x_stride;
    const int tid = threadIdx.x, lane = tid & 31;
    Soft acc{LOWEST, 0.f, 0.f};
    const int head = min(a.n, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
    const int packs = (a.n - head) / VEC;
    const Pack<T, VEC> *px = (const Pack<T, VEC> *)(x + head);
    for (int k = tid; k < packs; k += 2 * LOGP_THREADS) {
        Pack<T, VEC> p[2];
        p[0] = px[k];
        const bool two = k + LOGP_THREADS < packs;
        if (two) p[1] = px[k + LOGP_THREADS];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (h == 0 || two) {
                f2 v[VEC / 2];
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i) v[i] = to_f2(&p[h].v[2 * i]);
                acc.add_pairs(v);
            }
    }
    const int rest = a.n - packs * VEC;  // before the first pack and behind the last: at most 2 VEC - 2
    if (tid < rest) {
        float v[1] = {to_f(x[tid < head ? tid : tid + packs * VEC])};
        acc.add(v);
    }
    warp_join(acc);
    if (lane == 0) red[tid >> 5][0] = acc.m, red[tid >> 5][1] = acc.s, red[tid >> 5][2] = acc.t;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int i = 1; i < LOGP_THREADS / 32; ++i) acc.join(red[i][0], red[i][1], red[i][2]);
        logp_finish(a, row, acc, x, a.act[row], true);
    }
}

// Gradient.  With a mask: zeros over the row, then the legal places; what they
// need is fetched before the zeros are written, so that it arrives meanwhile.
// 33 us for 4,096 rows of 16,641 bfloat16 (136 MB written, 40 without fetching
// ahead), 127 us for 8,192 of float32 with up to 400 legal places (545 MB
// written, 218 MB of scattered logits and packed masks read: 5.6 TB/s); without
// a mask 50 us for 2,048 rows of 30,001 float16 (246 MB, 4.9 TB/s).
template <typename T, bool MASK>
__global__ void __launch_bounds__(LOGP_THREADS) logp_bwd_kernel(const LogpArgs a) {
    constexpr int VEC = 16 / sizeof(T), AHEAD = 4;
    pdl_enter();
    const int64_t row = blockIdx.x;
    const T *x = (const T *)a.x + row * a.x_stride;
    T *dx = (T *)a.dx + row * a.n;
    const int tid = threadIdx.x, lane = tid & 31;
    const uint32_t *bits = MASK ? a.bits + row * a.words : nullptr;
    uint32_t mine = MASK && tid < a.words ? bits[tid] : 0, more = MASK && tid + LOGP_THREADS < a.words ? bits[tid + LOGP_THREADS] : 0;
    const float4 st = a.stats[row];  // m, 1 / Z, H - log Z, the action
    const int act = __float_as_int(st.w);
    const bool inside = act >= 0 && act < a.n;
    const bool legal = inside && (!MASK || ((bits[act >> 5] >> (act & 31)) & 1));
    const float xa = inside ? to_f(x[act]) : 0.f;
    float u = a.glp ? a.glp[row * a.glp_stride] : 0.f;
    const float v = a.gent ? a.gent[row * a.gent_stride] : 0.f;
    // -p (u + v (log p + H)) = exp(c) (k0 + k1 c)
    float k0 = 0.f, k1 = -v * st.y;
    auto grad = [&](int j, float xj) {
        const float c = max_nan(xj - st.x, FAR);
        return ex2(c * LOG2E) * fmaf(k1, c, k0) + (j == act ? u : 0.f);
    };
    const int head = min(a.n, (int)((16 - ((uintptr_t)dx & 15)) & 15) / (int)sizeof(T));
    const int packs = (a.n - head) / VEC, rest = a.n - packs * VEC;
    Pack<T, VEC> *pd = (Pack<T, VEC> *)(dx + head);
    if (MASK) {
        // the first few legal places of this thread's first two words
        float xs[AHEAD];
        int at[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            at[i] = -1;
            if (mine) {
                at[i] = 32 * tid + __ffs(mine) - 1;
                mine &= mine - 1;
            } else if (more) {
                at[i] = 32 * (tid + LOGP_THREADS) + __ffs(more) - 1;
                more &= more - 1;
            }
            if (at[i] >= 0) xs[i] = to_f(x[at[i]]);
        }
        Pack<T, VEC> zero;
#pragma unroll
        for (int i = 0; i < VEC; ++i) zero.v[i] = from_f<T>(0.f);
        for (int k = tid; k < packs; k += LOGP_THREADS) pd[k] = zero;
        if (tid < rest) dx[tid < head ? tid : tid + packs * VEC] = zero.v[0];
        // the action's gradient: none without an action, or with one whose log-probability is -inf
        if (!legal || xa == -INFINITY) u = 0.f;
        k0 = -(u + v * st.z) * st.y;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (at[i] >= 0) dx[at[i]] = from_f<T>(grad(at[i], xs[i]));
        for (int w0 = tid - lane; w0 < a.words; w0 += LOGP_THREADS) {
            const int w = w0 + lane;
            uint32_t b = w == tid ? mine : w == tid + LOGP_THREADS ? more : w < a.words ? bits[w] : 0;
            // few legal places: each lane its own; many: the warp's words one after another, a lane per place
            if (__reduce_add_sync(ALL, __popc(b)) <= 128) {
                for (; b; b &= b - 1) {
                    const int j = 32 * w + __ffs(b) - 1;
                    dx[j] = from_f<T>(grad(j, to_f(x[j])));
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
        if (!legal || xa == -INFINITY) u = 0.f;
        k0 = -(u + v * st.z) * st.y;
        const bool same = (((uintptr_t)x ^ (uintptr_t)dx) & 15) == 0;  // x's packs start where dx's do
        const Pack<T, VEC> *px = (const Pack<T, VEC> *)(x + head);
        const f2 nm = both(-st.x), l = both(LOG2E), f0 = both(k0), f1 = both(k1);
#pragma unroll 2
        for (int k = tid; k < packs; k += LOGP_THREADS) {
            const int j = head + k * VEC;
            Pack<T, VEC> p;
            if (same)
                p = px[k];
            else
#pragma unroll
                for (int i = 0; i < VEC; ++i) p.v[i] = x[j + i];
            f2 g[VEC / 2];
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                float2 q = parts(to_f2(&p.v[2 * i]) + nm);
                q.x = max_nan(q.x, FAR), q.y = max_nan(q.y, FAR);
                const f2 c = make_f2(q.x, q.y);
                const float2 w = parts(c * l);
                g[i] = make_f2(ex2(w.x), ex2(w.y)) * fma2(c, f1, f0);
            }
            if ((unsigned)(act - j) < (unsigned)VEC)  // the action's pack
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i)
                    g[i] = g[i] + make_f2(j + 2 * i == act ? u : 0.f, j + 2 * i + 1 == act ? u : 0.f);
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) from_f2(&p.v[2 * i], g[i]);
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
// The places of a game are worked on at the same time, up to 16 of them, and
// the first that is not kept then draws: a game's chain is one place and one
// draw, whatever its drafts.  That reads places behind the first rejection in
// vain, but a game that goes place by place takes as long as its longest
// chain, and the others wait for it.
//
// That is with a mask, where a place is one warp's: it packs the mask, lists
// the legal actions in order, and does the rest on the list without a barrier;
// what bounds it is the mask's bytes (with many games) or the chain of some
// thousand cycles (with few).  Measured: 4,096 samples of 16,641 float32 with
// up to 80 legal actions 20 us (69 MB, 3.4 TB/s), 8 games of 4 drafts 8.9 us,
// 1,024 of up to 8 drafts 43 us; place by place and a CTA per game these took
// 89, 33 and 125.  1,024 games of 8 bare drafts 32 us.  Without a mask
// (verify_dense_kernel) 301 games of 5 drafts take 66 us, of which the 64-bit
// operations are about 15 at the chip's rate, and 64-bit exchanges, spills and
// the 32-bit pass over places behind a rejection the rest.

constexpr int VERIFY_WARPS = 36;  // of an SM, for the launch
constexpr double RESIDUAL_MIN = 1.0 / (double)(1ull << 40);  // less left after a rejection counts as none
constexpr int PLACES = 16;     // of a game at the same time, at most

struct VerifyArgs {
    jq_drafts d;
    int32_t share, own;     // masked: bytes of shared memory of a warp, and those of them before the list
};

// e^d for d <= 0 in 64 bits: d = k ln 2 / 16 + r, e^d = 2^(k / 16) e^r, from a
// table of 16 and five terms of the series (Tang's table-driven exponential,
// ACM TOMS 1989); |r| <= 0.0217, so the sixth is below 1.5e-13.  Below -700: 0.
// Good to 1.7e-13 relatively.  Ten operations, where the library's function has
// about three times that.  16 entries, because they lie in banks of their own.
constexpr int EXP_STEPS = 16;
__device__ __forceinline__ double exp_table(int i) { return exp2((double)i / EXP_STEPS); }
// 16 / ln 2, -ln 2 / 16, 1 / 5!, 1 / 4!, 1 / 3!: as constants in memory they are operands; written into the code,
// each use takes two more instructions to make one
__constant__ double c_exp[5] = {EXP_STEPS * 1.4426950408889634, -0.69314718055994531 / EXP_STEPS, 1.0 / 120, 1.0 / 24, 1.0 / 6};
__device__ __forceinline__ double exp_near(double d, const double *table) {  // d in [-700, 0]; elsewhere some number
    static_assert(EXP_STEPS == 16, "four bits of k are the table's");
    constexpr double MAGIC = 1.5 * 4503599627370496.0;  // 1.5 * 2^52: a sum's last bit is 1
    const double near = fma(d, c_exp[0], MAGIC);
    const uint32_t k = (uint32_t)__double2loint(near);  // k in two's complement
    const double r = fma(near - MAGIC, c_exp[1], d);
    const double e = r * fma(r, fma(r, fma(r, fma(r, c_exp[2], c_exp[3]), c_exp[4]), 0.5), 1.0);
    const double at = table[k & 15], v = fma(at, e, at);
    return __hiloint2double((int)((uint32_t)__double2hiint(v) + ((k & ~15u) << 16)), __double2loint(v));
}

// One row of logits and what its probabilities need.
struct Dist {
    enum { NONE = 0, SOME = 1, BROKEN = 2 };  // no legal place above -inf; a distribution; NaN or +inf at a legal place
    double m, z;  // the largest logit, and Z
    float low;    // logits below it have exp(x - m) = 0
    int state;
    static __device__ __forceinline__ Dist none() { return {0.0, 0.0, INFINITY, NONE}; }
    __device__ __forceinline__ void start(float top, bool there) {
        state = !there || top == -INFINITY ? NONE : top < INFINITY ? SOME : BROKEN;
        m = state == SOME ? top : 0.f;
        // rounded up: on the logits' own grid the nearest number may be as far as m - 1024, below what exp_near takes
        low = state == SOME ? __double2float_ru(m - 700.0) : INFINITY;
        z = 0;
    }
    __device__ __forceinline__ double weight(float x, const double *table) const {  // exp(x - m)
        const double e = exp_near((double)x - m, table);
        return x >= low ? e : 0.0;
    }
};

// What a place is, and whether its draft is kept.
template <typename T>
struct Place {
    const T *x, *y;       // logits; of the draft, or NULL
    const uint8_t *mask;
    int act;              // the drafted action; -1 behind the last
    bool drafted;         // i < len
    float u, xa, ya;      // the draft's random number, the drafted action's logits
    Dist p, q;
    __device__ __forceinline__ Place(const jq_drafts &d, int game, int i, int len)
        : x((const T *)d.logits + game * d.logits_game + i * d.logits_place), y(nullptr),
          mask(d.mask ? d.mask + game * d.mask_game + i * d.mask_place : nullptr), act(-1), drafted(i < len), u(0.f), xa(0.f), ya(0.f),
          p(Dist::none()), q(Dist::none()) {
        if (drafted) {
            act = d.drafted[(int64_t)game * d.drafts + i];
            u = d.accept_u[(int64_t)game * d.drafts + i];
            if (d.draft_logits) y = (const T *)d.draft_logits + game * d.draft_game + i * d.draft_place;
        }
        if (act >= d.actions) act = -1;
    }
    __device__ __forceinline__ void fetch() {  // the drafted action's logits, some time after the action itself
        if (act >= 0) {
            xa = to_f(x[act]);
            if (y) ya = to_f(y[act]);
        }
    }
    __device__ __forceinline__ bool broken() const { return (p.state | q.state) & Dist::BROKEN; }
    // probabilities are e / Z: compared and subtracted over the common denominator, without a division
    __device__ __forceinline__ bool kept(bool legal, const double *table) const {
        if (act < 0 || !legal || broken() || p.state != Dist::SOME) return false;
        const double ep = p.weight(xa, table);
        if (!y) return (double)u * p.z < ep;
        return q.state != Dist::SOME ? 0.0 < ep : __dmul_rn((double)u * q.weight(ya, table), p.z) < __dmul_rn(ep, q.z);
    }
    // whether `kept` might turn with sums that are off by `eps`
    __device__ __forceinline__ bool open(double eps, const double *table) const {
        if (act < 0 || broken() || p.state != Dist::SOME) return false;
        const double ep = p.weight(xa, table);
        if (!y) return fabs((double)u * p.z - ep) <= eps * ep;
        if (q.state != Dist::SOME) return false;
        const double l = (double)u * q.weight(ya, table) * p.z, r = ep * q.z;
        return fabs(l - r) <= eps * r && r > 0;
    }
    // what is drawn from, times `scale`: max(p - q, 0) while `residual`, else p; ep, eq are exp(x - m) at j
    __device__ __forceinline__ bool has_residual() const { return drafted && (y ? q.state == Dist::SOME : act >= 0); }
    __device__ __forceinline__ double scale(bool residual) const { return residual && y ? p.z * q.z : p.z; }
    __device__ __forceinline__ double draw(int j, double ep, double eq, bool residual) const {
        if (!residual) return ep;
        if (!y) return j == act ? 0.0 : ep;  // q is one-hot there
        const double w = __dmul_rn(ep, q.z) - __dmul_rn(eq, p.z);
        return w > 0 ? w : 0.0;
    }
    __device__ __forceinline__ double draw(int j, bool residual, const double *table) const {
        return draw(j, p.weight(to_f(x[j]), table), residual && y ? q.weight(to_f(y[j]), table) : 0.0, residual);
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
    for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(ALL, v, o));
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

// ALONE: no drafts, a game per warp.  Bounds: 32 and 24 warps an SM by registers.
template <typename T, bool ALONE>
__global__ void __launch_bounds__(ALONE ? 128 : 768, ALONE ? 8 : 1) verify_masked_kernel(const VerifyArgs a) {
    extern __shared__ __align__(16) char verify_smem[];
    __shared__ double table[EXP_STEPS];
    __shared__ int keeps[2][PLACES];
    const jq_drafts &d = a.d;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, n = d.actions;
    for (int i = threadIdx.x; i < EXP_STEPS; i += blockDim.x) table[i] = exp_table(i);
    pdl_enter();
    __syncthreads();
    // of the legal actions in order: exp(x - m), of the target and, where there are any, of the draft (until then their
    // logits), and the actions
    double *ep = (double *)(verify_smem + (size_t)warp * a.share + a.own), *eq = ep + LIST;
    int *list = (int *)(!ALONE && d.draft_logits ? eq + LIST : eq);
    Legal legal(verify_smem + (size_t)warp * a.share, ep, LIST);  // (the blocks found are done with when the list stands)
    const int game = ALONE ? blockIdx.x * warps + warp : blockIdx.x;
    if (game >= d.games) return;  // (ALONE: no barrier follows)
    int len = 0;
    if (!ALONE) {
        len = d.lengths ? d.lengths[game] : d.drafts;
        len = len < 0 ? 0 : len > d.drafts ? d.drafts : len;
    }
    int32_t *out = d.out_actions + (int64_t)game * (d.drafts + 1);
    float *out_lp = d.log_probs + (int64_t)game * (d.drafts + 1);
    for (int base = 0, round = 0;; base += warps, round ^= 1) {
        const int i = ALONE ? 0 : base + warp;
        const bool active = i <= len;
        bool kept = false;
        Place<T> at(d, game, active ? i : len, len);
        if (ALONE) at.y = nullptr, at.act = -1, at.drafted = false;
        int count = 0, w = 0;  // on the list; the mask's word behind it
        bool whole = true;     // the list has all legal actions, and stays; else it holds a part of them at a time
        float mx = -INFINITY, my = -INFINITY;
        double zx = 0, zy = 0;
        auto logits = [&]() {  // the list's, four scattered logits of each in flight
            for (int k0 = lane; k0 < count; k0 += 128) {
                float vx[4], vy[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (k0 + 32 * i < count) {
                        const int j = list[k0 + 32 * i];
                        vx[i] = to_f(at.x[j]);
                        if (at.y) vy[i] = to_f(at.y[j]);
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (k0 + 32 * i < count) {
                        mx = max_nan(mx, vx[i]);
                        ep[k0 + 32 * i] = __hiloint2double(0, __float_as_int(vx[i]));
                        if (at.y) {
                            my = max_nan(my, vy[i]);
                            eq[k0 + 32 * i] = __hiloint2double(0, __float_as_int(vy[i]));
                        }
                    }
            }
        };
        auto weights = [&]() {  // exp(x - m) in the logits' place
#pragma unroll 2
            for (int k = lane; k < count; k += 32) {
                const double e = at.p.weight(__int_as_float(__double2loint(ep[k])), table);
                ep[k] = e, zx += e;
                if (at.y) {
                    const double g = at.q.weight(__int_as_float(__double2loint(eq[k])), table);
                    eq[k] = g, zy += g;
                }
            }
            __syncwarp();  // other lanes read them
        };
        auto next_part = [&]() {
            count = legal.part(list, lane, w);
            if constexpr (ALONE) {
                logits();
            } else {
#pragma unroll 1
                for (int k = lane; k < count; k += 32) {  // one at a time, or the whole list's four lose registers
                    const float vx = to_f(at.x[list[k]]), vy = at.y ? to_f(at.y[list[k]]) : -INFINITY;
                    mx = max_nan(mx, vx), my = max_nan(my, vy);
                    ep[k] = __hiloint2double(0, __float_as_int(vx));
                    if (at.y) eq[k] = __hiloint2double(0, __float_as_int(vy));
                }
            }
        };
        if (active) {
            legal.read(at.mask, n, lane);
            at.fetch();
            count = legal.list(list, lane);
            whole = count <= LIST;
            if (whole)
                logits();
            else
                while (w < legal.words) next_part();
            at.p.start(warp_max(mx), true);
            at.q.start(warp_max(my), at.y != nullptr);
            if (whole)
                weights();
            else
                for (w = 0; w < legal.words;) next_part(), weights();
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) zx += __shfl_xor_sync(ALL, zx, o), zy += __shfl_xor_sync(ALL, zy, o);
            at.p.z = zx, at.q.z = zy;
            kept = at.kept(at.act >= 0 && legal.has(at.act), table);
        }
        int first = ALONE ? 0 : warps;  // the first place of this round that is not kept
        if (!ALONE) {
            if (lane == 0) keeps[round][warp] = kept;
            __syncthreads();
            for (int k = warps - 1; k >= 0; --k)
                if (!keeps[round][k]) first = k;
            if (kept && warp < first && lane == 0) out[i] = at.act, out_lp[i] = at.log_prob(at.act);
            if (first == warps) continue;
            if (warp != first) return;
        }
        int next = -1;
        if (at.p.state == Dist::SOME && !at.broken()) {
            const float rf = d.sample_u[game];
            const double r = rf > 0.f ? (double)rf : 0.0;
            auto draw = [&](bool residual) {  // false: nothing left to draw from
                double part, above, total = 0, below = 0;
                // this lane's actions are consecutive ones of the list: its weight, and with the lanes before
                auto sum_up = [&]() {
                    const int per = (count + 31) >> 5, lo = lane * per, hi = min(count, lo + per);
                    part = 0;
                    for (int k = lo; k < hi; ++k) part += at.draw(list[k], ep[k], at.y ? eq[k] : 0.0, residual);
                    above = warp_scan(part, lane);
                };
                if (whole)
                    sum_up(), total = __shfl_sync(ALL, above, 31);
                else
                    for (w = 0; w < legal.words; total += __shfl_sync(ALL, above, 31)) next_part(), weights(), sum_up();
                if (residual && !(total > RESIDUAL_MIN * at.scale(true))) return false;
                const double target = r * total;
                unsigned cross = 0;
                w = 0;
                do {
                    if (!whole) next_part(), weights(), sum_up();
                    // the first lane whose running sum is above the point; with none, the last that has weight
                    const double up = __shfl_up_sync(ALL, above, 1);
                    cross = __ballot_sync(ALL, part > 0 && below + above > target);
                    const unsigned some = __ballot_sync(ALL, part > 0);
                    const int who = cross ? __ffs(cross) - 1 : some ? 31 - __clz(some) : -1;
                    if (lane == who) {
                        const int per = (count + 31) >> 5, lo = lane * per, hi = min(count, lo + per);
                        double run = below + (lane ? up : 0.0);
                        bool crossed = false;
                        for (int k = lo; k < hi; ++k) {
                            const double v = at.draw(list[k], ep[k], at.y ? eq[k] : 0.0, residual);
                            run += v;
                            if (v > 0 && !crossed) next = list[k], crossed = run > target;
                        }
                    }
                    if (who >= 0) next = __shfl_sync(ALL, next, who);
                    below += __shfl_sync(ALL, above, 31);
                } while (!whole && !cross && w < legal.words);
                return true;
            };
            if (ALONE || !at.has_residual() || !draw(true)) draw(false);
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

// Without a mask: a cluster of CTAs per game, each a consecutive slice of every
// row.  For eight places at a time a warp takes the maximum and sum of one
// place's rows over the slice, in 32 bits (a ninth of the instructions of 64),
// and all tell all others once; warp w of each CTA then finds out about place
// w.  Where 32 bits leave it open whether a draft is kept, and for what is drawn
// from two rows, the sums are taken again in 64, every warp a chunk of the row.
// The draw is in 64 bits: weights of the chunks, told once, and the warp that
// has the point goes on alone.
constexpr int DENSE_THREADS = 256, DENSE_WARPS = DENSE_THREADS / 32, DENSE_CTAS = 8;
constexpr int DENSE_PLACES = DENSE_WARPS;  // of a round

// Every logit of x[0, n), by the warp: 8 bytes a load, the ends one by one.
template <typename T, typename F>
__device__ __forceinline__ void dense_each(const T *x, int n, int lane, F &&f) {
    constexpr int VEC = 8 / sizeof(T);
    const int head = min(n, (int)((8 - ((uintptr_t)x & 7)) & 7) / (int)sizeof(T)), packs = (n - head) / VEC;
    const Pack<T, VEC> *px = (const Pack<T, VEC> *)(x + head);
    int k = lane;
    for (; k + 96 < packs; k += 128) {
        Pack<T, VEC> p[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) p[u] = px[k + 32 * u];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) f(to_f(p[u].v[i]));
    }
    for (; k < packs; k += 32) {
        const Pack<T, VEC> p = px[k];
#pragma unroll
        for (int i = 0; i < VEC; ++i) f(to_f(p.v[i]));
    }
    const int rest = n - packs * VEC;  // before the first pack and behind the last
    if (lane < rest) f(to_f(x[lane < head ? lane : lane + packs * VEC]));
}

// Running maximum and sum of exp(x - m) in 32 bits, of a warp's part of a row.
struct Sum {
    float m, s;
    __device__ __forceinline__ void raise(float c) {
        if (c > m) s *= ex2((m - c) * LOG2E), m = c;
    }
    template <int N>
    __device__ __forceinline__ void add(const f2 (&x)[N]) {
        float c = m;
#pragma unroll
        for (int i = 0; i < N; ++i) c = fmaxf(c, fmaxf(parts(x[i]).x, parts(x[i]).y));
        raise(c);
        const f2 nm = both(-m), l = both(LOG2E);
        f2 ss = both(0.f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float2 w = parts((x[i] + nm) * l);
            ss = ss + make_f2(ex2(w.x), ex2(w.y));
        }
        s += parts(ss).x + parts(ss).y;
    }
    __device__ __forceinline__ void join(float m2, float s2) {
        const float top = fmaxf(m, m2);  // (of finite numbers, or +inf: then the sum is NaN)
        s = (s == 0.f ? 0.f : s * ex2((m - top) * LOG2E)) + (s2 == 0.f ? 0.f : s2 * ex2((m2 - top) * LOG2E));
        m = top;
    }
};
template <typename T>
__device__ __forceinline__ Sum chunk_sum(const T *x, int n, int lane) {
    constexpr int VEC = 8 / sizeof(T);
    const int head = min(n, (int)((8 - ((uintptr_t)x & 7)) & 7) / (int)sizeof(T)), packs = (n - head) / VEC;
    const Pack<T, VEC> *px = (const Pack<T, VEC> *)(x + head);
    Sum a{LOWEST, 0.f};
    const int rest = n - packs * VEC;  // before the first pack and behind the last
    const float end = lane < rest ? to_f(x[lane < head ? lane : lane + packs * VEC]) : -INFINITY;
    for (int k = lane; k < packs; k += 128) {
        f2 v[2 * VEC];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            Pack<T, VEC> p;
            const bool there = u == 0 || k + 32 * u < packs;
            if (there) p = px[k + 32 * u];
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) v[u * VEC / 2 + i] = there ? to_f2(&p.v[2 * i]) : both(-INFINITY);
        }
        a.add(v);
    }
    const f2 v[1] = {make_f2(end, -INFINITY)};
    a.add(v);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a.join(__shfl_xor_sync(ALL, a.m, o), __shfl_xor_sync(ALL, a.s, o));
    return a;
}

// The same sum in 64 bits, m being given.
template <typename T>
__device__ __forceinline__ double chunk_sum64(const T *x, int n, int lane, const Dist &d, const double *table) {
    double z = 0;
    if (d.state == Dist::SOME) dense_each(x, n, lane, [&](float v) { z += d.weight(v, table); });
    return warp_sum(z);
}

struct DenseSmem {
    double table[EXP_STEPS];
    float4 sums[2][DENSE_PLACES][DENSE_CTAS * DENSE_WARPS];  // by every warp at work on the place: m, sum of the target, of the draft
    double told[2][DENSE_CTAS * DENSE_WARPS][2];             // by every warp of the game, in 64 bits
    Dist p[DENSE_PLACES], q[DENSE_PLACES];
    int found[DENSE_PLACES];
};

template <typename T>
__global__ void __launch_bounds__(DENSE_THREADS, 4) verify_dense_kernel(const VerifyArgs a) {
    enum { KEPT, LEFT, OPEN };
    __shared__ DenseSmem sm;
    const jq_drafts &d = a.d;
    const double *table = sm.table;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = d.actions;
    const int rank = (int)cluster_rank(), ranks = (int)cluster_size(), game = blockIdx.x / ranks;
    const int warps = ranks * DENSE_WARPS, me = rank * DENSE_WARPS + warp;
    if (tid < EXP_STEPS) sm.table[tid] = exp_table(tid);
    pdl_enter();
    cluster_sync();  // the game's CTAs have all started: their shared memory may be written
    int len = d.lengths ? d.lengths[game] : d.drafts;
    len = len < 0 ? 0 : len > d.drafts ? d.drafts : len;
    int32_t *out = d.out_actions + (int64_t)game * (d.drafts + 1);
    float *out_lp = d.log_probs + (int64_t)game * (d.drafts + 1);
    const int chunk = (n + warps - 1) / warps, c0 = min(n, me * chunk), c1 = min(n, c0 + chunk);
    int turn = 0;
    // two numbers of this warp to every CTA
    auto tell = [&](double v0, double v1) {
        if (lane < 2 * ranks) cluster_store(&sm.told[turn][me][lane & 1], lane >> 1, lane & 1 ? v1 : v0);
        cluster_sync();
    };
    auto told = [&](int what) {  // their sum
        return warp_sum((lane < warps ? sm.told[turn][lane][what] : 0.0) + (lane + 32 < warps ? sm.told[turn][lane + 32][what] : 0.0));
    };
    const int slice = (n + ranks - 1) / ranks, s0 = min(n, rank * slice), s1 = min(n, s0 + slice);
    for (int base = 0, round = 0;; round ^= 1) {
        const int places = min(DENSE_PLACES, len - base + 1);
        // a place of this CTA's slice is one warp's, or several warps'
        const int split = DENSE_WARPS / places, k = warp / split, part_of = warp % split, share = (slice + split - 1) / split;
        // how far a 32-bit sum may be off, relatively: 2^-22 for an exponential, its argument's three roundings of at most
        // log2(n) <= 18 on average, one for each addition and 2^-22 for each time the maximum rose
        const double eps = (3.0 * ((share + 31) / 32) + 160.0) / (1 << 24);
        if (k < places) {
            const Place<T> at(d, game, base + k, len);
            const int b0 = min(s1, s0 + part_of * share), b1 = min(s1, b0 + share);
            const Sum sx = chunk_sum(at.x + b0, b1 - b0, lane);
            Sum sy{LOWEST, 0.f};
            if (at.y) sy = chunk_sum(at.y + b0, b1 - b0, lane);
            if (lane < ranks) cluster_store4(&sm.sums[round][k][rank * split + part_of], lane, make_float4(sx.m, sx.s, sy.m, sy.s));
        }
        cluster_sync();
        if (warp < places) {
            Place<T> at(d, game, base + warp, len);
            at.fetch();
            const float4 none = make_float4(0, 0, 0, 0);
            const int parts = ranks * split;
            const float4 t0 = lane < parts ? sm.sums[round][warp][lane] : none,
                         t1 = lane + 32 < parts ? sm.sums[round][warp][lane + 32] : none;
            // a chunk without a place above -inf has the sum 0, whatever its m; NaN or +inf make it NaN
            auto total = [&](float m0, float v0, float m1, float v1, Dist &dist, bool there) {
                m0 = v0 == 0.f ? -INFINITY : v0 != v0 ? v0 : m0;
                m1 = v1 == 0.f ? -INFINITY : v1 != v1 ? v1 : m1;
                dist.start(warp_max(max_nan(m0, m1)), there);
                dist.z = warp_sum((v0 == 0.f ? 0.0 : v0 * dist.weight(m0, table)) + (v1 == 0.f ? 0.0 : v1 * dist.weight(m1, table)));
            };
            total(t0.x, t0.y, t1.x, t1.y, at.p, true);
            total(t0.z, t0.w, t1.z, t1.w, at.q, at.y != nullptr);
            const int found = at.open(4 * eps, table) ? OPEN : at.kept(true, table) ? KEPT : LEFT;
            if (lane == 0) sm.p[warp] = at.p, sm.q[warp] = at.q, sm.found[warp] = found;
        }
        __syncthreads();
        // what all CTAs of the game have in the same numbers, they decide alike
        int first = places;
        for (int k = places - 1; k >= 0; --k)
            if (sm.found[k] != KEPT) first = k;
        if (rank == 0 && warp < first && lane == 0) {
            Place<T> at(d, game, base + warp, len);
            at.p = sm.p[warp];
            out[base + warp] = at.act, out_lp[base + warp] = at.log_prob(at.act);
        }
        if (first == places) {  // (the place behind the last draft is never kept)
            base += places;
            __syncthreads();
            continue;
        }
        const int i = base + first;
        Place<T> at(d, game, i, len);
        at.p = sm.p[first], at.q = sm.q[first];
        bool exact = false;  // Z is in 64 bits
        auto make_exact = [&]() {
            const double zx = chunk_sum64(at.x + c0, c1 - c0, lane, at.p, table);
            tell(zx, at.y ? chunk_sum64(at.y + c0, c1 - c0, lane, at.q, table) : 0.0);
            at.p.z = told(0), at.q.z = told(1);
            turn ^= 1;
            exact = true;
        };
        if (sm.found[first] == OPEN) {
            at.fetch();
            make_exact();
            if (at.kept(true, table)) {
                if (me == 0 && lane == 0) out[i] = at.act, out_lp[i] = at.log_prob(at.act);
                base = i + 1;
                __syncthreads();
                continue;
            }
        }
        int next = -1, who = 0;  // who: the warp whose chunk has the point
        if (at.p.state == Dist::SOME && !at.broken()) {
            const float rf = d.sample_u[game];
            const double r = rf > 0.f ? (double)rf : 0.0;
            if (at.has_residual() && at.y && !exact) make_exact();
            for (int pass = at.has_residual() ? 0 : 1; pass < 2; ++pass) {
                const bool residual = pass == 0;
                auto weight = [&](int j) { return at.draw(j, residual, table); };
                double part = 0;
                if (residual && at.y) {
#pragma unroll 4
                    for (int j = c0 + lane; j < c1; j += 32) part += weight(j);
                    part = warp_sum(part);
                } else {  // the target alone, but for the draft's action where that was certain
                    const int skip = residual && at.act >= c0 && at.act < c1 ? at.act : c1;
                    for (int from = c0, to = skip; from < c1; from = to + 1, to = c1)
                        part += chunk_sum64(at.x + from, to - from, lane, at.p, table);
                }
                tell(part, 0);
                // the first chunk whose running sum is above the point; with none, the last that has weight
                const int per = (warps + 31) / 32, k0 = lane * per, k1 = k0 + 1;
                const double t0 = k0 < warps ? sm.told[turn][k0][0] : 0.0, t1 = per > 1 && k1 < warps ? sm.told[turn][k1][0] : 0.0;
                turn ^= 1;
                const double above = warp_scan(t0 + t1, lane), total = __shfl_sync(ALL, above, 31);
                if (!exact && !residual) at.p.z = total;  // exp(x - m), summed up in 64 bits
                if (residual && !at.y && !exact) at.p.z = total + at.p.weight(to_f(at.x[at.act]), table);
                if (residual && !(total > RESIDUAL_MIN * at.scale(true))) continue;
                const double target = r * total, up = __shfl_up_sync(ALL, above, 1), before = lane ? up : 0.0;
                unsigned cross = __ballot_sync(ALL, t0 + t1 > 0 && above > target), some = __ballot_sync(ALL, t0 + t1 > 0);
                int owner = cross ? __ffs(cross) - 1 : 31 - __clz(some);
                const bool second = t1 > 0 && !(t0 > 0 && before + t0 > target);
                who = __shfl_sync(ALL, second ? k1 : k0, owner);
                double below = __shfl_sync(ALL, second ? before + t0 : before, owner);
                if (who != me) return;
                // 256 places at a time, eight consecutive ones a lane; whether the point is in them, or the last weight may be
                constexpr int STEP = 8;
                auto look = [&](int f, bool last) {
                    double w[STEP], s = 0;
#pragma unroll
                    for (int k = 0; k < STEP; ++k) {
                        const int j = f + STEP * lane + k;
                        w[k] = j < c1 ? weight(j) : 0.0;
                        s += w[k];
                    }
                    const double sum = warp_scan(s, lane), up = __shfl_up_sync(ALL, sum, 1);
                    cross = __ballot_sync(ALL, !last && s > 0 && below + sum > target), some = __ballot_sync(ALL, s > 0);
                    if (cross || last) {
                        double run = below + (lane ? up : 0.0);
                        bool crossed = false;
                        int at_j = -1;
#pragma unroll
                        for (int k = 0; k < STEP; ++k) {
                            run += w[k];
                            if (w[k] > 0 && !crossed) at_j = f + STEP * lane + k, crossed = !last && run > target;
                        }
                        next = __shfl_sync(ALL, at_j, cross ? __ffs(cross) - 1 : 31 - __clz(some));
                    }
                    below += __shfl_sync(ALL, sum, 31);
                };
                int held = c0;
                cross = 0;
                for (int f = c0; f < c1 && !cross; f += 32 * STEP) {
                    look(f, false);
                    if (some) held = f;
                }
                if (!cross) look(held, true);  // the point is at the end of the chunk's sum: its last place with weight
                break;
            }
        }
        if (who != me) return;
        if (lane == 0) {
            d.accepted[game] = i;
            out[i] = next;
            out_lp[i] = next >= 0 ? at.log_prob(next) : at.broken() ? __int_as_float(0x7fc00000) : 0.f;
        }
        for (int k = i + 1 + lane; k <= d.drafts; k += 32) out[k] = -1, out_lp[k] = 0.f;
        return;
    }
}

// Lets a kernel have `bytes` of an SM's shared memory on the current device.
template <typename K>
static cudaError_t allow_smem(K *kernel, int bytes, std::atomic<uint64_t> &raised) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (raised.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) raised.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

template <typename T>
static int logp_forward(LogpArgs &a, cudaStream_t s) {
    if (!a.mask) {
        CU(launch_pdl(logp_dense_kernel<T>, (unsigned)a.rows, LOGP_THREADS, 0, s, a));
        return JQ_OK;
    }
    a.share = (int)Legal::bytes(a.n) + 4 * BLOCKS;
    const size_t smem = (size_t)LOGP_WARPS * a.share;
    static std::atomic<uint64_t> raised{0};
    if (smem > 48 * 1024) CU(allow_smem(logp_masked_kernel<T>, 200 * 1024, raised));
    CU(launch_pdl(logp_masked_kernel<T>, (unsigned)((a.rows + LOGP_WARPS - 1) / LOGP_WARPS), 32 * LOGP_WARPS, smem, s, a));
    return JQ_OK;
}

template <typename T>
static int logp_backward(const LogpArgs &a, cudaStream_t s) {
    CU(a.bits ? launch_pdl(logp_bwd_kernel<T, true>, (unsigned)a.rows, LOGP_THREADS, 0, s, a)
              : launch_pdl(logp_bwd_kernel<T, false>, (unsigned)a.rows, LOGP_THREADS, 0, s, a));
    return JQ_OK;
}

template <typename T>
static int verify_launch(const jq_drafts &d, cudaStream_t s) {
    VerifyArgs a{d, 0, 0};
    if (!d.mask) {
        int sms, rc = device_sms(sms);
        if (rc) return rc;
        // CTAs of a thousand places or more until the SMs are full (4 each; up to twice that, and no step shows where it is
        // passed: 296 games 65.7 us, 297 66.1, 301 65.7): each place costs every warp an exchange
        int ctas = 1;
        while (ctas < DENSE_CTAS && (int64_t)d.games * ctas < 4 * (int64_t)sms && d.actions > 1024 * ctas) ctas *= 2;
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
    a.own = (int)Legal::bytes(d.actions);
    a.share = a.own + LIST * (d.draft_logits && d.drafts ? 20 : 12);
    static std::atomic<uint64_t> raised[2];
    if (d.drafts == 0) {
        int warps = 4;
        while (warps > 1 && warps * a.share > 200 * 1024) --warps;
        if (warps * a.share > 40 * 1024) CU(allow_smem(verify_masked_kernel<T, true>, 210 * 1024, raised[1]));
        CU(launch_pdl(verify_masked_kernel<T, true>, (unsigned)((d.games + warps - 1) / warps), 32 * warps, warps * a.share, s, a));
        return JQ_OK;
    }
    int sms, rc = device_sms(sms);
    if (rc) return rc;
    // places side by side: as few rounds as there are warps for, up to one and a half times what the SMs hold (24 each),
    // and no more places than those rounds need
    const int places = d.drafts + 1;
    int rounds = (places + PLACES - 1) / PLACES, warps = (places + rounds - 1) / rounds;
    while (warps > 2 && (int64_t)d.games * warps > VERIFY_WARPS * (int64_t)sms) ++rounds, warps = (places + rounds - 1) / rounds;
    while (warps > 1 && warps * a.share > 200 * 1024) --warps;
    if (warps * a.share > 40 * 1024) CU(allow_smem(verify_masked_kernel<T, false>, 210 * 1024, raised[0]));
    CU(launch_pdl(verify_masked_kernel<T, false>, (unsigned)d.games, 32 * warps, warps * a.share, s, a));
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
    a.rows = rows;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == JQ_F32) return logp_forward<float>(a, s);
    if (dtype == JQ_F16) return logp_forward<__half>(a, s);
    return logp_forward<__nv_bfloat16>(a, s);
}

int jq_action_log_prob_backward(const void *d_logits, int64_t row_stride, int32_t dtype, const uint32_t *d_bits,
                                const float *d_stats, const float *d_grad_log_prob, int64_t grad_log_prob_stride,
                                const float *d_grad_entropy, int64_t grad_entropy_stride, int64_t rows,
                                int32_t actions, void *d_dlogits, void *stream) {
    int rc = logp_check(d_logits, row_stride, dtype, rows, actions);
    if (rc) return rc;
    if (!d_stats || !d_dlogits) return fail(JQ_ERR_ARG, "action scores: statistics or output missing");
    if (grad_log_prob_stride < 0 || grad_entropy_stride < 0) return fail(JQ_ERR_ARG, "action scores: negative stride");
    if (((uintptr_t)d_bits | (uintptr_t)d_grad_log_prob | (uintptr_t)d_grad_entropy) & 3 || (uintptr_t)d_stats & 15 ||
        (uintptr_t)d_dlogits & (elem_size(dtype) - 1))
        return fail(JQ_ERR_ARG, "action scores: an array is not aligned to its elements");
    LogpArgs a{};
    a.x = d_logits, a.bits = const_cast<uint32_t *>(d_bits);
    a.stats = (float4 *)const_cast<float *>(d_stats), a.glp = d_grad_log_prob, a.gent = d_grad_entropy;
    a.glp_stride = grad_log_prob_stride, a.gent_stride = grad_entropy_stride, a.dx = d_dlogits;
    a.rows = rows, a.x_stride = row_stride, a.n = actions, a.words = (actions + 31) / 32;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == JQ_F32) return logp_backward<float>(a, s);
    if (dtype == JQ_F16) return logp_backward<__half>(a, s);
    return logp_backward<__nv_bfloat16>(a, s);
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
