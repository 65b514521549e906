// jq_norm.cu -- layer norm over the last axis, forward and backward.
//
//   mu = mean(x), s2 = mean((x - mu)^2), r = 1 / sqrt(s2 + eps)
//   xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum dy xh,  db = sum dy
//
// Bound: memory.  Forward moves 2 elements per place (x in, y out), backward
// 3 (x and dy in, dx out).  Two things stand in the way.  Instructions per
// row: the reductions, and loops over places that are not there.  So a thread
// holds up to E = 16 places of a row (few threads, few shuffles: two rows of
// 256 share a warp's), in groups of G that are skipped together where the row
// is shorter, and arithmetic is on pairs of floats.  And bytes in flight: a
// row's reductions are a chain of some hundred cycles, so the next rows come
// into a ring of shared memory by asynchronous copies of 16-byte blocks
// (whatever the rows' alignment) while it runs, without a register for them.
// A row belongs to TPR threads of a warp, whose rows and ring are its own, or
// from 513 places on to a CTA of as few warps as hold it (TPR = 0).  Threads
// keep their places' weights, and in the backward pass their two gradient
// sums, in registers while they walk the rows; these leave once per CTA and a
// second kernel adds them up in a fixed order, so equal calls give equal bits.
//
// Statistics are 32-bit.  The mean is taken twice: m, the rounded mean, then
// delta = mean(x - m), what the rounding left, so a row whose mean is large
// against its spread loses nothing (s2 = mean((x - m)^2) - delta^2, in which
// delta^2 is at rounding level).  Where it is not, because the row is all but
// constant, m takes delta in and the row is done once more, from memory, when a
// warp (CTA) has been through all of its rows: asked for in the walk itself, it
// cost every row 1 to 20 % by the registers.  The three numbers (m, delta, r)
// per row go to the backward pass.
//
// Measured (B200, 264,192 rows of 256 bfloat16): forward 47 us (5.8 TB/s, 0.89
// of a plain copy's rate), backward 70 us (5.8 TB/s) and 6.5 us for the second
// kernel after a flush; pass after pass 73 us without the weights' gradients and
// 79 with them.  Rows of a CTA wait for its barriers: 6,000 rows of 4,096
// float16 take 28 and 43 us (3.5 TB/s, 63 and 43 % of the issue slots), 8,191
// of 1,111 float32, whose rows start anywhere, 19 and 25 us (3.8 and 4.3 TB/s).
// Rows of one or two places, whose threads hold mostly nothing, spill up to 60
// bytes: 3,000,017 rows of 1 float32 take 70 and 70 us, of 16 bfloat16 (half as
// many) 30 and 42.
#include <atomic>

#include "jq_ops.cuh"

namespace jq {

struct NormArgs {
    const void *x, *w, *b, *dy;
    void *y;                  // forward: y; backward: dx (may be NULL)
    float *stats;             // (rows, 3): m, delta, r
    float *part;              // backward: (grid, 2, dim) sums of dw and db, or NULL
    int64_t x_stride, dy_stride, rows;
    int32_t dim, groups, wf32;
    int32_t chunk;            // rows of a ring slot
    int32_t x_bytes, slot_bytes;  // of a slot: x's share, and all
    float eps;
};

constexpr int NORM_E = 16, NORM_WARPS = 16;           // places of a thread, warps of the longest row
constexpr int NORM_FWD_SLOTS = 4, NORM_BWD_SLOTS = 3; // of a warp's ring; a CTA's rows have 3
constexpr int NORM_BWD_SLOT = 4688;                   // bytes, at most, where a slot has several rows: 2 x 8 x 3 of them on an SM

// Sums of N values over the threads of a row.  TPR = 0: the row is the whole
// CTA; two buffers, so one barrier per sum.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*sm)[NORM_WARPS][N], int &phase) {
#pragma unroll
    for (int o = (TPR ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(ALL, v[k], o);
    if (TPR == 0) {
        const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) sm[phase][warp][k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = 0.f;
#pragma unroll 4
        for (int i = 0; i < warps; ++i)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += sm[phase][i][k];
        phase ^= 1;
    }
}

// Whether the rounding of the mean is most of what the squares about it show,
// or made them overflow: a row that is all but constant.
__device__ __forceinline__ bool is_off(float var, float square) { return var < 0.75f * square || square == INFINITY; }

// A row's places in one thread, as pairs of floats: E / VEC packs, the row's
// threads apart, in groups of G places.  A row takes as few threads as hold
// it, so its first half is inside the row for every thread, and at most the
// last group is skipped; only rows of up to 32 places (TPR = 2) can be shorter.
// FULL: every place is inside (16 tpr places), and nothing is asked.
template <typename T, int VEC, int TPR, bool FULL>
struct Places {
    static constexpr int G = VEC > 4 ? VEC : 4, NG = NORM_E / G, PG = G / VEC;
    f2 v[NORM_E / 2];
    static __device__ __forceinline__ bool has(int g, int groups) {  // group g of a row has places (for some thread)
        return FULL || (TPR == 2 ? g < groups : G == NORM_E / 2 || g < NG - 1 || groups == NG);
    }
    static constexpr bool sure(int pack) { return FULL || (TPR != 2 && pack < NORM_E / VEC / 2); }
    // places outside the row: 0, or as its last ones
    template <bool LAST = false>
    __device__ __forceinline__ void load(const char *row, int t, int tpr, int dim, int groups) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if (has(g, groups)) {
                alignas(16) T e[G];
#pragma unroll
                for (int k = 0; k < PG; ++k) {
                    int j = (t + (g * PG + k) * tpr) * VEC;
                    if (LAST) j = min(j, dim - VEC);
                    Pack<T, VEC> p;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) p.v[i] = from_f<T>(0.f);
                    if (sure(g * PG + k) || j < dim) p = *(const Pack<T, VEC> *)(row + j * (int)sizeof(T));
#pragma unroll
                    for (int i = 0; i < VEC; ++i) e[k * VEC + i] = p.v[i];
                }
#pragma unroll
                for (int i = 0; i < G / 2; ++i) v[g * G / 2 + i] = to_f2(&e[2 * i]);
            }
        }
    }
};

// Group g of a row, rounded and stored.
template <typename T, int VEC, int TPR, bool FULL>
__device__ __forceinline__ void store_group(T *row, const f2 *v, int g, int t, int tpr, int dim) {
    using P = Places<T, VEC, TPR, FULL>;
    alignas(16) T o[P::G];
#pragma unroll
    for (int i = 0; i < P::G / 2; ++i) from_f2(&o[2 * i], v[i]);
#pragma unroll
    for (int k = 0; k < P::PG; ++k) {
        const int j = (t + (g * P::PG + k) * tpr) * VEC;
        if (P::sure(g * P::PG + k) || j < dim) {
            Pack<T, VEC> q;
#pragma unroll
            for (int i = 0; i < VEC; ++i) q.v[i] = o[k * VEC + i];
            *(Pack<T, VEC> *)(row + j) = q;
        }
    }
}

// A thread's weights and biases.
template <typename T, int VEC>
__device__ __forceinline__ void load_weights(f2 *to, const void *w, bool f32, float none, int t, int tpr, int dim) {
#pragma unroll
    for (int i = 0; i < NORM_E / 2; ++i) {
        float u[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int e = 2 * i + h, j = (t + e / VEC * tpr) * VEC + e % VEC;
            u[h] = w && j < dim ? load_as<T>(w, f32, j) : none;
        }
        to[i] = make_f2(u[0], u[1]);
    }
}

// An array's rows on their way through the ring.  Rows without a gap are one
// span of a slot, others a span each, in pitches of whole 16-byte blocks.
// ALIGNED: every row starts on 16 bytes.
template <typename T, bool ALIGNED>
struct RowStream {
    const char *x, *end, *at;  // the array, and the row that is fetched next
    int64_t stride, hop;       // bytes from row to row, from fetch to fetch
    int bytes, pitch;
    bool dense;
    __device__ __forceinline__ RowStream(const void *x, int64_t stride, int64_t rows, int dim, int64_t first, int64_t step)
        : x((const char *)x), end((const char *)x + ((rows - 1) * stride + dim) * (int64_t)sizeof(T)),
          at((const char *)x + first * stride * (int64_t)sizeof(T)), stride(stride * (int64_t)sizeof(T)),
          hop(step * stride * (int64_t)sizeof(T)), bytes(dim * (int)sizeof(T)), dense(stride == dim) {
        pitch = dense ? bytes : ((bytes + 15) & ~15) + 16;
    }
    __device__ __forceinline__ void fetch(char *slot, int n, int t, int threads) const {
        if (dense)
            copy_span<T, ALIGNED>(slot, at, n * bytes, x, end, t, threads);
        else
            for (int k = 0; k < n; ++k) copy_span<T, ALIGNED>(slot + k * pitch, at + k * stride, bytes, x, end, t, threads);
    }
    __device__ __forceinline__ void skip() { at += hop; }
    // where row k of the slot that starts with row r0 starts
    __device__ __forceinline__ const char *row(const char *slot, uint32_t r0, int k) const {
        const char *p = slot + k * pitch;
        if (ALIGNED) return p;
        const uint32_t from = (uint32_t)(uintptr_t)x + (r0 + (dense ? 0 : k)) * (uint32_t)stride;  // the low bits are right
        return p + (from & 15);
    }
};

extern __shared__ __align__(16) char norm_ring[];

template <typename T, int VEC, int TPR, bool FULL>
struct NormFwd {
    using P = Places<T, VEC, TPR, FULL>;
    const NormArgs &a;
    const int t, tpr;
    f2 w[NORM_E / 2], b[NORM_E / 2];
    float (*sm1)[NORM_WARPS][1];
    float (*sm2)[NORM_WARPS][2];
    int phase1 = 0, phase2 = 0;

    // x - m; the mean of that, and of its square
    __device__ __forceinline__ void centre(P &x, float m, float &delta, float &square) {
        const float inv = 1.f / (float)a.dim;
        const bool whole = FULL || NORM_E * tpr == a.dim;
        const f2 nm = both(-m);
        f2 u = both(0.f), v = both(0.f);
#pragma unroll
        for (int g = 0; g < P::NG; ++g)
            if (P::has(g, a.groups))
#pragma unroll
                for (int i = g * P::G / 2; i < (g + 1) * P::G / 2; ++i) {
                    x.v[i] = x.v[i] + nm;
                    if (!whole && !P::sure(2 * i / VEC)) {
                        float2 c = parts(x.v[i]);
                        if ((t + 2 * i / VEC * tpr) * VEC >= a.dim) c.x = 0.f;
                        if ((t + (2 * i + 1) / VEC * tpr) * VEC >= a.dim) c.y = 0.f;
                        x.v[i] = make_f2(c.x, c.y);
                    }
                    u = u + x.v[i];
                    v = fma2(x.v[i], x.v[i], v);
                }
        float s2[2] = {parts(u).x + parts(u).y, parts(v).x + parts(v).y};
        row_sum<TPR>(s2, sm2, phase2);
        delta = s2[0] * inv, square = s2[1] * inv;
    }
    // AGAIN: only rows that are off, with a better mean.  Whether the row is (behind the last row: whatever).
    template <bool AGAIN>
    __device__ __forceinline__ bool row(const char *from, uint32_t r, bool valid) {
        const int dim = a.dim, groups = a.groups;
        P x;
        x.load(from, t, tpr, dim, groups);
        f2 s = both(0.f);
#pragma unroll
        for (int g = 0; g < P::NG; ++g)
            if (P::has(g, groups))
#pragma unroll
                for (int i = g * P::G / 2; i < (g + 1) * P::G / 2; ++i) s = s + x.v[i];
        float s1[1] = {parts(s).x + parts(s).y};
        row_sum<TPR>(s1, sm1, phase1);
        float m = s1[0] * (1.f / (float)dim), delta, square;
        centre(x, m, delta, square);
        if (AGAIN) {
            valid = valid && is_off(fmaxf(square - delta * delta, 0.f), square);
            m += delta;
            x.load(from, t, tpr, dim, groups);
            centre(x, m, delta, square);
        }
        const float var = fmaxf(square - delta * delta, 0.f), q = rsqrtf(var + a.eps);  // 2 units: no more than the sums
        if (valid) {
            T *y = (T *)((char *)a.y + (uint64_t)r * (uint32_t)(dim * (int)sizeof(T)));
            const f2 rr = both(q), back = both(-delta * q);
#pragma unroll
            for (int g = 0; g < P::NG; ++g)
                if (P::has(g, groups)) {
                    f2 o[P::G / 2];
#pragma unroll
                    for (int i = 0; i < P::G / 2; ++i)
                        o[i] = fma2(fma2(x.v[g * P::G / 2 + i], rr, back), w[g * P::G / 2 + i], b[g * P::G / 2 + i]);
                    store_group<T, VEC, TPR, FULL>(y, o, g, t, tpr, dim);
                }
            if (a.stats && t == 0) {
                float *st = a.stats + (uint64_t)r * 3;
                st[0] = m, st[1] = delta, st[2] = q;
            }
        }
        return is_off(var, square);
    }
};

// 24 warps an SM by registers.
template <typename T, int VEC, int TPR, bool FULL>
__global__ void __launch_bounds__(TPR ? 256 : 768, TPR ? 3 : 1) norm_fwd_kernel(const NormArgs a) {
    __shared__ float sm1[TPR ? 1 : 2][NORM_WARPS][1], sm2[TPR ? 1 : 2][NORM_WARPS][2];
    pdl_enter();
    constexpr int S = TPR ? NORM_FWD_SLOTS : 3, PER = 32 / (TPR ? TPR : 32);
    const int lane = threadIdx.x & 31, warp = TPR ? threadIdx.x >> 5 : 0;
    const uint32_t rows = (uint32_t)a.rows, chunk = TPR ? a.chunk : 1;
    // this warp's (TPR = 0: CTA's) first row, and how far it is to its next slot's
    const uint32_t first = (TPR ? blockIdx.x * 8 + warp : blockIdx.x) * chunk, step = gridDim.x * (TPR ? 8 : 1) * chunk;
    NormFwd<T, VEC, TPR, FULL> k{a, TPR ? lane & (TPR - 1) : (int)threadIdx.x, TPR ? TPR : (int)blockDim.x};
    k.sm1 = sm1, k.sm2 = sm2;
    load_weights<T, VEC>(k.w, a.w, a.wf32, 1.f, k.t, k.tpr, a.dim);
    load_weights<T, VEC>(k.b, a.b, a.wf32, 0.f, k.t, k.tpr, a.dim);
    RowStream<T, sizeof(T) * VEC == 16> xs(a.x, a.x_stride, a.rows, a.dim, first, step);
    char *ring = norm_ring + warp * S * a.slot_bytes;
    uint32_t ahead = first;
    auto fetch = [&](int slot) {
        if (ahead < rows) xs.fetch(ring + slot * a.slot_bytes, (int)min(chunk, rows - ahead), TPR ? lane : threadIdx.x, TPR ? 32 : blockDim.x);
        copies_end_group();
        xs.skip(), ahead += step;
    };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) fetch(s);
    int slot = 0;
    bool again = false;
    for (uint32_t r0 = first; r0 < rows; r0 += step) {
        const int free = slot == 0 ? S - 1 : slot - 1;
        const char *at = ring + slot * a.slot_bytes;
        if (TPR) {
            fetch(free);
            copies_wait_but<S - 1>();
            __syncwarp();
            for (uint32_t q = 0; q < chunk; q += PER) {  // whole warps: every lane takes part in the shuffles
                const uint32_t mine = q + lane / (TPR ? TPR : 32);
                again |= k.template row<false>(xs.row(at, r0, mine), r0 + mine, r0 + mine < rows);  // behind the last row: whatever is there, for nobody
            }
            __syncwarp();
        } else {
            copies_wait_but<S - 2>();
            __syncthreads();  // this row has arrived, and the last one's slot has been read
            fetch(free);
            again |= k.template row<false>(xs.row(at, r0, 0), r0, true);
        }
        slot = slot + 1 == S ? 0 : slot + 1;
    }
    copies_wait_but<0>();
    if (!(TPR ? __any_sync(ALL, again) : again)) return;
    for (uint32_t r0 = first; r0 < rows; r0 += step)
        for (uint32_t q = 0; q < chunk; q += PER) {
            const uint32_t r = r0 + q + (TPR ? lane / (TPR ? TPR : 32) : 0);
            k.template row<true>((const char *)a.x + min(r, rows - 1) * a.x_stride * (int64_t)sizeof(T), r, r < rows);
        }
}

template <typename T, int VEC, int TPR, bool FULL>
struct NormBwd {
    using P = Places<T, VEC, TPR, FULL>;
    const NormArgs &a;
    const int t, tpr;
    f2 w[NORM_E / 2], aw[NORM_E / 2], ab[NORM_E / 2];
    float (*sm)[NORM_WARPS][2];
    int phase = 0;

    // Places outside the row have dy = 0 and x = 0, so no part in any sum while their xh is a number.  It is not where the
    // mean is that large against the spread; AGAIN: dx of such rows, with other places in theirs.  Whether the row may be one.
    template <bool AGAIN>
    __device__ __forceinline__ bool row(const char *fx, const char *fy, const float *st, uint32_t r, bool valid) {
        const int dim = a.dim, groups = a.groups;
        const float inv = 1.f / (float)dim;
        P x, d;
        x.template load<AGAIN>(fx, t, tpr, dim, groups);
        d.load(fy, t, tpr, dim, groups);
        const float q = st[2];
        if (AGAIN) valid = valid && !(fabsf(st[0] * q) < 1e38f);
        const f2 nm = both(-st[0]), rr = both(q), off = both(-st[1] * q);
        f2 s = both(0.f), v = both(0.f);
#pragma unroll
        for (int g = 0; g < P::NG; ++g)
            if (P::has(g, groups))
#pragma unroll
                for (int i = g * P::G / 2; i < (g + 1) * P::G / 2; ++i) {
                    x.v[i] = fma2(x.v[i] + nm, rr, off);
                    const f2 gg = d.v[i] * w[i];
                    s = s + gg;
                    v = fma2(gg, x.v[i], v);
                    if (AGAIN) continue;
                    aw[i] = fma2(d.v[i], x.v[i], aw[i]);
                    ab[i] = ab[i] + d.v[i];
                }
        if (!a.y) return false;
        float sums[2] = {parts(s).x + parts(s).y, parts(v).x + parts(v).y};
        row_sum<TPR>(sums, sm, phase);
        if (valid) {
            const f2 k1 = both(-q * (sums[0] * inv)), k2 = both(-q * (sums[1] * inv));
            T *dx = (T *)((char *)a.y + (uint64_t)r * (uint32_t)(dim * (int)sizeof(T)));
#pragma unroll
            for (int g = 0; g < P::NG; ++g)
                if (P::has(g, groups)) {
                    f2 o[P::G / 2];
#pragma unroll
                    for (int i = 0; i < P::G / 2; ++i) {
                        const int e = g * P::G / 2 + i;
                        o[i] = fma2(x.v[e], k2, fma2(d.v[e] * w[e], rr, k1));
                    }
                    store_group<T, VEC, TPR, FULL>(dx, o, g, t, tpr, dim);
                }
        }
        return !FULL && sums[1] != sums[1];
    }
};

// dx of the warp's (CTA's) rows whose xh is no number outside the row.  Out of line, the walk keeps its registers.
template <typename T, int VEC, int TPR>
__device__ __noinline__ void norm_bwd_again(const NormArgs a, uint32_t first, uint32_t step, float (*sm)[NORM_WARPS][2]) {
    constexpr int PER = 32 / (TPR ? TPR : 32);
    const uint32_t lane = threadIdx.x & 31, rows = (uint32_t)a.rows, chunk = TPR ? a.chunk : 1;
    if (!TPR) __syncthreads();  // the walk's sums have been read
    NormBwd<T, VEC, TPR, false> k{a, TPR ? (int)lane & (TPR - 1) : (int)threadIdx.x, TPR ? TPR : (int)blockDim.x};
    k.sm = sm;
    load_weights<T, VEC>(k.w, a.w, a.wf32, 1.f, k.t, k.tpr, a.dim);
    for (uint32_t r0 = first; r0 < rows; r0 += step)
        for (uint32_t q = 0; q < chunk; q += PER) {
            const uint32_t mine = r0 + q + (TPR ? lane / (TPR ? TPR : 32) : 0), r = min(mine, rows - 1);
            k.template row<true>((const char *)a.x + r * a.x_stride * (int64_t)sizeof(T), (const char *)a.dy + r * a.dy_stride * (int64_t)sizeof(T),
                                 a.stats + (uint64_t)r * 3, r, mine < rows);
        }
}

// 16 warps an SM by registers.
template <typename T, int VEC, int TPR, bool FULL>
__global__ void __launch_bounds__(TPR ? 256 : 512, TPR ? 2 : 1) norm_bwd_kernel(const NormArgs a) {
    constexpr int S = NORM_BWD_SLOTS, PER = 32 / (TPR ? TPR : 32);
    __shared__ float sm[TPR ? 1 : 2][NORM_WARPS][2];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = TPR ? threadIdx.x >> 5 : 0, dim = a.dim;
    const uint32_t rows = (uint32_t)a.rows, chunk = TPR ? a.chunk : 1;
    const uint32_t first = (TPR ? blockIdx.x * 8 + warp : blockIdx.x) * chunk, step = gridDim.x * (TPR ? 8 : 1) * chunk;
    NormBwd<T, VEC, TPR, FULL> k{a, TPR ? lane & (TPR - 1) : (int)threadIdx.x, TPR ? TPR : (int)blockDim.x};
    k.sm = sm;
    load_weights<T, VEC>(k.w, a.w, a.wf32, 1.f, k.t, k.tpr, dim);
#pragma unroll
    for (int i = 0; i < NORM_E / 2; ++i) k.aw[i] = k.ab[i] = both(0.f);
    float *out = a.part + (int64_t)blockIdx.x * 2 * dim;
    RowStream<T, sizeof(T) * VEC == 16> xs(a.x, a.x_stride, a.rows, dim, first, step), ys(a.dy, a.dy_stride, a.rows, dim, first, step);
    char *ring = norm_ring + warp * S * a.slot_bytes;
    uint32_t ahead = first;
    const int t = TPR ? lane : threadIdx.x, threads = TPR ? 32 : blockDim.x;
    // a slot: x's rows, dy's rows, three statistics each
    auto fetch = [&](int slot) {
        if (ahead < rows) {
            char *to = ring + slot * a.slot_bytes;
            const int n = (int)min(chunk, rows - ahead);
            if (TPR && n < (int)chunk) {  // behind the last row: zeros, which add nothing to any sum
                for (int i = 16 * lane; i < a.slot_bytes; i += 512) *(uint4 *)(to + i) = make_uint4(0, 0, 0, 0);
                __syncwarp();
            }
            xs.fetch(to, n, t, threads);
            ys.fetch(to + a.x_bytes, n, t, threads);
            const uint32_t st = (uint32_t)__cvta_generic_to_shared(to + 2 * a.x_bytes);
            for (int i = t; i < 3 * n; i += threads) copy4(st + 4 * i, a.stats + (uint64_t)ahead * 3 + i);
        }
        copies_end_group();
        xs.skip(), ys.skip(), ahead += step;
    };
    bool again = false;
    auto row = [&](const char *at, uint32_t r0, uint32_t q, bool valid) {
        again |= k.template row<false>(xs.row(at, r0, q), ys.row(at + a.x_bytes, r0, q), (const float *)(at + 2 * a.x_bytes) + 3 * q, r0 + q, valid);
    };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) fetch(s);
    int slot = 0;
    for (uint32_t r0 = first; r0 < rows; r0 += step) {
        const int free = slot == 0 ? S - 1 : slot - 1;
        const char *at = ring + slot * a.slot_bytes;
        if (TPR) {
            fetch(free);
            copies_wait_but<S - 1>();
            __syncwarp();
            for (uint32_t q = lane / (TPR ? TPR : 32); q < chunk; q += PER) row(at, r0, q, r0 + q < rows);
            __syncwarp();
        } else {
            copies_wait_but<S - 2>();
            __syncthreads();  // this row has arrived, and the last one's slot has been read
            fetch(free);
            row(at, r0, 0, true);
        }
        slot = slot + 1 == S ? 0 : slot + 1;
    }
    copies_wait_but<0>();
    if (a.part && TPR) {
        const int sub = lane / (TPR ? TPR : 32);
        // the CTA's rows: those of a warp by shuffles, then its eight warps, in the ring's memory
        __syncthreads();
        float *cw = (float *)norm_ring, *cb = cw + 8 * dim;
#pragma unroll
        for (int e = 0; e < NORM_E; ++e) {
            float u = e % 2 ? parts(k.aw[e / 2]).y : parts(k.aw[e / 2]).x;
            float v = e % 2 ? parts(k.ab[e / 2]).y : parts(k.ab[e / 2]).x;
#pragma unroll
            for (int o = TPR ? TPR : 32; o < 32; o <<= 1) {
                u += __shfl_xor_sync(ALL, u, o);
                v += __shfl_xor_sync(ALL, v, o);
            }
            const int j = (k.t + e / VEC * k.tpr) * VEC + e % VEC;
            if (sub == 0 && j < dim) cw[warp * dim + j] = u, cb[warp * dim + j] = v;
        }
        __syncthreads();
        for (int j = threadIdx.x; j < dim; j += 256) {
            float u = 0.f, v = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) u += cw[i * dim + j], v += cb[i * dim + j];
            out[j] = u, out[dim + j] = v;
        }
    } else if (a.part) {
#pragma unroll
        for (int e = 0; e < NORM_E; ++e) {
            const int j = (k.t + e / VEC * k.tpr) * VEC + e % VEC;
            const float2 u = parts(k.aw[e / 2]), v = parts(k.ab[e / 2]);
            if (j < dim) out[j] = e % 2 ? u.y : u.x, out[dim + j] = e % 2 ? v.y : v.x;
        }
    }
    if constexpr (!FULL)
        if (TPR ? __any_sync(ALL, again) : again) norm_bwd_again<T, VEC, TPR>(a, first, step, sm);
}

// Sums of the weights' gradients over the CTAs, in a fixed order and 64 bits;
// a CTA has COLS columns, so that short rows fill more than a few SMs.
template <typename T, int COLS>
__global__ void __launch_bounds__(512) norm_dw_kernel(const float *part, int parts, int dim, void *dw, void *db,
                                                      int wf32) {
    constexpr int LANES = 512 / COLS;
    __shared__ double red[LANES][COLS + 1];
    pdl_enter();
    const int c = threadIdx.x % COLS, l = threadIdx.x / COLS;
    const int64_t n = 2 * (int64_t)dim, j = (int64_t)blockIdx.x * COLS + c;
    double s = 0;
    if (j < n)
#pragma unroll 8
        for (int i = l; i < parts; i += LANES) s += (double)part[i * n + j];
    red[l][c] = s;
    __syncthreads();
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        if (l < o) red[l][c] += red[l + o][c];
        __syncthreads();
    }
    if (l == 0 && j < n) {
        const double v = red[0][c];
        void *to = j < dim ? dw : db;
        const int64_t at = j < dim ? j : j - dim;
        if (to) {
            if (wf32)
                ((float *)to)[at] = (float)v;
            else
                ((T *)to)[at] = from_f<T>((float)v);
        }
    }
}

// Rows longer than the registers hold: a CTA per row that reads it again for
// each sum (from L2, where one row stays), and for the weights' gradients a
// thread per column over a share of the rows.  One element a load: 4,096 rows
// of 8,200 bfloat16 take 80 us forward and 272 both ways, of 16,384 145 and 591
// (8,192 places, in registers: 42 and 101).
template <typename T>
__global__ void __launch_bounds__(512, 4) norm_fwd_long_kernel(const NormArgs a) {
    __shared__ float sm1[2][NORM_WARPS][1], sm2[2][NORM_WARPS][2];
    pdl_enter();
    const float inv = 1.f / (float)a.dim;
    int phase1 = 0, phase2 = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.x_stride;
        T *y = (T *)a.y + row * a.dim;
        float s1[1] = {0.f}, s2[2];
#pragma unroll 8
        for (int j = threadIdx.x; j < a.dim; j += 512) s1[0] += to_f(x[j]);
        row_sum<0>(s1, sm1, phase1);
        float m = s1[0] * inv;
        for (bool last = false;; last = true) {
            s2[0] = s2[1] = 0.f;
#pragma unroll 8
            for (int j = threadIdx.x; j < a.dim; j += 512) {
                const float c = to_f(x[j]) - m;
                s2[0] += c;
                s2[1] += c * c;
            }
            row_sum<0>(s2, sm2, phase2);
            const float delta = s2[0] * inv, square = s2[1] * inv;
            const float var = fmaxf(square - delta * delta, 0.f), r = 1.f / sqrtf(var + a.eps);
#pragma unroll 4
            for (int j = threadIdx.x; j < a.dim; j += 512)
                y[j] = from_f<T>(((to_f(x[j]) - m) - delta) * r * (a.w ? load_as<T>(a.w, a.wf32, j) : 1.f) +
                                 (a.b ? load_as<T>(a.b, a.wf32, j) : 0.f));
            if (a.stats && threadIdx.x == 0) {
                float *st = a.stats + row * 3;
                st[0] = m, st[1] = delta, st[2] = r;
            }
            if (__builtin_expect(last || !is_off(var, square), 1)) break;
            m += delta;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(512) norm_dx_long_kernel(const NormArgs a) {
    __shared__ float sm[2][NORM_WARPS][2];
    pdl_enter();
    const float inv = 1.f / (float)a.dim;
    int phase = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.x_stride, *dy = (const T *)a.dy + row * a.dy_stride;
        T *dx = (T *)a.y + row * a.dim;
        const float m = a.stats[row * 3], delta = a.stats[row * 3 + 1], r = a.stats[row * 3 + 2];
        float s[2] = {0.f, 0.f};
#pragma unroll 4
        for (int j = threadIdx.x; j < a.dim; j += 512) {
            const float g = to_f(dy[j]) * (a.w ? load_as<T>(a.w, a.wf32, j) : 1.f);
            s[0] += g;
            s[1] += g * (((to_f(x[j]) - m) - delta) * r);
        }
        row_sum<0>(s, sm, phase);
        const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll 4
        for (int j = threadIdx.x; j < a.dim; j += 512) {
            const float g = to_f(dy[j]) * (a.w ? load_as<T>(a.w, a.wf32, j) : 1.f);
            dx[j] = from_f<T>(r * (g - c1 - ((to_f(x[j]) - m) - delta) * r * c2));
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_part_long_kernel(const NormArgs a) {
    pdl_enter();
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t share = (a.rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * share;
    const int64_t r1 = r0 + share < a.rows ? r0 + share : a.rows;
    if (j >= a.dim) return;
    float u = 0.f, v = 0.f;
#pragma unroll 4
    for (int64_t row = r0; row < r1; ++row) {
        const float d = to_f(((const T *)a.dy)[row * a.dy_stride + j]);
        const float x = to_f(((const T *)a.x)[row * a.x_stride + j]);
        u += d * (((x - a.stats[row * 3]) - a.stats[row * 3 + 1]) * a.stats[row * 3 + 2]);
        v += d;
    }
    float *out = a.part + (int64_t)blockIdx.y * 2 * a.dim;
    out[j] = u, out[a.dim + j] = v;
}

// How a call is laid out.
struct NormPlan {
    int kind;     // 0: warp, 1: CTA, 2: long
    int tpr, groups, threads, chunk, x_bytes, slot_bytes;
    size_t smem;
    int64_t grid; // CTAs; kind 2: rows of partial sums
};

constexpr int NORM_LONG_PARTS = 64;

static NormPlan norm_plan(int64_t rows, int32_t dim, int es, int vec, int sms, bool dense, bool backward) {
    NormPlan p{};
    if (dim > 32 * NORM_WARPS * NORM_E) {
        p.kind = 2, p.threads = 512;
        p.grid = rows < NORM_LONG_PARTS ? rows : NORM_LONG_PARTS;
        return p;
    }
    const int64_t warps = (int64_t)sms * (backward ? 16 : 24);  // resident, by the kernels' registers
    const int row = ((dim * es + 15) & ~15) + 16;               // a slot's bytes for a row, wherever it starts
    if (dim <= 32 * NORM_E) {
        p.threads = 256, p.tpr = 2;
        while (p.tpr * NORM_E < dim) p.tpr *= 2;
        const int per = 32 / p.tpr;
        // slots of 2 KB of x: copies in flight cover the latency, and a slot's cost is shared by several rows;
        // but no more rows than there are for a warp, and in the backward pass, where a row has dy's and 12 bytes of
        // statistics too, no more than let two CTAs' rings stand on an SM (short rows are mostly statistics)
        const int bytes = dense ? dim * es : row;
        int64_t sets = 2048 / (per * bytes), most = rows / (warps * per);
        if (backward) most = min(most, (int64_t)(NORM_BWD_SLOT - 80) / (per * (2 * bytes + 12)));  // 80: three roundings up
        sets = min(sets, most);
        p.chunk = per * (int)(sets < 1 ? 1 : sets);
        const int64_t need = (rows + 8 * (int64_t)p.chunk - 1) / (8 * (int64_t)p.chunk);
        p.grid = need < warps / 8 ? need : warps / 8;
    } else {
        p.kind = 1, p.chunk = 1;
        p.threads = 32 * ((dim + 32 * NORM_E - 1) / (32 * NORM_E));
        p.tpr = p.threads;
        const int64_t cap = (int64_t)sms * ((backward ? 16 : 24) * 32 / p.threads);  // whole CTAs of an SM
        p.grid = rows < cap ? rows : cap;
    }
    const int group = p.tpr * (vec > 4 ? vec : 4);
    p.groups = (dim + group - 1) / group;
    p.x_bytes = dense ? ((p.chunk * dim * es + 15) & ~15) + 16 : p.chunk * row;
    p.slot_bytes = backward ? 2 * p.x_bytes + ((12 * p.chunk + 15) & ~15) : p.x_bytes;
    p.smem = (size_t)p.slot_bytes * (p.kind ? 3 : 8 * (backward ? NORM_BWD_SLOTS : NORM_FWD_SLOTS));
    if (backward && !p.kind && p.smem < 64 * (size_t)dim) p.smem = 64 * (size_t)dim;  // the eight warps' two sums
    return p;
}

// Elements of the widest load that every row of every operand allows; 0
// where one is not even aligned to its elements.
static int norm_vec(int es, int32_t dim, const void *const *ptrs, const int64_t *strides, int n) {
    uintptr_t bits = (uintptr_t)dim * es;
    for (int i = 0; i < n; ++i) bits |= (uintptr_t)ptrs[i] | (uintptr_t)(strides[i] * es);
    if (bits & (es - 1)) return 0;
    if ((bits & 15) == 0) return 16 / es;
    return es == 2 && (bits & 3) == 0 ? 2 : 1;
}

template <typename T, int VEC, int TPR, bool FULL, bool BWD>
static cudaError_t norm_launch_as(const NormPlan &p, const NormArgs &a, cudaStream_t s) {
    auto *kernel = BWD ? norm_bwd_kernel<T, VEC, TPR, FULL> : norm_fwd_kernel<T, VEC, TPR, FULL>;
    static std::atomic<uint64_t> raised{0};  // devices on which the kernel may have all of an SM's shared memory
    if (p.smem > 40 * 1024) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = 1ull << (dev & 63);
        if (!(raised.load(std::memory_order_relaxed) & bit)) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
            if (e != cudaSuccess) return e;
            raised.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    return launch_pdl(kernel, (unsigned)p.grid, (unsigned)p.threads, p.smem, s, a);
}

template <typename T, int VEC, int TPR, bool BWD>
static cudaError_t norm_launch_tpr(const NormPlan &p, const NormArgs &a, cudaStream_t s) {
    constexpr bool WIDE = VEC * sizeof(T) == 16;  // rows of other widths are seldom full
    if (WIDE && a.dim == NORM_E * p.tpr) return norm_launch_as<T, VEC, TPR, WIDE, BWD>(p, a, s);
    return norm_launch_as<T, VEC, TPR, false, BWD>(p, a, s);
}

template <typename T, int VEC, bool BWD>
static cudaError_t norm_launch(const NormPlan &p, const NormArgs &a, cudaStream_t s) {
    if (p.kind == 1) return norm_launch_tpr<T, VEC, 0, BWD>(p, a, s);
    switch (p.tpr) {
        case 2: return norm_launch_tpr<T, VEC, 2, BWD>(p, a, s);
        case 4: return norm_launch_tpr<T, VEC, 4, BWD>(p, a, s);
        case 8: return norm_launch_tpr<T, VEC, 8, BWD>(p, a, s);
        case 16: return norm_launch_tpr<T, VEC, 16, BWD>(p, a, s);
        default: return norm_launch_tpr<T, VEC, 32, BWD>(p, a, s);
    }
}

template <typename T, bool BWD>
static cudaError_t norm_rows(const NormPlan &p, const NormArgs &a, int vec, int sms, cudaStream_t s) {
    if (p.kind == 2) {
        const int64_t cap = (int64_t)sms * 4;
        const unsigned g = (unsigned)(a.rows < cap ? a.rows : cap);
        if (!BWD) return launch_pdl(norm_fwd_long_kernel<T>, g, 512, 0, s, a);
        cudaError_t e = a.y ? launch_pdl(norm_dx_long_kernel<T>, g, 512, 0, s, a) : cudaSuccess;
        if (e != cudaSuccess || !a.part) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((a.dim + 255) / 256), (unsigned)p.grid);
        cfg.blockDim = dim3(256);
        cfg.stream = s;
        return cudaLaunchKernelEx(&cfg, norm_part_long_kernel<T>, a);
    }
    if (vec == 16 / (int)sizeof(T)) return norm_launch<T, 16 / sizeof(T), BWD>(p, a, s);
    if (sizeof(T) == 2 && vec == 2) return norm_launch<T, sizeof(T) == 2 ? 2 : 1, BWD>(p, a, s);
    return norm_launch<T, 1, BWD>(p, a, s);
}

template <bool BWD>
static cudaError_t norm_typed(int dtype, const NormPlan &p, const NormArgs &a, int vec, int sms, cudaStream_t s) {
    if (dtype == JQ_F32) return norm_rows<float, BWD>(p, a, vec, sms, s);
    if (dtype == JQ_F16) return norm_rows<__half, BWD>(p, a, vec, sms, s);
    return norm_rows<__nv_bfloat16, BWD>(p, a, vec, sms, s);
}

static int norm_check(const void *x, int64_t x_stride, int64_t rows, int32_t dim, int32_t dtype, int32_t wdtype) {
    if (!x || rows <= 0 || dim <= 0) return fail(JQ_ERR_ARG, "layer norm needs at least one row of at least one place");
    if (!known_dtype(dtype)) return fail(JQ_ERR_ARG, "layer norm: unknown dtype");
    if (wdtype != JQ_F32 && wdtype != dtype) return fail(JQ_ERR_ARG, "layer norm: weights are float32 or of x's type");
    if (x_stride < 0) return fail(JQ_ERR_ARG, "layer norm: negative row stride");
    if (rows > INT32_MAX || dim > 1 << 30) return fail(JQ_ERR_CAPACITY, "layer norm: more than 2^31 - 1 rows or 2^30 places");
    return JQ_OK;
}

}  // namespace jq

using namespace jq;

extern "C" {

int64_t jq_layer_norm_scratch_floats(int64_t rows, int32_t dim) {
    int sms = 0;
    if (rows <= 0 || dim <= 0 || device_sms(sms)) return 0;
    // whatever the type and the strides will be
    int64_t g = 0;
    for (int es = 2; es <= 4; es += 2)
        for (int dense = 0; dense < 2; ++dense) {
            const int64_t h = norm_plan(rows, dim, es, 1, sms, dense, true).grid;
            g = h > g ? h : g;
        }
    return g * 2 * (int64_t)dim;
}

int jq_layer_norm(const void *d_x, int64_t x_stride, const void *d_weight, const void *d_bias, int64_t rows,
                  int32_t dim, int32_t dtype, int32_t wdtype, float eps, void *d_y, float *d_stats, void *stream) {
    int rc = norm_check(d_x, x_stride, rows, dim, dtype, wdtype), sms;
    if (rc) return rc;
    if (!d_y) return fail(JQ_ERR_ARG, "layer norm output missing");
    if (!(eps >= 0.f)) return fail(JQ_ERR_ARG, "layer norm: eps must not be negative");
    if ((rc = device_sms(sms))) return rc;
    NormArgs a{};
    a.x = d_x, a.w = d_weight, a.b = d_bias, a.y = d_y, a.stats = d_stats;
    a.x_stride = x_stride, a.rows = rows, a.dim = dim, a.wf32 = wdtype == JQ_F32, a.eps = eps;
    const void *ptrs[] = {d_x, d_y};
    const int64_t strides[] = {rows > 1 ? x_stride : 0, rows > 1 ? dim : 0};
    const int vec = norm_vec(elem_size(dtype), dim, ptrs, strides, 2);
    if (!vec || (((uintptr_t)d_weight | (uintptr_t)d_bias) & (elem_size(wdtype) - 1)) || ((uintptr_t)d_stats & 3))
        return fail(JQ_ERR_ARG, "layer norm: an array is not aligned to its elements");
    const NormPlan p = norm_plan(rows, dim, elem_size(dtype), vec, sms, x_stride == dim, false);
    a.groups = p.groups, a.chunk = p.chunk, a.x_bytes = p.x_bytes, a.slot_bytes = p.slot_bytes;
    CU(norm_typed<false>(dtype, p, a, vec, sms, (cudaStream_t)stream));
    return JQ_OK;
}

int jq_layer_norm_backward(const void *d_x, int64_t x_stride, const void *d_weight, const void *d_dy,
                           int64_t dy_stride, const float *d_stats, int64_t rows, int32_t dim, int32_t dtype,
                           int32_t wdtype, void *d_dx, void *d_dweight, void *d_dbias, float *d_scratch,
                           void *stream) {
    int rc = norm_check(d_x, x_stride, rows, dim, dtype, wdtype), sms;
    if (rc) return rc;
    if (!d_dy || !d_stats || dy_stride < 0) return fail(JQ_ERR_ARG, "layer norm: gradient or statistics missing");
    if ((d_dweight || d_dbias) && !d_scratch) return fail(JQ_ERR_ARG, "layer norm: scratch missing");
    if (!d_dx && !d_dweight && !d_dbias) return fail(JQ_ERR_ARG, "layer norm: no gradient asked for");
    if ((rc = device_sms(sms))) return rc;
    NormArgs a{};
    a.x = d_x, a.w = d_weight, a.dy = d_dy, a.y = d_dx, a.stats = const_cast<float *>(d_stats);
    a.part = d_dweight || d_dbias ? d_scratch : nullptr;
    a.x_stride = x_stride, a.dy_stride = dy_stride, a.rows = rows, a.dim = dim, a.wf32 = wdtype == JQ_F32;
    const void *ptrs[] = {d_x, d_dy, d_dx ? d_dx : d_x};
    const int64_t strides[] = {rows > 1 ? x_stride : 0, rows > 1 ? dy_stride : 0, rows > 1 ? dim : 0};
    const int vec = norm_vec(elem_size(dtype), dim, ptrs, strides, 3);
    if (!vec || (((uintptr_t)d_weight | (uintptr_t)d_dweight | (uintptr_t)d_dbias) & (elem_size(wdtype) - 1)) ||
        (((uintptr_t)d_stats | (uintptr_t)d_scratch) & 3))
        return fail(JQ_ERR_ARG, "layer norm: an array is not aligned to its elements");
    const NormPlan p = norm_plan(rows, dim, elem_size(dtype), vec, sms, x_stride == dim && dy_stride == dim, true);
    a.groups = p.groups, a.chunk = p.chunk, a.x_bytes = p.x_bytes, a.slot_bytes = p.slot_bytes;
    cudaStream_t s = (cudaStream_t)stream;
    CU(norm_typed<true>(dtype, p, a, vec, sms, s));
    if (!a.part) return JQ_OK;
    const int64_t sums = 2 * (int64_t)dim;
    const bool narrow = sums < 32 * (int64_t)sms;
    const unsigned g = (unsigned)(narrow ? (sums + 7) / 8 : (sums + 31) / 32);
    auto *add = dtype == JQ_F16 ? (narrow ? norm_dw_kernel<__half, 8> : norm_dw_kernel<__half, 32>)
                                : (narrow ? norm_dw_kernel<__nv_bfloat16, 8> : norm_dw_kernel<__nv_bfloat16, 32>);
    CU(launch_pdl(add, g, 512, 0, s, (const float *)a.part, (int)p.grid, (int)dim, d_dweight, d_dbias, (int)a.wf32));
    return JQ_OK;
}

}  // extern "C"
