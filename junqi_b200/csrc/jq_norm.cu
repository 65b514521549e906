// jq_norm.cu -- layer norm over the last axis, forward and backward.
//
//   mu = mean(x), s2 = mean((x - mu)^2), r = 1 / sqrt(s2 + eps)
//   xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum dy xh,  db = sum dy
//
// Bound: memory.  Forward moves 2 elements per place (x in, y out), backward
// 3 (x and dy in, dx out); 8 and 14 operations per place are far below what
// the SMs do meanwhile.  So every kernel reads a row once, keeps it in
// registers through its reductions, and has the next row's loads in flight
// while it works: a group of `tpr` threads (a power of two, part of a warp up
// to a whole CTA) holds E = 8 or 16 places of a row in each thread, walks the
// rows with a fixed stride, and keeps its places' weights, and in the
// backward pass their two gradient sums, in registers all the way.  The
// sums of the weights' gradients leave once per CTA and a second kernel adds
// them up in a fixed order, so equal calls give equal bits.
//
// Statistics are 32-bit.  The mean is taken twice: m, the rounded mean, then
// delta = mean(x - m), what the rounding left, so a row whose mean is large
// against its spread loses nothing (s2 = mean((x - m)^2) - delta^2, in which
// delta^2 is at rounding level).  The three numbers (m, delta, r) per row go
// to the backward pass.
#include "jq_ops.cuh"

namespace jq {

struct NormArgs {
    const void *x, *w, *b, *dy;
    void *y;                  // forward: y; backward: dx (may be NULL)
    float *stats;             // (rows, 3): m, delta, r
    float *part;              // backward: (grid, 2, dim) sums of dw and db, or NULL
    int64_t x_stride, dy_stride, rows;
    int32_t dim, tpr, wf32;
    float eps;
};

// Sums of N values over the `tpr` threads of a row.  BLOCK: the row is the
// whole CTA; two buffers, so one barrier per sum.
template <bool BLOCK, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int tpr, float (*sm)[16][N], int &phase) {
    if (BLOCK) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(ALL, v[k], o);
        const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) sm[phase][warp][k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = 0.f;
        for (int i = 0; i < warps; ++i)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += sm[phase][i][k];
        phase ^= 1;
    } else {
        for (int o = tpr >> 1; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(ALL, v[k], o);
    }
}

// A row's places in one thread: NV packs, `tpr` packs apart.
template <typename T, int VEC, int NV>
struct RowRegs {
    Pack<T, VEC> p[NV];
    __device__ __forceinline__ void load(const T *row, int t, int tpr, int dim, bool valid) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int j = (t + k * tpr) * VEC;
            if (valid && j < dim)
                p[k] = *(const Pack<T, VEC> *)(row + j);
            else
#pragma unroll
                for (int i = 0; i < VEC; ++i) p[k].v[i] = from_f<T>(0.f);
        }
    }
};

template <typename T, int VEC, int E, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : 256) norm_fwd_kernel(const NormArgs a) {
    constexpr int NV = E / VEC;
    __shared__ float sm1[2][16][1], sm2[2][16][2];
    pdl_enter();
    const int tpr = a.tpr, lane = threadIdx.x & 31;
    const int t = BLOCK ? threadIdx.x : lane & (tpr - 1);
    const int dim = a.dim;
    const float inv = 1.f / (float)dim;
    float w[E], b[E];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int j = (t + k * tpr) * VEC + i;
            w[k * VEC + i] = a.w && j < dim ? load_as<T>(a.w, a.wf32, j) : 1.f;
            b[k * VEC + i] = a.b && j < dim ? load_as<T>(a.b, a.wf32, j) : 0.f;
        }
    // rows are walked by whole warps (BLOCK: CTAs), so every lane takes part in the shuffles
    const int per = BLOCK ? 1 : 32 / tpr;
    const int64_t step = BLOCK ? (int64_t)gridDim.x : (int64_t)gridDim.x * 8 * per;
    int64_t first = BLOCK ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * per;
    const int sub = BLOCK ? 0 : lane / tpr;
    int phase1 = 0, phase2 = 0;
    RowRegs<T, VEC, NV> next;
    next.load((const T *)a.x + (first + sub) * a.x_stride, t, tpr, dim, first + sub < a.rows);
    for (; first < a.rows; first += step) {
        const int64_t row = first + sub;
        const bool valid = row < a.rows;
        RowRegs<T, VEC, NV> cur = next;
        next.load((const T *)a.x + (row + step) * a.x_stride, t, tpr, dim, row + step < a.rows);
        float s1[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) s1[0] += to_f(cur.p[k].v[i]);
        row_sum<BLOCK>(s1, tpr, sm1, phase1);
        const float m = s1[0] * inv;
        float s2[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float c = (t + k * tpr) * VEC < dim ? to_f(cur.p[k].v[i]) - m : 0.f;
                s2[0] += c;
                s2[1] += c * c;
            }
        row_sum<BLOCK>(s2, tpr, sm2, phase2);
        const float delta = s2[0] * inv;
        const float r = 1.f / sqrtf(fmaxf(s2[1] * inv - delta * delta, 0.f) + a.eps);
        if (valid) {
            T *y = (T *)a.y + row * dim;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = (t + k * tpr) * VEC;
                if (j >= dim) continue;
                Pack<T, VEC> o;
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    o.v[i] = from_f<T>(((to_f(cur.p[k].v[i]) - m) - delta) * r * w[k * VEC + i] + b[k * VEC + i]);
                *(Pack<T, VEC> *)(y + j) = o;
            }
            if (a.stats && t == 0) {
                float *st = a.stats + row * 3;
                st[0] = m, st[1] = delta, st[2] = r;
            }
        }
    }
}

template <typename T, int VEC, int E, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : 256) norm_bwd_kernel(const NormArgs a) {
    constexpr int NV = E / VEC;
    __shared__ float sm[2][16][2];
    pdl_enter();
    const int tpr = a.tpr, lane = threadIdx.x & 31;
    const int t = BLOCK ? threadIdx.x : lane & (tpr - 1);
    const int dim = a.dim;
    const float inv = 1.f / (float)dim;
    float w[E], aw[E], ab[E];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int j = (t + k * tpr) * VEC + i;
            w[k * VEC + i] = a.w && j < dim ? load_as<T>(a.w, a.wf32, j) : 1.f;
            aw[k * VEC + i] = ab[k * VEC + i] = 0.f;
        }
    const int per = BLOCK ? 1 : 32 / tpr;
    const int64_t step = BLOCK ? (int64_t)gridDim.x : (int64_t)gridDim.x * 8 * per;
    int64_t first = BLOCK ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * per;
    const int sub = BLOCK ? 0 : lane / tpr;
    int phase = 0;
    RowRegs<T, VEC, NV> nx, ny;
    nx.load((const T *)a.x + (first + sub) * a.x_stride, t, tpr, dim, first + sub < a.rows);
    ny.load((const T *)a.dy + (first + sub) * a.dy_stride, t, tpr, dim, first + sub < a.rows);
    for (; first < a.rows; first += step) {
        const int64_t row = first + sub;
        const bool valid = row < a.rows;
        RowRegs<T, VEC, NV> cx = nx, cy = ny;
        float m = 0.f, delta = 0.f, r = 0.f;
        if (valid) {
            const float *st = a.stats + row * 3;
            m = st[0], delta = st[1], r = st[2];
        }
        nx.load((const T *)a.x + (row + step) * a.x_stride, t, tpr, dim, row + step < a.rows);
        ny.load((const T *)a.dy + (row + step) * a.dy_stride, t, tpr, dim, row + step < a.rows);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const bool in = valid && (t + k * tpr) * VEC < dim;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = to_f(cy.p[k].v[i]);  // 0 outside the row
                const float xh = in ? ((to_f(cx.p[k].v[i]) - m) - delta) * r : 0.f;
                const float g = d * w[k * VEC + i];
                s[0] += g;
                s[1] += g * xh;
                aw[k * VEC + i] += d * xh;
                ab[k * VEC + i] += d;
            }
        }
        if (a.y) {
            row_sum<BLOCK>(s, tpr, sm, phase);
            const float c1 = s[0] * inv, c2 = s[1] * inv;
            if (valid) {
                T *dx = (T *)a.y + row * dim;
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int j = (t + k * tpr) * VEC;
                    if (j >= dim) continue;
                    Pack<T, VEC> o;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float xh = ((to_f(cx.p[k].v[i]) - m) - delta) * r;
                        const float g = to_f(cy.p[k].v[i]) * w[k * VEC + i];
                        o.v[i] = from_f<T>(r * (g - c1 - xh * c2));
                    }
                    *(Pack<T, VEC> *)(dx + j) = o;
                }
            }
        }
    }
    if (!a.part) return;
    float *out = a.part + (int64_t)blockIdx.x * 2 * dim;
    if (BLOCK) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int j = (t + k * tpr) * VEC + i;
                if (j < dim) out[j] = aw[k * VEC + i], out[dim + j] = ab[k * VEC + i];
            }
    } else {
        // the CTA's rows: groups of a warp by shuffles, then its eight warps
        __shared__ float cw[8][32 * E], cb[8][32 * E];
        const int warp = threadIdx.x >> 5;
#pragma unroll
        for (int k = 0; k < E; ++k)
            for (int o = tpr; o < 32; o <<= 1) {
                aw[k] += __shfl_xor_sync(ALL, aw[k], o);
                ab[k] += __shfl_xor_sync(ALL, ab[k], o);
            }
        if (sub == 0)
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const int j = (t + k * tpr) * VEC + i;
                    if (j < dim) cw[warp][j] = aw[k * VEC + i], cb[warp][j] = ab[k * VEC + i];
                }
        __syncthreads();
        for (int j = threadIdx.x; j < dim; j += blockDim.x) {
            float u = 0.f, v = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) u += cw[i][j], v += cb[i][j];
            out[j] = u, out[dim + j] = v;
        }
    }
}

// Sums of the weights' gradients over the CTAs, in a fixed order and 64 bits.
template <typename T>
__global__ void __launch_bounds__(512) norm_dw_kernel(const float *part, int parts, int dim, void *dw, void *db,
                                                      int wf32) {
    __shared__ double red[16][33];
    pdl_enter();
    const int c = threadIdx.x & 31, l = threadIdx.x >> 5;
    const int64_t n = 2 * (int64_t)dim, j = (int64_t)blockIdx.x * 32 + c;
    double s = 0;
    if (j < n)
#pragma unroll 4
        for (int i = l; i < parts; i += 16) s += (double)part[i * n + j];
    red[l][c] = s;
    __syncthreads();
    if (l == 0 && j < n) {
        double v = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) v += red[i][c];
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
// thread per column over a share of the rows.
template <typename T>
__global__ void __launch_bounds__(512) norm_fwd_long_kernel(const NormArgs a) {
    __shared__ float sm1[2][16][1], sm2[2][16][2];
    pdl_enter();
    const float inv = 1.f / (float)a.dim;
    int phase1 = 0, phase2 = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.x_stride;
        T *y = (T *)a.y + row * a.dim;
        float s1[1] = {0.f}, s2[2] = {0.f, 0.f};
#pragma unroll 8
        for (int j = threadIdx.x; j < a.dim; j += 512) s1[0] += to_f(x[j]);
        row_sum<true>(s1, 512, sm1, phase1);
        const float m = s1[0] * inv;
#pragma unroll 8
        for (int j = threadIdx.x; j < a.dim; j += 512) {
            const float c = to_f(x[j]) - m;
            s2[0] += c;
            s2[1] += c * c;
        }
        row_sum<true>(s2, 512, sm2, phase2);
        const float delta = s2[0] * inv;
        const float r = 1.f / sqrtf(fmaxf(s2[1] * inv - delta * delta, 0.f) + a.eps);
#pragma unroll 4
        for (int j = threadIdx.x; j < a.dim; j += 512)
            y[j] = from_f<T>(((to_f(x[j]) - m) - delta) * r * (a.w ? load_as<T>(a.w, a.wf32, j) : 1.f) +
                             (a.b ? load_as<T>(a.b, a.wf32, j) : 0.f));
        if (a.stats && threadIdx.x == 0) {
            float *st = a.stats + row * 3;
            st[0] = m, st[1] = delta, st[2] = r;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(512) norm_dx_long_kernel(const NormArgs a) {
    __shared__ float sm[2][16][2];
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
        row_sum<true>(s, 512, sm, phase);
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

// How a call is laid out.  Up to 256 places a row is part of a warp, up to
// 8,192 it is a CTA, beyond that it is read again for each sum.
struct NormPlan {
    int kind;     // 0: warp, 1: CTA of E = 8, 2: CTA of E = 16, 3: long
    int tpr, threads;
    int64_t grid; // CTAs; kind 3: rows of partial sums
};

constexpr int NORM_LONG_PARTS = 64;

static NormPlan norm_plan(int64_t rows, int32_t dim, int sms, bool backward) {
    NormPlan p{};
    if (dim > 8192) {
        p.kind = 3, p.tpr = p.threads = 512;
        p.grid = rows < NORM_LONG_PARTS ? rows : NORM_LONG_PARTS;
        return p;
    }
    const int e = dim > 4096 ? 16 : 8;
    p.tpr = 1;
    while (p.tpr * e < dim) p.tpr *= 2;
    if (p.tpr <= 32) {
        p.threads = 256;
        const int64_t per = 256 / p.tpr, need = (rows + per - 1) / per, cap = (int64_t)sms * (backward ? 3 : 5);
        p.grid = need < cap ? need : cap;
    } else {
        p.kind = e == 8 ? 1 : 2;
        p.threads = p.tpr;
        const int64_t cap = (int64_t)sms * (backward ? (e == 8 ? 1024 : 512) : (e == 8 ? 1536 : 1024)) / p.threads;
        p.grid = rows < cap ? rows : cap;
    }
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

template <typename T, int VEC, bool BWD>
static cudaError_t norm_launch(const NormPlan &p, const NormArgs &a, cudaStream_t s) {
    const unsigned g = (unsigned)p.grid, t = (unsigned)p.threads;
    if (p.kind == 0) return launch_pdl(BWD ? norm_bwd_kernel<T, VEC, 8, false> : norm_fwd_kernel<T, VEC, 8, false>, g, t, 0, s, a);
    if (p.kind == 1) return launch_pdl(BWD ? norm_bwd_kernel<T, VEC, 8, true> : norm_fwd_kernel<T, VEC, 8, true>, g, t, 0, s, a);
    return launch_pdl(BWD ? norm_bwd_kernel<T, VEC, 16, true> : norm_fwd_kernel<T, VEC, 16, true>, g, t, 0, s, a);
}

template <typename T, bool BWD>
static cudaError_t norm_rows(const NormPlan &p, const NormArgs &a, int vec, int sms, cudaStream_t s) {
    if (p.kind == 3) {
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
    return JQ_OK;
}

}  // namespace jq

using namespace jq;

extern "C" {

int64_t jq_layer_norm_scratch_floats(int64_t rows, int32_t dim) {
    int sms = 0;
    if (rows <= 0 || dim <= 0 || device_sms(sms)) return 0;
    return norm_plan(rows, dim, sms, true).grid * 2 * (int64_t)dim;
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
    const NormPlan p = norm_plan(rows, dim, sms, false);
    a.tpr = p.tpr;
    const void *ptrs[] = {d_x, d_y};
    const int64_t strides[] = {rows > 1 ? x_stride : 0, rows > 1 ? dim : 0};
    const int vec = norm_vec(elem_size(dtype), dim, ptrs, strides, 2);
    if (!vec || (((uintptr_t)d_weight | (uintptr_t)d_bias) & (elem_size(wdtype) - 1)) || ((uintptr_t)d_stats & 3))
        return fail(JQ_ERR_ARG, "layer norm: an array is not aligned to its elements");
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
    const NormPlan p = norm_plan(rows, dim, sms, true);
    a.tpr = p.tpr;
    const void *ptrs[] = {d_x, d_dy, d_dx ? d_dx : d_x};
    const int64_t strides[] = {rows > 1 ? x_stride : 0, rows > 1 ? dy_stride : 0, rows > 1 ? dim : 0};
    const int vec = norm_vec(elem_size(dtype), dim, ptrs, strides, 3);
    if (!vec || (((uintptr_t)d_weight | (uintptr_t)d_dweight | (uintptr_t)d_dbias) & (elem_size(wdtype) - 1)) ||
        (((uintptr_t)d_stats | (uintptr_t)d_scratch) & 3))
        return fail(JQ_ERR_ARG, "layer norm: an array is not aligned to its elements");
    cudaStream_t s = (cudaStream_t)stream;
    CU(norm_typed<true>(dtype, p, a, vec, sms, s));
    if (!a.part) return JQ_OK;
    const unsigned g = (unsigned)((2 * (int64_t)dim + 31) / 32);
    const float *part = a.part;
    if (dtype == JQ_F16)
        CU(launch_pdl(norm_dw_kernel<__half>, g, 512, 0, s, part, (int)p.grid, (int)dim, d_dweight, d_dbias, (int)a.wf32));
    else
        CU(launch_pdl(norm_dw_kernel<__nv_bfloat16>, g, 512, 0, s, part, (int)p.grid, (int)dim, d_dweight, d_dbias, (int)a.wf32));
    return JQ_OK;
}

}  // extern "C"
