// The norms before and after a residual block, with the block's gate and residual scale.
//
// A sample has D * F values x_i (all components of a hyper-complex sample; weights are shared by its components, as batch-norm's are here).
//   n(v) = v * r(v),  r(v) = 1 / sqrt(mean(v^2) + eps)
//   y = x + s * g * (n(branch) * post)          h = n(y) * pre
// g is a gate per value of a group of samples (one group: of every sample; a group each: per value), s a number.
// Backward, for dy (gradient of y from the residual path) and dh, with u = n(branch) and yn = n(y):
//   t = dh * pre,   dx = dy + r(y) * (t - yn * mean(t * yn)),   dpre = sum dh * yn
//   dn = s * g * dx,   dgate = sum over the group of s * dx * u * post,   dpost = sum dn * u
//   v = dn * post,   dbranch = r(branch) * (v - u * mean(v * u))
// One pass over the data in each direction: a row stays in registers between its reductions. Sums are fp32, results are rounded once.
// Sums over samples: a CTA takes whole pieces of a group and keeps its columns' sums in registers; pieces are added by a second kernel in a fixed order.
#include "common.cuh"
#include "tc_common.cuh"

namespace pcb {
namespace {

using namespace tc;

template <typename T, int VEC> struct Vec;                // VEC neighbours: as loaded, and as fp32
template <> struct Vec<float, 4> {
    typedef uint4 raw;
    static __device__ __forceinline__ void unpack(const raw& r, float* v) { v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w); }
    static __device__ __forceinline__ raw pack(const float* v) { return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])); }
};
template <> struct Vec<float, 1> {
    typedef uint32_t raw;
    static __device__ __forceinline__ void unpack(const raw& r, float* v) { v[0] = __uint_as_float(r); }
    static __device__ __forceinline__ raw pack(const float* v) { return __float_as_uint(v[0]); }
};
template <typename T> __device__ __forceinline__ float from16(uint32_t h);
template <> __device__ __forceinline__ float from16<__half>(uint32_t h) { return __half2float(__ushort_as_half((uint16_t)h)); }
template <> __device__ __forceinline__ float from16<__nv_bfloat16>(uint32_t h) { return __uint_as_float(h << 16); }
template <typename T> __device__ __forceinline__ uint32_t pack16(float a, float b);
template <> __device__ __forceinline__ uint32_t pack16<__half>(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
template <typename T> struct Vec<T, 8> {
    typedef uint4 raw;
    static __device__ __forceinline__ void unpack(const raw& r, float* v) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = from16<T>(w[i] & 0xffffu); v[2 * i + 1] = from16<T>(w[i] >> 16); }
    }
    static __device__ __forceinline__ raw pack(const float* v) { return make_uint4(pack16<T>(v[0], v[1]), pack16<T>(v[2], v[3]), pack16<T>(v[4], v[5]), pack16<T>(v[6], v[7])); }
};
template <typename T> struct Vec<T, 1> {
    typedef uint16_t raw;
    static __device__ __forceinline__ void unpack(const raw& r, float* v) { v[0] = from16<T>(r); }
    static __device__ __forceinline__ raw pack(const float* v) { return (uint16_t)pack16<T>(v[0], 0.f); }
};

// VEC weights (fp32, ones where there are none)
template <int VEC>
__device__ __forceinline__ void load_weights(const float* w, int f, bool ok, float* v) {
    if (!w) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = 1.f;
    } else if (VEC == 1) {
        v[0] = ld_chained(w + f, ok);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 a = ld_chained(reinterpret_cast<const float4*>(w + f + i), ok);
            v[i] = a.x; v[i + 1] = a.y; v[i + 2] = a.z; v[i + 3] = a.w;
        }
    }
}

// Sum over the threads of a row: a warp, or the whole CTA of WPR warps. `turn` alternates between two sets of words.
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float (*words)[32], int& turn) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (WPR == 1) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) words[turn][warp] = v;
    __syncthreads();
    v = lane < WPR ? words[turn][lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    turn ^= 1;
    return v;
}

struct RNParams {
    int comps, n, features, groups, per_group;     // groups: rows of the gate per component (0: no gate); per_group: samples of each
    uint32_t magic;                                // ceil(2^32 / features): e / features = umulhi(e, magic) for the widths below (0: features == 1)
    float scale, eps;
    const void *x, *branch, *gate;
    const float *post, *pre;
    void *y, *h;
    float* stats;                                  // [2][n]: r(branch), r(y)
    // backward
    const void *dy, *dh;
    void *dx, *dbranch, *dgate;
    float *dpost, *dpre;
    float *part_w;                                 // [CTAs][2][comps * features]: dpre, dpost
    float *part_gate;                              // [groups * parts][comps * features]
    int parts, items;                              // pieces per group
};

// Where value e of a sample lies: component e / F, feature e % F.
__device__ __forceinline__ int comp_of(const RNParams& p, int e) { return p.comps == 1 ? 0 : (p.magic ? (int)__umulhi((uint32_t)e, p.magic) : e); }

__host__ __device__ constexpr int rn_threads(int wpr) { return wpr == 1 ? 128 : 32 * wpr; }

template <typename T, int VEC, int NV, int WPR>
__global__ void __launch_bounds__(rn_threads(WPR)) residual_norm_fwd_kernel(const RNParams p) {
    typedef Vec<T, VEC> V;
    typedef typename V::raw raw;
    constexpr int TPR = 32 * WPR, ROWS = rn_threads(WPR) / TPR;
    __shared__ float words[2][32];
    const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR, width = p.comps * p.features;
    int turn = 0;
    chain_wait();
    chain_next();
    const float inv_width = 1.f / (float)width;
    for (int row0 = blockIdx.x * ROWS; row0 < p.n; row0 += gridDim.x * ROWS) {
        const int row = row0 + sub;
        const bool live = row < p.n;
        const T* x = static_cast<const T*>(p.x) + (size_t)row * p.features;
        const T* b = static_cast<const T*>(p.branch) + (size_t)row * p.features;
        const T* g = p.gate ? static_cast<const T*>(p.gate) + (size_t)(row / p.per_group) * p.features : nullptr;
        raw xr[NV], br[NV], gr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
            const bool ok = live && e < width;
            const size_t at = (size_t)c * (p.n - 1) * p.features + e;
            xr[i] = ld_chained(reinterpret_cast<const raw*>(x + at), ok);
            if (p.branch) br[i] = ld_chained(reinterpret_cast<const raw*>(b + at), ok);
            if (g) gr[i] = ld_chained(reinterpret_cast<const raw*>(g + (size_t)c * (p.groups - 1) * p.features + e), ok);
        }
        float y[NV][VEC];
#pragma unroll
        for (int i = 0; i < NV; ++i) V::unpack(xr[i], y[i]);
        float rb = 0.f;
        if (p.branch) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float v[VEC];
                V::unpack(br[i], v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum = fmaf(v[j], v[j], sum);
            }
            rb = rsqrtf(row_sum<WPR>(sum, words, turn) * inv_width + p.eps);
            const float f = p.scale * rb;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                float v[VEC], w[VEC], gv[VEC];
                V::unpack(br[i], v);
                load_weights<VEC>(p.post, e - c * p.features, live && e < width, w);
                if (g) V::unpack(gr[i], gv);
#pragma unroll
                for (int j = 0; j < VEC; ++j) y[i][j] = fmaf(v[j] * f, g ? w[j] * gv[j] : w[j], y[i][j]);
            }
        }
        T* yo = static_cast<T*>(p.y) + (size_t)row * p.features;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
            if (p.y && live && e < width) *reinterpret_cast<raw*>(yo + (size_t)c * (p.n - 1) * p.features + e) = V::pack(y[i]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum = fmaf(y[i][j], y[i][j], sum);
        }
        float ry = 0.f;
        if (p.h) {
            ry = rsqrtf(row_sum<WPR>(sum, words, turn) * inv_width + p.eps);
            T* ho = static_cast<T*>(p.h) + (size_t)row * p.features;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                if (!live || e >= width) continue;
                float w[VEC];
                load_weights<VEC>(p.pre, e - c * p.features, true, w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) w[j] *= y[i][j] * ry;
                *reinterpret_cast<raw*>(ho + (size_t)c * (p.n - 1) * p.features + e) = V::pack(w);
            }
        }
        if (p.stats && tid == 0 && live) { p.stats[row] = rb; p.stats[p.n + row] = ry; }
    }
}

// GATE: 0 none, 1 a gate for each value, 2 gates shared by the samples of a group
template <typename T, int VEC, int NV, int WPR, int GATE>
__global__ void __launch_bounds__(rn_threads(WPR)) residual_norm_bwd_kernel(const RNParams p) {
    typedef Vec<T, VEC> V;
    typedef typename V::raw raw;
    constexpr int TPR = 32 * WPR, ROWS = rn_threads(WPR) / TPR;
    __shared__ float words[2][32];
    const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR, width = p.comps * p.features;
    int turn = 0;
    chain_wait();
    chain_next();
    const float inv_width = 1.f / (float)width;
    float dpre[NV][VEC], dpost[NV][VEC], dgate[GATE == 2 ? NV : 1][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) dpre[i][j] = dpost[i][j] = 0.f;
    const int slots = gridDim.x * ROWS, slot = blockIdx.x * ROWS + sub;
    // an item is a piece of a group of samples; the threads of a row take items (WPR == 1: each warp its own)
    for (int item = slot; item < p.items; item += slots) {
        const int group = item / p.parts, part = item - group * p.parts;
        const int begin = group * p.per_group + (int)((long long)p.per_group * part / p.parts), end = group * p.per_group + (int)((long long)p.per_group * (part + 1) / p.parts);
        if (GATE == 2) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) dgate[i][j] = 0.f;
        }
        raw gr[NV];
        for (int row = begin; row < end; ++row) {
            const size_t row_at = (size_t)row * p.features;
            raw yr[NV], br[NV], tr[NV], dr[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                const bool ok = e < width;
                const size_t at = row_at + (size_t)c * (p.n - 1) * p.features + e;
                if (p.dh) { yr[i] = ld_chained(reinterpret_cast<const raw*>(static_cast<const T*>(p.y) + at), ok); tr[i] = ld_chained(reinterpret_cast<const raw*>(static_cast<const T*>(p.dh) + at), ok); }
                if (p.dy) dr[i] = ld_chained(reinterpret_cast<const raw*>(static_cast<const T*>(p.dy) + at), ok);
                if (p.branch) br[i] = ld_chained(reinterpret_cast<const raw*>(static_cast<const T*>(p.branch) + at), ok);
                if (GATE == 1 || (GATE == 2 && row == begin))
                    gr[i] = ld_chained(reinterpret_cast<const raw*>(static_cast<const T*>(p.gate) + (size_t)group * p.features + (size_t)c * (p.groups - 1) * p.features + e), ok);
            }
            const float rb = p.branch ? ld_chained(p.stats + row) : 0.f, ry = p.dh ? ld_chained(p.stats + p.n + row) : 0.f;
            float dx[NV][VEC];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (p.dy) V::unpack(dr[i], dx[i]);
                else
#pragma unroll
                    for (int j = 0; j < VEC; ++j) dx[i][j] = 0.f;
            }
            if (p.dh) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                    float y[VEC], t[VEC], w[VEC];
                    V::unpack(yr[i], y);
                    V::unpack(tr[i], t);
                    load_weights<VEC>(p.pre, e - c * p.features, e < width, w);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float yn = y[j] * ry;
                        dpre[i][j] = fmaf(t[j], yn, dpre[i][j]);
                        sum = fmaf(t[j] * w[j], yn, sum);
                        dx[i][j] = fmaf(t[j] * w[j], ry, dx[i][j]);
                    }
                }
                const float f = row_sum<WPR>(sum, words, turn) * inv_width * ry * ry;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    float y[VEC];
                    V::unpack(yr[i], y);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) dx[i][j] = fmaf(-f, y[j], dx[i][j]);
                }
            }
            T* dxo = static_cast<T*>(p.dx);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                if (e < width) *reinterpret_cast<raw*>(dxo + row_at + (size_t)c * (p.n - 1) * p.features + e) = V::pack(dx[i]);
            }
            if (p.branch) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                    float b[VEC], w[VEC], g[VEC];
                    V::unpack(br[i], b);
                    load_weights<VEC>(p.post, e - c * p.features, e < width, w);
                    if (GATE) V::unpack(gr[i], g);
                    float dg[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float u = b[j] * rb, sdx = p.scale * dx[i][j], dn = GATE ? sdx * g[j] : sdx;
                        dpost[i][j] = fmaf(dn, u, dpost[i][j]);
                        dg[j] = sdx * u * w[j];
                        if (GATE == 2) dgate[i][j] += dg[j];
                        dx[i][j] = dn * w[j];
                        sum = fmaf(dx[i][j], u, sum);
                    }
                    if (GATE == 1 && p.dgate && e < width) *reinterpret_cast<raw*>(static_cast<T*>(p.dgate) + row_at + (size_t)c * (p.n - 1) * p.features + e) = V::pack(dg);
                }
                const float f = row_sum<WPR>(sum, words, turn) * inv_width * rb;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                    float b[VEC];
                    V::unpack(br[i], b);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) b[j] = rb * fmaf(-f, b[j], dx[i][j]);
                    if (e < width) *reinterpret_cast<raw*>(static_cast<T*>(p.dbranch) + row_at + (size_t)c * (p.n - 1) * p.features + e) = V::pack(b);
                }
            }
        }
        if (GATE == 2 && p.dgate) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                if (e >= width) continue;
                if (p.parts == 1) {
                    *reinterpret_cast<raw*>(static_cast<T*>(p.dgate) + (size_t)group * p.features + (size_t)c * (p.groups - 1) * p.features + e) = V::pack(dgate[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) p.part_gate[(size_t)item * width + e + j] = dgate[i][j];
                }
            }
        }
    }
    if (p.part_w) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * TPR + tid) * VEC;
            if (e >= width) continue;
            float* out = p.part_w + (size_t)slot * 2 * width + e;
#pragma unroll
            for (int j = 0; j < VEC; ++j) { out[j] = dpre[i][j]; out[width + j] = dpost[i][j]; }
        }
    }
}

// Rows wider than the registers: the same sums, the row read again in each step. A CTA per row.
constexpr int RN_WIDE_THREADS = 512;
template <typename T> __device__ __forceinline__ float at(const void* p, size_t i) {
    float v;
    Vec<T, 1>::unpack(ld_chained(static_cast<const typename Vec<T, 1>::raw*>(p) + i), &v);
    return v;
}
template <typename T> __device__ __forceinline__ void put(void* p, size_t i, float v) { static_cast<typename Vec<T, 1>::raw*>(p)[i] = Vec<T, 1>::pack(&v); }

template <typename T>
__global__ void __launch_bounds__(RN_WIDE_THREADS) residual_norm_fwd_wide_kernel(const RNParams p) {
    constexpr int WPR = RN_WIDE_THREADS / 32;
    __shared__ float words[2][32];
    int turn = 0;
    chain_wait();
    chain_next();
    const size_t F = p.features, N = p.n;
    const float inv_width = 1.f / ((float)p.comps * (float)p.features);
    for (int row = blockIdx.x; row < p.n; row += gridDim.x) {
        const size_t group = p.gate ? row / p.per_group : 0;
        float rb = 0.f, ry = 0.f;
        if (p.branch) {
            float sum = 0.f;
            for (int c = 0; c < p.comps; ++c)
                for (size_t f = threadIdx.x; f < F; f += RN_WIDE_THREADS) { const float v = at<T>(p.branch, (c * N + row) * F + f); sum = fmaf(v, v, sum); }
            rb = rsqrtf(row_sum<WPR>(sum, words, turn) * inv_width + p.eps);
        }
        auto value = [&](int c, size_t f) {
            const size_t i = (c * N + row) * F + f;
            const float x = at<T>(p.x, i);
            if (!p.branch) return x;
            const float w = (p.post ? ld_chained(p.post + f) : 1.f) * (p.gate ? at<T>(p.gate, (c * (size_t)p.groups + group) * F + f) : 1.f);
            return fmaf(at<T>(p.branch, i) * (p.scale * rb), w, x);
        };
        if (p.h) {
            float sum = 0.f;
            for (int c = 0; c < p.comps; ++c)
                for (size_t f = threadIdx.x; f < F; f += RN_WIDE_THREADS) { const float v = value(c, f); sum = fmaf(v, v, sum); }
            ry = rsqrtf(row_sum<WPR>(sum, words, turn) * inv_width + p.eps);
        }
        for (int c = 0; c < p.comps; ++c)
            for (size_t f = threadIdx.x; f < F; f += RN_WIDE_THREADS) {
                const float v = value(c, f);
                if (p.y) put<T>(p.y, (c * N + row) * F + f, v);
                if (p.h) put<T>(p.h, (c * N + row) * F + f, v * ry * (p.pre ? ld_chained(p.pre + f) : 1.f));
            }
        if (p.stats && threadIdx.x == 0) { p.stats[row] = rb; p.stats[N + row] = ry; }
    }
}

template <typename T>
__global__ void __launch_bounds__(RN_WIDE_THREADS) residual_norm_bwd_wide_kernel(const RNParams p) {
    constexpr int WPR = RN_WIDE_THREADS / 32;
    __shared__ float words[2][32];
    int turn = 0;
    chain_wait();
    chain_next();
    const size_t F = p.features, N = p.n, width = (size_t)p.comps * F;
    const float inv_width = 1.f / (float)width;
    float* mine = p.part_w ? p.part_w + (size_t)blockIdx.x * 2 * width : nullptr;     // this CTA's sums, each element one thread's
    if (mine)
        for (int c = 0; c < p.comps; ++c)
            for (size_t f = threadIdx.x; f < F; f += RN_WIDE_THREADS) mine[c * F + f] = mine[width + c * F + f] = 0.f;
    for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
        const size_t group = item / p.parts;
        const int part = item - (int)group * p.parts;
        const int begin = (int)group * p.per_group + (int)((long long)p.per_group * part / p.parts), end = (int)group * p.per_group + (int)((long long)p.per_group * (part + 1) / p.parts);
        float* gates = p.part_gate ? p.part_gate + (size_t)item * width : nullptr;
        for (int row = begin; row < end; ++row) {
            const float rb = p.branch ? ld_chained(p.stats + row) : 0.f, ry = p.dh ? ld_chained(p.stats + N + row) : 0.f;
            float fy = 0.f, fb = 0.f;
            auto weight = [&](const float* w, size_t f) { return w ? ld_chained(w + f) : 1.f; };
            if (p.dh) {
                float sum = 0.f;
                for (int c = 0; c < p.comps; ++c)
                    for (size_t f = threadIdx.x; f < F; f += RN_WIDE_THREADS) {
                        const size_t i = (c * N + row) * F + f;
                        const float t = at<T>(p.dh, i), yn = at<T>(p.y, i) * ry;
                        if (mine) mine[c * F + f] = fmaf(t, yn, mine[c * F + f]);
                        sum = fmaf(t * weight(p.pre, f), yn, sum);
                    }
                fy = row_sum<WPR>(sum, words, turn) * inv_width * ry * ry;
            }
            auto grad = [&](size_t i, size_t f) {
                float d = p.dy ? at<T>(p.dy, i) : 0.f;
                if (p.dh) d = fmaf(-fy, at<T>(p.y, i), fmaf(at<T>(p.dh, i) * weight(p.pre, f), ry, d));
                return d;
            };
            if (p.branch) {
                float sum = 0.f;
                for (int c = 0; c < p.comps; ++c)
                    for (size_t f = threadIdx.x; f < F; f += RN_WIDE_THREADS) {
                        const size_t i = (c * N + row) * F + f;
                        const float u = at<T>(p.branch, i) * rb, sdx = p.scale * grad(i, f), w = weight(p.post, f);
                        const float dn = p.gate ? sdx * at<T>(p.gate, (c * (size_t)p.groups + group) * F + f) : sdx, dg = sdx * u * w;
                        if (mine) mine[width + c * F + f] = fmaf(dn, u, mine[width + c * F + f]);
                        if (gates) gates[c * F + f] = row == begin ? dg : gates[c * F + f] + dg;
                        sum = fmaf(dn * w, u, sum);
                    }
                fb = row_sum<WPR>(sum, words, turn) * inv_width * rb;
            }
            for (int c = 0; c < p.comps; ++c)
                for (size_t f = threadIdx.x; f < F; f += RN_WIDE_THREADS) {
                    const size_t i = (c * N + row) * F + f;
                    const float d = grad(i, f);
                    put<T>(p.dx, i, d);
                    if (p.branch) {
                        const float b = at<T>(p.branch, i), w = weight(p.post, f), g = p.gate ? at<T>(p.gate, (c * (size_t)p.groups + group) * F + f) : 1.f;
                        put<T>(p.dbranch, i, rb * fmaf(-fb, b, p.scale * d * g * w));
                    }
                }
        }
    }
}

// Adds the pieces: the weights' gradients over slots and components, the gates' over the pieces of their group. 32 columns per CTA.
template <typename T>
__global__ void __launch_bounds__(256) residual_norm_sum_kernel(const RNParams p, int slots, int weight_blocks) {
    __shared__ float sums[2][8][33];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5, width = p.comps * p.features;
    chain_wait();
    chain_next();
    if ((int)blockIdx.x < weight_blocks) {
        const int f = blockIdx.x * 32 + col;
        float a = 0.f, b = 0.f;
        if (f < p.features)
            for (int r = slice; r < slots * p.comps; r += 8) {
                const int s = r / p.comps, c = r - s * p.comps;
                const float* src = p.part_w + (size_t)s * 2 * width + (size_t)c * p.features + f;
                a += ld_chained(src);
                b += ld_chained(src + width);
            }
        sums[0][slice][col] = a;
        sums[1][slice][col] = b;
        __syncthreads();
        if (slice < 2 && f < p.features) {
            float v = 0.f;
#pragma unroll
            for (int s = 0; s < 8; ++s) v += sums[slice][s][col];
            float* out = slice == 0 ? p.dpre : p.dpost;
            if (out) out[f] = v;
        }
    } else {
        const int blocks = (width + 31) / 32, id = blockIdx.x - weight_blocks, group = id / blocks, e = (id - group * blocks) * 32 + col;
        float a = 0.f;
        if (e < width)
            for (int s = slice; s < p.parts; s += 8) a += ld_chained(p.part_gate + ((size_t)group * p.parts + s) * width + e);
        sums[0][slice][col] = a;
        __syncthreads();
        if (slice == 0 && e < width) {
            float v = 0.f;
#pragma unroll
            for (int s = 0; s < 8; ++s) v += sums[0][s][col];
            const int c = e / p.features;
            put<T>(p.dgate, (size_t)group * p.features + (size_t)c * (p.groups - 1) * p.features + e, v);
        }
    }
}

// Values per thread of a row and warps per row for a width; warps 0: wider than the registers.
struct RNShape { int warps, slots; };
RNShape fwd_shape(int width) {
    if (width <= 32 * 16) return {1, 1};
    if (width <= 128 * 16) return {4, 1};
    if (width <= 128 * 32) return {4, 2};
    if (width <= 512 * 16) return {16, 1};
    if (width <= 512 * 32) return {16, 2};
    return {0, 0};
}
RNShape bwd_shape(int width) {
    if (width <= 32 * 16) return {1, 2};
    if (width <= 128 * 8) return {4, 1};
    if (width <= 128 * 16) return {4, 2};
    if (width <= 512 * 8) return {16, 1};
    if (width <= 512 * 16) return {16, 2};
    return {0, 0};
}
constexpr int RN_PER_SM = 4;                              // rows in work per SM in the backward pass: CTAs, or four warps each

struct RNPlan { RNShape shape; int grid, slots, parts, items; size_t part_w, part_gate, total; };
RNPlan bwd_plan(int comps, int n, int features, int groups) {
    RNPlan q = {};
    const long long width = (long long)comps * features;
    q.shape = width > 512 * 16 ? RNShape{0, 0} : bwd_shape((int)width);
    const int rows_per_cta = q.shape.warps == 1 ? 4 : 1, most = device_sms() * RN_PER_SM * rows_per_cta;
    const bool shared = groups > 0 && groups < n;
    const int g = shared || (groups == n && n > 0) ? groups : 1;
    if (groups == n && groups > 1 && !shared) { q.parts = 1; q.items = n; }          // a gate for each value: every sample is an item
    else {
        // pieces per group: as many as fill the machine for one to eight rounds, whichever has the fewest rounds x samples per piece
        const int per = n / g;
        long long best = -1;
        for (long long rounds = 1; rounds <= 8; ++rounds) {
            const long long fit = rounds * most / g, parts = fit < 1 ? 1 : (fit < per ? fit : per);
            const long long cost = (g * parts + most - 1) / most * ((per + parts - 1) / parts);
            if (best < 0 || cost < best) { best = cost; q.parts = (int)parts; }
        }
        q.items = g * q.parts;
    }
    const int want = q.items < most ? q.items : most;
    q.grid = (want + rows_per_cta - 1) / rows_per_cta;
    q.slots = q.shape.warps == 0 ? q.grid : q.grid * rows_per_cta;
    q.part_w = (size_t)q.slots * 2 * width * 4;
    q.part_gate = shared && (q.parts > 1 || q.shape.warps == 0) ? (size_t)q.items * width * 4 : (groups == n && n > 0 && q.shape.warps == 0 ? (size_t)n * width * 4 : 0);
    q.total = q.part_w + q.part_gate;
    return q;
}

int check_norm(const pcb_norm_desc* d) {
    if (!d) { set_error("null descriptor"); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->dtype < PCB_F32 || d->dtype > PCB_BF16) { set_error("unknown dtype %d", d->dtype); return PCB_ERR_INVALID_ARGUMENT; }
    Geom g = {};
    if (!algebra_setup(d->algebra, g)) { set_error("unknown algebra %d", d->algebra); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->batch < 0 || d->features <= 0) { set_error("invalid norm geometry"); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->gate_rows < 0 || (d->gate_rows > 0 && d->batch > 0 && d->batch % d->gate_rows != 0)) {
        set_error("%d rows of the gate for %d samples", d->gate_rows, d->batch);
        return PCB_ERR_INVALID_ARGUMENT;
    }
    if (!(d->epsilon >= 0.f)) { set_error("epsilon must not be negative"); return PCB_ERR_INVALID_ARGUMENT; }
    if ((long long)g.nc * d->batch * d->features > 2147483647LL || (long long)g.nc * d->features > 2147483647LL) { set_error("tensor too large for 32-bit element offsets"); return PCB_ERR_TOO_LARGE; }
    return PCB_OK;
}
int norm_comps(const pcb_norm_desc* d) { Geom g = {}; algebra_setup(d->algebra, g); return g.nc; }

RNParams norm_params(const pcb_norm_desc* d) {
    RNParams p = {};
    p.comps = norm_comps(d); p.n = d->batch; p.features = d->features;
    p.groups = d->gate_rows; p.per_group = d->gate_rows > 0 ? d->batch / d->gate_rows : d->batch;
    p.magic = d->features > 1 ? (uint32_t)((0x100000000ull + d->features - 1) / d->features) : 0u;
    p.scale = d->residual_scale; p.eps = d->epsilon;
    return p;
}
bool vectors(const RNParams& p, int vec) {
    uintptr_t all = 0;
    for (const void* t : {p.x, p.branch, p.gate, (const void*)p.y, (const void*)p.h, p.dy, p.dh, (const void*)p.dx, (const void*)p.dbranch, (const void*)p.dgate, (const void*)p.post, (const void*)p.pre})
        all |= reinterpret_cast<uintptr_t>(t);
    return p.features % vec == 0 && all % 16 == 0;
}

template <typename T, int VEC, int EPT, int WPR>
cudaError_t fwd_launch(const RNParams& p, cudaStream_t s) {
    constexpr int NV = EPT / VEC, ROWS = rn_threads(WPR) / (32 * WPR);
    return launch_chained(residual_norm_fwd_kernel<T, VEC, NV, WPR>, grid_cap(p.n, ROWS, 2048 / rn_threads(WPR)), rn_threads(WPR), 0, s, p);
}
template <typename T, int VEC>
cudaError_t fwd_any(const RNParams& p, cudaStream_t s) {
    const RNShape k = fwd_shape(p.comps * p.features);
    if (k.warps == 1) return fwd_launch<T, VEC, 16, 1>(p, s);
    if (k.warps == 4) return k.slots == 1 ? fwd_launch<T, VEC, 16, 4>(p, s) : fwd_launch<T, VEC, 32, 4>(p, s);
    if (k.warps == 16) return k.slots == 1 ? fwd_launch<T, VEC, 16, 16>(p, s) : fwd_launch<T, VEC, 32, 16>(p, s);
    return launch_chained(residual_norm_fwd_wide_kernel<T>, grid_cap(p.n, 1, 4), RN_WIDE_THREADS, 0, s, p);
}
template <typename T, int VEC, int EPT, int WPR>
cudaError_t bwd_launch(const RNParams& p, const RNPlan& q, cudaStream_t s) {
    constexpr int NV = EPT / VEC;
    const int gate = !p.gate ? 0 : (p.groups == p.n ? 1 : 2);
    if (gate == 0) return launch_chained(residual_norm_bwd_kernel<T, VEC, NV, WPR, 0>, q.grid, rn_threads(WPR), 0, s, p);
    if (gate == 1) return launch_chained(residual_norm_bwd_kernel<T, VEC, NV, WPR, 1>, q.grid, rn_threads(WPR), 0, s, p);
    return launch_chained(residual_norm_bwd_kernel<T, VEC, NV, WPR, 2>, q.grid, rn_threads(WPR), 0, s, p);
}
template <typename T, int VEC>
cudaError_t bwd_any(const RNParams& p, const RNPlan& q, cudaStream_t s) {
    if (q.shape.warps == 1) return bwd_launch<T, VEC, 16, 1>(p, q, s);
    if (q.shape.warps == 4) return q.shape.slots == 1 ? bwd_launch<T, VEC, 8, 4>(p, q, s) : bwd_launch<T, VEC, 16, 4>(p, q, s);
    if (q.shape.warps == 16) return q.shape.slots == 1 ? bwd_launch<T, VEC, 8, 16>(p, q, s) : bwd_launch<T, VEC, 16, 16>(p, q, s);
    return launch_chained(residual_norm_bwd_wide_kernel<T>, q.grid, RN_WIDE_THREADS, 0, s, p);
}
template <typename T, int VEC>
int fwd_typed(const RNParams& p, cudaStream_t s) {
    if (vectors(p, VEC)) PCB_CUDA_TRY((fwd_any<T, VEC>(p, s)));
    else PCB_CUDA_TRY((fwd_any<T, 1>(p, s)));
    return PCB_OK;
}
template <typename T, int VEC>
int bwd_typed(const RNParams& p, const RNPlan& q, cudaStream_t s) {
    if (vectors(p, VEC)) PCB_CUDA_TRY((bwd_any<T, VEC>(p, q, s)));
    else PCB_CUDA_TRY((bwd_any<T, 1>(p, q, s)));
    const int weight_blocks = p.part_w ? (p.features + 31) / 32 : 0;
    const long long gate_blocks = p.part_gate ? (long long)p.groups * ((p.comps * p.features + 31) / 32) : 0;
    if (weight_blocks + gate_blocks > 0)
        PCB_CUDA_TRY(launch_chained(residual_norm_sum_kernel<T>, (unsigned)(weight_blocks + gate_blocks), 256, 0, s, p, q.slots, weight_blocks));
    return PCB_OK;
}

}  // namespace
}  // namespace pcb

using namespace pcb;

extern "C" {

size_t pcb_residual_norm_bwd_workspace_size(const pcb_norm_desc* d) {
    if (check_norm(d) != PCB_OK || d->batch == 0) return 0;
    return bwd_plan(norm_comps(d), d->batch, d->features, d->gate_rows).total;
}

int pcb_residual_norm_fwd(const pcb_norm_desc* d, const void* x, const void* branch, const void* gate, const float* post, const float* pre, void* y, void* h,
                          float* stats, void* stream) {
    const int rc = check_norm(d);
    if (rc != PCB_OK || d->batch == 0) return rc;
    if (!x || (branch && !y) || (!y && !h)) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    if ((gate != nullptr) != (d->gate_rows > 0) || (!branch && (gate || post)) || (!h && pre)) { set_error("gate or weights without what they apply to"); return PCB_ERR_INVALID_ARGUMENT; }
    RNParams p = norm_params(d);
    p.x = x; p.branch = branch; p.gate = gate; p.post = post; p.pre = pre; p.y = y; p.h = h; p.stats = stats;
    const cudaStream_t s = (cudaStream_t)stream;
    if (d->dtype == PCB_F32) return fwd_typed<float, 4>(p, s);
    return d->dtype == PCB_F16 ? fwd_typed<__half, 8>(p, s) : fwd_typed<__nv_bfloat16, 8>(p, s);
}

int pcb_residual_norm_bwd(const pcb_norm_desc* d, const void* y, const void* branch, const void* gate, const float* post, const float* pre, const float* stats,
                          const void* dy, const void* dh, void* dx, void* dbranch, void* dgate, float* dpost, float* dpre, void* workspace, size_t workspace_bytes,
                          void* stream) {
    int rc = check_norm(d);
    if (rc != PCB_OK) return rc;
    const cudaStream_t s = (cudaStream_t)stream;
    const int comps = norm_comps(d);
    if (d->batch == 0) {
        if (dpost) PCB_CUDA_TRY(cudaMemsetAsync(dpost, 0, (size_t)d->features * 4, s));
        if (dpre) PCB_CUDA_TRY(cudaMemsetAsync(dpre, 0, (size_t)d->features * 4, s));
        if (dgate) PCB_CUDA_TRY(cudaMemsetAsync(dgate, 0, (size_t)comps * d->gate_rows * d->features * dtype_size(d->dtype), s));
        return PCB_OK;
    }
    if (!stats || (!dy && !dh) || !dx || (dh && !y) || (branch && !dbranch)) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    if ((gate != nullptr) != (d->gate_rows > 0) || (!branch && (gate || post || dpost)) || (!dh && (pre || dpre)) || (dgate && !gate)) {
        set_error("gate, weights or their gradients without what they apply to");
        return PCB_ERR_INVALID_ARGUMENT;
    }
    RNPlan q = bwd_plan(comps, d->batch, d->features, d->gate_rows);
    if (!workspace || workspace_bytes < q.total) { set_error("workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, q.total); return PCB_ERR_WORKSPACE; }
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) { set_error("the workspace must be 16-byte aligned"); return PCB_ERR_INVALID_ARGUMENT; }
    RNParams p = norm_params(d);
    p.branch = branch; p.gate = gate; p.post = post; p.pre = pre; p.y = const_cast<void*>(y); p.stats = const_cast<float*>(stats);
    p.dy = dy; p.dh = dh; p.dx = dx; p.dbranch = dbranch; p.dgate = dgate; p.dpost = dpost; p.dpre = dpre;
    p.part_w = dpost || dpre ? static_cast<float*>(workspace) : nullptr;
    p.part_gate = dgate && q.part_gate ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + q.part_w) : nullptr;
    p.parts = q.parts; p.items = q.items;
    if (!gate) p.per_group = d->batch;
    if (d->dtype == PCB_F32) return bwd_typed<float, 4>(p, q, s);
    return d->dtype == PCB_F16 ? bwd_typed<__half, 8>(p, q, s) : bwd_typed<__nv_bfloat16, 8>(p, q, s);
}

}  // extern "C"
