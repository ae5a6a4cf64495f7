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
#pragma once

#include "common.cuh"
#include "residual_norm.h"
#include "tc_common.cuh"

namespace pcb {
namespace {

using namespace tc;
using umma::smem_u32;

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

// VEC weights (fp32, ones where there are none). Plain loads: nothing marks these pointers as read-only, and the compiler may place them.
template <int VEC>
__device__ __forceinline__ void load_weights(const float* w, int f, bool ok, float* v) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = 1.f;
    if (!w || !ok) return;
    if (VEC == 1) {
        v[0] = w[f];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 a = *reinterpret_cast<const float4*>(w + f + i);
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

// Where value e of a sample lies: component e / F, feature e % F.
__device__ __forceinline__ int comp_of(const RNParams& p, int e) { return p.comps == 1 ? 0 : (p.magic ? (int)__umulhi((uint32_t)e, p.magic) : e); }

// Threads of a CTA: four rows of one warp each, or one row.
__host__ __device__ constexpr int rn_threads(int wpr) { return wpr == 1 ? 128 : 32 * wpr; }

// ---- rows on their way in: a ring of row buffers in shared memory, filled by cp.async some rows ahead, so that the loads in flight cost no registers.
// With VEC > 1 a thread copies exactly the 16 bytes that it reads later and nobody else's (its slots lie 16 * threads bytes apart), so that no barrier is needed. With
// VEC == 1 (rows that start anywhere) the threads of a row copy the aligned 16-byte units that cover each component's values; units are cut where the tensor ends.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// bytes of one component's values of a row in the ring, VEC == 1
__host__ __device__ inline int segment_bytes(int features, int size) { return (features * size + 14 + 15) / 16 * 16; }

constexpr int RN_RING_BYTES = 220 * 1024;      // of all CTAs of an SM
template <typename T, int VEC, int NV, int WPR, int MAX_TENSORS, int MAX_STAGES, int PER_SM>
struct Ring {
    static constexpr int TPR = 32 * WPR, THREADS = rn_threads(WPR);
    static constexpr int MOST = MAX_TENSORS * (VEC > 1 ? NV * THREADS * 16 : (THREADS / TPR) * (TPR * NV * (int)sizeof(T) + 8 * 32));   // bytes of a stage at most
    static constexpr int FIT = RN_RING_BYTES / PER_SM / MOST, STAGES = FIT < 1 ? 1 : (FIT < MAX_STAGES ? FIT : MAX_STAGES);
    uint32_t base;          // this row's part of the ring
    int stage_bytes, tensor_bytes, seg;
    __device__ __forceinline__ Ring(uint32_t smem, const RNParams& p, int tensors) {
        if (VEC > 1) {
            tensor_bytes = NV * THREADS * 16;
            stage_bytes = tensors * tensor_bytes;
            base = smem + threadIdx.x * 16;
            seg = 0;
        } else {
            seg = segment_bytes(p.features, sizeof(T));
            tensor_bytes = p.comps * seg;
            stage_bytes = tensors * tensor_bytes;
            base = smem + (threadIdx.x / TPR) * STAGES * stage_bytes;
        }
    }
    static size_t bytes(const RNParams& p, int tensors) {
        return VEC > 1 ? (size_t)STAGES * tensors * NV * THREADS * 16 : (size_t)(THREADS / TPR) * STAGES * tensors * p.comps * segment_bytes(p.features, sizeof(T));
    }
    // starts the copy of a row of tensor k ([comps][rows of the tensor][features]) into a stage
    __device__ __forceinline__ void fetch(const RNParams& p, int stage, int k, const void* tensor, int row, int rows) const {
        const int tid = threadIdx.x % TPR, width = p.comps * p.features;
        const uint32_t dst = base + stage * stage_bytes + k * tensor_bytes;
        if (VEC > 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                if (e < width) copy16(dst + i * THREADS * 16, static_cast<const T*>(tensor) + (size_t)row * p.features + (size_t)c * (rows - 1) * p.features + e, 16);
            }
        } else {
            const size_t end = (size_t)p.comps * rows * p.features * sizeof(T);
            const int units = seg / 16;
            for (int u = tid; u < p.comps * units; u += TPR) {
                const int c = p.comps == 1 ? 0 : u / units, in = u - c * units;
                const size_t first = ((size_t)c * rows + row) * p.features * sizeof(T), at = (first & ~size_t(15)) + (size_t)in * 16;
                if (at < first + (size_t)p.features * sizeof(T)) copy16(dst + c * seg + in * 16, static_cast<const uint8_t*>(tensor) + at, (uint32_t)(end - at < 16 ? end - at : 16));
            }
        }
    }
    // value (VEC > 1: vector) i of this thread, of a row fetched before
    __device__ __forceinline__ typename Vec<T, VEC>::raw get(const RNParams& p, int stage, int k, int i, int row, int rows) const {
        typedef typename Vec<T, VEC>::raw raw;
        const int tid = threadIdx.x % TPR;
        uint32_t at = base + stage * stage_bytes + k * tensor_bytes;
        raw r = raw();
        if constexpr (VEC > 1) {
            at += i * THREADS * 16;
            if ((i * TPR + tid) * VEC < p.comps * p.features) r = ld_shared_v4(at);
        } else {
            const int e = i * TPR + tid, c = comp_of(p, e);
            if (e < p.comps * p.features) {
                const uint32_t shift = ((uint32_t)c * (uint32_t)rows + (uint32_t)row) * (uint32_t)p.features * (uint32_t)sizeof(T) & 15u;
                at += c * seg + shift + (e - c * p.features) * sizeof(T);
                if constexpr (sizeof(T) == 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(at) : "memory");
                else asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(at) : "memory");
            }
        }
        return r;
    }
};

// Rows of a group of threads: piece `slot` of `slots` nearly equal runs of consecutive rows.
__device__ __forceinline__ int run_start(int rows, int slot, int slots) { return (int)((long long)rows * slot / slots); }

template <int WPR>
__device__ __forceinline__ void row_sync() {
    if (WPR == 1) __syncwarp();
    else __syncthreads();
}

constexpr int RN_FWD_STAGES = 4, RN_BWD_STAGES = 3;
template <typename T, int VEC, int NV, int WPR, int PER_SM> using FwdRing = Ring<T, VEC, NV, WPR, 3, RN_FWD_STAGES, PER_SM>;   // x, branch, a gate for each value
template <typename T, int VEC, int NV, int WPR, int PER_SM> using BwdRing = Ring<T, VEC, NV, WPR, 5, RN_BWD_STAGES, PER_SM>;   // y, dh, dy, branch, a gate for each value

template <typename T, int VEC, int NV, int WPR, int PER_SM>
__global__ void __launch_bounds__(rn_threads(WPR), PER_SM) residual_norm_fwd_kernel(const RNParams p) {
    typedef Vec<T, VEC> V;
    typedef typename V::raw raw;
    typedef FwdRing<T, VEC, NV, WPR, PER_SM> R;
    constexpr int TPR = 32 * WPR, ROWS = rn_threads(WPR) / TPR, STAGES = R::STAGES;
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ float words[2][32];
    const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR, width = p.comps * p.features;
    const bool own_gates = p.gate && p.groups == p.n;            // a gate for each value
    const R ring(smem_u32(ring_smem), p, own_gates ? 3 : 2);
    int turn = 0;
    chain_wait();
    chain_next();
    const float inv_width = 1.f / (float)width;
    const int slots = gridDim.x * ROWS, slot = blockIdx.x * ROWS + sub;
    const int begin = run_start(p.n, slot, slots), end = run_start(p.n, slot + 1, slots);
    auto fetch = [&](int row) {
        if (row < end) {
            const int stage = (row - begin) % STAGES;
            ring.fetch(p, stage, 0, p.x, row, p.n);
            if (p.branch) ring.fetch(p, stage, 1, p.branch, row, p.n);
            if (own_gates) ring.fetch(p, stage, 2, p.gate, row, p.n);
        }
        copies_commit();
    };
    for (int i = 0; i < STAGES; ++i) fetch(begin + i);
    raw gr[NV];
    int group = -1;
    // (with a CTA per row the runs of all its threads are one; with a warp per row there are no barriers)
    for (int row = begin; row < end; ++row) {
        const int stage = (row - begin) % STAGES;
        copies_wait<STAGES - 1>();
        if (VEC == 1) row_sync<WPR>();
        if (p.gate && !own_gates && row / p.per_group != group) {
            group = row / p.per_group;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                gr[i] = ld_chained(reinterpret_cast<const raw*>(static_cast<const T*>(p.gate) + (size_t)group * p.features + (size_t)c * (p.groups - 1) * p.features + e), e < width);
            }
        }
        const size_t row_at = (size_t)row * p.features;
        float y[NV][VEC];
        raw br[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            V::unpack(ring.get(p, stage, 0, i, row, p.n), y[i]);
            if (p.branch) br[i] = ring.get(p, stage, 1, i, row, p.n);
            if (own_gates) gr[i] = ring.get(p, stage, 2, i, row, p.n);
        }
        float rb = 0.f;
        if (!p.branch) row_sync<WPR>();
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
        }
        fetch(row + STAGES);                    // into the stage that every thread of the row has read by now
        if (p.branch) {
            const float f = p.scale * rb;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                float v[VEC], w[VEC], gv[VEC];
                V::unpack(br[i], v);
                load_weights<VEC>(p.post, e - c * p.features, e < width, w);
                if (p.gate) V::unpack(gr[i], gv);
#pragma unroll
                for (int j = 0; j < VEC; ++j) y[i][j] = fmaf(v[j] * f, p.gate ? w[j] * gv[j] : w[j], y[i][j]);
            }
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
            if (p.y && e < width) *reinterpret_cast<raw*>(static_cast<T*>(p.y) + row_at + (size_t)c * (p.n - 1) * p.features + e) = V::pack(y[i]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum = fmaf(y[i][j], y[i][j], sum);
        }
        float ry = 0.f;
        if (p.h) {
            ry = rsqrtf(row_sum<WPR>(sum, words, turn) * inv_width + p.eps);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                float w[VEC];
                load_weights<VEC>(p.pre, e - c * p.features, e < width, w);
#pragma unroll
                for (int j = 0; j < VEC; ++j) w[j] *= y[i][j] * ry;
                if (e < width) *reinterpret_cast<raw*>(static_cast<T*>(p.h) + row_at + (size_t)c * (p.n - 1) * p.features + e) = V::pack(w);
            }
        }
        if (p.stats && tid == 0) { p.stats[row] = rb; p.stats[p.n + row] = ry; }
    }
    copies_wait<0>();
}

// SHARED: gates shared by the samples of a group, whose gradients are sums
template <typename T, int VEC, int NV, int WPR, bool SHARED, int PER_SM>
__global__ void __launch_bounds__(rn_threads(WPR), PER_SM) residual_norm_bwd_kernel(const RNParams p) {
    typedef Vec<T, VEC> V;
    typedef typename V::raw raw;
    typedef BwdRing<T, VEC, NV, WPR, PER_SM> R;
    constexpr int TPR = 32 * WPR, ROWS = rn_threads(WPR) / TPR, STAGES = R::STAGES;
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ float words[2][32];
    const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR, width = p.comps * p.features;
    const bool own_gates = !SHARED && p.gate;                    // a gate for each value
    const R ring(smem_u32(ring_smem), p, own_gates ? 5 : 4);
    int turn = 0;
    chain_wait();
    chain_next();
    const float inv_width = 1.f / (float)width;
    float dpre[NV][VEC], dpost[NV][VEC], dgate[SHARED ? NV : 1][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) dpre[i][j] = dpost[i][j] = 0.f;
    const int slots = gridDim.x * ROWS, slot = blockIdx.x * ROWS + sub;
    // an item is a piece of a group of samples; the threads of a row take a run of items, whose rows follow each other
    const int item_begin = run_start(p.items, slot, slots), item_end = run_start(p.items, slot + 1, slots);
    auto item_row = [&](int item) {
        const int group = item / p.parts, part = item - group * p.parts;
        return group * p.per_group + (int)((long long)p.per_group * part / p.parts);
    };
    const int begin = item_row(item_begin), end = item_begin < item_end ? item_row(item_end) : begin;
    auto fetch = [&](int row) {
        if (row < end) {
            const int stage = (row - begin) % STAGES;
            if (p.dh) { ring.fetch(p, stage, 0, p.y, row, p.n); ring.fetch(p, stage, 1, p.dh, row, p.n); }
            if (p.dy) ring.fetch(p, stage, 2, p.dy, row, p.n);
            if (p.branch) ring.fetch(p, stage, 3, p.branch, row, p.n);
            if (own_gates) ring.fetch(p, stage, 4, p.gate, row, p.n);
        }
        copies_commit();
    };
    for (int i = 0; i < STAGES; ++i) fetch(begin + i);
    raw gr[NV];
    for (int item = item_begin; item < item_end; ++item) {
        const int group = item / p.parts, last = item_row(item + 1);
        if (SHARED) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                gr[i] = ld_chained(reinterpret_cast<const raw*>(static_cast<const T*>(p.gate) + (size_t)group * p.features + (size_t)c * (p.groups - 1) * p.features + e), e < width);
#pragma unroll
                for (int j = 0; j < VEC; ++j) dgate[i][j] = 0.f;
            }
        }
        for (int row = item_row(item); row < last; ++row) {
            const int stage = (row - begin) % STAGES;
            const size_t row_at = (size_t)row * p.features;
            const float rb = p.branch ? ld_chained(p.stats + row) : 0.f, ry = p.dh ? ld_chained(p.stats + p.n + row) : 0.f;
            copies_wait<STAGES - 1>();
            if (VEC == 1) row_sync<WPR>();
            raw br[NV];
            float dx[NV][VEC], y[NV][VEC];
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                if (p.dy) V::unpack(ring.get(p, stage, 2, i, row, p.n), dx[i]);
                else
#pragma unroll
                    for (int j = 0; j < VEC; ++j) dx[i][j] = 0.f;
                if (p.branch) br[i] = ring.get(p, stage, 3, i, row, p.n);
                if (own_gates) gr[i] = ring.get(p, stage, 4, i, row, p.n);
                if (p.dh) {
                    float t[VEC], w[VEC];
                    V::unpack(ring.get(p, stage, 0, i, row, p.n), y[i]);
                    V::unpack(ring.get(p, stage, 1, i, row, p.n), t);
                    load_weights<VEC>(p.pre, e - c * p.features, e < width, w);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float yn = y[i][j] * ry;
                        dpre[i][j] = fmaf(t[j], yn, dpre[i][j]);
                        t[j] *= w[j];
                        sum = fmaf(t[j], yn, sum);
                        dx[i][j] = fmaf(t[j], ry, dx[i][j]);
                    }
                }
            }
            float f = 0.f;
            if (p.dh) f = row_sum<WPR>(sum, words, turn) * inv_width * ry * ry;
            else row_sync<WPR>();
            fetch(row + STAGES);                // into the stage that every thread of the row has read by now
            if (p.dh) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) dx[i][j] = fmaf(-f, y[i][j], dx[i][j]);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                if (e < width) *reinterpret_cast<raw*>(static_cast<T*>(p.dx) + row_at + (size_t)c * (p.n - 1) * p.features + e) = V::pack(dx[i]);
            }
            if (p.branch) {
                sum = 0.f;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int e = (i * TPR + tid) * VEC, c = comp_of(p, e);
                    float b[VEC], w[VEC], g[VEC], dg[VEC];
                    V::unpack(br[i], b);
                    load_weights<VEC>(p.post, e - c * p.features, e < width, w);
                    if (SHARED || own_gates) V::unpack(gr[i], g);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float u = b[j] * rb, sdx = p.scale * dx[i][j], dn = SHARED || own_gates ? sdx * g[j] : sdx;
                        dpost[i][j] = fmaf(dn, u, dpost[i][j]);
                        dg[j] = sdx * u * w[j];
                        if (SHARED) dgate[i][j] += dg[j];
                        dx[i][j] = dn * w[j];
                        sum = fmaf(dx[i][j], u, sum);
                    }
                    if (own_gates && p.dgate && e < width) *reinterpret_cast<raw*>(static_cast<T*>(p.dgate) + row_at + (size_t)c * (p.n - 1) * p.features + e) = V::pack(dg);
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
        if (SHARED && p.dgate) {
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
    copies_wait<0>();
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

// Adds the pieces. Weights: eight columns (a sector) per CTA, the slots and components over 32 threads of each column. Gates: a thread per value.
constexpr int RN_SUM_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(RN_SUM_THREADS) residual_norm_sum_kernel(const RNParams p, int slots, int weight_blocks) {
    const int width = p.comps * p.features;
    chain_wait();
    chain_next();
    if ((int)blockIdx.x < weight_blocks) {
        __shared__ float sums[2][RN_SUM_THREADS / 8][8];
        const int col = threadIdx.x & 7, slice = threadIdx.x >> 3, f = blockIdx.x * 8 + col;
        float a = 0.f, b = 0.f;
        if (f < p.features) {
#pragma unroll 4
            for (int r = slice; r < slots * p.comps; r += RN_SUM_THREADS / 8) {
                const int s = r / p.comps, c = r - s * p.comps;
                const float* src = p.part_w + (size_t)s * 2 * width + (size_t)c * p.features + f;
                a += src[0];
                b += src[width];
            }
        }
        sums[0][slice][col] = a;
        sums[1][slice][col] = b;
        __syncthreads();
        if (threadIdx.x < 16 && blockIdx.x * 8 + (threadIdx.x & 7) < p.features) {
            const int which = threadIdx.x >> 3;
            float v = 0.f;
#pragma unroll
            for (int s = 0; s < RN_SUM_THREADS / 8; ++s) v += sums[which][s][col];
            float* out = which == 0 ? p.dpre : p.dpost;
            if (out) out[f] = v;
        }
    } else {
        const long long i = (long long)(blockIdx.x - weight_blocks) * RN_SUM_THREADS + threadIdx.x;
        if (i >= (long long)p.groups * width) return;
        const int group = (int)(i / width), e = (int)(i - (long long)group * width);
        float v = 0.f;
#pragma unroll 4
        for (int s = 0; s < p.parts; ++s) v += p.part_gate[((size_t)group * p.parts + s) * width + e];
        const int c = e / p.features;
        put<T>(p.dgate, (size_t)group * p.features + (size_t)c * (p.groups - 1) * p.features + e, v);
    }
}

// Whether the rows of every tensor are read 16 bytes at a time (vec values), and whether the tensors start on 16 bytes at all.
inline void alignment(const RNParams& p, int vec, bool& vectors, bool& bases) {
    uintptr_t tensors = 0;
    for (const void* t : {p.x, p.branch, p.gate, (const void*)p.y, (const void*)p.h, p.dy, p.dh, (const void*)p.dx, (const void*)p.dbranch, (const void*)p.dgate}) tensors |= reinterpret_cast<uintptr_t>(t);
    bases = tensors % 16 == 0;
    vectors = bases && p.features % vec == 0 && (reinterpret_cast<uintptr_t>(p.post) | reinterpret_cast<uintptr_t>(p.pre)) % 16 == 0;
}

template <typename K>
cudaError_t norm_launch(K kernel, int grid, int threads, size_t smem, cudaStream_t s, const RNParams& p) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_CTA_SMEM - 1024);     // (a limit, not what the launch asks for)
    return e != cudaSuccess ? e : launch_chained(kernel, grid, threads, smem, s, p);
}
template <typename T, int VEC, int EPT, int WPR, int PER_SM>
cudaError_t fwd_launch(const RNParams& p, cudaStream_t s) {
    constexpr int NV = EPT / VEC, THREADS = rn_threads(WPR), ROWS = THREADS / (32 * WPR);
    return norm_launch(residual_norm_fwd_kernel<T, VEC, NV, WPR, PER_SM>, grid_cap(p.n, ROWS, PER_SM), THREADS,
                       FwdRing<T, VEC, NV, WPR, PER_SM>::bytes(p, p.gate && p.groups == p.n ? 3 : 2), s, p);
}
template <typename T, int VEC>
cudaError_t fwd_any(const RNParams& p, cudaStream_t s) {
    constexpr int H = VEC == 1 ? 2 : 1;                         // (addresses of single values cost registers: half the CTAs)
    const RNShape k = fwd_shape((long long)p.comps * p.features);
    if (k.warps == 1) return fwd_launch<T, VEC, 16, 1, 6 / H>(p, s);
    if (k.warps == 8) return fwd_launch<T, VEC, 8, 8, 4 / H>(p, s);
    if (k.values == 8) return fwd_launch<T, VEC, 8, 16, 2 / H>(p, s);
    if (k.values == 16) return fwd_launch<T, VEC, 16, 16, 1>(p, s);
    return fwd_launch<T, VEC, 32, 16, 1>(p, s);
}
template <typename T, int VEC, int NV, int WPR, int PER_SM>
cudaError_t bwd_launch(const RNParams& p, const RNPlan& q, cudaStream_t s) {
    const bool shared = p.gate && p.groups != p.n;
    const size_t smem = BwdRing<T, VEC, NV, WPR, PER_SM>::bytes(p, p.gate && !shared ? 5 : 4);
    return shared ? norm_launch(residual_norm_bwd_kernel<T, VEC, NV, WPR, true, PER_SM>, q.grid, rn_threads(WPR), smem, s, p)
                  : norm_launch(residual_norm_bwd_kernel<T, VEC, NV, WPR, false, PER_SM>, q.grid, rn_threads(WPR), smem, s, p);
}
template <typename T, int VEC>
cudaError_t bwd_any(const RNParams& p, const RNPlan& q, cudaStream_t s) {
    switch (q.shape.warps) {
        case 1: return bwd_launch<T, VEC, 8 / VEC, 1, 4>(p, q, s);
        case 4: return bwd_launch<T, VEC, 8 / VEC, 4, 4>(p, q, s);
        case 8: return bwd_launch<T, VEC, 8 / VEC, 8, 2>(p, q, s);
        default: return q.shape.values == 8 ? bwd_launch<T, VEC, 8 / VEC, 16, 1>(p, q, s) : bwd_launch<T, VEC, 16 / VEC, 16, 1>(p, q, s);
    }
}
template <typename T, int VEC>
int fwd_typed(const RNParams& p, cudaStream_t s) {
    bool vec, bases;
    alignment(p, VEC, vec, bases);
    const RNShape k = fwd_shape((long long)p.comps * p.features);
    if (k.warps == 0 || !bases) PCB_CUDA_TRY(launch_chained(residual_norm_fwd_wide_kernel<T>, grid_cap(p.n, 1, 4), RN_WIDE_THREADS, 0, s, p));
    else if (vec) PCB_CUDA_TRY((fwd_any<T, VEC>(p, s)));
    else PCB_CUDA_TRY((fwd_any<T, 1>(p, s)));
    return PCB_OK;
}
template <typename T, int VEC>
int bwd_typed(const RNParams& p, const RNPlan& q, cudaStream_t s) {
    bool vec, bases;
    alignment(p, VEC, vec, bases);
    if (q.shape.warps == 0) PCB_CUDA_TRY(launch_chained(residual_norm_bwd_wide_kernel<T>, q.grid, RN_WIDE_THREADS, 0, s, p));
    else if (vec) PCB_CUDA_TRY((bwd_any<T, VEC>(p, q, s)));
    else PCB_CUDA_TRY((bwd_any<T, 1>(p, q, s)));
    const long long weight_blocks = p.part_w ? (p.features + 7) / 8 : 0;
    const long long gate_blocks = p.part_gate ? ((long long)p.groups * p.comps * p.features + RN_SUM_THREADS - 1) / RN_SUM_THREADS : 0;
    if (weight_blocks + gate_blocks > 0)
        PCB_CUDA_TRY(launch_chained(residual_norm_sum_kernel<T>, (unsigned)(weight_blocks + gate_blocks), RN_SUM_THREADS, 0, s, p, q.slots, (int)weight_blocks));
    return PCB_OK;
}

}  // namespace
}  // namespace pcb
