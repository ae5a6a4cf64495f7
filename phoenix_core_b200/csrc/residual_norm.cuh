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
#include "packed.cuh"
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

// The threads of a row (WPR warps; a CTA may hold several rows) wait for each other: barrier 1 + row of the CTA.
template <int WPR>
__device__ __forceinline__ void row_sync() {
    if (WPR == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / (32 * WPR)), "n"(32 * WPR) : "memory");
}
// Sum over the threads of a row. `words`: two sets of a word per warp, used in turn.
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* words, int& turn) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (WPR == 1) return v;
    const int warp = (threadIdx.x >> 5) % WPR, lane = threadIdx.x & 31;
    if (lane == 0) words[turn * WPR + warp] = v;
    row_sync<WPR>();
    constexpr int SPREAD = WPR <= 2 ? 2 : (WPR <= 4 ? 4 : (WPR <= 8 ? 8 : 16));      // lanes that the words are spread over, in a power of two
    const int word = lane & (SPREAD - 1);
    v = SPREAD == WPR || word < WPR ? words[turn * WPR + word] : 0.f;
#pragma unroll
    for (int o = SPREAD / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    turn ^= 1;
    return v;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A thread's values of a row, EPT of them in pairs, and the ring of row buffers in shared memory that cp.async fills some rows ahead, so that loads in flight cost
// no registers. A thread owns aligned vectors of 16 bytes and copies exactly what it reads later, so that no barrier is needed for that. Everything that does not change from
// row to row is worked out once: with 8 values per thread and that arithmetic in the loop a row took 44 instructions a value, and the pass was bound by issue slots.
//
// Rows whose length is no multiple of 16 bytes (!ALIGNED) start at one of `period` places within 16 bytes, and rows `period` apart at the same one. A CTA takes rows of
// one such class only, so that its threads' vectors hold the same features in every row; vectors that reach into a neighbouring row are masked, and
// stored value by value. (Value by value throughout, 3001 quaternion rows of 4 x 509 took 61 us backward.)
//
// One CTA per SM holds ROWS rows at a time, and the weights in shared memory: the ring leaves no L1 to speak of, and weights that came from L2 for every row were as
// many bytes as the rows (16384 x 4096 bf16: 115 us forward, 190 backward).
constexpr int RN_SMEM = 218 * 1024;
template <typename T, int VEC, bool ALIGNED, int EPT, int WPR, int ROWS_, int TENSORS, int MAX_STAGES>
struct Row {
    static constexpr int ROWS = ROWS_, TPR = 32 * WPR, THREADS = ROWS * TPR, NV = EPT / VEC, PAIRS = EPT / 2, SIZE = sizeof(T);
    static constexpr int TENSOR = NV * TPR * 16, STAGE = TENSORS * TENSOR, WEIGHTS = 2 * EPT * TPR * 4;   // bytes of a tensor's row, of a stage of one row, of both weights
    static constexpr bool HELD = WEIGHTS + ROWS * STAGE <= RN_SMEM;                           // weights in shared memory
    static constexpr int FIT = (RN_SMEM - (HELD ? WEIGHTS : 0)) / (ROWS * STAGE), STAGES = FIT < MAX_STAGES ? FIT : MAX_STAGES;
    static_assert(STAGES >= 1, "a row of every tensor fits");
    static_assert(EPT <= 32, "a bit for every value");
    static constexpr size_t SMEM = (size_t)ROWS * STAGES * STAGE + (HELD ? WEIGHTS : 0);
    static constexpr int RAW = NV * 4;                                                        // registers of a tensor's values as loaded
    static constexpr uint32_t FULL = (1u << VEC) - 1u;
    uint32_t base, held;                    // this thread's first vector in its row's ring; its weights: four at a time, TPR * 16 bytes apart
    int tid, width;
    int off[NV], feature[NV], comp[NV];     // first element of vector i relative to row * F; its feature (negative where it reaches back) and component
    uint32_t mask;                          // bit i * VEC + j: value j of vector i is one of the row's

    __device__ __forceinline__ Row(uint32_t smem, const RNParams& p, int row) {      // row: any of this CTA's
        tid = threadIdx.x % TPR;
        width = p.comps * p.features;
        base = smem + (HELD ? WEIGHTS : 0) + (threadIdx.x / TPR) * STAGES * STAGE + tid * 16;
        held = smem + tid * 16;
        mask = 0;
        const int per = ALIGNED ? p.features / VEC : (p.features + 2 * VEC - 2) / VEC;        // vectors of a component
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int v = i * TPR + tid, c = p.comps == 1 ? 0 : v / per;
            const long long first = ((long long)c * p.n + row) * p.features;
            const int shift = ALIGNED ? 0 : (int)(first & (VEC - 1));
            feature[i] = (v - c * per) * VEC - shift;
            off[i] = (int)((long long)c * p.n * p.features + feature[i]);
            comp[i] = c;
            if (c < p.comps && v - c * per < per) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (ALIGNED || (feature[i] + j >= 0 && feature[i] + j < p.features)) mask |= 1u << (i * VEC + j);
            }
        }
    }
    __device__ __forceinline__ uint32_t some(int i) const { return mask >> (i * VEC) & FULL; }
    // starts the copies of a row of each tensor (null: none)
    __device__ __forceinline__ void fetch(const RNParams& p, int stage, int row, const void* const (&tensors)[TENSORS]) const {
        const uint32_t dst = base + stage * STAGE;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!some(i)) continue;
            const long long element = (long long)row * p.features + off[i];
            uint32_t bytes = 16;
            if (!ALIGNED) {                                      // the last vector of a tensor ends where the tensor does
                const long long left = ((long long)p.n * width - element) * SIZE;
                bytes = left < 16 ? (uint32_t)left : 16u;
            }
#pragma unroll
            for (int k = 0; k < TENSORS; ++k)
                if (tensors[k]) copy16(dst + k * TENSOR + i * TPR * 16, static_cast<const T*>(tensors[k]) + element, bytes);
        }
    }
    // this thread's values of tensor k of a row that has arrived, as loaded (zeros where there are none)
    __device__ __forceinline__ void get(int stage, int k, uint32_t (&raw)[RAW]) const {
        const uint32_t src = base + stage * STAGE + k * TENSOR;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (some(i)) v = ld_shared_v4(src + i * TPR * 16);
            if (!ALIGNED && some(i) != FULL) {
                uint32_t* w = &v.x;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (VEC == 8) w[j] &= (mask >> (i * VEC + 2 * j) & 1 ? 0xffffu : 0u) | (mask >> (i * VEC + 2 * j + 1) & 1 ? 0xffff0000u : 0u);
                    else w[j] = mask >> (i * VEC + j) & 1 ? w[j] : 0u;
                }
            }
            raw[4 * i] = v.x; raw[4 * i + 1] = v.y; raw[4 * i + 2] = v.z; raw[4 * i + 3] = v.w;
        }
    }
    __device__ __forceinline__ static Pair value(const uint32_t (&raw)[RAW], int q) {
        if constexpr (SIZE == 4) return pair(__uint_as_float(raw[2 * q]), __uint_as_float(raw[2 * q + 1]));
        else return pair(from16<T>(raw[q] & 0xffffu), from16<T>(raw[q] >> 16));
    }
    // a row of the gate (once for a group)
    __device__ __forceinline__ void load_gate(const RNParams& p, int group, Pair (&v)[PAIRS]) const {
#pragma unroll
        for (int q = 0; q < PAIRS; ++q) {
            const int i = 2 * q / VEC, j = 2 * q % VEC;
            const typename Vec<T, 1>::raw* src = static_cast<const typename Vec<T, 1>::raw*>(p.gate) + ((size_t)comp[i] * p.groups + group) * p.features + feature[i] + j;
            float a, b;
            Vec<T, 1>::unpack(ld_chained(src, mask >> (2 * q) & 1), &a);
            Vec<T, 1>::unpack(ld_chained(src + 1, mask >> (2 * q + 1) & 1), &b);
            v[q] = pair(a, b);
        }
    }
    __device__ __forceinline__ void store_at(T* dst, int i, const Pair (&v)[PAIRS]) const {
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) halves(v[i * (VEC / 2) + j], f[2 * j], f[2 * j + 1]);
        if (ALIGNED || some(i) == FULL) {
            *reinterpret_cast<uint4*>(dst) = Vec<T, VEC>::pack(f);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (mask >> (i * VEC + j) & 1) reinterpret_cast<typename Vec<T, 1>::raw*>(dst)[j] = Vec<T, 1>::pack(&f[j]);
        }
    }
    __device__ __forceinline__ void store(void* tensor, const RNParams& p, int row, const Pair (&v)[PAIRS]) const {
        T* line = static_cast<T*>(tensor) + (size_t)row * p.features;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (some(i)) store_at(line + off[i], i, v);
    }
    // a row of the gate's gradient (value by value where its rows start elsewhere than the samples')
    __device__ __forceinline__ void store_gate(const RNParams& p, int group, const Pair (&v)[PAIRS]) const {
#pragma unroll
        for (int q = 0; q < PAIRS; ++q) {
            const int i = 2 * q / VEC, j = 2 * q % VEC;
            typename Vec<T, 1>::raw* dst = static_cast<typename Vec<T, 1>::raw*>(p.dgate) + ((size_t)comp[i] * p.groups + group) * p.features + feature[i] + j;
            float a, b;
            halves(v[q], a, b);
            if (mask >> (2 * q) & 1) dst[0] = Vec<T, 1>::pack(&a);
            if (mask >> (2 * q + 1) & 1) dst[1] = Vec<T, 1>::pack(&b);
        }
    }
    // Weights of this thread's features (ones where there are none), from global memory: plain loads, nothing marks these pointers as read-only.
    __device__ __forceinline__ void load_weights(const float* w, Pair (&v)[PAIRS]) const {
#pragma unroll
        for (int q = 0; q < PAIRS; ++q) {
            v[q] = pair(1.f);
            const int at = feature[2 * q / VEC] + 2 * q % VEC;
            if (w) v[q] = pair(mask >> (2 * q) & 1 ? w[at] : 1.f, mask >> (2 * q + 1) & 1 ? w[at + 1] : 1.f);
        }
    }
    // the first row's threads put them into shared memory (followed by a barrier of the CTA); `which`: 0 post, 1 pre
    __device__ __forceinline__ void hold_weights(const RNParams& p) const {
        if (!HELD) return;
        if (threadIdx.x < TPR) {
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                Pair v[PAIRS];
                load_weights(which ? p.pre : p.post, v);
                const uint32_t dst = held + which * (WEIGHTS / 2);
#pragma unroll
                for (int q = 0; q < PAIRS; ++q) asm volatile("st.shared.b64 [%0], %1;" ::"r"(dst + (q / 2) * TPR * 16 + (q & 1) * 8), "l"(v[q].v) : "memory");
            }
        }
        __syncthreads();
    }
    __device__ __forceinline__ void weights(const RNParams& p, int which, Pair (&v)[PAIRS]) const {
        if constexpr (!HELD) load_weights(which ? p.pre : p.post, v);
        else {
            const uint32_t src = held + which * (WEIGHTS / 2);
#pragma unroll
            for (int q = 0; q < PAIRS; q += 2) asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(v[q].v), "=l"(v[q + 1].v) : "r"(src + (q / 2) * TPR * 16));
        }
    }
    // this thread's sums to out[component * F + feature]
    __device__ __forceinline__ void store_sums(const RNParams& p, float* out, const Pair (&v)[PAIRS]) const {
#pragma unroll
        for (int q = 0; q < PAIRS; ++q) {
            const int i = 2 * q / VEC;
            float* dst = out + (size_t)comp[i] * p.features + feature[i] + 2 * q % VEC;
            float a, b;
            halves(v[q], a, b);
            if (mask >> (2 * q) & 1) dst[0] = a;
            if (mask >> (2 * q + 1) & 1) dst[1] = b;
        }
    }
};

// Class of a CTA (where its rows start within 16 bytes), its rank within the class, and the class's CTAs.
__device__ __forceinline__ void class_of(int period, int& cls, int& rank, int& of) {
    cls = blockIdx.x % period;
    rank = blockIdx.x / period;
    of = (gridDim.x - cls + period - 1) / period;
}

// Where run `slot` of `slots` nearly equal runs of `rows` things starts.
__device__ __forceinline__ int run_start(int rows, int slot, int slots) { return (int)((long long)rows * slot / slots); }

constexpr int RN_FWD_STAGES = 4, RN_BWD_STAGES = 3;
// OWN, GATE 1: a gate for each value
template <typename T, int VEC, bool ALIGNED, int EPT, int WPR, int ROWS, bool OWN> using FwdRow = Row<T, VEC, ALIGNED, EPT, WPR, ROWS, OWN ? 3 : 2, RN_FWD_STAGES>;        // x, branch, gate
template <typename T, int VEC, bool ALIGNED, int EPT, int WPR, int ROWS, int GATE> using BwdRow = Row<T, VEC, ALIGNED, EPT, WPR, ROWS, GATE == 1 ? 5 : 4, RN_BWD_STAGES>;  // y, dh, dy, branch, gate

template <typename T, int VEC, bool ALIGNED, int EPT, int WPR, int ROWS, bool OWN>
__global__ void __launch_bounds__(32 * WPR * ROWS, 1) residual_norm_fwd_kernel(const RNParams p) {
    typedef FwdRow<T, VEC, ALIGNED, EPT, WPR, ROWS, OWN> R;
    constexpr int STAGES = R::STAGES, PAIRS = R::PAIRS;
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ float all_words[R::ROWS][2 * WPR];
    float* words = all_words[threadIdx.x / R::TPR];
    const int period = ALIGNED ? 1 : p.period;
    int cls, rank, of, turn = 0;
    class_of(period, cls, rank, of);
    const R r(smem_u32(ring_smem), p, cls);
    chain_wait();
    chain_next();
    r.hold_weights(p);
    const float inv_width = 1.f / (float)r.width;
    const int count = cls < p.n ? (p.n - cls + period - 1) / period : 0;        // rows of the class
    const int slots = of * R::ROWS, slot = rank * R::ROWS + threadIdx.x / R::TPR;
    const int begin = run_start(count, slot, slots), end = run_start(count, slot + 1, slots);
    const void* tensors[OWN ? 3 : 2];
    tensors[0] = p.x; tensors[1] = p.branch;
    if constexpr (OWN) tensors[2] = p.gate;
    auto fetch = [&](int t, int stage) {
        if (t < end) r.fetch(p, stage, cls + period * t, *reinterpret_cast<const void* const(*)[OWN ? 3 : 2]>(&tensors));
        copies_commit();
    };
    for (int i = 0; i < STAGES; ++i) fetch(begin + i, i);
    Pair gate[OWN ? 1 : PAIRS];
    int group_end = 0, stage = 0;                                // (shared gates: the row behind the present group)
    // (the threads of a row run through the same rows; different rows of a CTA have no barrier in common)
    for (int t = begin; t < end; ++t) {
        const int row = cls + period * t;
        copies_wait<STAGES - 1>();
        if constexpr (!OWN) {
            if (p.gate && row >= group_end) {
                const int group = row / p.per_group;
                group_end = (group + 1) * p.per_group;
                r.load_gate(p, group, gate);
            }
        }
        Pair y[PAIRS];
        float rb = 0.f;
        {
            uint32_t xraw[R::RAW], braw[R::RAW], graw[OWN ? R::RAW : 1];
            r.get(stage, 0, xraw);
            if (p.branch) r.get(stage, 1, braw);
            if constexpr (OWN) r.get(stage, 2, graw);
            if (p.branch) {
                Pair s = pair(0.f);
#pragma unroll
                for (int q = 0; q < PAIRS; ++q) { const Pair b = R::value(braw, q); s = fma2(b, b, s); }
                rb = rsqrtf(row_sum<WPR>(sum(s), words, turn) * inv_width + p.eps);
            } else row_sync<WPR>();
            fetch(t + STAGES, stage);                            // into the stage that has been read by now
            if (p.branch) {
                const Pair f = pair(p.scale * rb);
                Pair w[PAIRS];
                r.weights(p, 0, w);
                if constexpr (OWN) {
#pragma unroll
                    for (int q = 0; q < PAIRS; ++q) w[q] = w[q] * R::value(graw, q);
                } else if (p.gate) {
#pragma unroll
                    for (int q = 0; q < PAIRS; ++q) w[q] = w[q] * gate[q];
                }
#pragma unroll
                for (int q = 0; q < PAIRS; ++q) y[q] = fma2(R::value(braw, q) * f, w[q], R::value(xraw, q));
            } else {
#pragma unroll
                for (int q = 0; q < PAIRS; ++q) y[q] = R::value(xraw, q);
            }
        }
        if (p.y) r.store(p.y, p, row, y);
        float ry = 0.f;
        if (p.h) {
            Pair s = pair(0.f), w[PAIRS];
#pragma unroll
            for (int q = 0; q < PAIRS; ++q) s = fma2(y[q], y[q], s);
            r.weights(p, 1, w);
            ry = rsqrtf(row_sum<WPR>(sum(s), words, turn) * inv_width + p.eps);
            const Pair f = pair(ry);
#pragma unroll
            for (int q = 0; q < PAIRS; ++q) y[q] = y[q] * f * w[q];
            r.store(p.h, p, row, y);
        }
        if (p.stats && r.tid == 0) { p.stats[row] = rb; p.stats[p.n + row] = ry; }
        if (++stage == STAGES) stage = 0;
    }
    copies_wait<0>();
}

// GATE: 0 none, 1 a gate for each value, 2 gates shared by the samples of a group, whose gradients are sums
template <typename T, int VEC, bool ALIGNED, int EPT, int WPR, int ROWS, int GATE>
__global__ void __launch_bounds__(32 * WPR * ROWS, 1) residual_norm_bwd_kernel(const RNParams p) {
    typedef BwdRow<T, VEC, ALIGNED, EPT, WPR, ROWS, GATE> R;
    constexpr int STAGES = R::STAGES, PAIRS = R::PAIRS;
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ float all_words[R::ROWS][2 * WPR];
    float* words = all_words[threadIdx.x / R::TPR];
    const int period = ALIGNED ? 1 : p.period;
    int cls, rank, of, turn = 0;
    class_of(period, cls, rank, of);
    const R r(smem_u32(ring_smem), p, cls);
    chain_wait();
    chain_next();
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.status = 0;
    r.hold_weights(p);
    const float inv_width = 1.f / (float)r.width;
    const int slots = of * R::ROWS, slot = rank * R::ROWS + threadIdx.x / R::TPR;
    // Shared gates: an item is a piece of a group's rows of this class; the threads of a row take a run of items, whose rows follow each other. Otherwise a run of rows.
    const int items = GATE == 2 ? p.groups * p.pieces : (cls < p.n ? (p.n - cls + period - 1) / period : 0);
    const int item_begin = run_start(items, slot, slots), item_end = run_start(items, slot + 1, slots);
    auto rows_before = [&](int row) { return row > cls ? (row - cls + period - 1) / period : 0; };           // rows of the class in front of `row`
    auto item_start = [&](int item) {
        if (GATE != 2) return item;
        const int group = item / p.pieces, piece = item - group * p.pieces, a = rows_before(group * p.per_group);
        return group == p.groups ? rows_before(p.n) : a + run_start(rows_before((group + 1) * p.per_group) - a, piece, p.pieces);
    };
    const int begin = item_start(item_begin), end = item_begin < item_end ? item_start(item_end) : begin;
    const void* tensors[GATE == 1 ? 5 : 4];
    tensors[0] = p.dh ? p.y : nullptr; tensors[1] = p.dh; tensors[2] = p.dy; tensors[3] = p.branch;
    if constexpr (GATE == 1) tensors[4] = p.gate;
    auto fetch = [&](int t, int stage) {
        if (t < end) r.fetch(p, stage, cls + period * t, *reinterpret_cast<const void* const(*)[GATE == 1 ? 5 : 4]>(&tensors));
        copies_commit();
    };
    for (int i = 0; i < STAGES; ++i) fetch(begin + i, i);
    // What a gate that stays the same over rows multiplies can wait for its last row: with a = scale * gate and G = sum of dx * u over the rows,
    //   dpost += a * G,   dgate = scale * post * G,   v = dx * (a * post)
    Pair dpre[PAIRS], dpost[PAIRS], g_sum[PAIRS], factor[GATE == 1 ? 1 : PAIRS];
#pragma unroll
    for (int q = 0; q < PAIRS; ++q) dpre[q] = dpost[q] = g_sum[q] = pair(0.f);
    if constexpr (GATE == 0) {
        r.weights(p, 0, factor);
#pragma unroll
        for (int q = 0; q < PAIRS; ++q) factor[q] = factor[q] * pair(p.scale);
    }
    int item = item_begin - 1, last = begin, stage = 0;          // last: behind the rows of the present item
    for (int t = begin; t < end; ++t) {
        const int row = cls + period * t;
        if (GATE == 2 && t == last) {
            ++item;
            last = item_start(item + 1);
            if constexpr (GATE == 2) {
                Pair w[PAIRS];
                r.load_gate(p, item / p.pieces, factor);
                r.weights(p, 0, w);
#pragma unroll
                for (int q = 0; q < PAIRS; ++q) { factor[q] = factor[q] * pair(p.scale) * w[q]; g_sum[q] = pair(0.f); }
            }
        }
        const float rb = p.branch ? ld_chained(p.stats + row) : 0.f, ry = p.dh ? ld_chained(p.stats + p.n + row) : 0.f;
        copies_wait<STAGES - 1>();
        uint32_t braw[R::RAW], graw[GATE == 1 ? R::RAW : 1];
        Pair dx[PAIRS];
        if (p.dy) {
            uint32_t raw[R::RAW];
            r.get(stage, 2, raw);
#pragma unroll
            for (int q = 0; q < PAIRS; ++q) dx[q] = R::value(raw, q);
        } else {
#pragma unroll
            for (int q = 0; q < PAIRS; ++q) dx[q] = pair(0.f);
        }
        if (p.branch) r.get(stage, 3, braw);
        if constexpr (GATE == 1) r.get(stage, 4, graw);
        if (p.dh) {
            uint32_t raw[R::RAW], yraw[R::RAW];
            Pair w[PAIRS], s = pair(0.f);
            r.get(stage, 0, yraw);
            r.get(stage, 1, raw);
            r.weights(p, 1, w);
            const Pair f = pair(ry);
#pragma unroll
            for (int q = 0; q < PAIRS; ++q) {
                const Pair y = R::value(yraw, q), z = R::value(raw, q) * f, v = z * w[q];        // dh * r(y), t * r(y)
                dpre[q] = fma2(z, y, dpre[q]);
                s = fma2(v, y, s);
                dx[q] = dx[q] + v;
            }
            const Pair m = pair(-(row_sum<WPR>(sum(s), words, turn) * inv_width * ry * ry));
            fetch(t + STAGES, stage);                            // into the stage that has been read by now
#pragma unroll
            for (int q = 0; q < PAIRS; ++q) dx[q] = fma2(m, R::value(yraw, q), dx[q]);
        } else {
            row_sync<WPR>();
            fetch(t + STAGES, stage);
        }
        r.store(p.dx, p, row, dx);
        if (p.branch) {
            Pair s = pair(0.f);
            const Pair f = pair(rb);
            if constexpr (GATE == 1) {
                Pair w[PAIRS], dg[PAIRS];
                const Pair scale = pair(p.scale);
                r.weights(p, 0, w);
#pragma unroll
                for (int q = 0; q < PAIRS; ++q) {
                    const Pair u = R::value(braw, q) * f, sdx = scale * dx[q], dn = sdx * R::value(graw, q);
                    dg[q] = sdx * u * w[q];
                    dpost[q] = fma2(dn, u, dpost[q]);
                    dx[q] = dn * w[q];
                    s = fma2(dx[q], u, s);
                }
                if (p.dgate) r.store(p.dgate, p, row, dg);
            } else {
#pragma unroll
                for (int q = 0; q < PAIRS; ++q) {
                    const Pair u = R::value(braw, q) * f;
                    g_sum[q] = fma2(dx[q], u, g_sum[q]);
                    dx[q] = dx[q] * factor[q];
                    s = fma2(dx[q], u, s);
                }
            }
            const Pair m = pair(-(row_sum<WPR>(sum(s), words, turn) * inv_width * rb));
#pragma unroll
            for (int q = 0; q < PAIRS; ++q) dx[q] = f * fma2(m, R::value(braw, q), dx[q]);
            r.store(p.dbranch, p, row, dx);
        }
        if constexpr (GATE == 2) {
            if (t + 1 == last) {
                const int group = item / p.pieces, piece = item - group * p.pieces;
                const Pair scale = pair(p.scale);
                Pair w[PAIRS], gate[PAIRS];
                r.load_gate(p, group, gate);
                r.weights(p, 0, w);
#pragma unroll
                for (int q = 0; q < PAIRS; ++q) {
                    dpost[q] = fma2(gate[q] * scale, g_sum[q], dpost[q]);
                    g_sum[q] = g_sum[q] * scale * w[q];
                }
                if (p.dgate) {
                    if (p.part_gate) r.store_sums(p, p.part_gate + ((size_t)group * p.parts + cls * p.pieces + piece) * r.width, g_sum);
                    else r.store_gate(p, group, g_sum);
                }
            }
        }
        if (++stage == STAGES) stage = 0;
    }
    copies_wait<0>();
    if (GATE == 0) {
#pragma unroll
        for (int q = 0; q < PAIRS; ++q) dpost[q] = g_sum[q] * pair(p.scale);
    }
    if (p.part_w) {
        // the rows of the CTA together, in shared memory (nothing reads the ring any more)
        float* out = p.part_w + (size_t)blockIdx.x * 2 * r.width;
        if constexpr (R::ROWS > 1) {
            static_assert((size_t)R::ROWS * 2 * EPT * R::TPR * 4 <= R::SMEM, "sums of the rows");
            float* sums = reinterpret_cast<float*>(ring_smem);
            __syncthreads();
            float* mine = sums + (size_t)(threadIdx.x / R::TPR) * 2 * r.width;
            r.store_sums(p, mine, dpre);
            r.store_sums(p, mine + r.width, dpost);
            __syncthreads();
            for (int e = threadIdx.x; e < 2 * r.width; e += R::THREADS) {
                float v = sums[e];
                for (int k = 1; k < R::ROWS; ++k) v += sums[(size_t)k * 2 * r.width + e];
                out[e] = v;
            }
        } else {
            r.store_sums(p, out, dpre);
            r.store_sums(p, out + r.width, dpost);
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
    __shared__ float words[2 * WPR];
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

template <typename T, bool OWN>
__global__ void __launch_bounds__(RN_WIDE_THREADS) residual_norm_bwd_wide_kernel(const RNParams p) {
    constexpr int WPR = RN_WIDE_THREADS / 32;
    __shared__ float words[2 * WPR];
    int turn = 0;
    chain_wait();
    chain_next();
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.status = 0;
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
                        if constexpr (OWN) {
                            if (p.dgate) put<T>(p.dgate, (c * (size_t)p.groups + group) * F + f, dg);
                        } else if (gates) gates[c * F + f] = row == begin ? dg : gates[c * F + f] + dg;
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

// Adds the pieces. Weights: eight columns (a sector) per CTA, the slots and components over 64 threads of each column. Gates: 1 to 64 threads per value.
constexpr int RN_SUM_THREADS = 512;
template <typename T>
__global__ void __launch_bounds__(RN_SUM_THREADS) residual_norm_sum_kernel(const RNParams p, int slots, int weight_blocks, int slices) {
    const int width = p.comps * p.features;
    chain_wait();
    chain_next();
    if ((int)blockIdx.x < weight_blocks) {
        __shared__ float sums[2][RN_SUM_THREADS / 8][8];
        const int col = threadIdx.x & 7, slice = threadIdx.x >> 3, f = blockIdx.x * 8 + col;
        float a = 0.f, b = 0.f;
        if (f < p.features) {
#pragma unroll 8
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
        // `slices` threads of a value each add up their share of the parts
        __shared__ float parts[RN_SUM_THREADS];
        const int values = RN_SUM_THREADS / slices, col = threadIdx.x % values, slice = threadIdx.x / values;
        const long long i = (long long)(blockIdx.x - weight_blocks) * values + col;
        const bool live = i < (long long)p.groups * width;
        const int group = live ? (int)(i / width) : 0, e = live ? (int)(i - (long long)group * width) : 0;
        float v = 0.f;
        if (live) {
#pragma unroll 4
            for (int s = slice; s < p.parts; s += slices) v += p.part_gate[((size_t)group * p.parts + s) * width + e];
        }
        parts[threadIdx.x] = v;
        __syncthreads();
        if (slice == 0 && live) {
            for (int s = 1; s < slices; ++s) v += parts[s * values + col];
            const int c = e / p.features;
            put<T>(p.dgate, (size_t)group * p.features + (size_t)c * (p.groups - 1) * p.features + e, v);
        }
    }
}

// Whether every tensor starts on 16 bytes.
inline bool aligned_bases(const RNParams& p) {
    uintptr_t tensors = 0;
    for (const void* t : {p.x, p.branch, (const void*)p.y, (const void*)p.h, p.dy, p.dh, (const void*)p.dx, (const void*)p.dbranch}) tensors |= reinterpret_cast<uintptr_t>(t);
    if (p.gate && p.groups == p.n) tensors |= reinterpret_cast<uintptr_t>(p.gate) | reinterpret_cast<uintptr_t>(p.dgate);
    return tensors % 16 == 0;
}

template <auto Kernel>
cudaError_t norm_launch(int grid, int threads, size_t smem, cudaStream_t s, const RNParams& p) {
    const cudaError_t e = allow_cta_smem<Kernel>(MAX_CTA_SMEM - 1024);             // (the sums' words are static)
    return e != cudaSuccess ? e : launch_chained(Kernel, grid, threads, smem, s, p);
}
template <typename T, int VEC, bool ALIGNED, int EPT, int WPR, int ROWS, bool OWN>
cudaError_t fwd_own(const RNParams& p, cudaStream_t s) {
    typedef FwdRow<T, VEC, ALIGNED, EPT, WPR, ROWS, OWN> R;
    const int least = p.n < p.period ? p.n : p.period, grid = grid_cap(p.n, ROWS, 1);          // a CTA for each place that rows start at
    return norm_launch<residual_norm_fwd_kernel<T, VEC, ALIGNED, EPT, WPR, ROWS, OWN>>(grid < least ? least : grid, R::THREADS, R::SMEM, s, p);
}
template <typename T, int VEC, bool ALIGNED, int EPT, int WPR, int ROWS>
cudaError_t fwd_launch(const RNParams& p, cudaStream_t s) {
    return p.gate && p.groups == p.n ? fwd_own<T, VEC, ALIGNED, EPT, WPR, ROWS, true>(p, s) : fwd_own<T, VEC, ALIGNED, EPT, WPR, ROWS, false>(p, s);
}
template <typename T, int VEC, bool ALIGNED>
cudaError_t fwd_any(const RNParams& p, const RNShape& k, cudaStream_t s) {
    if (k.warps == 1) return k.values == 8 ? fwd_launch<T, VEC, ALIGNED, 8, 1, 16>(p, s) : fwd_launch<T, VEC, ALIGNED, 32, 1, 12>(p, s);
    if (k.warps == 4) return k.values == 16 ? fwd_launch<T, VEC, ALIGNED, 16, 4, 4>(p, s) : fwd_launch<T, VEC, ALIGNED, 32, 4, 3>(p, s);
    if (k.warps == 5) return fwd_launch<T, VEC, ALIGNED, 16, 5, 3>(p, s);
    return k.warps == 8 ? fwd_launch<T, VEC, ALIGNED, 32, 8, 1>(p, s) : fwd_launch<T, VEC, ALIGNED, 32, 16, 1>(p, s);
}
template <typename T, int VEC, bool ALIGNED, int EPT, int WPR, int ROWS, int GATE>
cudaError_t bwd_gate(const RNParams& p, int grid, cudaStream_t s) {
    typedef BwdRow<T, VEC, ALIGNED, EPT, WPR, ROWS, GATE> R;
    return norm_launch<residual_norm_bwd_kernel<T, VEC, ALIGNED, EPT, WPR, ROWS, GATE>>(grid, R::THREADS, R::SMEM, s, p);
}
template <typename T, int VEC, bool ALIGNED, int EPT, int WPR, int ROWS>
cudaError_t bwd_launch(const RNParams& p, int grid, cudaStream_t s) {
    if (!p.gate) return bwd_gate<T, VEC, ALIGNED, EPT, WPR, ROWS, 0>(p, grid, s);
    return p.groups == p.n ? bwd_gate<T, VEC, ALIGNED, EPT, WPR, ROWS, 1>(p, grid, s) : bwd_gate<T, VEC, ALIGNED, EPT, WPR, ROWS, 2>(p, grid, s);
}
template <typename T, int VEC, bool ALIGNED>
cudaError_t bwd_any(const RNParams& p, const RNShape& k, int grid, cudaStream_t s) {
    switch (k.warps) {
        case 1: return k.values == 8 ? bwd_launch<T, VEC, ALIGNED, 8, 1, 16>(p, grid, s) : bwd_launch<T, VEC, ALIGNED, 16, 1, 12>(p, grid, s);
        case 2: return bwd_launch<T, VEC, ALIGNED, 16, 2, 6>(p, grid, s);
        case 3: return bwd_launch<T, VEC, ALIGNED, 16, 3, 4>(p, grid, s);
        case 4: return bwd_launch<T, VEC, ALIGNED, 16, 4, 3>(p, grid, s);
        case 5: return bwd_launch<T, VEC, ALIGNED, 16, 5, 3>(p, grid, s);
        case 8: return bwd_launch<T, VEC, ALIGNED, 16, 8, 2>(p, grid, s);
        default: return bwd_launch<T, VEC, ALIGNED, 16, 16, 1>(p, grid, s);
    }
}
template <typename T, int VEC>
int fwd_typed(RNParams p, cudaStream_t s) {
    p.period = row_period(p.features, sizeof(T));
    const RNShape k = fwd_shape(padded_width(p.comps, p.features, sizeof(T)));
    if (k.warps == 0 || !aligned_bases(p)) PCB_CUDA_TRY(launch_chained(residual_norm_fwd_wide_kernel<T>, grid_cap(p.n, 1, 4), RN_WIDE_THREADS, 0, s, p));
    else if (p.period == 1) PCB_CUDA_TRY((fwd_any<T, VEC, true>(p, k, s)));
    else PCB_CUDA_TRY((fwd_any<T, VEC, false>(p, k, s)));
    return PCB_OK;
}
template <typename T, int VEC>
int bwd_typed(RNParams p, RNPlan q, cudaStream_t s) {
    p.period = row_period(p.features, sizeof(T));
    const bool wide = q.shape.warps == 0 || !aligned_bases(p);
    if (wide) q = q.shape.warps == 0 ? q : wide_plan(p.comps, p.n, p.features, p.gate ? p.groups : 0);
    p.parts = q.parts; p.pieces = q.pieces; p.items = q.items;
    // (beside an SM margin fewer CTAs take the same pieces: the plan, and with it the workspace, is that of the whole device)
    const int grid = wide ? (q.grid < 4 * sm_count() ? q.grid : 4 * sm_count()) : ctas_beside(q.grid, p.period, sm_count());
    p.part_w = p.dpost || p.dpre ? reinterpret_cast<float*>(p.workspace) : nullptr;
    p.part_gate = p.dgate && q.part_gate ? reinterpret_cast<float*>(p.workspace + q.part_w) : nullptr;
    if (wide && p.gate && p.groups == p.n) PCB_CUDA_TRY((launch_chained(residual_norm_bwd_wide_kernel<T, true>, grid, RN_WIDE_THREADS, 0, s, p)));
    else if (wide) PCB_CUDA_TRY((launch_chained(residual_norm_bwd_wide_kernel<T, false>, grid, RN_WIDE_THREADS, 0, s, p)));
    else if (p.period == 1) PCB_CUDA_TRY((bwd_any<T, VEC, true>(p, q.shape, grid, s)));
    else PCB_CUDA_TRY((bwd_any<T, VEC, false>(p, q.shape, grid, s)));
    const long long weight_blocks = p.part_w ? (p.features + 7) / 8 : 0;
    // threads per value of a gate: up to two values' worth for every SM's 2048, while each has two parts at least (5358 x 174, one gate: 17 us, 177 by one thread each; 16384 x 4096,
    // 16 gates of 111 parts: 13 us, 47 with 64 each)
    int slices = 1;
    while (slices < 64 && slices * 4 <= q.parts && (long long)p.groups * p.comps * p.features * slices < 2048LL * device_sms()) slices *= 2;
    const int values = RN_SUM_THREADS / slices;
    const long long gate_blocks = p.part_gate ? ((long long)p.groups * p.comps * p.features + values - 1) / values : 0;
    if (weight_blocks + gate_blocks > 0)
        PCB_CUDA_TRY(launch_chained(residual_norm_sum_kernel<T>, (unsigned)(weight_blocks + gate_blocks), RN_SUM_THREADS, 0, s, p, grid, (int)weight_blocks, slices));
    return PCB_OK;
}

}  // namespace
}  // namespace pcb
