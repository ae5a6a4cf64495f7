// Distillation from a teacher's largest logits, mixed with the cross-entropy of the labels.
//
// A sample has V = D * U logits z (U units of each of D components, class = component * U + unit), a label c, and for k classes i the teacher's logits t_i.
//   p = softmax(t / T) over the k classes, q = softmax(z / T) over all of them
//   loss = (1 - a) * (log sum_j exp z_j - z_c) + a * T^2 * sum_i p_i (log p_i - log q_i)
//   dz_j = g * ((1 - a) * (softmax(z)_j - [j = c]) + a * T * (q_j - p_j))
// Both sums over the vocabulary are taken in one pass with a running maximum; the gradient reads the logits once more and writes
// them once. With T = 2 the exponentials of T = 1 are the squares of the others: one exponential per logit, which keeps the pass bound by memory
// (16 exponentials per clock and SM are two thirds of what a pass over 16-bit logits takes at full bandwidth). 4096 x 131072 bf16: 192 us forward (5.6 TB/s), 346
// backward (6.2 TB/s both ways) from cold caches, 178 and 337 behind themselves; bound by memory.
// Few rows are cut over the CTAs of a cluster, whose maxima and sums are joined through distributed shared memory.
#include "class_shares.h"
#include "common.cuh"
#include "packed.cuh"
#include "tc_common.cuh"

namespace pcb {
namespace {

using namespace tc;

constexpr int DI_MAX_ENTRIES = 4096;
constexpr float LOG2E = 1.4426950408889634f;

enum { DI_HARD = 0, DI_SOFT = 1, DI_SAME = 2, DI_SQUARE = 3, DI_BOTH = 4 };   // exponentials: at 1, at T, T == 1, T == 2, both

struct DIParams {
    int comps, n, units, entries, splits;
    float alpha, temp, inv_temp;
    const void *logits, *teacher;
    const long long *labels, *index;
    float *loss, *stats;                 // stats [3][n]: maximum, sum at 1, sum at T (infinity: no entry of the teacher's)
    const float* grad;
    void* dlogits;
};

template <typename T> struct Bits;       // one value, and 16 bytes of them
template <> struct Bits<float> {
    static constexpr int VEC = 4;
    static constexpr uint32_t NOTHING = 0xff800000u;              // minus infinity throughout a word
    static __device__ __forceinline__ float one(const float* p, bool ok) { return __uint_as_float(ld_chained(reinterpret_cast<const uint32_t*>(p), ok)); }
    static __device__ __forceinline__ void unpack(const uint4& r, float* v) { v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w); }
    static __device__ __forceinline__ uint4 pack(const float* v) { return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])); }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
    template <int N> static __device__ __forceinline__ float largest(const uint4 (&raw)[N]) {      // (of what is a number)
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < N; ++u) m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(raw[u].x), __uint_as_float(raw[u].y)), fmaxf(__uint_as_float(raw[u].z), __uint_as_float(raw[u].w))));
        return m;
    }
};
template <> struct Bits<__half> {
    static constexpr int VEC = 8;
    static constexpr uint32_t NOTHING = 0xfc00fc00u;
    static __device__ __forceinline__ float one(const __half* p, bool ok) { return __half2float(__ushort_as_half(ld_chained(reinterpret_cast<const uint16_t*>(p), ok))); }
    static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i])); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&h); }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
    template <int N> static __device__ __forceinline__ float largest(const uint4 (&raw)[N]) {
        __half2 m = *reinterpret_cast<const __half2*>(&raw[0].x);
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __hmax2(m, *reinterpret_cast<const __half2*>(&w[i]));
        }
        const float2 f = __half22float2(m);
        return fmaxf(f.x, f.y);
    }
};
template <> struct Bits<__nv_bfloat16> {
    static constexpr int VEC = 8;
    static constexpr uint32_t NOTHING = 0xff80ff80u;
    static __device__ __forceinline__ float one(const __nv_bfloat16* p, bool ok) { return __uint_as_float((uint32_t)ld_chained(reinterpret_cast<const uint16_t*>(p), ok) << 16); }
    static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ uint4 pack(const float* v) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&h); }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
    template <int N> static __device__ __forceinline__ float largest(const uint4 (&raw)[N]) {
        __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&raw[0].x);
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&w[i]));
        }
        const float2 f = __bfloat1622float2(m);
        return fmaxf(f.x, f.y);
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// (Packed pairs: a pass over 16-bit logits at full bandwidth is 11.5 logits per clock and SM, and one value per instruction, nine instructions a logit, left it bound by
// issue slots at 4.6 TB/s.)
__device__ __forceinline__ Pair ex2(Pair x) {
    float a, b;
    halves(x, a, b);
    return pair(ex2(a), ex2(b));
}
// exponentials of d = z - max <= 0 at temperature 1 and T
template <int KIND>
__device__ __forceinline__ void exps(Pair d, float c_temp, Pair& e1, Pair& et) {
    const Pair one = pair(LOG2E, LOG2E), ct = pair(c_temp, c_temp);
    if (KIND == DI_HARD) { e1 = ex2(d * one); et = pair(0.f, 0.f); }
    else if (KIND == DI_SOFT) { et = ex2(d * ct); e1 = pair(0.f, 0.f); }
    else if (KIND == DI_SAME) { e1 = et = ex2(d * one); }
    else if (KIND == DI_SQUARE) { et = ex2(d * ct); e1 = et * et; }
    else { e1 = ex2(d * one); et = ex2(d * ct); }
}
template <int KIND>
__device__ __forceinline__ void exps(float d, float c_temp, float& e1, float& et) {
    Pair a, b;
    float unused;
    exps<KIND>(pair(d, 0.f), c_temp, a, b);
    halves(a, e1, unused);
    halves(b, et, unused);
}

struct Sums { float m, s1, st; };
template <int KIND>
__device__ __forceinline__ void raise(Sums& a, float m, float c_temp) {          // the sums relative to a larger maximum
    float f1, ft;
    exps<KIND>(a.m - m, c_temp, f1, ft);
    a.s1 *= f1;
    a.st *= ft;
    a.m = m;
}
template <int KIND>
__device__ __forceinline__ void join(Sums& a, Sums b, float c_temp) {
    if (b.m > a.m) { const Sums s = a; a = b; b = s; }
    if (b.m == -INFINITY) { a.s1 += b.s1; a.st += b.st; return; }                 // nothing there (or not a number)
    raise<KIND>(b, a.m, c_temp);
    a.s1 += b.s1;
    a.st += b.st;
}
// The running sums of a thread: two of each, added up at the end.
struct Running { float m; Pair s1, st; };
template <int KIND, typename T, int UNROLL>
__device__ __forceinline__ void add(Running& a, const uint4 (&raw)[UNROLL], float c_temp) {
    const float top = Bits<T>::largest(raw);
    if (top > a.m) {
        float f1, ft;
        exps<KIND>(a.m - top, c_temp, f1, ft);
        a.s1 = a.s1 * pair(f1, f1);
        a.st = a.st * pair(ft, ft);
        a.m = top;
    }
    const float m = a.m == -INFINITY ? 0.f : a.m;
    const Pair minus = pair(-m, -m);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        float v[Bits<T>::VEC];
        Bits<T>::unpack(raw[u], v);
#pragma unroll
        for (int i = 0; i < Bits<T>::VEC; i += 2) {
            Pair e1, et;
            exps<KIND>(pair(v[i], v[i + 1]) + minus, c_temp, e1, et);
            if (KIND != DI_SOFT) a.s1 = a.s1 + e1;
            if (KIND != DI_HARD && KIND != DI_SAME) a.st = a.st + et;
        }
    }
}
template <int KIND>
__device__ __forceinline__ void add(Running& a, float v, float c_temp) {
    if (v > a.m) {
        float f1, ft;
        exps<KIND>(a.m - v, c_temp, f1, ft);
        a.s1 = a.s1 * pair(f1, f1);
        a.st = a.st * pair(ft, ft);
        a.m = v;
    }
    float e1, et;
    exps<KIND>(v - (a.m == -INFINITY ? 0.f : a.m), c_temp, e1, et);
    a.s1 = a.s1 + pair(e1, 0.f);
    if (KIND != DI_SAME) a.st = a.st + pair(et, 0.f);
}
template <int KIND>
__device__ __forceinline__ Sums sums_of(const Running& a) {
    float x, y;
    Sums r;
    r.m = a.m;
    halves(a.s1, x, y);
    r.s1 = x + y;
    halves(a.st, x, y);
    r.st = KIND == DI_SAME ? r.s1 : x + y;
    return r;
}

// Over classes [lo, hi) of a sample, all THREADS threads of a CTA together: vec(1 or 4 times 16 bytes, where the first of them lies, vectors between them, vectors
// from the first one to the end) and one(value, where it lies) for what is not whole 16 bytes of the row. Past the end there is minus infinity. BESIDE: a whole row's components are
// read side by side, each by its share of the threads (1000 rows of 8 x 10654 bf16: 58 us, 80 one behind another). In short rows what a thread reads is on its way before it looks at
// the first of it; in long ones that would only cost registers (4096 x 131072 bf16: 227 us, 190 without).
template <typename T, bool VECTORS, int THREADS, bool BESIDE, typename VecFn, typename OneFn>
__device__ __forceinline__ void over_classes(const T* logits, const DIParams& p, int row, int lo, int hi, VecFn vec, OneFn one) {
    constexpr int VEC = Bits<T>::VEC, UNROLL = 4;
    constexpr bool LONG = THREADS == 512;
    const int threads = BESIDE ? THREADS / p.comps : THREADS, tid = BESIDE ? threadIdx.x % threads : threadIdx.x;
    for (int c = BESIDE ? threadIdx.x / threads : lo / p.units, end = BESIDE ? c + 1 : components_below(hi, p.units); c < end; ++c) {
        const int a = max(lo, c * p.units), b = min(hi, (c + 1) * p.units);
        const T* first = logits + ((size_t)c * p.n + row) * p.units + (a - c * p.units);
        if (!VECTORS) {
            for (int i = tid; i < b - a; i += threads) one(Bits<T>::one(first + i, true), first + i);
            continue;
        }
        const int head = min(b - a, (int)((16 - (reinterpret_cast<uintptr_t>(first) & 15)) & 15) / (int)sizeof(T)), body = (b - a - head) / VEC;
        const T* start = first + head;
        int v = tid;
        if constexpr (LONG) {
            if (tid < head) one(Bits<T>::one(first + tid, true), first + tid);
            for (; v + (UNROLL - 1) * threads < body; v += UNROLL * threads) {
                uint4 raw[UNROLL];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) raw[u] = ld_chained(reinterpret_cast<const uint4*>(start) + v + u * threads);
                vec(raw, start + (size_t)v * VEC, threads, UNROLL * threads);
            }
            for (; v < body; v += threads) {
                const uint4 raw[1] = {ld_chained(reinterpret_cast<const uint4*>(start) + v)};
                vec(raw, start + (size_t)v * VEC, threads, threads);
            }
            for (int i = head + body * VEC + tid; i < b - a; i += threads) one(Bits<T>::one(first + i, true), first + i);
        } else {
            const int tail = b - a - head - body * VEC;        // (at most seven values at either end: fewer than the threads)
            const T* rest = start + body * VEC + tid;
            const float early = Bits<T>::one(first + tid, tid < head), late = Bits<T>::one(rest, tid < tail);
            for (; v < body; v += UNROLL * threads) {
                uint4 raw[UNROLL];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    const bool ok = v + u * threads < body;
                    raw[u] = ld_chained(reinterpret_cast<const uint4*>(start) + v + u * threads, ok);
                    if (!ok) raw[u] = make_uint4(Bits<T>::NOTHING, Bits<T>::NOTHING, Bits<T>::NOTHING, Bits<T>::NOTHING);
                }
                vec(raw, start + (size_t)v * VEC, threads, body - v);
            }
            if (tid < head) one(early, first + tid);
            if (tid < tail) one(late, rest);
        }
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <typename T>
__device__ __forceinline__ float logit(const DIParams& p, int row, int cls) {
    const int c = cls / p.units;
    return Bits<T>::one(static_cast<const T*>(p.logits) + ((size_t)c * p.n + row) * p.units + (cls - c * p.units), true);
}
// The class of the teacher's entry i of a row, or -1 where it names none, and its logit over T.
template <typename T>
__device__ __forceinline__ int entry(const DIParams& p, int row, int i, float& t) {
    const long long at = (long long)row * p.entries + i;
    const uint2 w = ld_chained(reinterpret_cast<const uint2*>(p.index + at));
    const long long cls = (long long)(((unsigned long long)w.y << 32) | w.x);
    if (cls < 0 || cls >= (long long)p.comps * p.units) { t = -INFINITY; return -1; }
    t = Bits<T>::one(static_cast<const T*>(p.teacher) + at, true) * p.inv_temp;
    return (int)cls;
}
// Has a row's entries (up to four for each lane of a warp) brought near before they are due, and the logits that they name: a short row's time is a chain of such loads.
template <typename T>
__device__ __forceinline__ void fetch_entries(const DIParams& p, int row, int lane) {
    for (int i = lane; i < min(p.entries, 128); i += 32) {
        const long long at = (long long)row * p.entries + i;
        ld_chained(reinterpret_cast<const uint2*>(p.index + at));
        Bits<T>::one(static_cast<const T*>(p.teacher) + at, true);
    }
}
template <typename T>
__device__ __forceinline__ void fetch_their_logits(const DIParams& p, int row, int lane) {
    for (int i = lane; i < min(p.entries, 128); i += 32) {
        float x;
        const int cls = entry<T>(p, row, i, x);
        if (cls >= 0) logit<T>(p, row, cls);
    }
}
__device__ __forceinline__ int label_of(const DIParams& p, int row) {
    if (!p.labels) return -1;
    const uint2 w = ld_chained(reinterpret_cast<const uint2*>(p.labels + row));
    const long long cls = (long long)(((unsigned long long)w.y << 32) | w.x);
    return cls < 0 || cls >= (long long)p.comps * p.units ? -1 : (int)cls;
}

// CTAs of a size that an SM is to hold: long rows (512 threads each) need 1536 threads with four vectors on their way, short ones are latency after latency
constexpr int di_ctas(int threads) { return threads == 512 ? 3 : (threads == 128 ? 8 : (threads == 64 ? 20 : 32)); }

template <typename T, bool VECTORS, int KIND, int THREADS, bool BESIDE>
__global__ void __launch_bounds__(THREADS, di_ctas(THREADS)) distill_fwd_kernel(const DIParams p) {
    constexpr int WARPS = THREADS / 32;
    __shared__ Sums words[WARPS];
    __shared__ Sums whole;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int row = blockIdx.x / p.splits, split = blockIdx.x - row * p.splits;
    const int classes = p.comps * p.units;
    const int lo = share_start(classes, split, p.splits), hi = share_start(classes, split + 1, p.splits);
    const float c_temp = LOG2E * p.inv_temp;
    chain_wait();
    chain_next();
    Running run = {-INFINITY, pair(0.f, 0.f), pair(0.f, 0.f)};
    const bool last = split == 0 && warp == 0;                 // the warp that writes the row's loss
    constexpr bool LONG = THREADS == 512;
    int label = -1;
    float labelled = 0.f;
    if (!LONG && KIND != DI_SOFT && last) label = label_of(p, row);
    if (!LONG && KIND != DI_HARD && last) fetch_entries<T>(p, row, lane);
    over_classes<T, VECTORS, THREADS, BESIDE>(static_cast<const T*>(p.logits), p, row, lo, hi,
        [&](const auto& raw, const T*, int, int) { add<KIND, T>(run, raw, c_temp); },
        [&](float v, const T*) { add<KIND>(run, v, c_temp); });
    if (!LONG && label >= 0) labelled = logit<T>(p, row, label);
    if (!LONG && KIND != DI_HARD && last) fetch_their_logits<T>(p, row, lane);
    Sums a = sums_of<KIND>(run);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        Sums b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o); b.s1 = __shfl_xor_sync(0xffffffffu, a.s1, o); b.st = __shfl_xor_sync(0xffffffffu, a.st, o);
        join<KIND>(a, b, c_temp);
    }
    if (lane == 0) words[warp] = a;
    __syncthreads();
    if (warp == 0) {
        a = lane < WARPS ? words[lane] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
        for (int o = WARPS / 2; o; o >>= 1) {
            Sums b;
            b.m = __shfl_xor_sync(0xffffffffu, a.m, o); b.s1 = __shfl_xor_sync(0xffffffffu, a.s1, o); b.st = __shfl_xor_sync(0xffffffffu, a.st, o);
            join<KIND>(a, b, c_temp);
        }
        if (lane == 0) whole = a;
    }
    if (p.splits > 1) {
        __syncthreads();
        cluster_sync_all();
        if (split == 0 && warp == 0) {
            a = {-INFINITY, 0.f, 0.f};
            if (lane < p.splits) {
                const uint32_t src = map_to_cta((uint32_t)__cvta_generic_to_shared(&whole), lane);
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(a.m) : "r"(src) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(a.s1) : "r"(src + 4) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(a.st) : "r"(src + 8) : "memory");
            }
#pragma unroll
            for (int o = 4; o; o >>= 1) {
                Sums b;
                b.m = __shfl_xor_sync(0xffffffffu, a.m, o); b.s1 = __shfl_xor_sync(0xffffffffu, a.s1, o); b.st = __shfl_xor_sync(0xffffffffu, a.st, o);
                join<KIND>(a, b, c_temp);
            }
        }
        cluster_sync_all();                       // nobody leaves while its sums are read
    }
    if (!last) return;
    a.m = __shfl_sync(0xffffffffu, a.m, 0); a.s1 = __shfl_sync(0xffffffffu, a.s1, 0); a.st = __shfl_sync(0xffffffffu, a.st, 0);
    const bool none = a.m == -INFINITY && a.s1 == 0.f && a.st == 0.f;    // no class left: the row counts for nothing
    float loss = 0.f;
    if (LONG && KIND != DI_SOFT && !none) {
        label = label_of(p, row);
        if (label >= 0) labelled = logit<T>(p, row, label);
    }
    if (label >= 0 && !none) loss = (1.f - p.alpha) * (logf(a.s1) - (labelled - a.m));
    bool any = false;
    if (KIND != DI_HARD && !none) {
        float peak = -INFINITY;
        // (entries with weight: minus infinity has none, and a NaN, which is no maximum, is to be seen)
        for (int i = lane; i < p.entries; i += 32) { float x; if (entry<T>(p, row, i, x) >= 0) { any = any || x != -INFINITY; peak = fmaxf(peak, x); } }
        peak = warp_max(peak);
        any = __any_sync(0xffffffffu, any);
        float total = 0.f;
        for (int i = lane; i < p.entries; i += 32) { float x; if (entry<T>(p, row, i, x) >= 0 && any) total += ex2((x - peak) * LOG2E); }
        total = warp_sum(total);
        const float log_total = logf(total), log_st = logf(a.st);
        float sum = 0.f;
        for (int i = lane; i < p.entries; i += 32) {
            float x;
            const int cls = entry<T>(p, row, i, x);
            if (cls < 0 || !any) continue;
            const float pi = ex2((x - peak) * LOG2E) / total;
            if (pi > 0.f || pi != pi) sum += pi * ((x - peak - log_total) - ((logit<T>(p, row, cls) - a.m) * p.inv_temp - log_st));
        }
        loss += p.alpha * p.temp * p.temp * warp_sum(sum);
    }
    if (lane == 0) {
        p.loss[row] = loss;
        if (p.stats) {
            p.stats[row] = none || a.m > -INFINITY ? a.m : NAN;            // (minus infinity: nothing there; NaN: nothing but that)
            p.stats[p.n + row] = KIND == DI_SOFT ? INFINITY : a.s1;
            p.stats[2 * p.n + row] = KIND == DI_HARD || !any ? INFINITY : a.st;
        }
    }
}

template <typename T, bool VECTORS, int KIND, int THREADS, bool BESIDE>
__global__ void __launch_bounds__(THREADS, di_ctas(THREADS)) distill_bwd_kernel(const DIParams p) {
    extern __shared__ __align__(16) float shared[];            // [places] classes of the teacher's entries, [places] probabilities; places: entries in whole fours
    const int places = (p.entries + 3) & ~3;
    int* classes_of = reinterpret_cast<int*>(shared);
    float* probs = shared + places;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    // from the last row on: the forward pass has left the last rows in L2
    const int back = blockIdx.x / p.splits, row = p.n - 1 - back, split = blockIdx.x - back * p.splits;
    const int classes = p.comps * p.units;
    const int lo = share_start(classes, split, p.splits), hi = share_start(classes, split + 1, p.splits);
    const float c_temp = LOG2E * p.inv_temp;
    chain_wait();
    chain_next();
    const float g = ld_chained(p.grad + row), m = ld_chained(p.stats + row), s1 = ld_chained(p.stats + p.n + row), st = ld_chained(p.stats + 2 * p.n + row);
    const int label = KIND == DI_SOFT ? -1 : label_of(p, row);
    if (THREADS < 512 && KIND != DI_HARD && warp == 0) fetch_entries<T>(p, row, lane);
    const bool none = m == -INFINITY, soft = KIND != DI_HARD && st != INFINITY;
    const float c1 = label >= 0 && !none ? g * (1.f - p.alpha) / s1 : 0.f, ct = soft && !none ? g * p.alpha * p.temp / st : 0.f;
    const float base = none ? 0.f : m;
    auto value = [&](float z) {
        float e1, et;
        exps<KIND>(z - base, c_temp, e1, et);
        if (none) return 0.f;
        if (KIND == DI_HARD) return c1 * e1;
        if (KIND == DI_SOFT) return ct * et;
        if (KIND == DI_SAME) return (c1 + ct) * e1;
        return fmaf(c1, e1, ct * et);
    };
    T* out = static_cast<T*>(p.dlogits);
    const T* in = static_cast<const T*>(p.logits);
    const Pair minus = pair(-base, -base), p1 = pair(c1, c1), pt = pair(ct, ct);
    auto values = [&](const uint4& raw, T* at) {
        float v[Bits<T>::VEC];
        Bits<T>::unpack(raw, v);
#pragma unroll
        for (int i = 0; i < Bits<T>::VEC; i += 2) {
            Pair e1, et, d;
            exps<KIND>(pair(v[i], v[i + 1]) + minus, c_temp, e1, et);
            if (KIND == DI_HARD) d = p1 * e1;
            else if (KIND == DI_SOFT) d = pt * et;
            else if (KIND == DI_SAME) d = (p1 + pt) * e1;
            else d = fma2(p1, e1, pt * et);
            halves(d, v[i], v[i + 1]);
        }
        if (none) {
#pragma unroll
            for (int i = 0; i < Bits<T>::VEC; ++i) v[i] = 0.f;
        }
        *reinterpret_cast<uint4*>(at) = Bits<T>::pack(v);
    };
    over_classes<T, VECTORS, THREADS, BESIDE>(in, p, row, lo, hi,
        [&](const auto& raw, const T* at, int step, int left) {
            constexpr int VECTORS_AT_ONCE = sizeof(raw) / sizeof(uint4);
#pragma unroll
            for (int u = 0; u < VECTORS_AT_ONCE; ++u)
                if (u * step < left) values(raw[u], out + (at - in) + (size_t)u * step * Bits<T>::VEC);
        },
        [&](float v, const T* at) { Bits<T>::put(out + (at - in), value(v)); });
    // the classes of the label and of the teacher's entries once more, with their own terms
    if (soft && !none && warp == 0) {
        float peak = -INFINITY;
        for (int i = lane; i < p.entries; i += 32) {
            float x;
            classes_of[i] = entry<T>(p, row, i, x);
            probs[i] = x;
            peak = fmaxf(peak, x);
        }
        peak = warp_max(peak);
        float total = 0.f;
        for (int i = lane; i < p.entries; i += 32) { const float e = classes_of[i] >= 0 ? ex2((probs[i] - peak) * LOG2E) : 0.f; probs[i] = e; total += e; }
        total = warp_sum(total);
        for (int i = lane; i < p.entries; i += 32) probs[i] /= total;
        if (lane < places - p.entries) { classes_of[p.entries + lane] = -1; probs[p.entries + lane] = 0.f; }
    }
    __syncthreads();
    if (none) return;
    const int entries = soft ? p.entries : 0;
    for (int i = t; i <= entries; i += THREADS) {
        const int cls = i < entries ? classes_of[i] : label;
        if (cls < lo || cls >= hi) continue;
        const float z = logit<T>(p, row, cls);
        float prob = 0.f;
        for (int j = 0; j < entries; j += 4) {                    // (a class may be named twice; all who write it write the same)
            const int4 c4 = *reinterpret_cast<const int4*>(classes_of + j);
            const float4 p4 = *reinterpret_cast<const float4*>(probs + j);
            prob += c4.x == cls ? p4.x : 0.f;
            prob += c4.y == cls ? p4.y : 0.f;
            prob += c4.z == cls ? p4.z : 0.f;
            prob += c4.w == cls ? p4.w : 0.f;
        }
        float v = value(z) - g * p.alpha * p.temp * prob;
        if (cls == label) v -= g * (1.f - p.alpha);
        const int c = cls / p.units;
        Bits<T>::put(out + ((size_t)c * p.n + row) * p.units + (cls - c * p.units), v);
    }
}

int check_distill(const pcb_distill_desc* d, int& comps) {
    if (!d) { set_error("null descriptor"); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->dtype < PCB_F32 || d->dtype > PCB_BF16) { set_error("unknown dtype %d", d->dtype); return PCB_ERR_INVALID_ARGUMENT; }
    Geom g = {};
    if (!algebra_setup(d->algebra, g)) { set_error("unknown algebra %d", d->algebra); return PCB_ERR_INVALID_ARGUMENT; }
    comps = g.nc;
    if (d->batch < 0 || d->units <= 0 || d->entries < 0) { set_error("invalid distillation geometry"); return PCB_ERR_INVALID_ARGUMENT; }
    // (log2(e) / T multiplies the logits and T^2 the second term, both in fp32)
    if (!(d->alpha >= 0.f && d->alpha <= 1.f) || !(d->temperature > 0.f) || LOG2E * (1.f / d->temperature) == INFINITY || d->temperature * d->temperature == INFINITY) {
        set_error("alpha in [0, 1] and a positive temperature with 1.45 / T and T^2 in fp32's range expected");
        return PCB_ERR_INVALID_ARGUMENT;
    }
    if (d->entries > DI_MAX_ENTRIES) { set_error("%d entries of the teacher's, %d at most", d->entries, DI_MAX_ENTRIES); return PCB_ERR_UNSUPPORTED; }
    if ((long long)comps * d->units > 2147483647LL || (long long)comps * d->units * d->batch > (1LL << 40) || (long long)d->batch * 8 > 2147483647LL) {
        set_error("too many classes or rows");
        return PCB_ERR_TOO_LARGE;
    }
    return PCB_OK;
}
DIParams distill_params(const pcb_distill_desc* d, int comps) {
    DIParams p = {};
    p.comps = comps; p.n = d->batch; p.units = d->units; p.entries = d->entries;
    p.alpha = d->alpha; p.temp = d->temperature; p.inv_temp = 1.f / d->temperature;
    return p;
}
int kind_of(const DIParams& p, bool hard, bool soft) {
    if (!soft || p.alpha == 0.f) return DI_HARD;
    if (!hard || p.alpha == 1.f) return DI_SOFT;
    return p.temp == 1.f ? DI_SAME : (p.temp == 2.f ? DI_SQUARE : DI_BOTH);
}
// CTAs that share a row: enough for four CTAs on every SM, with 4096 classes each
int row_splits(const DIParams& p) {
    const long long classes = (long long)p.comps * p.units;
    int s = 1;
    while (s < 8 && (long long)p.n * s * 2 <= 4LL * sm_count() && classes >= 4096LL * s * 2) s *= 2;
    return s;
}
template <typename T, bool VECTORS, int KIND>
cudaError_t launch_kind(bool forward, const DIParams& p, cudaStream_t s) {
    const long long per = (long long)p.comps * p.units / p.splits;
    const unsigned grid = (unsigned)p.n * (unsigned)p.splits;
    const size_t smem = forward ? 0 : (size_t)((p.entries + 3) & ~3) * 8;
    auto launch = [&](auto threads, auto beside) {
        constexpr int THREADS = decltype(threads)::value;
        constexpr bool BESIDE = decltype(beside)::value;
        auto kernel = forward ? distill_fwd_kernel<T, VECTORS, KIND, THREADS, BESIDE> : distill_bwd_kernel<T, VECTORS, KIND, THREADS, BESIDE>;
        return launch_clusters(forward ? p.splits : 1, true, kernel, grid, THREADS, smem, s, p);
    };
    const std::true_type beside;
    // A short row is a chain of latencies, and its threads count for nothing but the rows that an SM can hold: forward 4030 x 103 f32 8.5 us with a warp each, 17 with 128
    // threads; 2637 x (8 x 189) bf16 11.8 us with 64, 16 with 128. (A component's share is eight threads at least.)
    if (per <= 512 && p.comps <= 4) return launch(std::integral_constant<int, 32>(), beside);
    if (per <= 2048) return launch(std::integral_constant<int, 64>(), beside);
    if (per <= 4096 && p.splits == 1) return launch(std::integral_constant<int, 128>(), beside);
    if (p.comps > 1 && p.splits == 1) return launch(std::integral_constant<int, 512>(), beside);
    return launch(std::integral_constant<int, 512>(), std::false_type());
}
template <typename T, bool VECTORS>
cudaError_t launch_any(bool forward, int kind, const DIParams& p, cudaStream_t s) {
    switch (kind) {
        case DI_HARD: return launch_kind<T, VECTORS, DI_HARD>(forward, p, s);
        case DI_SOFT: return launch_kind<T, VECTORS, DI_SOFT>(forward, p, s);
        case DI_SAME: return launch_kind<T, VECTORS, DI_SAME>(forward, p, s);
        case DI_SQUARE: return launch_kind<T, VECTORS, DI_SQUARE>(forward, p, s);
        default: return launch_kind<T, VECTORS, DI_BOTH>(forward, p, s);
    }
}
template <typename T>
int launch_typed(bool forward, const DIParams& p, cudaStream_t s) {
    const int kind = kind_of(p, p.labels != nullptr, p.entries > 0);
    const uintptr_t a = reinterpret_cast<uintptr_t>(p.logits), b = reinterpret_cast<uintptr_t>(p.dlogits);
    const bool vec = forward || a % 16 == b % 16;              // rows may start anywhere, but a row and its gradient at the same place in 16 bytes
    if (vec) PCB_CUDA_TRY((launch_any<T, true>(forward, kind, p, s)));
    else PCB_CUDA_TRY((launch_any<T, false>(forward, kind, p, s)));
    return PCB_OK;
}
int launch_distill(bool forward, int dtype, const DIParams& p, cudaStream_t s) {
    if (dtype == PCB_F32) return launch_typed<float>(forward, p, s);
    return dtype == PCB_F16 ? launch_typed<__half>(forward, p, s) : launch_typed<__nv_bfloat16>(forward, p, s);
}

}  // namespace
}  // namespace pcb

using namespace pcb;

extern "C" {

int pcb_distill_fwd(const pcb_distill_desc* d, const void* logits, const long long* labels, const void* teacher, const long long* index, float* loss,
                    float* stats, void* stream) {
    int comps;
    const int rc = check_distill(d, comps);
    if (rc != PCB_OK || d->batch == 0) return rc;
    if (!logits || !loss || (d->entries > 0 && (!teacher || !index))) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    DIParams p = distill_params(d, comps);
    p.logits = logits; p.labels = labels; p.teacher = teacher; p.index = index; p.loss = loss; p.stats = stats;
    p.splits = row_splits(p);
    return launch_distill(true, d->dtype, p, (cudaStream_t)stream);
}

int pcb_distill_bwd(const pcb_distill_desc* d, const void* logits, const long long* labels, const void* teacher, const long long* index, const float* stats,
                    const float* grad_loss, void* dlogits, void* stream) {
    int comps;
    const int rc = check_distill(d, comps);
    if (rc != PCB_OK || d->batch == 0) return rc;
    if (!logits || !stats || !grad_loss || !dlogits || (d->entries > 0 && (!teacher || !index))) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    const size_t bytes = (size_t)comps * d->batch * d->units * dtype_size(d->dtype);
    if (overlaps(logits, bytes, dlogits, bytes)) { set_error("the gradient must not share memory with the logits"); return PCB_ERR_INVALID_ARGUMENT; }
    DIParams p = distill_params(d, comps);
    p.logits = logits; p.labels = labels; p.teacher = teacher; p.index = index; p.stats = const_cast<float*>(stats); p.grad = grad_loss; p.dlogits = dlogits;
    p.splits = row_splits(p);
    return launch_distill(false, d->dtype, p, (cudaStream_t)stream);
}

}  // extern "C"
