// Quantisation to e4m3 with a power-of-two scale for each block of 128 values (see dense8.cuh).
//
//   e = min { e : max|x| <= 448 * 2^e },   q = rn_e4m3(x * 2^-e)
//
// With max|x| = m * 2^p, 1 <= m < 2, and 448 = 1.75 * 2^8: e = p - 8 where m <= 1.75, else p - 7, read off the bits of the fp32 maximum. x * 2^-e is
// exact, so the result is one rounding of x and the same whatever computes it. Infinities and NaN become the type's NaN and do not
// enter the maximum.
//
// A CTA takes a tile of 128 x 128 values in registers, 8 x 8 per thread: the blocks of 1 x 128, of 128 x 1 and of 128 x 128 all lie within it, so the
// backward pass reads dy once for both of its products.
#include <cuda_fp8.h>

#include "dense8.cuh"
#include "tc_common.cuh"

namespace pcb {
namespace {

using namespace tc;

constexpr int QT_THREADS = 256;

__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {            // e + 127 of a block with that fp32 maximum (finite)
    if (amax_bits == 0) return 127;
    int p = (int)(amax_bits >> 23);
    uint32_t m = amax_bits & 0x7fffffu;
    if (p == 0) return 1;                                                  // below 2^-126: e = -126
    const int e = p - 8 + (m > 0x600000u ? 1 : 0);                         // p is biased by 127 already
    return e < 1 ? 1 : e;
}
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }   // 2^-e, byte in [1, 247]

// |v| as bits, or zero for what is no finite number
__device__ __forceinline__ uint32_t finite_abs(float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ float finite_or_nan(float v) {                  // (the conversion would saturate an infinity)
    return (__float_as_uint(v) & 0x7fffffffu) == 0x7f800000u ? __uint_as_float(0x7fffffffu) : v;
}

template <typename T> __device__ __forceinline__ void unpack8(const uint4& raw, float (&v)[8]);
template <> __device__ __forceinline__ void unpack8<__half>(const uint4& raw, float (&v)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 f = __half22float2(h[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
}
template <> __device__ __forceinline__ void unpack8<__nv_bfloat16>(const uint4& raw, float (&v)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ float load1(const float* p) { return ld_chained(p); }
__device__ __forceinline__ float load1(const __half* p) { return __half2float(__ushort_as_half(ld_chained(reinterpret_cast<const uint16_t*>(p)))); }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __uint_as_float((uint32_t)ld_chained(reinterpret_cast<const uint16_t*>(p)) << 16); }

// Eight neighbours of a row; `valid` of them exist. VEC: the row starts on 16 bytes and valid is 0 or 8.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int valid, float (&v)[8]) {
    if (VEC) {
        if (valid <= 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
        } else if (sizeof(T) == 4) {
            const float4 a = ld_chained(reinterpret_cast<const float4*>(p)), b = ld_chained(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            if constexpr (sizeof(T) == 2) unpack8<T>(ld_chained(reinterpret_cast<const uint4*>(p)), v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < valid ? load1(p + i) : 0.f;
    }
}

enum { QT_ROWS = 1, QT_COLS = 2, QT_BLOCKS = 4 };

struct QTParams {
    int rows, cols, pitch;
    uint8_t *row_values, *col_values;            // QT_BLOCKS: row_values
    uint32_t *row_words, *col_words;             // QT_BLOCKS: row_words is the byte array
    int row_groups, col_groups;                  // groups of four blocks along the columns (row scales) and along the rows (column scales)
    int* status;                                 // cleared by the first CTA, or null
};

// Thread t holds columns 8 * (t % 16) .. + 7 of rows (t / 16) + 16 * i: the lanes of half a warp hold one row.
template <typename T, int MODE, bool VEC>
__global__ void __launch_bounds__(QT_THREADS) quantize_tile_kernel(const T* x, QTParams p) {
    __shared__ uint32_t col_max[8][Q8_BLOCK];
    __shared__ uint32_t warp_max[8];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, c8 = (t & 15) * 8, r0 = t >> 4;
    const int comp = blockIdx.z, row_block = blockIdx.y, col_block = blockIdx.x;
    const int col = col_block * Q8_BLOCK + c8;
    chain_wait();
    chain_next();
    if (p.status && t == 0 && comp == 0 && row_block == 0 && col_block == 0) *p.status = 0;
    const int valid = min(8, p.cols - col);
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = row_block * Q8_BLOCK + r0 + 16 * i;
        load8<T, VEC>(x + ((size_t)comp * p.rows + row) * p.cols + col, row < p.rows ? valid : 0, v[i]);
    }
    auto store = [&](uint8_t* values, int i, const float (&s)[8]) {
        const int row = row_block * Q8_BLOCK + r0 + 16 * i;
        if (row >= p.rows || col >= p.pitch) return;
        uint2 w;
        w.x = to_e4m3x4(finite_or_nan(v[i][0]) * s[0], finite_or_nan(v[i][1]) * s[1], finite_or_nan(v[i][2]) * s[2], finite_or_nan(v[i][3]) * s[3]);
        w.y = to_e4m3x4(finite_or_nan(v[i][4]) * s[4], finite_or_nan(v[i][5]) * s[5], finite_or_nan(v[i][6]) * s[6], finite_or_nan(v[i][7]) * s[7]);
        *reinterpret_cast<uint2*>(values + ((size_t)comp * p.rows + row) * p.pitch + col) = w;
    };
    if (MODE & (QT_ROWS | QT_BLOCKS)) {
        uint32_t tile = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, finite_abs(v[i][j]));
            if constexpr ((MODE & QT_BLOCKS) != 0) {
                tile = max(tile, m);
            } else {
#pragma unroll
                for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                const int byte = scale_byte(m), row = row_block * Q8_BLOCK + r0 + 16 * i;
                const float f = inverse_scale(byte);
                const float s[8] = {f, f, f, f, f, f, f, f};
                store(p.row_values, i, s);
                if ((t & 15) == 0 && row < p.rows)
                    reinterpret_cast<uint8_t*>(p.row_words + ((size_t)comp * p.row_groups + (col_block >> 2)) * p.rows + row)[col_block & 3] = (uint8_t)byte;
            }
        }
        if constexpr ((MODE & QT_BLOCKS) != 0) {
            tile = __reduce_max_sync(0xffffffffu, tile);
            if (lane == 0) warp_max[warp] = tile;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 8; ++w) tile = max(tile, warp_max[w]);
            const int byte = scale_byte(tile);
            const float f = inverse_scale(byte);
            const float s[8] = {f, f, f, f, f, f, f, f};
#pragma unroll
            for (int i = 0; i < 8; ++i) store(p.row_values, i, s);
            if (t == 0) reinterpret_cast<uint8_t*>(p.row_words)[((size_t)comp * gridDim.y + row_block) * gridDim.x + col_block] = (uint8_t)byte;
        }
    }
    if (MODE & QT_COLS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, finite_abs(v[i][j]));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));                // the warp's other half holds other rows of these columns
            if (lane < 16) col_max[warp][c8 + j] = m;
        }
        __syncthreads();
        float s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t m = 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) m = max(m, col_max[w][c8 + j]);
            const int byte = scale_byte(m);
            s[j] = inverse_scale(byte);
            if (t < 16 && col + j < p.cols)
                reinterpret_cast<uint8_t*>(p.col_words + ((size_t)comp * p.col_groups + (row_block >> 2)) * p.cols + col + j)[row_block & 3] = (uint8_t)byte;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) store(p.col_values, i, s);
    }
}

template <typename T, int MODE>
cudaError_t launch_tile(const void* x, const QTParams& p, int comps, cudaStream_t stream) {
    const dim3 grid(q8_blocks(p.cols), q8_blocks(p.rows), comps);
    const bool vec = p.cols % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(QT_THREADS); cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    const T* xt = static_cast<const T*>(x);
    return vec ? cudaLaunchKernelEx(&cfg, quantize_tile_kernel<T, MODE, true>, xt, p) : cudaLaunchKernelEx(&cfg, quantize_tile_kernel<T, MODE, false>, xt, p);
}
template <int MODE>
int launch_typed(int dtype, const void* x, const QTParams& p, int comps, cudaStream_t stream) {
    if (q8_blocks(p.rows) > 65535) { set_error("more than 65535 blocks of 128 rows"); return PCB_ERR_TOO_LARGE; }
    if (dtype == PCB_F32) PCB_CUDA_TRY((launch_tile<float, MODE>(x, p, comps, stream)));
    else if (dtype == PCB_F16) PCB_CUDA_TRY((launch_tile<__half, MODE>(x, p, comps, stream)));
    else PCB_CUDA_TRY((launch_tile<__nv_bfloat16, MODE>(x, p, comps, stream)));
    return PCB_OK;
}

}  // namespace

int q8_quantize(int dtype, int comps, int rows, int cols, const void* x, Q8Target by_rows, Q8Target by_cols, int* status, cudaStream_t stream) {
    const QTParams p = {rows, cols, q8_pitch(cols), by_rows.values, by_cols.values, by_rows.words, by_cols.words, q8_groups(cols), q8_groups(rows), status};
    if (by_rows.values && by_cols.values) return launch_typed<QT_ROWS | QT_COLS>(dtype, x, p, comps, stream);
    return by_rows.values ? launch_typed<QT_ROWS>(dtype, x, p, comps, stream) : launch_typed<QT_COLS>(dtype, x, p, comps, stream);
}

int q8_quantize_blocks(int dtype, int comps, int rows, int cols, const void* x, uint8_t* values, uint8_t* scales, cudaStream_t stream) {
    const QTParams p = {rows, cols, q8_pitch(cols), values, nullptr, reinterpret_cast<uint32_t*>(scales), nullptr, 0, 0, nullptr};
    return launch_typed<QT_BLOCKS>(dtype, x, p, comps, stream);
}

}  // namespace pcb
