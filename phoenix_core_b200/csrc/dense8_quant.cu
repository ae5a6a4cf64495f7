// Quantisation to e4m3 with a power-of-two scale for each block of 128 values (see dense8.cuh).
//
//   e = min { e : max|x| <= 448 * 2^e },   q = rn_e4m3(x * 2^-e)
//
// With max|x| = m * 2^p, 1 <= m < 2, and 448 = 1.75 * 2^8: e = p - 8 where m <= 1.75, else p - 7, read off the bits of the fp32 maximum. x * 2^-e is
// exact, so the result is one rounding of x and the same whatever computes it. Infinities and NaN become the type's NaN and do not
// enter the maximum.
//
// A CTA takes a tile of 128 x 128 values in registers, 4 x 8 per thread: the blocks of 1 x 128, of 128 x 1 and of 128 x 128 all lie within it, so the
// backward pass reads dy once for both of its products. The tile stays as it was loaded (as fp32 it took 176 registers, and one CTA per SM moved 2.2 TB/s);
// maxima are taken over the bits of the magnitudes, two 16-bit values at a time. Three CTAs of 512 threads on an SM (fp32, and rows that start anywhere, whose words take registers: two), whose loads and stores lie beside each other, though
// some words spill for it. 8192 x 4096 bf16: by rows 23.5 to 27.4 us by the machine (3.7 to 4.3 TB/s read and written), both orientations of one and the columns of another 46 to 48 (54 with two CTAs); 2420 x 8096 fp32 by rows
// 21.5 (26.5 with one). What is left is latency: a CTA's loads are over before its stores begin.
#include "dense8.cuh"
#include "e4m3.cuh"
#include "tc_common.cuh"

namespace pcb {
namespace {

using namespace tc;

constexpr int QT_THREADS = 512, QT_WARPS = QT_THREADS / 32, QT_PER = 4, QT_STEP = QT_THREADS / 16;   // rows per thread, and between them

// Eight neighbours as loaded. A key is a value's magnitude as bits (monotonic); a 32-bit word holds the keys of two 16-bit values or of one fp32 value.
template <typename T> struct Eight;
template <> struct Eight<float> {
    static constexpr int WORDS = 8;
    static constexpr uint32_t INF_KEY = 0x7f800000u;
    uint32_t w[8];
    static __device__ __forceinline__ uint32_t keys(uint32_t w) { return w & 0x7fffffffu; }
    static __device__ __forceinline__ uint32_t finite_keys(uint32_t w) { const uint32_t k = keys(w); return k < INF_KEY ? k : 0u; }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
    static __device__ __forceinline__ uint32_t whole(uint32_t keys) { return keys; }                       // the largest key of a word
    static __device__ __forceinline__ uint32_t bits(uint32_t key) { return key; }                           // as fp32
    __device__ __forceinline__ void two(int j, float& a, float& b) const { a = __uint_as_float(w[2 * j]); b = __uint_as_float(w[2 * j + 1]); }
    __device__ __forceinline__ void numbers(int j) { if (keys(w[j]) == INF_KEY) w[j] = 0x7fffffffu; }             // infinities to NaN: the conversion would saturate them
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const float* p) {
        const uint4 a = ld_chained(reinterpret_cast<const uint4*>(p)), b = ld_chained(reinterpret_cast<const uint4*>(p) + 1);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    __device__ __forceinline__ void load(const float* p, int valid) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = ld_chained(reinterpret_cast<const uint32_t*>(p) + i, i < valid);
    }
};
template <typename T> struct Eight16 {
    static constexpr int WORDS = 4;
    uint32_t w[4];
    static __device__ __forceinline__ uint32_t keys(uint32_t w) { return w & 0x7fff7fffu; }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
    static __device__ __forceinline__ uint32_t whole(uint32_t keys) { return max(keys & 0xffffu, keys >> 16); }
    __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
    __device__ __forceinline__ void load(const T* p) {
        const uint4 a = ld_chained(reinterpret_cast<const uint4*>(p));
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
    __device__ __forceinline__ void load(const T* p, int valid) {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)ld_chained(h + 2 * i, 2 * i < valid) | ((uint32_t)ld_chained(h + 2 * i + 1, 2 * i + 1 < valid) << 16);
    }
    // eight values `odd` (0 or 1) values behind the word x[0]
    __device__ __forceinline__ void from(const uint32_t (&x)[5], uint32_t odd) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(x[i], x[i + 1], odd * 16u);
    }
};
template <> struct Eight<__half> : Eight16<__half> {
    static constexpr uint32_t INF_KEY = 0x7c00u;
    static __device__ __forceinline__ uint32_t finite_keys(uint32_t w) {
        const uint32_t k = keys(w), lo = k & 0xffffu, hi = k >> 16;
        return (lo < INF_KEY ? lo : 0u) | ((hi < INF_KEY ? hi : 0u) << 16);
    }
    static __device__ __forceinline__ uint32_t bits(uint32_t key) { return __float_as_uint(__half2float(__ushort_as_half((uint16_t)key))); }
    __device__ __forceinline__ void two(int j, float& a, float& b) const { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j])); a = f.x; b = f.y; }
    __device__ __forceinline__ void numbers(int j) { w[j] |= ((keys(w[j]) & 0xffffu) == INF_KEY ? 0x7fffu : 0u) | (keys(w[j]) >> 16 == INF_KEY ? 0x7fff0000u : 0u); }
};
template <> struct Eight<__nv_bfloat16> : Eight16<__nv_bfloat16> {
    static constexpr uint32_t INF_KEY = 0x7f80u;
    static __device__ __forceinline__ uint32_t finite_keys(uint32_t w) {
        const uint32_t k = keys(w), lo = k & 0xffffu, hi = k >> 16;
        return (lo < INF_KEY ? lo : 0u) | ((hi < INF_KEY ? hi : 0u) << 16);
    }
    static __device__ __forceinline__ uint32_t bits(uint32_t key) { return key << 16; }
    __device__ __forceinline__ void two(int j, float& a, float& b) const { a = __uint_as_float(w[j] << 16); b = __uint_as_float(w[j] & 0xffff0000u); }
    __device__ __forceinline__ void numbers(int j) { w[j] |= ((keys(w[j]) & 0xffffu) == INF_KEY ? 0x7fffu : 0u) | (keys(w[j]) >> 16 == INF_KEY ? 0x7fff0000u : 0u); }
};

enum { QT_ROWS = 1, QT_COLS = 2, QT_BLOCKS = 4 };

struct QTParams {
    const void* x;
    int rows, cols, pitch;
    int row_blocks, col_blocks, tiles;           // tiles: of all components
    uint8_t *row_values, *col_values;            // QT_BLOCKS: row_values; with QT_ROWS and QT_COLS either may be null
    uint32_t *row_words, *col_words;             // QT_BLOCKS: row_words is the byte array
    int row_groups, col_groups;                  // groups of four blocks along the columns (row scales) and along the rows (column scales)
    int vectors;                                 // rows start on 16 bytes and end on them
};

// Thread t holds columns 8 * (t % 16) .. + 7 of rows (t / 16) + 32 * i: the lanes of half a warp hold one row.
// VEC: every tensor's rows are whole eights and start on 16 bytes. A launch takes the tiles of one tensor or of two, one behind the other; status: cleared by the first CTA, or null.
template <typename T, int MODE, bool VEC>
__global__ void __launch_bounds__(QT_THREADS, sizeof(T) == 2 && VEC ? 3 : 2) quantize_tile_kernel(const __grid_constant__ QTParams p0, const __grid_constant__ QTParams p1, int* status) {
    typedef Eight<T> E;
    __shared__ uint32_t col_max[QT_WARPS][16 * E::WORDS];
    __shared__ uint32_t warp_max[QT_WARPS];
    __shared__ __align__(16) float col_scale[Q8_BLOCK];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, c8 = (t & 15) * 8, r0 = t >> 4;
    const QTParams& p = (int)blockIdx.x < p0.tiles ? p0 : p1;
    const unsigned tile = blockIdx.x - ((int)blockIdx.x < p0.tiles ? 0u : (unsigned)p0.tiles), line = tile / (unsigned)p.col_blocks;
    const int col_block = (int)(tile - line * (unsigned)p.col_blocks), comp = (int)(line / (unsigned)p.row_blocks), row_block = (int)line - comp * p.row_blocks;
    const int col = col_block * Q8_BLOCK + c8, first_row = row_block * Q8_BLOCK + r0;
    chain_wait();
    chain_next();
    if (status && t == 0 && blockIdx.x == 0) *status = 0;
    const int valid = min(8, p.cols - col);
    E v[QT_PER];
    {
        const T* x = static_cast<const T*>(p.x);
        const T* src = x + ((size_t)comp * p.rows + first_row) * p.cols + col;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < QT_PER; ++i) {
                if (first_row + QT_STEP * i < p.rows && valid > 0) v[i].load(src + (size_t)QT_STEP * i * p.cols);
                else v[i].zero();
            }
        } else if (p.vectors) {
            // (one tensor of the launch may be so without the other; an fp32 row may end in the middle of an eight)
#pragma unroll
            for (int i = 0; i < QT_PER; ++i) {
                const uint4* at = reinterpret_cast<const uint4*>(src + (size_t)QT_STEP * i * p.cols);
                const bool live = first_row + QT_STEP * i < p.rows;
                const uint4 a = ld_chained(at, live && valid > 0);
                v[i].w[0] = a.x; v[i].w[1] = a.y; v[i].w[2] = a.z; v[i].w[3] = a.w;
                if constexpr (sizeof(T) == 4) {
                    const uint4 b = ld_chained(at + 1, live && valid > 4);
                    v[i].w[4] = b.x; v[i].w[5] = b.y; v[i].w[6] = b.z; v[i].w[7] = b.w;
                }
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < QT_PER; ++i) v[i].load(src + (size_t)QT_STEP * i * p.cols, first_row + QT_STEP * i < p.rows ? valid : 0);
        } else {
            // Rows that start on two bytes: as the words around them, five for eight values, but for the ends of rows (and of the tensor). Every load is on its way before the
            // first value is looked at.
            uint32_t word[QT_PER][5], odd_start[QT_PER];
            const bool inside = valid == 8 && col > 0 && col + 8 < p.cols;
#pragma unroll
            for (int i = 0; i < QT_PER; ++i) {
                const T* at = src + (size_t)QT_STEP * i * p.cols;
                odd_start[i] = (uint32_t)(reinterpret_cast<uintptr_t>(at) >> 1) & 1u;
                const uint32_t* u = reinterpret_cast<const uint32_t*>(at - odd_start[i]);
                const bool live = inside && first_row + QT_STEP * i < p.rows;
#pragma unroll
                for (int k = 0; k < 5; ++k) word[i][k] = ld_chained(u + k, live && (k < 4 || odd_start[i]));
            }
#pragma unroll
            for (int i = 0; i < QT_PER; ++i) v[i].from(word[i], odd_start[i]);
            if (__any_sync(0xffffffffu, !inside)) {
#pragma unroll
                for (int i = 0; i < QT_PER; ++i)
                    if (!inside && first_row + QT_STEP * i < p.rows && valid > 0) v[i].load(src + (size_t)QT_STEP * i * p.cols, valid);
            }
        }
    }
    uint32_t row_keys[QT_PER], most = 0;
#pragma unroll
    for (int i = 0; i < QT_PER; ++i) {
        row_keys[i] = 0;
#pragma unroll
        for (int j = 0; j < E::WORDS; ++j) row_keys[i] = E::larger(row_keys[i], E::keys(v[i].w[j]));
        row_keys[i] = E::whole(row_keys[i]);
        most = max(most, row_keys[i]);
    }
    // whether the tile holds infinities or NaN, which are kept out of the maxima and become NaN (the conversion would saturate an infinity)
    const bool odd = __syncthreads_or(most >= E::INF_KEY);
    if (odd) {
        most = 0;
#pragma unroll
        for (int i = 0; i < QT_PER; ++i) {
            row_keys[i] = 0;
#pragma unroll
            for (int j = 0; j < E::WORDS; ++j) row_keys[i] = E::larger(row_keys[i], E::finite_keys(v[i].w[j]));
            row_keys[i] = E::whole(row_keys[i]);
            most = max(most, row_keys[i]);
        }
    }
    // Rounds and stores the tile with a scale for each row (ROW) or each column.
    auto store = [&](uint8_t* values, auto scale_of) {
        if (col >= p.pitch) return;
        uint8_t* dst = values + ((size_t)comp * p.rows + first_row) * p.pitch + col;
        if (odd) {
#pragma unroll
            for (int i = 0; i < QT_PER; ++i) {
#pragma unroll
                for (int j = 0; j < E::WORDS; ++j) v[i].numbers(j);
            }
        }
#pragma unroll
        for (int i = 0; i < QT_PER; ++i) {
            if (first_row + QT_STEP * i >= p.rows) break;
            uint32_t lo = 0, hi = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float a, b;
                v[i].two(j, a, b);
                const float2 s = scale_of(i, j);
                const uint32_t q = to_e4m3x2(a, b, s);
                if (j < 2) lo |= q << (16 * j);
                else hi |= q << (16 * (j - 2));
            }
            *reinterpret_cast<uint2*>(dst + (size_t)QT_STEP * i * p.pitch) = make_uint2(lo, hi);
        }
    };
    if ((MODE & QT_ROWS) && p.row_values) {
        float f[QT_PER];
#pragma unroll
        for (int i = 0; i < QT_PER; ++i) {
            uint32_t m = row_keys[i];
#pragma unroll
            for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const int byte = scale_byte(E::bits(m)), row = first_row + QT_STEP * i;
            f[i] = inverse_scale(byte);
            if ((t & 15) == 0 && row < p.rows)
                reinterpret_cast<uint8_t*>(p.row_words + ((size_t)comp * p.row_groups + (col_block >> 2)) * p.rows + row)[col_block & 3] = (uint8_t)byte;
        }
        store(p.row_values, [&](int i, int) { return make_float2(f[i], f[i]); });
    }
    if constexpr ((MODE & QT_BLOCKS) != 0) {
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) warp_max[warp] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < QT_WARPS; ++w) most = max(most, warp_max[w]);
        const int byte = scale_byte(E::bits(most));
        const float f = inverse_scale(byte);
        store(p.row_values, [&](int, int) { return make_float2(f, f); });
        if (t == 0) reinterpret_cast<uint8_t*>(p.row_words)[((size_t)comp * p.row_blocks + row_block) * p.col_blocks + col_block] = (uint8_t)byte;
    }
    if constexpr ((MODE & QT_COLS) != 0) {
        uint32_t m[E::WORDS];
#pragma unroll
        for (int j = 0; j < E::WORDS; ++j) {
            m[j] = 0;
            if (odd) {
#pragma unroll
                for (int i = 0; i < QT_PER; ++i) m[j] = E::larger(m[j], E::finite_keys(v[i].w[j]));
            } else {
#pragma unroll
                for (int i = 0; i < QT_PER; ++i) m[j] = E::larger(m[j], E::keys(v[i].w[j]));
            }
            m[j] = E::larger(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));       // the warp's other half holds other rows of these columns
            if (lane < 16) col_max[warp][lane * E::WORDS + j] = m[j];
        }
        __syncthreads();
        // the first eight warps' threads each join a word of the sixteen warps' and leave the inverse scales of its columns
        constexpr int PER = 8 / E::WORDS;                                          // columns per word
        if (t < 16 * E::WORDS) {
            uint32_t k = 0;
#pragma unroll
            for (int w = 0; w < QT_WARPS; ++w) k = E::larger(k, col_max[w][t]);
#pragma unroll
            for (int h = 0; h < PER; ++h) {
                const int byte = scale_byte(E::bits(PER == 1 ? k : (h ? k >> 16 : k & 0xffffu))), e = t * PER + h, at = col_block * Q8_BLOCK + e;
                col_scale[e] = inverse_scale(byte);
                if (at < p.cols) reinterpret_cast<uint8_t*>(p.col_words + ((size_t)comp * p.col_groups + (row_block >> 2)) * p.cols + at)[row_block & 3] = (uint8_t)byte;
            }
        }
        __syncthreads();
        const float4 sa = *reinterpret_cast<const float4*>(&col_scale[c8]), sb = *reinterpret_cast<const float4*>(&col_scale[c8 + 4]);
        store(p.col_values, [&](int, int j) {
            return j == 0 ? make_float2(sa.x, sa.y) : (j == 1 ? make_float2(sa.z, sa.w) : (j == 2 ? make_float2(sb.x, sb.y) : make_float2(sb.z, sb.w)));
        });
    }
}

template <typename T, int MODE>
cudaError_t launch_tile(const QTParams& p0, const QTParams& p1, int* status, cudaStream_t stream) {
    auto vectors = [](const QTParams& p) { return p.tiles == 0 || (p.vectors && p.cols % 8 == 0); };
    const unsigned grid = (unsigned)p0.tiles + (unsigned)p1.tiles;
    return vectors(p0) && vectors(p1) ? launch_chained(quantize_tile_kernel<T, MODE, true>, grid, QT_THREADS, 0, stream, p0, p1, status)
                                      : launch_chained(quantize_tile_kernel<T, MODE, false>, grid, QT_THREADS, 0, stream, p0, p1, status);
}
template <int MODE>
int launch_typed(int dtype, const QTParams& p0, const QTParams& p1, int* status, cudaStream_t stream) {
    if (dtype == PCB_F32) PCB_CUDA_TRY((launch_tile<float, MODE>(p0, p1, status, stream)));
    else if (dtype == PCB_F16) PCB_CUDA_TRY((launch_tile<__half, MODE>(p0, p1, status, stream)));
    else PCB_CUDA_TRY((launch_tile<__nv_bfloat16, MODE>(p0, p1, status, stream)));
    return PCB_OK;
}
QTParams tile_params(int dtype, int comps, int rows, int cols, const void* x, Q8Target by_rows, Q8Target by_cols) {
    const int row_blocks = q8_blocks(rows), col_blocks = q8_blocks(cols);
    return {x, rows, cols, q8_pitch(cols), row_blocks, col_blocks, comps * row_blocks * col_blocks, by_rows.values, by_cols.values, by_rows.words, by_cols.words,
            q8_groups(cols), q8_groups(rows), cols * dtype_size(dtype) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0};
}

}  // namespace

int q8_quantize_rows(int dtype, int comps, int rows, int cols, const void* x, Q8Target by_rows, int* status, cudaStream_t stream) {
    return launch_typed<QT_ROWS>(dtype, tile_params(dtype, comps, rows, cols, x, by_rows, Q8Target{}), QTParams{}, status, stream);
}

int q8_quantize_backward(int dtype, int comps, int rows, int x_cols, int dy_cols, const void* x, const void* dy, Q8Target x_by_cols, Q8Target dy_by_rows, Q8Target dy_by_cols, int* status,
                         cudaStream_t stream) {
    return launch_typed<QT_ROWS | QT_COLS>(dtype, tile_params(dtype, comps, rows, dy_cols, dy, dy_by_rows, dy_by_cols), tile_params(dtype, comps, rows, x_cols, x, Q8Target{}, x_by_cols), status, stream);
}

int q8_quantize_blocks(int dtype, int comps, int rows, int cols, const void* x, uint8_t* values, uint8_t* scales, cudaStream_t stream) {
    return launch_typed<QT_BLOCKS>(dtype, tile_params(dtype, comps, rows, cols, x, Q8Target{values, reinterpret_cast<uint32_t*>(scales)}, Q8Target{}), QTParams{}, nullptr, stream);
}

}  // namespace pcb
