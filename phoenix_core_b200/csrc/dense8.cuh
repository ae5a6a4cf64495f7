// Operands of the dense layer in 8-bit floating point, and the launchers of its kernels.
//
// An operand is a matrix per component, held as e4m3 numbers in rows of `pitch` bytes (a multiple of 16, as the copies that
// read it need), with a power-of-two scale 2^e for each block of 128 values along the axis that a product sums over, kept as the byte e + 127:
//   vector scales   one block of 128 x 1 for each row (or column): words[comp][group][row], byte j of a word belongs to the block 4 * group + j of
//                   the summed axis, so that a word is what the tensor cores take for 512 values of that axis
//   block scales    one block of 128 x 128 (filters): bytes[comp][row block][column block]
// e is the smallest whole number with max|x| <= 448 * 2^e, so nothing saturates and the division by the scale is exact: the one rounding is the
// one to e4m3. Blocks of zeros have e = 0, and e >= -126.
#pragma once

#include "common.cuh"

namespace pcb {

constexpr int Q8_BLOCK = 128;
inline int q8_pitch(int cols) { return (cols + 15) / 16 * 16; }
inline int q8_blocks(int n) { return (n + Q8_BLOCK - 1) / Q8_BLOCK; }
inline int q8_groups(int n) { return (q8_blocks(n) + 3) / 4; }

struct Q8Operand {
    const uint8_t* values;
    const void* scales;          // words (vector) or bytes (block)
    int pitch;                   // bytes between rows of `values`
    int block_scales;            // 0: one word per index of the operand's own axis; 1: bytes
    int bytes_k, bytes_mn;       // block scales: strides of the byte over blocks of the summed axis and of the operand's own axis
    int mn_major;                // rows of `values` run along the operand's own axis (else along the summed one)
};

// out[c][m][n] = sum over components and k of sign * a[m][k] * b[n][k] (+ bias), rounded once to `dtype`.
struct Q8Product {
    Pass pass;
    int swapped;                 // forward and backward-data: the filter is operand A (few tokens)
    int m, n, k;                 // per component
    Q8Operand a, b;
    void* out;
    int dtype;
    const void* bias;            // [components][features], forward only
    int* status;
    const void* tokens = nullptr;       // the tokens as the caller has them: quantised by the product itself (then operand b is not read)
};

// Quantises x ([components][rows][cols], dense) with blocks of 1 x 128; of the backward pass's tensors x with blocks of 128 x 1 and dy with those and, unless its values
// are null, with blocks of 1 x 128, in one launch; a filter with blocks of 128 x 128. The status word is cleared by the first two.
struct Q8Target { uint8_t* values; uint32_t* words; };
int q8_quantize_rows(int dtype, int comps, int rows, int cols, const void* x, Q8Target by_rows, int* status_to_clear, cudaStream_t stream);
int q8_quantize_backward(int dtype, int comps, int rows, int x_cols, int dy_cols, const void* x, const void* dy, Q8Target x_by_cols, Q8Target dy_by_rows, Q8Target dy_by_cols,
                         int* status_to_clear, cudaStream_t stream);
int q8_quantize_blocks(int dtype, int comps, int rows, int cols, const void* x, uint8_t* values, uint8_t* scales, cudaStream_t stream);
int q8_product(const Geom& g, const Q8Product& p, cudaStream_t stream);
// The form (pcb_dense8_form) that q8_product takes, and the CTAs that share a tile: of the product's sizes alone.
int q8_form(const Geom& g, const Q8Product& p, int* splits);
// The two gradients of a backward call, in one launch or two.
int q8_two_products(const Geom& g, const Q8Product& first, const Q8Product& second, cudaStream_t stream);
bool q8_together(const Geom& g, const Q8Product& first, const Q8Product& second);
// Whether a forward or backward-data product of that many tokens takes the filter as operand A.
bool q8_swapped(int tokens);
// Whether the product quantises that many tokens itself.
bool q8_raw_tokens(int tokens);

}  // namespace pcb
