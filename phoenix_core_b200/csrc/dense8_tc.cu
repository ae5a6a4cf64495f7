// Products of 8-bit operands with block scales on the tensor cores: forward, backward-data and filter gradient of the dense layer (dense8.cuh).
//
//   out[c][m][n] = sum over (component j of the reduction, k) of sign(c, j) * 2^(ea + eb) * qa[m][k] * qb[n][k]      (+ bias)
//
// The algebra's block is a choice of operand components and a sign per (c, j); the sign is the negation bit of the instruction, so a quaternion
// layer is sixteen products of the same tiles and no operand is changed. The scales are powers of two, which tcgen05.mma.kind::mxf8f6f4
// multiplies in itself: one e8m0 byte per operand row and 32 values, here the same byte four times over (the blocks have 128). Products are
// exact and sums are held in fp32 in tensor memory over the whole reduction.
//
// Roles: warp 0 copies the operand tiles (TMA; both majornesses are read where they lie), warp 1 issues, warps 2 and 3 lay the scales out (a word per
// row holds the bytes of four blocks; 32 x 4 words are 512 bytes in the order that tcgen05.cp takes to tensor memory), warps 4-11 drain the accumulators.
// Four forms:
//   PAIR      256 x 256 tiles on pairs of SMs, half of either operand in each one's shared memory. An 8-bit MMA of 128 x 256 x 32 takes 128 clocks and reads 12 KB of
//             shared memory, into which TMA writes as much again: more than the 128 bytes a clock that shared memory moves. On one SM a block of 128 took
//             0.53 us where the MMAs alone take 0.27; a pair moves a third less. 8192 x 4096 -> 4096: 100 us, 2.75 PFLOP/s (84 % of twice the bf16 burst rate); with the clocks that
//             this load leaves, a block takes 589 clocks of which the MMAs take 512: one accumulator of 256 columns is all that tensor memory holds beside the scales, so the epilogue
//             is not covered.
//   single    128 x 128 tiles; a tile's reduction is cut over the CTAs of a cluster where there are fewer tiles than SMs, whose partial sums are added in a
//             fixed order through distributed shared memory.
//   SWAP      few tokens: the filter is operand A, a tile is 128 features x 16 or 64 tokens; bound by the filter's bytes.
//   RAW       the same for up to four tokens, which are quantised here: four warps each take a block of 128 of the reduction at a time straight from the caller's tensor
//             into the stage and the scales' words, so that the call is one launch.
#include "dense8.cuh"
#include "e4m3.cuh"
#include "tc_common.cuh"

namespace pcb {
namespace {

using namespace umma;
using namespace tc;

constexpr int D8_BM = 128, D8_BK = 128;
constexpr int D8_THREADS = 384, D8_EPI_WARPS = 8;
constexpr uint32_t D8_A_BYTES = D8_BM * D8_BK;
constexpr int D8_SF_STAGES = 4;
constexpr int D8_RAW = 4;                                       // tokens that a product quantises itself, at most
constexpr uint32_t D8_SF_BYTES = 512 * 3;                       // one set of 128 rows for A, up to two for B
constexpr int ST_D8_PRODUCER = 0x100, ST_D8_MMA = 0x200, ST_D8_SCALES = 0x400, ST_D8_EPILOGUE = 0x800;

template <int BN, bool SWAP, bool PAIR> struct D8Config {
    static constexpr int B_ROWS = PAIR ? BN / 2 : (BN < 32 ? 32 : BN);   // rows of B in a CTA's shared memory (tiles start on 1024 bytes: 8 rows)
    static constexpr uint32_t B_BYTES = B_ROWS * D8_BK;
    static constexpr uint32_t STAGE = D8_A_BYTES + B_BYTES;
    static constexpr int STAGES = BN >= 128 ? (SWAP ? 6 : 5) : (BN >= 64 ? 8 : 10);
    static constexpr int ACC = BN >= 256 ? 1 : 2;                // accumulators in tensor memory
    static constexpr uint32_t ACC_COLS = BN < 32 ? 32 : BN;
    static constexpr uint32_t SF_COL = 496;                      // scales: 4 columns for A, 8 for B
    static constexpr int CTAS = PAIR ? 2 : 1;
    static constexpr int M = D8_BM * CTAS;                       // rows of a tile
    static constexpr uint32_t OUT_BYTES = SWAP ? 0 : 4096;       // per epilogue warp: 32 rows of 128 bytes on their way out
    static constexpr int PART_PITCH = SWAP ? D8_BM : BN + 4;     // words between rows of partial sums (16-byte accesses of eight rows meet no bank twice)
    static constexpr uint32_t BARS = 512;
    static constexpr size_t SMEM = 1024 + STAGES * STAGE + D8_EPI_WARPS * OUT_BYTES + D8_SF_STAGES * D8_SF_BYTES + BARS;
};

struct D8Params {
    int pass, ga, comps;
    unsigned long long neg;
    int m, n, k;
    int chunks, groups;                 // blocks of 128 and groups of four of them per component of the reduction
    int m_tiles, n_tiles, tiles;        // tiles: over all output components
    int out_map;                        // the output is written through its tensor map
    int splits;                         // CTAs of the cluster that share a tile
    int a_mn, b_mn;                     // operands run along their own axis
    int a_blocks, b_blocks;             // scales are bytes per 128 x 128 block, else words
    const uint8_t *a_scales, *b_scales;
    int a_bk, a_bm, a_bc, b_bk, b_bm, b_bc;   // strides of the bytes: blocks of the reduction, blocks of the own axis, components
    int dtype;
    long long out_comp; int out_ld;     // element (c, slow, fast) of the output at c * out_comp + slow * out_ld + fast
    void* out;
    const void* bias;                   // [comps][fast extent], or null
    const void* tokens;                 // RAW: the tokens as the caller has them, [comps][n][k]
    int* clear;                         // the call's status word, if this launch is to reset it
};

// What a launch computes: a product, or both of the backward pass, whose tiles follow one another.
template <int N> struct D8Args {
    CUtensorMap a[N], b[N], out[N];
    D8Params p[N];
    __device__ __forceinline__ int tiles() const { return N > 1 ? p[0].tiles + p[N - 1].tiles : p[0].tiles; }
    __device__ __forceinline__ int product(int tile) const { return N > 1 && tile >= p[0].tiles ? 1 : 0; }
    __device__ __forceinline__ int local(int tile) const { return N > 1 && tile >= p[0].tiles ? tile - p[0].tiles : tile; }
};

// Operand components and sign of term j of output component c.
__device__ __forceinline__ void d8_term(const D8Params& p, int c, int j, int& x_comp, int& other, bool& neg) {
    if (p.pass == PASS_FWD)           { x_comp = j; other = alg_pair(p.ga, j, c); neg = alg_negative(p.neg, j, c); }                       // x_l, w_r
    else if (p.pass == PASS_BWD_DATA) { x_comp = j; other = alg_pair(p.ga, c, j); neg = alg_negative(p.neg, c, j); }                       // dy_d, w_r
    else                              { x_comp = j; other = alg_pair(p.ga, j, c); neg = alg_negative(p.neg, j, other); }                   // x_l, dy_d
}

// kind::mxf8f6f4, e4m3 operands, e8m0 scales, fp32 sums
__device__ __forceinline__ uint32_t d8_idesc(int M, int N, bool a_mn, bool b_mn, bool a_neg) {
    return ((uint32_t)a_neg << 13) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void mma_mxf8(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
            "mov.b64 da, {%1, %2};\n\t"
            "mov.b64 db, {%3, %4};\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %5, [%7], [%8], p;\n\t}"
            ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
            "mov.b64 da, {%1, %2};\n\t"
            "mov.b64 db, {%3, %4};\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %5, [%7], [%8], p;\n\t}"
            ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
}
// 32 rows of 16 bytes to four columns of tensor memory, in each of the four groups of 32 lanes (PAIR: in both CTAs, each from its own shared memory)
template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem_addr) {
    const uint64_t desc = (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | DESC_VERSION_SM100;
    if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// The scales of the odd CTA are written by its own threads: the arrival that announces them in the even CTA releases at cluster scope (what its thread has waited for included), the
// wait acquires there.
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool warp_wait_acquire_cluster(uint32_t bar, uint32_t parity, int* status, int code) {
    const bool ok = warp_wait_bounded(bar, parity, status, code);
    if (ok) {
        [[maybe_unused]] uint32_t done;                          // (complete already: this one orders)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    }
    return ok;
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ float ld_typed(const void* p, int dtype, size_t i) {
    if (dtype == PCB_F32) return ld_chained(static_cast<const float*>(p) + i);
    const uint16_t h = ld_chained(static_cast<const uint16_t*>(p) + i);
    return dtype == PCB_F16 ? __half2float(__ushort_as_half(h)) : __uint_as_float((uint32_t)h << 16);
}
__device__ __forceinline__ uint16_t to_16(float v, int dtype) {
    return dtype == PCB_F16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
__device__ __forceinline__ void st_typed(void* p, int dtype, size_t i, float v) {
    if (dtype == PCB_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = to_16(v, dtype);
}
__device__ __forceinline__ uint32_t pack_16(float a, float b, int dtype) {
    if (dtype == PCB_F16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp's 32 rows (one per lane) whose lines start anywhere, through 4 KB of shared memory so that the lanes of an instruction write neighbours: words w of row r lie at
// r * 32 + (w ^ r), which meets no bank twice in either direction. rows, cols: how many exist; ld: elements between rows.
__device__ __forceinline__ void park_words(uint32_t buf, int first, const uint32_t* v, int n, int lane) {
#pragma unroll
    for (int e = 0; e < 32; ++e)
        if (e < n) asm volatile("st.shared.u32 [%0], %1;" ::"r"(buf + (uint32_t)(lane * 32 + ((first + e) ^ lane)) * 4u), "r"(v[e]) : "memory");
}
// 32 columns of floats per row (eight reads in flight before the first of their stores, here and below)
__device__ __forceinline__ void store_parked_floats(uint32_t buf, float* out, int rows, int cols, int ld, int lane) {
    __syncwarp();
    out += lane;
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 8) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x[i]) : "r"(buf + (uint32_t)((r0 + i) * 32 + (lane ^ (r0 + i))) * 4u));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (r0 + i < rows && lane < cols) out[(long long)(r0 + i) * ld] = x[i];
    }
    __syncwarp();
}
// 64 columns of 16-bit values per row, in words of two: stored as words where the row starts on four bytes, else as the words between (whose halves come from two
// parked ones) and a value at either end
__device__ __forceinline__ void store_parked_halves(uint32_t buf, uint16_t* out, int rows, int cols, int ld, int lane) {
    __syncwarp();
    cols = min(cols, 64);
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 8) {
        uint32_t w[8], next[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(buf + (uint32_t)((r0 + i) * 32 + (lane ^ (r0 + i))) * 4u));
#pragma unroll
        for (int i = 0; i < 8; ++i) next[i] = __shfl_down_sync(0xffffffffu, w[i], 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint16_t* line = out + (long long)(r0 + i) * ld;
            const uint32_t odd = (uint32_t)(reinterpret_cast<uintptr_t>(line) >> 1) & 1u, word = __funnelshift_r(w[i], next[i], odd * 16u);
            const int col = 2 * lane + (int)odd;
            const bool live = r0 + i < rows;
            if (live && col + 1 < cols) *reinterpret_cast<uint32_t*>(line + col) = word;
            if (live && col + 1 == cols) line[col] = (uint16_t)word;             // the last column of the tensor, or of the block
            if (live && odd && lane == 0) line[0] = (uint16_t)w[i];
        }
    }
    __syncwarp();
}

// Where a warp is in its CTA's part of a reduction: group `group` of component j, with the operands' components and the sign. Stepped, not computed anew: the
// divisions of one step took a warp about as long as the MMAs of a block.
struct D8Walk {
    int left, j, group, first, second;       // groups left, component of the reduction, its group; components of x (or dy) and of the other operand
    bool neg;
    __device__ __forceinline__ void start(const D8Params& p, int c, int g_begin, int g_end, int j_begin) {
        left = g_end - g_begin;
        j = j_begin;
        group = g_begin - j_begin * p.groups;
        term(p, c);
    }
    __device__ __forceinline__ void term(const D8Params& p, int c) {
        if (j < p.comps) d8_term(p, c, j, first, second, neg);
    }
    __device__ __forceinline__ void step(const D8Params& p, int c) {
        --left;
        if (++group == p.groups) { group = 0; ++j; term(p, c); }
    }
    __device__ __forceinline__ int blocks(const D8Params& p) const { return min(4, p.chunks - 4 * group); }
};

// Tile order: the tiles of eight rows of tiles together, so that the CTAs at work share both operands' tiles in L2.
__device__ __forceinline__ void d8_tile(const D8Params& p, int tile, int& c, int& mt, int& nt) {
    const unsigned per = (unsigned)(p.m_tiles * p.n_tiles), t = (unsigned)tile;
    const unsigned comp = per > t ? 0u : t / per, r = t - comp * per, band = 8u * (unsigned)p.n_tiles, b = band > r ? 0u : r / band, in = r - b * band;
    const unsigned height = min(8u, (unsigned)p.m_tiles - b * 8u), col = in / height;
    c = (int)comp;
    mt = (int)(b * 8u + in - col * height);
    nt = (int)col;
}

// RAW: warp 8 + j quantises block j of every group of the reduction for up to D8_RAW tokens. It leaves byte j of the tokens' words before it waits for the stage, as the
// products of the group wait for the words of all four.
template <int STAGES, uint32_t STAGE>
__device__ __forceinline__ void d8_quantize_tokens(const D8Params& p, uint32_t base, uint32_t sf, uint32_t full, uint32_t empty, uint32_t sf_full, uint32_t sf_empty, int first, int stride,
                                                   int g_begin, int g_end, int j_begin, int* status) {
    const int lane = threadIdx.x & 31, j = (threadIdx.x >> 5) & 3;
    const bool quads = p.k % 4 == 0 && reinterpret_cast<uintptr_t>(p.tokens) % 16 == 0;          // four values per load
    D8Walk w;
    int q = 0, block0 = 0;                                       // block0: blocks of the groups behind us (their stages follow each other)
    uint32_t par = 1;
    for (int tile = first; tile < p.tiles; tile += stride) {
        int c, mt, nt;
        d8_tile(p, tile, c, mt, nt);
        for (w.start(p, c, g_begin, g_end, j_begin); w.left > 0; w.step(p, c)) {
            const int blocks = w.blocks(p), k = (w.group * 4 + j) * D8_BK + lane * 4;
            // (every load is on its way before the first value is looked at)
            uint4 raw[D8_RAW];
            if (j < blocks) {
#pragma unroll
                for (int r = 0; r < D8_RAW; ++r) {
                    const bool live = r < p.n && k < p.k;
                    const size_t at = ((size_t)w.first * p.n + r) * p.k + k;
                    if (quads && p.dtype == PCB_F32) raw[r] = ld_chained(static_cast<const uint4*>(p.tokens) + at / 4, live);
                    else if (quads) {
                        const uint2 x = ld_chained(static_cast<const uint2*>(p.tokens) + at / 4, live);
                        raw[r].x = x.x; raw[r].y = x.y;
                    } else if (p.dtype == PCB_F32) {
                        const uint32_t* x = static_cast<const uint32_t*>(p.tokens) + at;
                        raw[r] = make_uint4(ld_chained(x, live), ld_chained(x + 1, live && k + 1 < p.k), ld_chained(x + 2, live && k + 2 < p.k), ld_chained(x + 3, live && k + 3 < p.k));
                    } else {
                        const uint16_t* x = static_cast<const uint16_t*>(p.tokens) + at;
                        raw[r].x = (uint32_t)ld_chained(x, live) | (uint32_t)ld_chained(x + 1, live && k + 1 < p.k) << 16;
                        raw[r].y = (uint32_t)ld_chained(x + 2, live && k + 2 < p.k) | (uint32_t)ld_chained(x + 3, live && k + 3 < p.k) << 16;
                    }
                }
            }
            if (!warp_wait_bounded(sf_empty + 8 * q, par, status, ST_D8_SCALES)) return;
            uint32_t data[D8_RAW];
            if (j < blocks) {
#pragma unroll
                for (int r = 0; r < D8_RAW; ++r) {
                    if (r >= p.n) break;
                    float v[4];
                    if (p.dtype == PCB_F32) {
                        v[0] = __uint_as_float(raw[r].x); v[1] = __uint_as_float(raw[r].y); v[2] = __uint_as_float(raw[r].z); v[3] = __uint_as_float(raw[r].w);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t h = (e < 2 ? raw[r].x : raw[r].y) >> (16 * (e & 1)) & 0xffffu;
                            v[e] = p.dtype == PCB_F16 ? __half2float(__ushort_as_half((uint16_t)h)) : __uint_as_float(h << 16);
                        }
                    }
                    uint32_t top = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t key = __float_as_uint(v[e]) & 0x7fffffffu;
                        if (key < 0x7f800000u) top = max(top, key);
                        else v[e] = __uint_as_float(0x7fffffffu);                   // infinities too: the conversion would saturate them
                    }
                    const int byte = scale_byte(__reduce_max_sync(0xffffffffu, top));
                    const float f = inverse_scale(byte);
                    data[r] = to_e4m3x2(v[0], v[1], make_float2(f, f)) | to_e4m3x2(v[2], v[3], make_float2(f, f)) << 16;
                    if (lane == 0) asm volatile("st.shared.u8 [%0], %1;" ::"r"(sf + q * D8_SF_BYTES + 512u + r * 16u + j), "r"(byte) : "memory");
                }
                fence_proxy_async_smem();
            }
            __syncwarp();
            if (elect_one()) mbar_arrive(sf_full + 8 * q);
            __syncwarp();
            if (j < blocks) {
                const int block = block0 + j, s = block % STAGES;
                if (!warp_wait_bounded(empty + 8 * s, ((uint32_t)(block / STAGES) & 1u) ^ 1u, status, ST_D8_PRODUCER)) return;
                const uint32_t b = base + s * STAGE + D8_A_BYTES + (uint32_t)(lane & 3) * 4u;
#pragma unroll
                for (int r = 0; r < D8_RAW; ++r) {
                    if (r >= p.n) break;
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(b + r * 128u + (uint32_t)(((lane >> 2) ^ (r & 7)) << 4)), "r"(data[r]) : "memory");
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (elect_one()) mbar_arrive(full + 8 * s);
                __syncwarp();
            }
            block0 += blocks;
            if (++q == D8_SF_STAGES) { q = 0; par ^= 1u; }
        }
    }
}

// SWAP: operand A is the filter, so that tile rows run along the output's fast axis. PAIR: clusters of two; the even CTA issues for both.
// The waits look at a status word of the CTA's own; the call's gets it at the end.
template <int BN, bool SWAP, bool PAIR, bool RAW, int N>
__global__ void __launch_bounds__(D8_THREADS, 1) dense8_kernel(const __grid_constant__ D8Args<N> args, int* call_status) {
    static_assert(!RAW || (SWAP && BN == 16 && D8_RAW <= BN), "raw tokens lie in one narrow tile");
    using C = D8Config<BN, SWAP, PAIR>;
    extern __shared__ uint8_t smem_raw[];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* staged = base + C::STAGES * C::STAGE;               // (on 1024 bytes, as the swizzle of the output's boxes needs)
    uint8_t* sf = staged + D8_EPI_WARPS * C::OUT_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sf + D8_SF_STAGES * D8_SF_BYTES);
    const uint32_t rank = PAIR ? cluster_ctarank() : 0;
    const uint32_t base_addr = smem_u32(base), sf_addr = smem_u32(sf);
    const uint32_t full = smem_u32(bars), empty = full + 8 * C::STAGES, sf_full = empty + 8 * C::STAGES, sf_empty = sf_full + 8 * D8_SF_STAGES;
    const uint32_t acc_full = sf_empty + 8 * D8_SF_STAGES, acc_empty = acc_full + 8 * C::ACC, slot = acc_empty + 8 * C::ACC;
    int* status = reinterpret_cast<int*>(bars + 2 * C::STAGES + 2 * D8_SF_STAGES + 2 * C::ACC + 1);

    // (the first copies would wait for their maps)
    if (warp == 2 && lane < 3 * N) {
        const int of = lane / N, i = lane % N;
        const CUtensorMap* map = of == 0 ? &args.a[i] : (of == 1 ? &args.b[i] : &args.out[i]);
        if (of == 0 || (of == 1 && !RAW) || (of == 2 && args.p[i].out_map)) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    }
    if (t == 0) {
        *status = 0;
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(full + 8 * s, RAW ? 2 : 1); mbar_init(empty + 8 * s, 1); }
        for (int s = 0; s < D8_SF_STAGES; ++s) { mbar_init(sf_full + 8 * s, RAW ? 5 : (PAIR && rank == 0 ? 3 : 2)); mbar_init(sf_empty + 8 * s, 1); }
        for (int s = 0; s < C::ACC; ++s) { mbar_init(acc_full + 8 * s, 1); mbar_init(acc_empty + 8 * s, RAW ? 4 : D8_EPI_WARPS * C::CTAS); }
        fence_barrier_init();
    }
    if (warp == 1) {
        if (PAIR) tmem_alloc_pair(slot, 512);
        else tmem_alloc(slot, 512);
    }
    if (RAW) {
        // rows of tokens that do not exist: zeros with a scale of one
        for (int i = t; i < C::STAGES * (BN * D8_BK / 16); i += D8_THREADS)
            st_shared_v4(base_addr + (uint32_t)(i / (BN * D8_BK / 16)) * C::STAGE + D8_A_BYTES + (uint32_t)(i % (BN * D8_BK / 16)) * 16u, 0u, 0u, 0u, 0u);
        for (int i = t; i < D8_SF_STAGES * 32; i += D8_THREADS)
            st_shared_v4(sf_addr + (uint32_t)(i / 32) * D8_SF_BYTES + 512u + (uint32_t)(i % 32) * 16u, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
        fence_proxy_async_smem();
    }
    tc_fence_before_sync();
    __syncthreads();
    if (PAIR) cluster_sync_all();                                // both CTAs' barriers exist before anything signals them
    tc_fence_after_sync();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
    chain_wait();
    chain_next();
    if (args.p[0].clear && t == 0 && blockIdx.x == 0) *args.p[0].clear = 0;

    const int splits = N > 1 ? 1 : args.p[0].splits, split = splits > 1 ? (int)cluster_ctarank() : 0;
    const int share = PAIR ? 2 : splits, first = blockIdx.x / share, stride = gridDim.x / share, tiles = args.tiles();
    // this CTA's groups of the reduction (numbered over all its components)
    const int all_groups = args.p[0].comps * args.p[0].groups;
    const int g_begin = N > 1 ? 0 : (int)((long long)all_groups * split / splits), j_begin = N > 1 ? 0 : g_begin / args.p[0].groups;
    const int g_end_of_one = (int)((long long)all_groups * (split + 1) / splits);
    auto end_of = [&](const D8Params& p) { return N > 1 ? p.comps * p.groups : g_end_of_one; };
    D8Walk w;

    if (warp == 0) {
        int s = 0;
        uint32_t par = 1;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += stride) {
            const int product = args.product(tile);
            const D8Params& p = args.p[product];
            const CUtensorMap &map_a = args.a[product], &map_b = args.b[product];
            int c, mt, nt;
            d8_tile(p, args.local(tile), c, mt, nt);
            for (w.start(p, c, g_begin, end_of(p), j_begin); w.left > 0 && ok; w.step(p, c)) {
                const int k0 = w.group * 4, k1 = k0 + w.blocks(p), ca = SWAP ? w.second : w.first, cb = SWAP ? w.first : w.second;
                for (int k = k0; k < k1; ++k) {
                    ok = warp_wait_bounded(empty + 8 * s, par, status, ST_D8_PRODUCER);
                    if (!ok) break;
                    if (elect_one()) {
                        const uint32_t a = base_addr + s * C::STAGE, b = a + D8_A_BYTES, bar = full + 8 * s;
                        const int m0 = mt * C::M + (int)rank * D8_BM, n0 = nt * BN + (PAIR ? (int)rank * C::B_ROWS : 0);
                        if constexpr (PAIR) {
                            // one box of either operand per CTA; the even CTA's barrier counts the bytes of both
                            const uint32_t lead = map_to_cta(bar, 0);
                            if (rank == 0) mbar_arrive_expect_tx(bar, 2 * C::STAGE);
                            tma_load_3d_pair(a, &map_a, p.a_mn ? m0 : k * D8_BK, p.a_mn ? k * D8_BK : m0, ca, lead);
                            tma_load_3d_pair(b, &map_b, p.b_mn ? n0 : k * D8_BK, p.b_mn ? k * D8_BK : n0, cb, lead);
                        } else {
                            mbar_arrive_expect_tx(bar, D8_A_BYTES + (RAW ? 0 : BN * D8_BK));
                            tma_load_3d(a, &map_a, p.a_mn ? m0 : k * D8_BK, p.a_mn ? k * D8_BK : m0, ca, bar);
                            if constexpr (!RAW) tma_load_3d(b, &map_b, p.b_mn ? n0 : k * D8_BK, p.b_mn ? k * D8_BK : n0, cb, bar);
                        }
                    }
                    __syncwarp();
                    if (++s == C::STAGES) { s = 0; par ^= 1u; }
                }
            }
        }
    } else if (warp == 1 && rank != 0) {
        // The odd CTA's word to the even one that its scales are laid out. (The release at cluster scope waits for every load that its thread has under way: in the warps
        // that load the scales it took 1000 to 1800 clocks a group.)
        int q = 0, left = 0;
        uint32_t par = 0;
        for (int i = first; i < tiles; i += stride) left += end_of(args.p[args.product(i)]) - g_begin;
        for (; left > 0 && warp_wait_bounded(sf_full + 8 * q, par, status, ST_D8_SCALES); --left) {
            if (elect_one()) mbar_arrive_release_cluster(map_to_cta(sf_full + 8 * q, 0));
            __syncwarp();
            if (++q == D8_SF_STAGES) { q = 0; par ^= 1u; }
        }
    } else if (warp == 1) {
        const bool elected = elect_one();              // one lane issues and commits throughout
        int s = 0, q = 0, acc = 0;
        uint32_t par = 0, sf_par = 0, acc_par = 1;
        bool ok = true;
        // a barrier of both CTAs, by its address in the even one
        auto commit_both = [&](uint32_t bar) {
            if constexpr (PAIR) { mma_commit_pair(map_to_cta(bar, 0)); mma_commit_pair(map_to_cta(bar, 1)); }
            else mma_commit(bar);
        };
        const uint32_t sfa = tmem + C::SF_COL, sfb = sfa + 4;
        for (int tile = first; tile < tiles && ok; tile += stride) {
            const D8Params& p = args.p[args.product(tile)];
            const bool a_mn = p.a_mn, b_mn = BN >= 128 && p.b_mn;
            const uint32_t a_step = a_mn ? 32 * 128 / 16 : 32 / 16, b_step = b_mn ? 32 * 128 / 16 : 32 / 16;
            int c, mt, nt;
            d8_tile(p, args.local(tile), c, mt, nt);
            ok = warp_wait_bounded(acc_empty + 8 * acc, acc_par, status, ST_D8_MMA);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t d = tmem + acc * C::ACC_COLS;
            uint32_t accumulate = 0;
            for (w.start(p, c, g_begin, end_of(p), j_begin); w.left > 0 && ok; w.step(p, c)) {
                const int blocks = w.blocks(p);
                const uint32_t idesc = d8_idesc(C::M, BN, a_mn, b_mn, w.neg);
                ok = PAIR ? warp_wait_acquire_cluster(sf_full + 8 * q, sf_par, status, ST_D8_MMA) : warp_wait_bounded(sf_full + 8 * q, sf_par, status, ST_D8_MMA);
                if (!ok) break;
                tc_fence_after_sync();
                if (elected) {
                    const uint32_t src = sf_addr + q * D8_SF_BYTES;
                    copy_scales<PAIR>(sfa, src);
                    copy_scales<PAIR>(sfb, src + 512);
                    if (BN > 128) copy_scales<PAIR>(sfb + 4, src + 1024);
                }
                __syncwarp();
                for (int k = 0; k < blocks; ++k) {
                    ok = warp_wait_bounded(full + 8 * s, par, status, ST_D8_MMA);
                    if (!ok) break;
                    tc_fence_after_sync();
                    if (elected) {
                        const uint32_t a = base_addr + s * C::STAGE, b = a + D8_A_BYTES;
                        const uint64_t da = make_desc_kmajor(a), db = make_desc_kmajor(b);      // (tiles of 128 rows: one block of 128 bytes in either majorness)
                        const uint32_t id = idesc | ((uint32_t)k << 4) | ((uint32_t)k << 29);      // byte k of the scales' words
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mma_mxf8<PAIR>(d, (uint32_t)da + i * a_step, (uint32_t)(da >> 32), (uint32_t)db + i * b_step, (uint32_t)(db >> 32), id, sfa, sfb, accumulate);
                            accumulate = 1;
                        }
                        commit_both(empty + 8 * s);
                    }
                    accumulate = 1;
                    __syncwarp();
                    if (++s == C::STAGES) { s = 0; par ^= 1u; }
                }
                if (!ok) break;
                if (elected) commit_both(sf_empty + 8 * q);
                __syncwarp();
                if (++q == D8_SF_STAGES) { q = 0; sf_par ^= 1u; }
            }
            if (!ok) break;
            if (elected) commit_both(acc_full + 8 * acc);
            __syncwarp();
            if (++acc == C::ACC) { acc = 0; acc_par ^= 1u; }
        }
    } else if (RAW && (warp == 3 || warp >= 8)) {
        if (warp >= 8)
            d8_quantize_tokens<C::STAGES, C::STAGE>(args.p[0], base_addr, sf_addr, full, empty, sf_full, sf_empty, first, stride, g_begin, g_end_of_one, j_begin, status);
    } else if (warp < 4) {
        // Warp 2 the scales of A, warp 3 those of B, a group of the reduction at a time. The words of the next group are loaded before those of this one are waited for: one
        // warp that loaded them when they were due took 2600 clocks a group, where the MMAs of a group take 2048.
        const bool b_side = warp == 3;
        bool blocks = false;
        const uint8_t* scales = nullptr;
        int bk = 0, bm = 0, extent = 0, product = 0;
        uint32_t per_group = 0, per_comp = 0;                    // bytes (fewer than 2^31: a word for 128 values, and those have fewer)
        auto operand = [&]() {
            const D8Params& p = args.p[product];
            blocks = b_side ? p.b_blocks : p.a_blocks;
            scales = b_side ? p.b_scales : p.a_scales;
            bk = b_side ? p.b_bk : p.a_bk; bm = b_side ? p.b_bm : p.a_bm; extent = b_side ? p.n : p.m;
            per_group = blocks ? 4u * bk : 4u * extent;
            per_comp = blocks ? (uint32_t)(b_side ? p.b_bc : p.a_bc) : per_group * p.groups;
        };
        operand();
        constexpr int SETS = BN > 128 ? 2 : 1;                   // sets of 128 rows of B
        struct Words { uint32_t w[SETS][4]; bool blocks; };
        int tile = first, c = 0, row0[SETS];
        const uint8_t* at[SETS];                                 // where this lane's words (blocks: byte) of the walk's group lie
        const uint8_t* origin[SETS];                             // the same of component 0 and group 0
        auto aim = [&]() {
            const uint32_t comp = SWAP == b_side ? w.first : w.second;
#pragma unroll
            for (int h = 0; h < SETS; ++h) at[h] = origin[h] + (size_t)(comp * per_comp + (uint32_t)w.group * per_group);
        };
        auto begin = [&]() {
            if (tile >= tiles) return;
            if (N > 1 && args.product(tile) != product) { product = 1; operand(); }
            const D8Params& p = args.p[product];
            int mt, nt;
            d8_tile(p, args.local(tile), c, mt, nt);
#pragma unroll
            for (int h = 0; h < SETS; ++h) row0[h] = b_side ? nt * BN + h * 128 : mt * C::M + (int)rank * D8_BM;
#pragma unroll
            for (int h = 0; h < SETS; ++h) origin[h] = scales + (blocks ? (row0[h] / 128) * bm + (lane & 3) * bk : (row0[h] + lane) * 4);
            w.start(p, c, g_begin, end_of(p), j_begin);
            aim();
        };
        begin();
        // the words of rows row0 + lane + 32 i: what lane puts at byte 16 * lane of a set of 128 rows
        auto load = [&](Words& out) {
            if (tile >= tiles) return;
            const D8Params& p = args.p[product];
            out.blocks = blocks;
#pragma unroll
            for (int h = 0; h < SETS; ++h) {
                if (h > 0 && !b_side) break;
                if (blocks) {
                    // (a set of 128 rows that starts on a multiple of 128 lies in one block: lane e loads the byte of block e of the reduction)
                    out.w[h][0] = row0[h] < extent && w.group * 4 + (lane & 3) < p.chunks ? *reinterpret_cast<const volatile uint8_t*>(at[h]) : 127u;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) out.w[h][i] = ld_chained(reinterpret_cast<const uint32_t*>(at[h]) + 32 * i, row0[h] + lane + 32 * i < extent);
                }
            }
            w.step(p, c);
            if (w.left == 0) { tile += stride; begin(); }
            else aim();
        };
        int q = 0;
        uint32_t par = 1;
        bool ok = true;
        Words next, now;
        load(next);
        for (int t_ = first; t_ < tiles && ok; t_ += stride)
            for (int i = g_begin, last = end_of(args.p[args.product(t_)]); i < last && ok; ++i) {
                now = next;
                load(next);
                ok = warp_wait_bounded(sf_empty + 8 * q, par, status, ST_D8_SCALES);
                if (!ok) break;
                const uint32_t dst = sf_addr + q * D8_SF_BYTES + (b_side ? 512 : 0) + lane * 16;
#pragma unroll
                for (int h = 0; h < SETS; ++h) {
                    if (h > 0 && !b_side) break;
                    uint32_t* v = now.w[h];
                    if (now.blocks) {
                        const uint32_t word = __shfl_sync(0xffffffffu, v[0], 0) | (__shfl_sync(0xffffffffu, v[0], 1) << 8) | (__shfl_sync(0xffffffffu, v[0], 2) << 16) |
                                              (__shfl_sync(0xffffffffu, v[0], 3) << 24);
                        v[0] = v[1] = v[2] = v[3] = word;
                    }
                    st_shared_v4(dst + h * 512, v[0], v[1], v[2], v[3]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (elect_one()) mbar_arrive(sf_full + 8 * q);
                __syncwarp();
                if (++q == D8_SF_STAGES) { q = 0; par ^= 1u; }
            }
    } else if (warp >= 4) {
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        constexpr int COLS = BN < 64 ? 32 : BN / 2;               // columns per warp; with a narrow tile the second four warps have none
        constexpr int BLOCKS = COLS / 32;
        const bool idle = BN < 64 && half > 0;
        const int col0 = half * COLS;
        const uint32_t buf = smem_u32(staged) + (warp - 4) * C::OUT_BYTES;
        int acc = 0;
        uint32_t par = 0;
        bool ok = true;
        for (int tile = first; tile < tiles && ok; tile += stride) {
            const int product = args.product(tile);
            const D8Params& p = args.p[product];
            const CUtensorMap& map_out = args.out[product];
            const int fast = SWAP ? p.m : p.n;
            int c, mt, nt;
            d8_tile(p, args.local(tile), c, mt, nt);
            const int before = read_status(status);
            ok = warp_may_store(warp_wait_bounded(acc_full + 8 * acc, par, status, ST_D8_EPILOGUE), before);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t src = tmem + ((uint32_t)(quarter * 32) << 16) + acc * C::ACC_COLS + col0;
            uint32_t v[BLOCKS][32];
            if (!idle) {
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) tmem_ld_32x32b_x32(src + 32 * b, v[b]);
                tmem_ld_wait();
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) tmem_regs_ready(v[b]);
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(map_to_cta(acc_empty + 8 * acc, 0));
                else mbar_arrive(acc_empty + 8 * acc);
            }
            if (++acc == C::ACC) { acc = 0; par ^= 1u; }
            if (idle) continue;
            const int row = quarter * 32 + lane, row0 = mt * C::M + (int)rank * D8_BM + quarter * 32, m = row0 + lane, n0 = nt * BN + col0;
            if (splits > 1) {
                // partial sums to shared memory (the ring: every MMA has read it), the fast axis of the output contiguous
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) {
                    if constexpr (SWAP) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const int n = col0 + 32 * b + e;
                            if (n < BN) asm volatile("st.shared.u32 [%0], %1;" ::"r"(base_addr + (uint32_t)(n * C::PART_PITCH + row) * 4u), "r"(v[b][e]) : "memory");
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) st_shared_v4(base_addr + (uint32_t)(row * C::PART_PITCH + col0 + 32 * b + e) * 4u, v[b][e], v[b][e + 1], v[b][e + 2], v[b][e + 3]);
                    }
                }
                continue;
            }
            const long long comp0 = (long long)c * p.out_comp;
            if (SWAP) {
                const float add = p.bias && m < p.m ? ld_typed(p.bias, p.dtype, (size_t)c * fast + m) : 0.f;
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const int n = n0 + 32 * b + e;
                        if (m < p.m && n < p.n && 32 * b + e < BN - col0) st_typed(p.out, p.dtype, comp0 + (long long)n * p.out_ld + m, __uint_as_float(v[b][e]) + add);
                    }
            } else {
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) {
                    const int n = n0 + 32 * b;
                    if (n >= p.n) break;
                    if (p.bias) {
                        const float add = n + lane < p.n ? ld_typed(p.bias, p.dtype, (size_t)c * fast + n + lane) : 0.f;
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[b][e] = __float_as_uint(__uint_as_float(v[b][e]) + __shfl_sync(0xffffffffu, add, e));
                    }
                    uint32_t packed[16];
                    if (p.dtype != PCB_F32) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) packed[e] = pack_16(__uint_as_float(v[b][2 * e]), __uint_as_float(v[b][2 * e + 1]), p.dtype);
                    }
                    if (p.out_map) {
                        // rows of 128 bytes (64 or 32 columns), swizzled as the output's boxes are; the copy leaves out what lies beyond the output
                        const bool f32 = p.dtype == PCB_F32;
                        if (f32 || (b & 1) == 0) {
                            if (lane == 0) bulk_wait_read_all();
                            __syncwarp();
                        }
                        const uint32_t line = buf + lane * 128;
                        if (f32) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) st_shared_v4(line + ((e ^ (lane & 7)) << 4), v[b][4 * e], v[b][4 * e + 1], v[b][4 * e + 2], v[b][4 * e + 3]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) st_shared_v4(line + (((e + 4 * (b & 1)) ^ (lane & 7)) << 4), packed[4 * e], packed[4 * e + 1], packed[4 * e + 2], packed[4 * e + 3]);
                        }
                        if (f32 || (b & 1) || n + 32 >= p.n) {
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0 && row0 < p.m) {
                                tma_store_3d(&map_out, buf, f32 ? n : n - 32 * (b & 1), row0, c);
                                bulk_commit_group();
                            }
                        }
                    } else if (p.dtype == PCB_F32) {
                        park_words(buf, 0, v[b], 32, lane);
                        store_parked_floats(buf, static_cast<float*>(p.out) + comp0 + (long long)row0 * p.out_ld + n, p.m - row0, p.n - n, p.out_ld, lane);
                    } else {
                        park_words(buf, 16 * (b & 1), packed, 16, lane);
                        if ((b & 1) || n + 32 >= p.n)
                            store_parked_halves(buf, static_cast<uint16_t*>(p.out) + comp0 + (long long)row0 * p.out_ld + n - 32 * (b & 1), p.m - row0, p.n - n + 32 * (b & 1), p.out_ld, lane);
                    }
                }
            }
        }
        if (!SWAP && lane == 0) bulk_wait_all();
    }
    if (N == 1 && splits > 1) {
        const D8Params& p = args.p[0];
        // one tile per cluster: every CTA adds its share of the tile's elements, in the order of the ranks
        __syncthreads();
        cluster_sync_all();
        int c, mt, nt;
        d8_tile(p, first, c, mt, nt);
        const int ms = min(D8_BM, p.m - mt * D8_BM), ns = min(BN, p.n - nt * BN);
        const int fast_n = SWAP ? ms : ns, slow_n = SWAP ? ns : ms, fast0 = SWAP ? mt * D8_BM : nt * BN, slow0 = SWAP ? nt * BN : mt * D8_BM, extent = SWAP ? p.m : p.n;
        bool good = true;                   // no wait ran out in any CTA of the tile
        for (int r = 0; r < p.splits; ++r) {
            uint32_t word;
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(word) : "r"(map_to_cta(smem_u32(status), r)) : "memory");
            good = good && word == 0u;
        }
        const size_t size = p.dtype == PCB_F32 ? 4 : 2;
        const bool quads = p.out_ld % 4 == 0 && p.out_comp % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % (4 * size) == 0;
        constexpr int F4 = (SWAP ? D8_BM : BN) / 4;
        if (good) {
            // four neighbours of the output at a time (one by one, a tile of 128 x 128 took ten microseconds to add up)
            for (int e = split * D8_THREADS + t; e < slow_n * F4; e += p.splits * D8_THREADS) {
                const int slow = e / F4, fast = e % F4 * 4;
                if (fast >= fast_n) continue;
                const uint32_t local = base_addr + (uint32_t)(slow * C::PART_PITCH + fast) * 4u;
                float part[8][4];
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < p.splits)
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(part[r][0]), "=f"(part[r][1]), "=f"(part[r][2]), "=f"(part[r][3]) : "r"(map_to_cta(local, r)) : "memory");
                float out[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < p.splits) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) out[i] += part[r][i];
                    }
                if (p.bias) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (fast + i < fast_n) out[i] += ld_typed(p.bias, p.dtype, (size_t)c * extent + fast0 + fast + i);
                }
                const size_t at = (size_t)((long long)c * p.out_comp + (long long)(slow0 + slow) * p.out_ld + fast0 + fast);
                if (quads && fast + 4 <= fast_n) {
                    if (p.dtype == PCB_F32) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(out[0], out[1], out[2], out[3]);
                    else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(pack_16(out[0], out[1], p.dtype), pack_16(out[2], out[3], p.dtype));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (fast + i < fast_n) st_typed(p.out, p.dtype, at + i, out[i]);
                }
            }
        }
        cluster_sync_all();                 // nobody leaves while its partial sums are read
    }
    tc_fence_before_sync();
    __syncthreads();
    if (t == 0 && *status != 0) atomicOr(call_status, *status);
    if (PAIR) cluster_sync_all();
    if (warp == 1) {
        tc_fence_after_sync();
        if (PAIR) tmem_dealloc_pair(tmem, 512);
        else tmem_dealloc(tmem, 512);
    }
}

int operand_map(CUtensorMap* map, const Q8Operand& o, int extent, int k, int comps, int box_rows, const char* what) {
    const int inner = o.mn_major ? extent : k, outer = o.mn_major ? k : extent;
    const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)comps};
    const cuuint64_t strides[2] = {(cuuint64_t)o.pitch, (cuuint64_t)o.pitch * outer};
    const cuuint32_t box[3] = {128, (cuuint32_t)(o.mn_major ? 128 : box_rows), 1};
    return make_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, o.values, 3, dims, strides, box, nullptr, CU_TENSOR_MAP_SWIZZLE_128B, what);
}

template <int BN, bool SWAP, bool PAIR, bool RAW, int N>
int describe(const Geom& g, const Q8Product& q, int splits, D8Args<N>& args, int i) {
    using C = D8Config<BN, SWAP, PAIR>;
    D8Params& p = args.p[i];
    p.pass = q.pass; p.ga = g.ga; p.comps = g.nc; p.neg = g.neg;
    p.m = q.m; p.n = q.n; p.k = q.k;
    p.chunks = q8_blocks(q.k); p.groups = q8_groups(q.k);
    p.m_tiles = (q.m + C::M - 1) / C::M; p.n_tiles = (q.n + BN - 1) / BN; p.tiles = p.m_tiles * p.n_tiles * g.nc;
    p.splits = splits;
    p.a_mn = q.a.mn_major; p.b_mn = q.b.mn_major;
    p.a_blocks = q.a.block_scales; p.b_blocks = q.b.block_scales;
    p.a_scales = static_cast<const uint8_t*>(q.a.scales); p.b_scales = static_cast<const uint8_t*>(q.b.scales);
    p.a_bk = q.a.bytes_k; p.a_bm = q.a.bytes_mn; p.b_bk = q.b.bytes_k; p.b_bm = q.b.bytes_mn;
    p.a_bc = q8_blocks(q.m) * q8_blocks(q.k); p.b_bc = q8_blocks(q.n) * q8_blocks(q.k);
    p.dtype = q.dtype; p.out = q.out; p.bias = q.bias;
    p.out_ld = SWAP ? q.m : q.n;
    p.out_comp = (long long)q.m * q.n;
    p.tokens = q.tokens; p.clear = RAW ? q.status : nullptr;
    int rc = operand_map(&args.a[i], q.a, q.m, q.k, g.nc, D8_BM, "8-bit operand A");
    if (rc == PCB_OK && !RAW) rc = operand_map(&args.b[i], q.b, q.n, q.k, g.nc, PAIR ? C::B_ROWS : BN, "8-bit operand B");
    const size_t size = dtype_size(q.dtype);
    p.out_map = !SWAP && splits == 1 && q.n * size % 16 == 0 && reinterpret_cast<uintptr_t>(q.out) % 16 == 0;
    if (rc == PCB_OK && p.out_map) {
        const cuuint64_t dims[3] = {(cuuint64_t)q.n, (cuuint64_t)q.m, (cuuint64_t)g.nc}, strides[2] = {q.n * size, (cuuint64_t)q.n * q.m * size};
        const cuuint32_t box[3] = {(cuuint32_t)(128 / size), 32, 1};
        const CUtensorMapDataType type = q.dtype == PCB_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : (q.dtype == PCB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
        rc = make_tensor_map(&args.out[i], type, q.out, 3, dims, strides, box, nullptr, CU_TENSOR_MAP_SWIZZLE_128B, "8-bit product's output");
    }
    return rc;
}
template <int BN, bool SWAP, bool PAIR, bool RAW, int N>
int start(const D8Args<N>& args, int splits, int* status, cudaStream_t stream) {
    using C = D8Config<BN, SWAP, PAIR>;
    const size_t smem = C::SMEM > ONE_CTA_SMEM ? C::SMEM : ONE_CTA_SMEM;
    static_assert(C::SMEM <= MAX_CTA_SMEM, "shared memory of a CTA");
    PCB_CUDA_TRY((allow_cta_smem<dense8_kernel<BN, SWAP, PAIR, RAW, N>>()));
    int tiles = 0;
    for (int i = 0; i < N; ++i) tiles += args.p[i].tiles;
    const int grid = PAIR ? 2 * (tiles < sm_pairs() ? tiles : sm_pairs()) : (splits > 1 ? tiles * splits : (tiles < sm_count() ? tiles : sm_count()));
    PCB_CUDA_TRY(launch_clusters(PAIR ? 2 : splits, true, dense8_kernel<BN, SWAP, PAIR, RAW, N>, grid, D8_THREADS, smem, stream, args, status));
    return PCB_OK;
}
template <int BN, bool SWAP, bool PAIR, bool RAW = false>
int launch(const Geom& g, const Q8Product& q, int splits, cudaStream_t stream) {
    D8Args<1> args = {};
    const int rc = describe<BN, SWAP, PAIR, RAW>(g, q, splits, args, 0);
    return rc != PCB_OK ? rc : start<BN, SWAP, PAIR, RAW>(args, splits, q.status, stream);
}
template <int BN>
int launch_two(const Geom& g, const Q8Product& first, const Q8Product& second, cudaStream_t stream) {
    D8Args<2> args = {};
    int rc = describe<BN, false, false, false>(g, first, 1, args, 0);
    if (rc == PCB_OK) rc = describe<BN, false, false, false>(g, second, 1, args, 1);
    return rc != PCB_OK ? rc : start<BN, false, false, false>(args, 1, first.status, stream);
}

// CTAs that share a tile of 128 rows and bn columns, up to a portable cluster and the SMs there are
int splits_for(const Geom& g, const Q8Product& q, int bn, double* cost = nullptr) {
    const int groups = g.nc * q8_groups(q.k);
    const long long tiles = (long long)q8_blocks(q.m) * ((q.n + bn - 1) / bn) * g.nc;
    int best = 1;
    double least = groups;                               // a group of four blocks takes about a microsecond
    for (int s = 2; s <= 8 && s <= groups && tiles * s <= sm_count(); s *= 2) {
        const double c = 3.5 + (groups + s - 1) / s;
        if (c < least) { least = c; best = s; }
    }
    if (cost) *cost = best == 1 ? 7.5 + (double)((tiles + sm_count() - 1) / sm_count()) * g.nc * q8_blocks(q.k) * 0.27 : 7.5 + least;
    return best;
}
double pair_cost(const Geom& g, const Q8Product& q) {
    const long long tiles = (long long)((q.m + 255) / 256) * ((q.n + 255) / 256) * g.nc;
    return sm_pairs() > 0 ? 12.0 + (double)((tiles + sm_pairs() - 1) / sm_pairs()) * g.nc * q8_blocks(q.k) * 0.34 : 1e30;
}

}  // namespace

bool q8_swapped(int tokens) { return tokens <= 64; }
// Each token adds its loads and a maximum over a warp to the way to the first product: 4096 -> 4096 by itself took 14.2 us for one token and 24 to 27 for 8 and 16
// (in registers for 16), where quantising first takes 3.7 + 11 us and 3 us more of the host.
bool q8_raw_tokens(int tokens) { return tokens <= D8_RAW; }

// Measured on cold inputs, us (fitted to 1 to 4 rounds of tiles and reductions of 5 to 128 blocks): a single tile of 128 x 128 takes 0.27 a block behind 7.5 for launch, first
// copies and epilogue; a pair's of 256 x 256 0.34 a block behind 12; a reduction cut over a cluster 3.5 more. 2048 x 4096 -> 4096: pairs 33.9, single 44.4;
// 1024 x 4096 -> 4096 24.4 / 25.5; 2048 x 1024 -> 4096 18.0 / 17.4; 512 x 4096 -> 4096 23.0 / 16.1; GA(3,0,0) 4608 x 512 -> 768 85.5 / 129.8. Cut in two and not, 300 x 4096 -> 2048 14.0 / 14.6; 512 x 1024 ->
// 1024 10.6 / 8.6.
int q8_form(const Geom& g, const Q8Product& q, int* splits) {
    *splits = 1;
    if (q.swapped) {
        *splits = splits_for(g, q, q.n <= 16 ? 16 : 64);
        return q8_raw_tokens(q.n) && q.pass == PASS_FWD ? PCB_DENSE8_TOKENS : PCB_DENSE8_FILTER_FIRST;
    }
    double single = 0.0;
    const int cut = splits_for(g, q, 128, &single);
    if (pair_cost(g, q) < single) return PCB_DENSE8_PAIRS;
    *splits = cut;
    return PCB_DENSE8_TILES;
}
int q8_product(const Geom& g, const Q8Product& q, cudaStream_t stream) {
    int splits;
    switch (q8_form(g, q, &splits)) {
        case PCB_DENSE8_TOKENS: return launch<16, true, false, true>(g, q, splits, stream);
        case PCB_DENSE8_FILTER_FIRST: return q.n <= 16 ? launch<16, true, false>(g, q, splits, stream) : launch<64, true, false>(g, q, splits, stream);
        case PCB_DENSE8_PAIRS: return launch<256, false, true>(g, q, 1, stream);
        default: return launch<128, false, false>(g, q, splits, stream);
    }
}

// Both gradients in one launch where that is the cheaper by the costs above: tiles of 128 x 128, dealt to the CTAs in turn. A second launch costs its 7.5 us less some 2 that lie
// beside the end of the first. Measured, f16, with the quantisation in front: quaternion 777 x 500 -> 1001 36.6 us, 42.7 in two launches; 256 x 512 -> 512 13.2 / 19.7; real 4096 x 1024 -> 1024
// 25.7 / 29.9; complex 6096 x 389 -> 3136, which the costs call equal, 156.8 / 146.8: hence the margin.
bool q8_together(const Geom& g, const Q8Product& first, const Q8Product& second) {
    if (first.swapped || second.swapped) return false;
    double a = 0.0, b = 0.0;
    splits_for(g, first, 128, &a);
    splits_for(g, second, 128, &b);
    const double apart = fmin(a, pair_cost(g, first)) + fmin(b, pair_cost(g, second)) - 2.0;
    const long long sms = sm_count(), t0 = (long long)q8_blocks(first.m) * q8_blocks(first.n) * g.nc, all = t0 + (long long)q8_blocks(second.m) * q8_blocks(second.n) * g.nc;
    // the CTA with the most to do is the first, or the first that has one tile fewer of either
    double most = 0.0;
    for (long long i : {0LL, t0 % sms, all % sms}) {
        const long long ours = (t0 - i + sms - 1) / sms, both = (all - i + sms - 1) / sms;
        most = fmax(most, (double)(ours * q8_blocks(first.k) + (both - ours) * q8_blocks(second.k)) * g.nc);
    }
    return 7.5 + most * 0.27 < 0.85 * apart;
}
int q8_two_products(const Geom& g, const Q8Product& first, const Q8Product& second, cudaStream_t stream) {
    if (q8_together(g, first, second)) return launch_two<128>(g, first, second, stream);
    const int rc = q8_product(g, first, stream);
    return rc != PCB_OK ? rc : q8_product(g, second, stream);
}

}  // namespace pcb
