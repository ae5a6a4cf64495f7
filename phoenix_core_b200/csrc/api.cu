// C ABI of the backend: argument validation, geometry, kernel-family selection and dispatch.
// Nothing here allocates device memory; scratch comes from the caller's workspace.
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <unordered_map>

#include "common.cuh"
#include "dense8.cuh"
#include "tc_common.cuh"
#include "tensor_path.cuh"
#include "umma.cuh"

namespace pcb {
// (a kernel and not a memset, so that the kernel behind it can be chained to it)
static __global__ void clear_status_kernel(int* word) {
    tc::chain_wait();
    tc::chain_next();
    if (threadIdx.x == 0) *word = 0;
}
int clear_status_word(int* word, cudaStream_t stream) {
    if (reinterpret_cast<uintptr_t>(word) % sizeof(int) != 0) PCB_CUDA_TRY(cudaMemsetAsync(word, 0, sizeof(int), stream));   // any workspace address is taken
    else PCB_CUDA_TRY(tc::launch_chained(clear_status_kernel, 1, 32, 0, stream, word));
    return PCB_OK;
}

int g_sm_margin = 0;         // SMs the persistent kernels leave free (pcb_set_sm_margin)

static thread_local char g_error[512] = {0};

void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
}

// Status words that lie elsewhere than at the head of their workspace (pcb_set_status_word), by workspace address.
static std::mutex g_word_mutex;
static std::unordered_map<const void*, int*> g_words;
static std::atomic<int> g_word_count{0};            // (looked at first: a program without such words takes no lock)
int* status_of(const void* workspace) {
    if (workspace && g_word_count.load(std::memory_order_acquire) > 0) {
        std::lock_guard<std::mutex> lock(g_word_mutex);
        const auto it = g_words.find(workspace);
        if (it != g_words.end()) return it->second;
    }
    return static_cast<int*>(const_cast<void*>(workspace));
}

// Staged inputs kept by forward calls, by workspace address (host-side bookkeeping; the data itself lives in that workspace).
// A forward call that stages x in the layout its filter gradient reads records (x, problem signature) under its workspace;
// every later call that is given the same workspace erases the record before it writes there. pcb_qconv2d_bwd_kept reads the
// staged copy only when the record still matches its own x and problem, and stages x itself otherwise.
struct KeptInput { const void* x; unsigned long long signature; };
static std::mutex g_kept_mutex;
static std::unordered_map<const void*, KeptInput> g_kept;
void forget_kept(const void* workspace) {
    if (!workspace) return;
    std::lock_guard<std::mutex> lock(g_kept_mutex);
    g_kept.erase(workspace);
}

namespace {

constexpr long long MAX_NUMEL = 2147483647LL;   // tensor offsets are 32-bit element indices inside kernels

int out_size(int in, int k, int dil, int stride, int before, int after) {
    const int eff = (k - 1) * dil + 1;
    return (in + before + after - eff + stride) / stride;
}

// Validates a convolution descriptor and fills the kernel geometry.
int conv_geom(const pcb_conv2d_desc* d, Geom& g) {
    if (!d) { set_error("null descriptor"); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->dtype < PCB_F32 || d->dtype > PCB_BF16) { set_error("unknown dtype %d", d->dtype); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->n < 0 || d->ci <= 0 || d->co <= 0 || d->h <= 0 || d->w <= 0 || d->kh <= 0 || d->kw <= 0 || d->stride_h <= 0 ||
        d->stride_w <= 0 || d->pad_top < 0 || d->pad_left < 0 || d->pad_bottom < 0 || d->pad_right < 0) {
        set_error("invalid convolution geometry");
        return PCB_ERR_INVALID_ARGUMENT;
    }
    if (d->groups < 1 || d->co % d->groups != 0) { set_error("invalid groups (%d groups, %d output channels)", d->groups, d->co); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->groups != 1 && (d->data_format != PCB_LAYOUT_NCHW || d->filter_layout != PCB_FILTER_OIHW)) {
        set_error("grouped convolution takes NCHW tensors and OIHW filters only (groups = %d)", d->groups);
        return PCB_ERR_UNSUPPORTED;
    }
    if (d->dilation_h < 1 || d->dilation_w < 1) { set_error("dilation must be >= 1"); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->variant != PCB_VARIANT_16_PRODUCT && d->variant != PCB_VARIANT_8_PRODUCT) { set_error("unknown variant"); return PCB_ERR_INVALID_ARGUMENT; }
    if (!algebra_setup(d->algebra, g)) { set_error("unknown algebra %d", d->algebra); return PCB_ERR_INVALID_ARGUMENT; }
    // groups: the descriptor's ci is the filters' input channels (the input tensor holds ci * groups), co the total
    g.groups = d->groups;
    g.Nb = d->n; g.Ci = d->ci; g.Co = d->co / d->groups; g.H = d->h; g.W = d->w;
    g.KH = d->kh; g.KW = d->kw; g.SH = d->stride_h; g.SW = d->stride_w; g.DH = d->dilation_h; g.DW = d->dilation_w;
    g.PT = d->pad_top; g.PL = d->pad_left;
    g.HO = out_size(d->h, d->kh, d->dilation_h, d->stride_h, d->pad_top, d->pad_bottom);
    g.WO = out_size(d->w, d->kw, d->dilation_w, d->stride_w, d->pad_left, d->pad_right);
    if (g.HO <= 0 || g.WO <= 0) { set_error("empty convolution output (%d x %d)", g.HO, g.WO); return PCB_ERR_INVALID_ARGUMENT; }
    g.w_io = 0; g.dw_io = 0; g.real_in = d->real_valued_input ? 1 : 0; g.has_bias = d->has_bias ? 1 : 0;
    if (d->data_format < PCB_LAYOUT_NCHW || d->data_format > PCB_LAYOUT_NHWC || d->filter_layout < PCB_FILTER_OIHW || d->filter_layout > PCB_FILTER_HWIO) {
        set_error("unknown tensor layout (data format %d, filter layout %d)", d->data_format, d->filter_layout);
        return PCB_ERR_INVALID_ARGUMENT;
    }
    set_conv_strides(g, d->data_format, d->filter_layout, g.Ci * g.groups, g.Co * g.groups);
    g.plain = (d->data_format == PCB_LAYOUT_NCHW && d->filter_layout == PCB_FILTER_OIHW && g.groups == 1) ? 1 : 0;
    const long long xn = (long long)(g.real_in ? 1 : g.nc) * g.Nb * g.Ci * g.groups * g.H * g.W;
    const long long yn = (long long)g.nc * g.Nb * g.Co * g.groups * g.HO * g.WO;
    const long long wn = (long long)g.nc * g.Co * g.groups * g.Ci * g.KH * g.KW;
    if (xn > MAX_NUMEL || yn > MAX_NUMEL || wn > MAX_NUMEL || g.H > 32767 || g.W > 32767) {
        set_error("tensor too large for 32-bit element offsets");
        return PCB_ERR_TOO_LARGE;
    }
    return PCB_OK;
}

int dense_geom(const pcb_dense_desc* d, Geom& g) {
    if (!d) { set_error("null descriptor"); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->dtype < PCB_F32 || d->dtype > PCB_BF16) { set_error("unknown dtype %d", d->dtype); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->batch < 0 || d->in_features <= 0 || d->out_features <= 0) { set_error("invalid dense geometry"); return PCB_ERR_INVALID_ARGUMENT; }
    if (d->variant != PCB_VARIANT_16_PRODUCT && d->variant != PCB_VARIANT_8_PRODUCT) { set_error("unknown variant"); return PCB_ERR_INVALID_ARGUMENT; }
    if (!algebra_setup(d->algebra, g)) { set_error("unknown algebra %d", d->algebra); return PCB_ERR_INVALID_ARGUMENT; }
    g.Nb = d->batch; g.Ci = d->in_features; g.Co = d->out_features;
    g.H = g.W = g.HO = g.WO = 1; g.KH = g.KW = 1; g.SH = g.SW = 1; g.DH = g.DW = 1; g.PT = g.PL = 0;
    g.w_io = d->filter_oi ? 0 : 1;
    g.dw_io = 1;   // both reference backends emit the filter gradient input-major (src/backend/cudnn/dense.hpp:187-195)
    g.real_in = 0; g.has_bias = d->has_bias ? 1 : 0;
    // x [D*B, I], y [D*B, O]; filters [D, I, O] or [D, O, I]; the filter gradient always [D, I, O]
    g.xp = g.Ci; g.xc = 1; g.xh = g.xw = 0; g.yp = g.Co; g.yc = 1; g.yh = g.yw = 0;
    g.wr = g.Ci * g.Co; g.wh = g.ww = 0; g.wo = g.w_io ? 1 : g.Ci; g.wi = g.w_io ? g.Co : 1;
    g.dr = g.wr; g.dkh = g.dkw = 0; g.dco = 1; g.dci = g.Co;
    g.bias_ld = g.Co; g.plain = 1; g.groups = 1;
    if ((long long)g.nc * g.Nb * g.Ci > MAX_NUMEL || (long long)g.nc * g.Nb * g.Co > MAX_NUMEL || (long long)g.nc * g.Ci * g.Co > MAX_NUMEL) {
        set_error("tensor too large for 32-bit element offsets");
        return PCB_ERR_TOO_LARGE;
    }
    return PCB_OK;
}

// The factorised 8-product form exists for quaternions only (reference: src/conv2d.hpp:167, :433); every other
// algebra runs the generic product whatever the variant says.
int variant_for(const Geom& g, int variant) { return g.nc == 4 ? variant : (int)PCB_VARIANT_16_PRODUCT; }

// The formulation the tensor-core kernels are asked for. With PCB_ENGINE_AUTO the 8-product request is read the way the
// reference means it -- "prefer speed to memory" (Context::preferSpeedToMemory, src/backend/backend.hpp:58): where a
// tensor-core kernel exists it is the fast choice (its one formulation needs no lane temporaries either), and the factorised
// kernels keep the problems the tensor cores do not take. PCB_ENGINE_TENSOR and PCB_ENGINE_SIMT take the variant literally.
int tensor_variant(int variant, int engine) { return engine == PCB_ENGINE_AUTO ? (int)PCB_VARIANT_16_PRODUCT : variant; }

// Clears the device wait status at the start of an API call. Every kernel launched by the call only ORs into the
// word, so pcb_check_device_status afterwards reports an expiry in ANY launch of the call, not just the last one.
// A call that hands the reset to its first launch (StatusClear) settles it with finish_status: a call that launched nothing
// resets the word all the same.
int reset_status(void* workspace, size_t ws_bytes, cudaStream_t stream) {
    return workspace && ws_bytes >= sizeof(int) ? clear_status_word(status_of(workspace), stream) : (int)PCB_OK;
}

StatusClear owe_status(void* workspace, size_t ws_bytes) {
    StatusClear sc;
    sc.word = status_of(workspace);
    sc.pending = workspace && ws_bytes >= sizeof(int);
    return sc;
}
int finish_status(StatusClear& sc, int rc, cudaStream_t stream) {
    const int rs = sc.now(stream);
    return rc != PCB_OK ? rc : rs;
}

unsigned long long problem_signature(int dtype, const Geom& g) {
    const int v[] = {dtype, g.nc, g.ga, g.real_in, g.Nb, g.Ci, g.Co, g.H, g.W, g.KH, g.KW, g.SH, g.SW, g.DH, g.DW, g.PT, g.PL, g.HO, g.WO};
    unsigned long long h = 1469598103934665603ull;                   // FNV-1a over the geometry
    for (int x : v) { h ^= (unsigned long long)(unsigned)x; h *= 1099511628211ull; }
    return h;
}
void remember_kept(const void* workspace, const void* x, unsigned long long signature) {
    std::lock_guard<std::mutex> lock(g_kept_mutex);
    if (g_kept.size() >= 4096) g_kept.clear();                       // bounded: callers that never run the backward pass
    g_kept[workspace] = KeptInput{x, signature};
}
bool kept_matches(const void* workspace, const void* x, unsigned long long signature) {
    std::lock_guard<std::mutex> lock(g_kept_mutex);
    const auto it = g_kept.find(workspace);
    return it != g_kept.end() && it->second.x == x && it->second.signature == signature;
}

size_t workspace_bytes(Pass pass, int dtype, int variant, int engine, const Geom& g) {
    size_t s = simt_scratch_bytes(pass, dtype, variant, g);
    const size_t t = tensor_scratch_bytes(pass, dtype, tensor_variant(variant, engine), engine, g);
    if (t > s) s = t;
    return WS_HEADER + ((s + 255) / 256) * 256;
}

// `full`: the problem as described; where the workspace is too small for it the kernels take the tight layout (Geom), so that a workspace
// of a size that once was enough still is.
int run_pass(Pass pass, int dtype, int variant, int engine, const Geom& full, const void* a, const void* b, const void* bias,
             void* out, void* workspace, size_t ws_bytes, cudaStream_t stream, const PassExtras* extras = nullptr, StatusClear* sc = nullptr) {
    forget_kept(workspace);
    Geom g = full;
    const size_t offset = extras ? extras->scratch_offset : 0;       // scratch another pass of the same call still needs
    size_t need = workspace_bytes(pass, dtype, variant, engine, g) + offset;
    if (workspace && ws_bytes < need) {
        g.tight = 1;
        need = workspace_bytes(pass, dtype, variant, engine, g) + offset;
    }
    const int tv = tensor_variant(variant, engine);
    const bool needs_ws = need > WS_HEADER || tensor_path_supported(pass, dtype, tv, g);
    if (needs_ws && (workspace == nullptr || ws_bytes < need)) {
        set_error("workspace of %zu bytes required, %zu given", need, workspace ? ws_bytes : (size_t)0);
        return PCB_ERR_WORKSPACE;
    }
    float* scratch = workspace ? reinterpret_cast<float*>(static_cast<char*>(workspace) + WS_HEADER + offset) : nullptr;
    int* status = status_of(workspace);
    // the tensor-core kernels move 16-byte chunks of NCHW / OIHW tensors: every tensor (and the workspace) must be 16-byte
    // aligned. Tensors of other layouts and the channel slices of grouped layers are addressed element by element (staged
    // operands, strided stores), so there only the workspace has to be.
    const uintptr_t tensors = g.plain ? (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(out)) : 0;
    const bool aligned = ((tensors | reinterpret_cast<uintptr_t>(workspace)) & 15u) == 0;
    if (engine != PCB_ENGINE_SIMT && aligned && tensor_path_supported(pass, dtype, tv, g)) {
        const int rc = tensor_launch(pass, dtype, tv, g, a, b, bias, out, scratch, status, stream, extras, sc);
        // (a reset behind the kernels would hide what they reported, and they would have waited against an old word)
        if (rc == PCB_OK && sc && sc->pending) { set_error("status word not reset in front of the kernels"); return PCB_ERR_CUDA; }
        if (rc == PCB_OK && pass == PASS_FWD && forward_keeps_staged_input(dtype, tv, g)) remember_kept(workspace, b, problem_signature(dtype, g));
        return rc;
    }
    if (engine == PCB_ENGINE_TENSOR) {
        set_error("no tensor-core kernel for this problem");
        return PCB_ERR_UNSUPPORTED;
    }
    if (sc) { const int rc = sc->now(stream); if (rc != PCB_OK) return rc; }
    return simt_launch(pass, dtype, variant, g, a, b, bias, out, scratch, stream);
}

// How far a dense call runs on the kernels that take the caller's tensors as they are (qgemm_tc.cu). `tensors`: the OR of all
// tensor addresses of the call; `apart`: no result shares memory with an operand, which these kernels read while they write (the
// staged kernels copy their operands first, so a gradient may replace the tensor it belongs to). The workspace must be large enough for
// the staged kernels (in their tight layout), which take the call where these do not.
DenseRoute dense_route(const pcb_dense_desc* desc, const Geom& g, uintptr_t tensors, bool apart, bool backward, void* workspace, size_t ws_bytes) {
    const int v = variant_for(g, desc->variant), tv = tensor_variant(v, desc->engine);
    Geom tight = g;
    tight.tight = 1;
    size_t need = workspace_bytes(backward ? PASS_BWD_FILTER : PASS_FWD, desc->dtype, v, desc->engine, tight);
    if (backward) {
        const size_t data = workspace_bytes(PASS_BWD_DATA, desc->dtype, v, desc->engine, tight);
        if (data > need) need = data;
    }
    const bool direct = desc->engine != PCB_ENGINE_SIMT && apart && workspace && ws_bytes >= need &&
                        ((tensors | reinterpret_cast<uintptr_t>(workspace)) & 15u) == 0 && dense_tc_supported(desc->dtype, tv, g);
    return direct ? dense_tc_route(desc->dtype, g, backward, backward && desc->require_input_grad) : DENSE_STAGED;
}
// Bytes of a dense layer's tensors.
struct DenseBytes { size_t x, y, w; };
DenseBytes dense_bytes(int dtype, const Geom& g) {
    const size_t e = (size_t)g.nc * dtype_size(dtype);
    return {e * g.Nb * g.Ci, e * g.Nb * g.Co, e * g.Ci * g.Co};
}

// Grouped convolution (reference: the groups argument of the scalar convolutions, src/backend/cudnn/conv2d.hpp:126-127):
// one pass per group on the CUDA-core kernels, which address every tensor through strides -- a group is a channel slice
// of x, y and the filters. The filter gradient of a group is produced contiguously in the workspace and copied into its
// slice (component r of the gradient is Co_total * Ci * taps elements apart, a group's slice Co * Ci * taps wide).
size_t group_slice_bytes(int dtype, const Geom& g) {
    return (((size_t)g.nc * g.Co * g.Ci * g.KH * g.KW * dtype_size(dtype)) + 255) / 256 * 256;
}

size_t conv_workspace_bytes(Pass pass, int dtype, int variant, int engine, const Geom& g) {
    if (g.groups == 1) return workspace_bytes(pass, dtype, variant, engine, g);
    return workspace_bytes(pass, dtype, variant, engine, g) + (pass == PASS_BWD_FILTER ? group_slice_bytes(dtype, g) : 0);
}

int run_conv_pass(Pass pass, int dtype, int variant, int engine, const Geom& full, const void* a, const void* b, const void* bias,
                  void* out, void* workspace, size_t ws_bytes, cudaStream_t stream, const PassExtras* extras = nullptr, StatusClear* sc = nullptr) {
    if (full.groups == 1) return run_pass(pass, dtype, variant, engine, full, a, b, bias, out, workspace, ws_bytes, stream, extras, sc);
    const size_t es = dtype_size(dtype);
    Geom g = full;
    size_t need = conv_workspace_bytes(pass, dtype, variant, engine, g);
    if (workspace && ws_bytes < need) {
        g.tight = 1;
        need = conv_workspace_bytes(pass, dtype, variant, engine, g);
    }
    if (need > WS_HEADER && (workspace == nullptr || ws_bytes < need)) {
        set_error("workspace of %zu bytes required, %zu given", need, workspace ? ws_bytes : (size_t)0);
        return PCB_ERR_WORKSPACE;
    }
    const size_t taps = (size_t)g.KH * g.KW;
    const size_t x_step = (size_t)g.Ci * g.H * g.W * es, y_step = (size_t)g.Co * g.HO * g.WO * es;
    const size_t w_step = (size_t)g.Co * g.Ci * taps * es, bias_step = (size_t)g.Co * es;
    const char* ca = static_cast<const char*>(a);
    const char* cb = static_cast<const char*>(b);
    char* co = static_cast<char*>(out);
    for (int gi = 0; gi < g.groups; ++gi) {
        int rc;
        if (pass == PASS_FWD) {            // a = filters, b = x, out = y
            rc = run_pass(pass, dtype, variant, engine, g, ca + gi * w_step, cb + gi * x_step,
                          bias ? static_cast<const char*>(bias) + gi * bias_step : nullptr, co + gi * y_step, workspace, ws_bytes, stream, nullptr, sc);
        } else if (pass == PASS_BWD_DATA) { // a = filters, b = dy, out = dx
            rc = run_pass(pass, dtype, variant, engine, g, ca + gi * w_step, cb + gi * y_step, nullptr, co + gi * x_step, workspace, ws_bytes, stream, nullptr, sc);
        } else {                           // a = dy, b = x, out = dw: contiguous slice first
            Geom gs = g;
            gs.dr = g.Co * g.Ci * (int)taps;
            const size_t inner = workspace_bytes(pass, dtype, variant, engine, g);   // a multiple of 256 bytes
            char* tmp = static_cast<char*>(workspace) + inner;                             // the slice follows the pass's own scratch
            rc = run_pass(pass, dtype, variant, engine, gs, ca + gi * y_step, cb + gi * x_step, nullptr, tmp, workspace, inner, stream, nullptr, sc);
            if (rc == PCB_OK) {
                const size_t row = (size_t)g.Co * g.Ci * taps * es;
                PCB_CUDA_TRY(cudaMemcpy2DAsync(co + gi * w_step, row * g.groups, tmp, row, row, g.nc, cudaMemcpyDeviceToDevice, stream));
            }
        }
        if (rc != PCB_OK) return rc;
    }
    return PCB_OK;
}

// One thread waits, with the given clock limit, on an mbarrier that nothing ever signals: the wait runs out, the
// status word gets its bit and the kernel returns normally. No tensor memory, no copies, nothing left in flight.
constexpr int ST_SELFTEST = 0x40000000;
__global__ void wait_expiry_kernel(int* status, long long limit_clocks) {
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) {
        umma::mbar_init(umma::smem_u32(&bar), 1);
        umma::fence_barrier_init();
        umma::mbar_wait_bounded(umma::smem_u32(&bar), 0, status, ST_SELFTEST, limit_clocks);
    }
}

// The three convolution passes without the status reset (an API call clears the word once, then runs one or more of these).
int conv_fwd(const pcb_conv2d_desc* desc, const void* x, const void* w, const void* bias, void* y,
             void* workspace, size_t workspace_bytes_, cudaStream_t stream, StatusClear* sc = nullptr) {
    Geom g;
    int rc = conv_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (g.Nb == 0) return PCB_OK;   // empty input: silent no-op, as the reference (src/conv2d.hpp:81-82)
    if (!x || !w || !y || (g.has_bias && !bias)) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    if (g.real_in && g.has_bias) { set_error("bias addition is not supported for real-valued inputs"); return PCB_ERR_UNSUPPORTED; }
    return run_conv_pass(PASS_FWD, desc->dtype, variant_for(g, desc->variant), desc->engine, g, w, x, bias, y, workspace, workspace_bytes_, stream, nullptr, sc);
}

int conv_bwd_data(const pcb_conv2d_desc* desc, const void* w, const void* dy, void* dx,
                  void* workspace, size_t workspace_bytes_, cudaStream_t stream, StatusClear* sc = nullptr) {
    Geom g;
    int rc = conv_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (g.Nb == 0) return PCB_OK;
    if (g.real_in) { set_error("input gradient required for a real-valued input tensor"); return PCB_ERR_UNSUPPORTED; }
    if (!w || !dy || !dx) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    return run_conv_pass(PASS_BWD_DATA, desc->dtype, variant_for(g, desc->variant), desc->engine, g, w, dy, nullptr, dx, workspace, workspace_bytes_, stream, nullptr, sc);
}

int conv_bwd_filter(const pcb_conv2d_desc* desc, const void* x, const void* dy, void* dw,
                    void* workspace, size_t workspace_bytes_, cudaStream_t stream, const PassExtras* extras = nullptr, StatusClear* sc = nullptr) {
    Geom g;
    int rc = conv_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (!dw) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    if (g.Nb == 0) {   // empty input: zero filter gradient, as the reference (src/conv2d.hpp:341-344)
        PCB_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)g.nc * g.Co * g.groups * g.Ci * g.KH * g.KW * dtype_size(desc->dtype), stream));
        return PCB_OK;
    }
    if (!x || !dy) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    return run_conv_pass(PASS_BWD_FILTER, desc->dtype, variant_for(g, desc->variant), desc->engine, g, dy, x, nullptr, dw, workspace, workspace_bytes_, stream, extras, sc);
}

// Staged dy shared by the two gradients of one call: the copy that backward-data makes at the start of the scratch stays where it
// is, and the filter gradient -- run second, its own scratch placed behind that copy -- reads it through a tensor map instead of
// staging dy again. Applies to 16-bit layers whose backward-data pass reads an uninserted copy (stride 1, or 2 x 2 by pixel
// classes) and whose two kernels agree on the layout.
bool bwd_shares_dy(const pcb_conv2d_desc* desc, const Geom& g, StagedView* view, size_t* offset) {
    if (desc->engine == PCB_ENGINE_SIMT || !desc->require_input_grad || g.Nb == 0 || g.groups != 1) return false;
    size_t bytes = 0;
    if (!backward_shares_staged_dy(desc->dtype, tensor_variant(variant_for(g, desc->variant), desc->engine), g, view, &bytes)) return false;
    *offset = (bytes + 1023) / 1024 * 1024;
    return true;
}

// dw and dx of one call. `kept_x`: see pcb_qconv2d_bwd_kept.
int conv_bwd_both(const pcb_conv2d_desc* desc, const void* x, const void* w, const void* dy, void* dw, void* dx,
                  void* workspace, size_t workspace_bytes_, cudaStream_t stream, const void* kept_x, StatusClear* sc) {
    Geom g;
    int rc = conv_geom(desc, g);
    if (rc != PCB_OK) return rc;
    PassExtras extras;
    extras.kept_x = kept_x;
    StagedView view;
    size_t offset = 0;
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(dy) |
                          reinterpret_cast<uintptr_t>(dw) | reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(workspace);
    // (not where dx replaces x: the filter gradient, run second, reads x)
    const size_t x_bytes = (size_t)g.nc * g.Nb * g.Ci * g.groups * g.H * g.W * dtype_size(desc->dtype);
    if (x && w && dy && dw && dx && workspace && (all & 15u) == 0 && !overlaps(dx, x_bytes, x, x_bytes) && bwd_shares_dy(desc, g, &view, &offset) &&
        workspace_bytes_ >= conv_workspace_bytes(PASS_BWD_DATA, desc->dtype, variant_for(g, desc->variant), desc->engine, g) &&
        workspace_bytes_ >= conv_workspace_bytes(PASS_BWD_FILTER, desc->dtype, variant_for(g, desc->variant), desc->engine, g) + offset) {
        // backward-data first: it leaves dy in [WS_HEADER, WS_HEADER + offset), in the layout of a workspace that is large enough
        rc = conv_bwd_data(desc, w, dy, dx, workspace, workspace_bytes_, stream, sc);
        if (rc != PCB_OK) return rc;
        view.base = static_cast<const char*>(workspace) + WS_HEADER;
        extras.dy = view;
        extras.scratch_offset = offset;
        return conv_bwd_filter(desc, x, dy, dw, workspace, workspace_bytes_, stream, &extras, sc);
    }
    rc = conv_bwd_filter(desc, x, dy, dw, workspace, workspace_bytes_, stream, &extras, sc);
    if (rc != PCB_OK) return rc;
    if (desc->require_input_grad && desc->n > 0) rc = conv_bwd_data(desc, w, dy, dx, workspace, workspace_bytes_, stream, sc);
    return rc;
}

// ---- dense layer in 8-bit floating point: where its copies of the operands lie in the workspace
struct Dense8Space {
    size_t x_rows, x_words, dy_rows, dy_row_words, dy_cols, dy_col_words, x_cols, x_col_words, total;
};
size_t align256(size_t v) { return (v + 255) / 256 * 256; }
size_t q8_value_bytes(int comps, int rows, int cols) { return (size_t)comps * rows * q8_pitch(cols); }
size_t q8_word_bytes(int comps, int extent, int summed) { return (size_t)comps * q8_groups(summed) * extent * 4; }
Dense8Space dense8_space(const Geom& g, bool backward, bool need_dx) {
    Dense8Space s = {};
    size_t at = WS_HEADER;
    auto take = [&](size_t bytes) { const size_t here = at; at = align256(at + bytes); return here; };
    if (!backward) {
        s.x_rows = take(q8_value_bytes(g.nc, g.Nb, g.Ci));
        s.x_words = take(q8_word_bytes(g.nc, g.Nb, g.Ci));
    } else {
        if (need_dx) {
            s.dy_rows = take(q8_value_bytes(g.nc, g.Nb, g.Co));
            s.dy_row_words = take(q8_word_bytes(g.nc, g.Nb, g.Co));
        }
        s.dy_cols = take(q8_value_bytes(g.nc, g.Nb, g.Co));
        s.dy_col_words = take(q8_word_bytes(g.nc, g.Co, g.Nb));
        s.x_cols = take(q8_value_bytes(g.nc, g.Nb, g.Ci));
        s.x_col_words = take(q8_word_bytes(g.nc, g.Ci, g.Nb));
    }
    s.total = at;
    return s;
}
int dense8_geom(const pcb_dense_desc* d, Geom& g) {
    const int rc = dense_geom(d, g);
    if (rc != PCB_OK) return rc;
    if (d->engine != PCB_ENGINE_AUTO && d->engine != PCB_ENGINE_TENSOR) {
        set_error("8-bit dense layers run on the tensor cores only");
        return PCB_ERR_UNSUPPORTED;
    }
    // (the 8-bit copies have rows of whole 16 bytes)
    if ((long long)g.nc * g.Nb * q8_pitch(g.Ci) > MAX_NUMEL || (long long)g.nc * g.Nb * q8_pitch(g.Co) > MAX_NUMEL ||
        (long long)g.nc * g.Ci * q8_pitch(g.Co) > MAX_NUMEL || (long long)g.nc * q8_pitch(g.Ci) * g.Co > MAX_NUMEL) {
        set_error("tensor too large for 32-bit element offsets");
        return PCB_ERR_TOO_LARGE;
    }
    return PCB_OK;
}
int dense8_workspace(const void* workspace, size_t have, size_t need) {
    if (!workspace || have < need) { set_error("workspace of %zu bytes, %zu needed", workspace ? have : (size_t)0, need); return PCB_ERR_WORKSPACE; }
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) { set_error("the workspace of an 8-bit dense layer must be 16-byte aligned"); return PCB_ERR_INVALID_ARGUMENT; }
    return PCB_OK;
}
// The filter as an operand whose own axis is `out_features` (forward) or in_features (backward-data).
Q8Operand dense8_filter(const Geom& g, const void* values, const void* scales, bool forward) {
    const int cols = g.w_io ? g.Co : g.Ci;
    Q8Operand o = {static_cast<const uint8_t*>(values), scales, q8_pitch(cols), 1, 0, 0, 0};
    o.mn_major = forward ? g.w_io : !g.w_io;                            // rows of the filter run along the operand's own axis
    const int row_stride = q8_blocks(cols);
    o.bytes_k = o.mn_major ? row_stride : 1;
    o.bytes_mn = o.mn_major ? 1 : row_stride;
    return o;
}
// A product of the layer: tokens by the filter, or for the filter gradient x by dy (both as they lie).
Q8Product dense8_product(const Geom& g, Pass pass, const Q8Operand& first, const Q8Operand& second, void* out, int dtype, int* status) {
    if (pass == PASS_BWD_FILTER) return {pass, 0, g.Ci, g.Co, g.Nb, first, second, out, dtype, nullptr, status};
    const int features = pass == PASS_FWD ? g.Co : g.Ci, summed = pass == PASS_FWD ? g.Ci : g.Co;
    if (q8_swapped(g.Nb)) return {pass, 1, features, g.Nb, summed, second, first, out, dtype, nullptr, status};
    return {pass, 0, g.Nb, features, summed, first, second, out, dtype, nullptr, status};
}
int dense8_check_filter(const void* values) {
    if (reinterpret_cast<uintptr_t>(values) % 16 != 0) { set_error("8-bit filter values must be 16-byte aligned"); return PCB_ERR_INVALID_ARGUMENT; }
    return PCB_OK;
}

}  // namespace
}  // namespace pcb

using namespace pcb;

extern "C" {

int pcb_set_sm_margin(int sms) {
    if (sms < 0 || sms > 64) return PCB_ERR_INVALID_ARGUMENT;
    pcb::g_sm_margin = sms;
    return PCB_OK;
}
int pcb_get_sm_margin(void) { return pcb::g_sm_margin; }


const char* pcb_version(void) { return "phoenix_core_b200 0.1 (sm_100a)"; }

const char* pcb_status_string(int status) {
    switch (status) {
        case PCB_OK: return "ok";
        case PCB_ERR_INVALID_ARGUMENT: return "invalid argument";
        case PCB_ERR_UNSUPPORTED: return "unsupported configuration";
        case PCB_ERR_WORKSPACE: return "workspace missing or too small";
        case PCB_ERR_CUDA: return "CUDA runtime error";
        case PCB_ERR_DEVICE_TIMEOUT: return "device-side wait expired";
        case PCB_ERR_TOO_LARGE: return "size beyond supported maximum";
    }
    return "unknown status";
}

const char* pcb_last_error_message(void) { return g_error; }

int pcb_conv2d_output_size(const pcb_conv2d_desc* desc, int32_t* out_h, int32_t* out_w) {
    Geom g;
    const int rc = conv_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (out_h) *out_h = g.HO;
    if (out_w) *out_w = g.WO;
    return PCB_OK;
}

size_t pcb_qconv2d_fwd_workspace_size(const pcb_conv2d_desc* desc) {
    Geom g;
    if (conv_geom(desc, g) != PCB_OK) return 0;
    return conv_workspace_bytes(PASS_FWD, desc->dtype, variant_for(g, desc->variant), desc->engine, g);
}

size_t pcb_qconv2d_bwd_workspace_size(const pcb_conv2d_desc* desc) {
    Geom g;
    if (conv_geom(desc, g) != PCB_OK) return 0;
    const size_t a = conv_workspace_bytes(PASS_BWD_DATA, desc->dtype, variant_for(g, desc->variant), desc->engine, g);
    size_t b = conv_workspace_bytes(PASS_BWD_FILTER, desc->dtype, variant_for(g, desc->variant), desc->engine, g);
    StagedView view;
    size_t offset = 0;
    if (bwd_shares_dy(desc, g, &view, &offset)) b += offset;          // the filter gradient's scratch lies behind the shared copy of dy
    return a > b ? a : b;
}

size_t pcb_qdense_fwd_workspace_size(const pcb_dense_desc* desc) {
    Geom g;
    if (dense_geom(desc, g) != PCB_OK) return 0;
    return workspace_bytes(PASS_FWD, desc->dtype, variant_for(g, desc->variant), desc->engine, g);
}

size_t pcb_qdense_bwd_workspace_size(const pcb_dense_desc* desc) {
    Geom g;
    if (dense_geom(desc, g) != PCB_OK) return 0;
    const size_t a = workspace_bytes(PASS_BWD_DATA, desc->dtype, variant_for(g, desc->variant), desc->engine, g);
    const size_t b = workspace_bytes(PASS_BWD_FILTER, desc->dtype, variant_for(g, desc->variant), desc->engine, g);
    return a > b ? a : b;
}

int pcb_qconv2d_fwd(const pcb_conv2d_desc* desc, const void* x, const void* w, const void* bias, void* y,
                    void* workspace, size_t workspace_bytes_, void* stream) {
    StatusClear sc = owe_status(workspace, workspace_bytes_);
    return finish_status(sc, conv_fwd(desc, x, w, bias, y, workspace, workspace_bytes_, (cudaStream_t)stream, &sc), (cudaStream_t)stream);
}

int pcb_qconv2d_bwd_data(const pcb_conv2d_desc* desc, const void* w, const void* dy, void* dx,
                         void* workspace, size_t workspace_bytes_, void* stream) {
    StatusClear sc = owe_status(workspace, workspace_bytes_);
    return finish_status(sc, conv_bwd_data(desc, w, dy, dx, workspace, workspace_bytes_, (cudaStream_t)stream, &sc), (cudaStream_t)stream);
}

int pcb_qconv2d_bwd_filter(const pcb_conv2d_desc* desc, const void* x, const void* dy, void* dw,
                           void* workspace, size_t workspace_bytes_, void* stream) {
    StatusClear sc = owe_status(workspace, workspace_bytes_);
    return finish_status(sc, conv_bwd_filter(desc, x, dy, dw, workspace, workspace_bytes_, (cudaStream_t)stream, nullptr, &sc), (cudaStream_t)stream);
}

int pcb_qconv2d_bwd_filter_noalloc(const pcb_conv2d_desc* desc, const void* x, const void* dy, void* dw, void* stream) {
    Geom g;
    int rc = conv_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (!dw) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    if (g.groups != 1) { set_error("the allocation-free filter gradient takes one group"); return PCB_ERR_UNSUPPORTED; }
    if ((size_t)g.nc * g.Co * g.Ci * g.KH * g.KW > simt_static_scratch_capacity()) {
        set_error("filter gradient of %zu elements exceeds the built-in scratch of %zu elements",
                  (size_t)g.nc * g.Co * g.Ci * g.KH * g.KW, simt_static_scratch_capacity());
        return PCB_ERR_TOO_LARGE;
    }
    if (g.Nb == 0) {
        PCB_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)g.nc * g.Co * g.Ci * g.KH * g.KW * dtype_size(desc->dtype), (cudaStream_t)stream));
        return PCB_OK;
    }
    if (!x || !dy) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    return simt_bwd_filter_static(desc->dtype, variant_for(g, desc->variant), g, dy, x, dw, (cudaStream_t)stream);
}

int pcb_qconv2d_bwd(const pcb_conv2d_desc* desc, const void* x, const void* w, const void* dy, void* dw, void* dx,
                    void* workspace, size_t workspace_bytes_, void* stream) {
    StatusClear sc = owe_status(workspace, workspace_bytes_);
    return finish_status(sc, conv_bwd_both(desc, x, w, dy, dw, dx, workspace, workspace_bytes_, (cudaStream_t)stream, nullptr, &sc), (cudaStream_t)stream);
}

int pcb_qconv2d_fwd_keeps_input(const pcb_conv2d_desc* desc) {
    Geom g;
    if (conv_geom(desc, g) != PCB_OK || desc->engine == PCB_ENGINE_SIMT || g.Nb == 0) return 0;
    return forward_keeps_staged_input(desc->dtype, tensor_variant(variant_for(g, desc->variant), desc->engine), g) ? 1 : 0;
}

int pcb_qconv2d_bwd_kept(const pcb_conv2d_desc* desc, const void* x, const void* w, const void* dy, void* dw, void* dx,
                         const void* fwd_workspace, size_t fwd_workspace_bytes, void* workspace, size_t workspace_bytes_, void* stream) {
    StatusClear sc = owe_status(workspace, workspace_bytes_);
    const void* kept_x = nullptr;
    Geom g;
    if (fwd_workspace && fwd_workspace != workspace && (reinterpret_cast<uintptr_t>(fwd_workspace) & 15u) == 0 && conv_geom(desc, g) == PCB_OK &&
        pcb_qconv2d_fwd_keeps_input(desc) && fwd_workspace_bytes >= pcb_qconv2d_fwd_workspace_size(desc) &&
        kept_matches(fwd_workspace, x, problem_signature(desc->dtype, g)))
        kept_x = static_cast<const char*>(fwd_workspace) + WS_HEADER;
    return finish_status(sc, conv_bwd_both(desc, x, w, dy, dw, dx, workspace, workspace_bytes_, (cudaStream_t)stream, kept_x, &sc), (cudaStream_t)stream);
}

int pcb_qdense_fwd(const pcb_dense_desc* desc, const void* x, const void* w, const void* bias, void* y,
                   void* workspace, size_t workspace_bytes_, void* stream) {
    Geom g;
    int rc = dense_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (g.Nb == 0) return PCB_OK;
    if (!x || !w || !y || (g.has_bias && !bias)) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    StatusClear sc = owe_status(workspace, workspace_bytes_);
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(y);
    const DenseBytes n = dense_bytes(desc->dtype, g);
    const bool apart = !overlaps(y, n.y, x, n.x) && !overlaps(y, n.y, w, n.w);
    if (dense_route(desc, g, all, apart, false, workspace, workspace_bytes_) == DENSE_DIRECT) {
        forget_kept(workspace);
        rc = dense_tc_fwd(desc->dtype, g, x, w, bias, y, status_of(workspace), (cudaStream_t)stream, sc);
    } else {
        rc = run_pass(PASS_FWD, desc->dtype, variant_for(g, desc->variant), desc->engine, g, w, x, bias, y, workspace, workspace_bytes_, (cudaStream_t)stream, nullptr, &sc);
    }
    return finish_status(sc, rc, (cudaStream_t)stream);
}

int pcb_qdense_bwd(const pcb_dense_desc* desc, const void* x, const void* w, const void* dy, void* dw, void* dx,
                   void* workspace, size_t workspace_bytes_, void* stream) {
    Geom g;
    int rc = dense_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (!dw) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    if (g.Nb == 0) {   // src/dense.hpp:226-229
        PCB_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)g.nc * g.Co * g.Ci * dtype_size(desc->dtype), (cudaStream_t)stream));
        return PCB_OK;
    }
    if (!x || !w || !dy || (desc->require_input_grad && !dx)) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    StatusClear sc = owe_status(workspace, workspace_bytes_);
    void* gx = desc->require_input_grad ? dx : nullptr;
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(dy) |
                          reinterpret_cast<uintptr_t>(dw) | reinterpret_cast<uintptr_t>(gx);
    const DenseBytes n = dense_bytes(desc->dtype, g);
    auto free_of_operands = [&](const void* out, size_t bytes) { return !overlaps(out, bytes, x, n.x) && !overlaps(out, bytes, w, n.w) && !overlaps(out, bytes, dy, n.y); };
    const bool apart = free_of_operands(dw, n.w) && free_of_operands(gx, n.x) && !overlaps(dw, n.w, gx, n.x);
    const DenseRoute route = dense_route(desc, g, all, apart, true, workspace, workspace_bytes_);
    if (route != DENSE_STAGED) {
        forget_kept(workspace);
        rc = dense_tc_bwd(desc->dtype, g, x, w, dy, dw, route == DENSE_DIRECT ? gx : nullptr, status_of(workspace), (cudaStream_t)stream, sc);
    } else {
        rc = run_pass(PASS_BWD_FILTER, desc->dtype, variant_for(g, desc->variant), desc->engine, g, dy, x, nullptr, dw, workspace, workspace_bytes_, (cudaStream_t)stream, nullptr, &sc);
    }
    if (rc == PCB_OK && route != DENSE_DIRECT && desc->require_input_grad)
        rc = run_pass(PASS_BWD_DATA, desc->dtype, variant_for(g, desc->variant), desc->engine, g, w, dy, nullptr, dx, workspace, workspace_bytes_, (cudaStream_t)stream, nullptr, &sc);
    return finish_status(sc, rc, (cudaStream_t)stream);
}

int pcb_qconv2d_engine_for(const pcb_conv2d_desc* desc, int pass) {
    Geom g;
    const int rc = conv_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (pass < 0 || pass > 2) { set_error("pass must be 0, 1 or 2"); return PCB_ERR_INVALID_ARGUMENT; }
    if (desc->engine != PCB_ENGINE_SIMT && tensor_path_supported((Pass)pass, desc->dtype, tensor_variant(variant_for(g, desc->variant), desc->engine), g)) return PCB_ENGINE_TENSOR;
    return desc->engine == PCB_ENGINE_TENSOR ? (int)PCB_ERR_UNSUPPORTED : (int)PCB_ENGINE_SIMT;
}

int pcb_qdense_engine_for(const pcb_dense_desc* desc, int pass) {
    Geom g;
    const int rc = dense_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (pass < 0 || pass > 2) { set_error("pass must be 0, 1 or 2"); return PCB_ERR_INVALID_ARGUMENT; }
    if (desc->engine != PCB_ENGINE_SIMT && tensor_path_supported((Pass)pass, desc->dtype, tensor_variant(variant_for(g, desc->variant), desc->engine), g)) return PCB_ENGINE_TENSOR;
    return desc->engine == PCB_ENGINE_TENSOR ? (int)PCB_ERR_UNSUPPORTED : (int)PCB_ENGINE_SIMT;
}

int pcb_selftest_wait_expiry(const pcb_conv2d_desc* desc, const void* x, const void* w, void* y, void* workspace,
                             size_t workspace_bytes_, long long limit_clocks, void* stream) {
    if (!workspace || workspace_bytes_ < WS_HEADER) { set_error("the self-test needs a workspace"); return PCB_ERR_WORKSPACE; }
    if (limit_clocks < 1 || limit_clocks > (1ll << 24)) { set_error("limit_clocks must be in [1, 2^24]"); return PCB_ERR_INVALID_ARGUMENT; }
    int rc = reset_status(workspace, workspace_bytes_, (cudaStream_t)stream);
    if (rc != PCB_OK) return rc;
    wait_expiry_kernel<<<1, 32, 0, (cudaStream_t)stream>>>(status_of(workspace), limit_clocks);
    PCB_CUDA_TRY(cudaGetLastError());
    // a further launch of the same call: it must leave the recorded expiry in place
    if (desc) rc = conv_fwd(desc, x, w, nullptr, y, workspace, workspace_bytes_, (cudaStream_t)stream);
    return rc;
}

int pcb_set_status_word(const void* workspace, void* word) {
    if (!workspace) { set_error("null workspace"); return PCB_ERR_INVALID_ARGUMENT; }
    if (reinterpret_cast<uintptr_t>(word) % sizeof(int) != 0) { set_error("a status word must be 4-byte aligned"); return PCB_ERR_INVALID_ARGUMENT; }
    std::lock_guard<std::mutex> lock(g_word_mutex);
    if (word) g_words[workspace] = static_cast<int*>(word);
    else g_words.erase(workspace);
    g_word_count.store((int)g_words.size(), std::memory_order_release);
    return PCB_OK;
}

int pcb_check_device_status(const void* workspace, size_t workspace_bytes_, void* stream) {
    if (!workspace || workspace_bytes_ < sizeof(int)) return PCB_OK;
    int word = 0;
    PCB_CUDA_TRY(cudaMemcpyAsync(&word, status_of(workspace), sizeof(int), cudaMemcpyDeviceToHost, (cudaStream_t)stream));
    PCB_CUDA_TRY(cudaStreamSynchronize((cudaStream_t)stream));
    if (word != 0) {
        set_error("device-side wait expired (status word 0x%08x)", word);
        return PCB_ERR_DEVICE_TIMEOUT;
    }
    return PCB_OK;
}

size_t pcb_filter8_values_size(const pcb_dense_desc* desc) {
    Geom g;
    if (dense8_geom(desc, g) != PCB_OK) return 0;
    return q8_value_bytes(g.nc, g.w_io ? g.Ci : g.Co, g.w_io ? g.Co : g.Ci);
}
size_t pcb_filter8_scales_size(const pcb_dense_desc* desc) {
    Geom g;
    if (dense8_geom(desc, g) != PCB_OK) return 0;
    return (size_t)g.nc * q8_blocks(g.Ci) * q8_blocks(g.Co);
}
int pcb_quantize_filter8(const pcb_dense_desc* desc, const void* w, void* values, void* scales, void* stream) {
    Geom g;
    int rc = dense8_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (!w || !values || !scales) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    if ((rc = dense8_check_filter(values)) != PCB_OK) return rc;
    return q8_quantize_blocks(desc->dtype, g.nc, g.w_io ? g.Ci : g.Co, g.w_io ? g.Co : g.Ci, w, static_cast<uint8_t*>(values), static_cast<uint8_t*>(scales),
                              (cudaStream_t)stream);
}
size_t pcb_qdense8_fwd_workspace_size(const pcb_dense_desc* desc) {
    Geom g;
    return dense8_geom(desc, g) == PCB_OK ? dense8_space(g, false, false).total : 0;
}
size_t pcb_qdense8_bwd_workspace_size(const pcb_dense_desc* desc) {
    Geom g;
    return dense8_geom(desc, g) == PCB_OK ? dense8_space(g, true, desc->require_input_grad != 0).total : 0;
}
int pcb_qdense8_form_for(const pcb_dense_desc* desc, int pass) {
    Geom g;
    const int rc = dense8_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (pass < 0 || pass > 2 || (pass == 1 && !desc->require_input_grad)) { set_error("pass must be 0, 2 or, with an input gradient, 1"); return PCB_ERR_INVALID_ARGUMENT; }
    if (g.Nb == 0) { set_error("no samples: nothing is launched"); return PCB_ERR_INVALID_ARGUMENT; }
    auto sizes = [&](Pass p) { return dense8_product(g, p, Q8Operand{}, Q8Operand{}, nullptr, desc->dtype, nullptr); };
    if (pass != 0 && desc->require_input_grad && q8_together(g, sizes(PASS_BWD_FILTER), sizes(PASS_BWD_DATA))) return PCB_DENSE8_BOTH_GRADIENTS;
    int splits;
    return q8_form(g, sizes(pass == 0 ? PASS_FWD : (pass == 1 ? PASS_BWD_DATA : PASS_BWD_FILTER)), &splits);
}
int pcb_qdense8_fwd(const pcb_dense_desc* desc, const void* x, const void* w8, const void* w8_scales, const void* bias, void* y, void* workspace,
                    size_t workspace_bytes_, void* stream) {
    Geom g;
    int rc = dense8_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (g.Nb == 0) return PCB_OK;
    if (!x || !w8 || !w8_scales || !y || (g.has_bias && !bias)) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    const Dense8Space at = dense8_space(g, false, false);
    if ((rc = dense8_workspace(workspace, workspace_bytes_, at.total)) != PCB_OK || (rc = dense8_check_filter(w8)) != PCB_OK) return rc;
    const size_t size = dtype_size(desc->dtype);
    if (overlaps(y, (size_t)g.nc * g.Nb * g.Co * size, x, (size_t)g.nc * g.Nb * g.Ci * size)) { set_error("y must not share memory with x"); return PCB_ERR_INVALID_ARGUMENT; }
    forget_kept(workspace);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    int* status = status_of(workspace);
    const Q8Target rows = {ws + at.x_rows, reinterpret_cast<uint32_t*>(ws + at.x_words)};
    const bool raw = q8_raw_tokens(g.Nb);
    if (!raw && (rc = q8_quantize_rows(desc->dtype, g.nc, g.Nb, g.Ci, x, rows, status, (cudaStream_t)stream)) != PCB_OK) return rc;
    const Q8Operand tokens = {rows.values, rows.words, q8_pitch(g.Ci), 0, 0, 0, 0}, filter = dense8_filter(g, w8, w8_scales, true);
    Q8Product q = dense8_product(g, PASS_FWD, tokens, filter, y, desc->dtype, status);
    if (g.has_bias) q.bias = bias;
    if (raw) q.tokens = x;
    return q8_product(g, q, (cudaStream_t)stream);
}
int pcb_qdense8_bwd(const pcb_dense_desc* desc, const void* x, const void* w8, const void* w8_scales, const void* dy, void* dw, void* dx, void* workspace,
                    size_t workspace_bytes_, void* stream) {
    Geom g;
    int rc = dense8_geom(desc, g);
    if (rc != PCB_OK) return rc;
    if (!dw) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    if (g.Nb == 0) {
        PCB_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)g.nc * g.Co * g.Ci * dtype_size(desc->dtype), (cudaStream_t)stream));
        return PCB_OK;
    }
    const bool need_dx = desc->require_input_grad != 0;
    if (!x || !dy || (need_dx && (!dx || !w8 || !w8_scales))) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    const Dense8Space at = dense8_space(g, true, need_dx);
    if ((rc = dense8_workspace(workspace, workspace_bytes_, at.total)) != PCB_OK || (need_dx && (rc = dense8_check_filter(w8)) != PCB_OK)) return rc;
    forget_kept(workspace);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    int* status = status_of(workspace);
    const cudaStream_t st = (cudaStream_t)stream;
    const Q8Target dy_rows = {need_dx ? ws + at.dy_rows : nullptr, reinterpret_cast<uint32_t*>(ws + at.dy_row_words)};
    const Q8Target dy_cols = {ws + at.dy_cols, reinterpret_cast<uint32_t*>(ws + at.dy_col_words)};
    const Q8Target x_cols = {ws + at.x_cols, reinterpret_cast<uint32_t*>(ws + at.x_col_words)};
    if ((rc = q8_quantize_backward(desc->dtype, g.nc, g.Nb, g.Ci, g.Co, x, dy, x_cols, dy_rows, dy_cols, status, st)) != PCB_OK) return rc;
    const Q8Operand a = {x_cols.values, x_cols.words, q8_pitch(g.Ci), 0, 0, 0, 1}, b = {dy_cols.values, dy_cols.words, q8_pitch(g.Co), 0, 0, 0, 1};
    const Q8Product of_filter = dense8_product(g, PASS_BWD_FILTER, a, b, dw, desc->dtype, status);
    if (!need_dx) return q8_product(g, of_filter, st);
    const Q8Operand tokens = {dy_rows.values, dy_rows.words, q8_pitch(g.Co), 0, 0, 0, 0}, filter = dense8_filter(g, w8, w8_scales, false);
    const Q8Product q = dense8_product(g, PASS_BWD_DATA, tokens, filter, dx, desc->dtype, status);
    return q8_two_products(g, of_filter, q, st);
}

}  // extern "C"
