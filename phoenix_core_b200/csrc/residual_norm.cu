// C entry points of the norms before and after a residual block (formulas and kernels: residual_norm.cuh).
#include "residual_norm.h"

namespace pcb {
namespace {

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
// No result may lie where an operand or another result does: rows are read ahead of those that are written.
struct Span { const void* at; size_t bytes; };
int check_apart(const Span* results, int n, const Span* operands, int m) {
    for (int i = 0; i < n; ++i) {
        if (!results[i].at) continue;
        for (int k = 0; k < m + i; ++k) {
            const Span& o = k < m ? operands[k] : results[k - m];
            if (o.at && overlaps(results[i].at, results[i].bytes, o.at, o.bytes)) { set_error("a result shares memory with another tensor of the call"); return PCB_ERR_INVALID_ARGUMENT; }
        }
    }
    return PCB_OK;
}
int norm_comps(const pcb_norm_desc* d) { Geom g = {}; algebra_setup(d->algebra, g); return g.nc; }

RNParams norm_params(const pcb_norm_desc* d) {
    RNParams p = {};
    p.comps = norm_comps(d); p.n = d->batch; p.features = d->features;
    p.groups = d->gate_rows; p.per_group = d->gate_rows > 0 ? d->batch / d->gate_rows : d->batch;
    p.scale = d->residual_scale; p.eps = d->epsilon;
    return p;
}
}  // namespace
}  // namespace pcb

using namespace pcb;

extern "C" {

size_t pcb_residual_norm_bwd_workspace_size(const pcb_norm_desc* d) {
    if (check_norm(d) != PCB_OK || d->batch == 0) return 0;
    return WS_HEADER + bwd_plan(norm_comps(d), d->batch, d->features, d->gate_rows, (int)dtype_size(d->dtype)).total;
}

int pcb_residual_norm_fwd(const pcb_norm_desc* d, const void* x, const void* branch, const void* gate, const float* post, const float* pre, void* y, void* h,
                          float* stats, void* stream) {
    const int rc = check_norm(d);
    if (rc != PCB_OK || d->batch == 0) return rc;
    if (!x || (branch && !y) || (!y && !h)) { set_error("null tensor pointer"); return PCB_ERR_INVALID_ARGUMENT; }
    if ((gate != nullptr) != (d->gate_rows > 0) || (!branch && (gate || post)) || (!h && pre)) { set_error("gate or weights without what they apply to"); return PCB_ERR_INVALID_ARGUMENT; }
    RNParams p = norm_params(d);
    const size_t size = dtype_size(d->dtype), row = (size_t)p.comps * d->batch * d->features * size, gates = (size_t)p.comps * d->gate_rows * d->features * size, weight = (size_t)d->features * 4;
    const Span results[] = {{y, row}, {h, row}, {stats, (size_t)d->batch * 8}}, operands[] = {{x, row}, {branch, row}, {gate, gates}, {post, weight}, {pre, weight}};
    if (const int apart = check_apart(results, 3, operands, 5)) return apart;
    p.x = x; p.branch = branch; p.gate = gate; p.post = post; p.pre = pre; p.y = y; p.h = h; p.stats = stats;
    const cudaStream_t s = (cudaStream_t)stream;
    if (d->dtype == PCB_F32) return norm_fwd_f32(p, s);
    return d->dtype == PCB_F16 ? norm_fwd_f16(p, s) : norm_fwd_bf16(p, s);
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
    const RNPlan q = bwd_plan(comps, d->batch, d->features, d->gate_rows, (int)dtype_size(d->dtype));
    const size_t need = WS_HEADER + q.total;
    if (!workspace || workspace_bytes < need) { set_error("workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need); return PCB_ERR_WORKSPACE; }
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) { set_error("the workspace must be 16-byte aligned"); return PCB_ERR_INVALID_ARGUMENT; }
    RNParams p = norm_params(d);
    const size_t size = dtype_size(d->dtype), row = (size_t)comps * d->batch * d->features * size, gates = (size_t)comps * d->gate_rows * d->features * size, weight = (size_t)d->features * 4;
    const Span results[] = {{dx, row}, {dbranch, branch ? row : 0}, {dgate, gates}, {dpost, weight}, {dpre, weight}, {workspace, need}};
    const Span operands[] = {{dh ? y : nullptr, row}, {branch, row}, {gate, gates}, {post, weight}, {pre, weight}, {stats, (size_t)d->batch * 8}, {dy, row}, {dh, row}};
    if (const int apart = check_apart(results, 6, operands, 8)) return apart;
    p.branch = branch; p.gate = gate; p.post = post; p.pre = pre; p.y = const_cast<void*>(y); p.stats = const_cast<float*>(stats);
    p.dy = dy; p.dh = dh; p.dx = dx; p.dbranch = dbranch; p.dgate = dgate; p.dpost = dpost; p.dpre = dpre;
    forget_kept(workspace);
    p.workspace = static_cast<uint8_t*>(workspace) + WS_HEADER;
    p.status = status_of(workspace);
    if (!gate) p.per_group = d->batch;
    if (d->dtype == PCB_F32) return norm_bwd_f32(p, q, s);
    return d->dtype == PCB_F16 ? norm_bwd_f16(p, q, s) : norm_bwd_bf16(p, q, s);
}

}  // extern "C"
