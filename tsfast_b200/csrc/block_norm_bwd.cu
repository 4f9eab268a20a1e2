// Adjoint of the block norms: rows on 16-byte boundaries, and the C entry points.
#include "block_norm_bwd.cuh"

namespace b200 {
namespace norm {
int bwd_aligned(const Args& p, const Sums& o, int dtype, bool layer, bool post, bool res, cudaStream_t st) { return bwd_of<true>(p, o, dtype, layer, post, res, st); }
}  // namespace norm
}  // namespace b200

extern "C" {

size_t b200_block_norm_bwd_workspace_bytes(int64_t M, int64_t D, int kind) {
    using namespace b200::norm;
    if (M <= 0 || D < 1 || D > kMaxWidth) return 256;
    return b200::align_up((size_t)grid_of(M, (int)D) * (kind == 1 ? 5 : 3) * (size_t)D * 4, 256);
}

int b200_block_norm_bwd(int dtype, int64_t M, int64_t D, int kind, int act, float eps, int params_f32, const void* gy, int64_t ldgy,
                        const void* gres, int64_t ldgr, const void* x, int64_t ldx, const void* gate, int64_t ldg, const void* residual,
                        int64_t ldr, const void* w1, const void* b1, const void* scale, const void* w2, const void* b2, const void* stats,
                        void* gx, void* ggate, void* gresidual, void* gw1, void* gb1, void* gscale, void* gw2, void* gb2, void* workspace,
                        size_t workspace_bytes, void* stream) {
    using namespace b200;
    using namespace b200::norm;
    if (D > kMaxWidth) return B200_ERR_UNSUPPORTED;
    Args p = {};
    p.M = M, p.D = (int)D, p.x = x, p.ldx = ldx, p.gate = act == kActNone ? nullptr : gate, p.ldg = ldg, p.res = residual, p.ldr = ldr;
    p.par[kGW1] = w1, p.par[kGB1] = b1, p.par[kGScale] = scale, p.par[kGW2] = w2, p.par[kGB2] = b2, p.pf32 = params_f32, p.act = act, p.eps = eps;
    p.gy = gy, p.ldgy = ldgy, p.gres = gres, p.ldgr = ldgr, p.gx = gx, p.ggate = act == kActNone ? nullptr : ggate, p.gresid = gresidual;
    p.stats = (float*)const_cast<void*>(stats), p.part = (float*)workspace;
    const bool res = w2 != nullptr;
    const int rc = check(p, dtype, kind, res);
    if (rc != B200_OK) return rc;
    if (kind == 0 && (gb1 || gb2)) return B200_ERR_ARG;
    if ((gw1 && !w1) || (gb1 && !w1) || (gscale && !scale) || ((gw2 || gb2) && !res) || (ggate && !gate)) return B200_ERR_ARG;
    if (!on_boundary(params_f32 ? 4 : block_elem_size(dtype), gw1, gb1, gscale, gw2, gb2) || !on_boundary(block_elem_size(dtype), ggate)) return B200_ERR_ARG;
    if (M > 0 && (!x || !gy || !stats || (res && (!residual || !gresidual)))) return B200_ERR_ARG;
    if (M > 0 && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < b200_block_norm_bwd_workspace_bytes(M, D, kind)))
        return B200_ERR_WORKSPACE;
    const int e = block_elem_size(dtype);
    const bool al = set_shape(p, e);
    Sums o = {};
    o.out[kGW2] = gw2, o.out[kGScale] = gscale, o.out[kGW1] = gw1, o.out[kGB2] = gb2, o.out[kGB1] = gb1, o.f32 = params_f32;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // a gate that is not used has the gradient zero
    if (act == kActNone && ggate && M > 0 && cudaMemsetAsync(ggate, 0, (size_t)M * D * e, st) != cudaSuccess) return B200_ERR_LAUNCH;
    return al ? bwd_aligned(p, o, dtype, kind == 1, w1 != nullptr, res, st) : bwd_unaligned(p, o, dtype, kind == 1, w1 != nullptr, res, st);
}

}  // extern "C"
