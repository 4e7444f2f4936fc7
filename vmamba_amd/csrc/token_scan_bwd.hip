// Gradients of the selective scan of token sequences: the C entries (kernels in token_scan_bwd.h).
#include "token_scan.h"

namespace ss2d {

// ---- host ------------------------------------------------------------------------------------------------------------------------
int ts_read(const ss2d_token_scan_params *p, TsArgs &a);
int ts_copy(const float *from, float *to, int64_t n, hipStream_t st);

static int ts_bwd_read(const ss2d_token_scan_bwd_params *p, TsBwdArgs &q) {
    q = {};
    if (!p) return SS2D_EINVAL;
    const int rc = ts_read(&p->fwd, q.f);
    if (rc != SS2D_OK) return rc;
    TsArgs &a = q.f;
    q.dout = p->dout; q.dfinal = p->dfinal_state; q.du = p->du; q.ddelta = p->ddelta; q.dz = p->dz; q.dinitial = p->dinitial_state;
    q.do_b = p->dout_batch_stride; q.do_t = p->dout_token_stride;
    a.near = a.near && q.do_t >= 0 && q.do_t < 1 << 24;
    if (a.dim == 0 || a.tokens == 0) return SS2D_OK;
    const int ch = kWave / (a.N <= 4 ? 1 : a.N <= 8 ? 2 : 4) * (a.N <= 32 ? kTsBwdWaves<1> : kTsBwdWaves<4>);
    a.wgs = (a.per_group + ch - 1) / ch;
    // Segments: two workgroups to a CU are what the gradients' registers leave room for, so that their rounds are of 512, and what is handed from one segment to the next
    // costs a fifth of what goes into it.  (4 x 2048 tokens of 2048 channels, forward and gradients: 4 segments 414 us, 6 474, 7 460, 8 422; 8 x 784 of 768, 8 states: 4 205, 6 179, 7 161, 13 166.)
    const int64_t wgs = (int64_t)a.batch * a.groups * a.wgs, most = (a.tokens + (int64_t)kTsGrid - 1) / kTsGrid;
    int64_t n = 1;
    double least = 0;
    for (int64_t k = 1; k <= most && k <= 512 && (k == 1 || wgs * (k - 1) < 4096); ++k) {
        const double cost = (double)((wgs * k + 511) / 512) / (double)k * (1.0 + 0.2 * (double)(k - 1) / (double)k);
        if (k == 1 || cost < 0.99 * least) { least = cost; n = k; }
    }
    a.seg_len = ts_seg_len(a.tokens, n, a.keep);
    a.n_segs = (int)((a.tokens + (int64_t)a.seg_len - 1) / a.seg_len);
    if (wgs * a.n_segs > kTsLaunch / kBlock || (a.n_segs > 1 && a.batch > 65535) || !ts_sums_fit(a)) return SS2D_ENOTSUP;
    // What is handed from behind keeps fewer registers: as many workgroups, of four wavefronts always, as come to four on a CU (4 x 2048 tokens of 2048 channels: 768 in place
    // of 384, 59 -> 42 us)
    const int left_ch = kWave / ts_sets(a.N) * kWavesPerWg;
    q.left_wgs = (a.per_group + left_ch - 1) / left_ch;
    const auto slots = [&](int each) { return (int)((a.tokens + (int64_t)a.seg_len / each - 1) / (a.seg_len / each)) - each; };
    q.each = 1;
    while (a.n_segs > 1 && a.seg_len % (2 * q.each * kTsTile) == 0 && a.seg_len / (2 * q.each) >= kTsGrid && (int64_t)a.batch * a.groups * q.left_wgs * slots(2 * q.each) <= 1024) q.each *= 2;
    q.slots = a.n_segs > 1 ? slots(q.each) : 0;
    return SS2D_OK;
}

static int64_t ts_bwd_carve(TsBwdArgs &q, uint8_t *base) {
    const TsArgs &a = q.f;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { uint8_t *p = base ? base + at : nullptr; at += (bytes + 255) / 256 * 256; return p; };
    const int64_t cuts = (int64_t)a.batch * q.slots, parts = (int64_t)a.batch * a.n_segs, states = (int64_t)a.dim * a.N;
    q.left = (float *)take(cuts * states * 4);
    q.behind = (float *)take(cuts * states * 4);
    q.gsums = (float *)take(cuts * a.dim * 4);
    q.gflags = (int32_t *)take(cuts * 4);
    q.pBC = (float *)take((int64_t)a.wgs * a.batch * a.tokens * a.groups * a.N * 8);
    q.pA = (float *)take(parts * states * 4);
    q.pD = (float *)take(parts * 2 * a.dim * 4);
    return at;
}

template <typename T> int ts_bwd_run(const ss2d_token_scan_bwd_params *p, const TsBwdArgs &q, hipStream_t st);

}  // namespace ss2d

using namespace ss2d;

extern "C" int64_t ss2d_token_scan_bwd_workspace_bytes(const ss2d_token_scan_bwd_params *params) {
    TsBwdArgs q;
    const int rc = ts_bwd_read(params, q);
    if (rc != SS2D_OK) return rc;
    return q.f.dim && q.f.batch && q.f.tokens ? ts_bwd_carve(q, nullptr) : 0;
}

extern "C" int ss2d_token_scan_bwd(const ss2d_token_scan_bwd_params *params, void *workspace, int64_t workspace_bytes, void *stream) {
    TsBwdArgs q;
    const int rc = ts_bwd_read(params, q);
    if (rc != SS2D_OK) return rc;
    const TsArgs &a = q.f;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (a.dim == 0) return SS2D_OK;
    if (a.batch == 0 || a.tokens == 0) {                             // no tokens: the weights' gradients are zeros, the states' what came in
        for (const auto &[to, n] : {std::pair<float *, int64_t>{params->dA, (int64_t)a.dim * a.N}, {params->dD, a.dim}, {params->ddelta_bias, a.dim}}) {
            const int status = ts_copy(nullptr, to, n, st);
            if (status != SS2D_OK) return status;
        }
        return ts_copy(q.dfinal, q.dinitial, (int64_t)a.n_seqs * a.dim * a.N, st);
    }
    if (!a.u || !a.delta || !a.A || !a.B || !a.C || !q.dout || !a.kept || !q.du || !q.ddelta || !params->dB || !params->dC || (a.z && !q.dz)) return SS2D_EINVAL;
    const int64_t need = ts_bwd_carve(q, (uint8_t *)workspace);
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16) return SS2D_EINVAL;
    if (workspace_bytes < need) return SS2D_ENOMEM;
    switch (params->fwd.dtype) {
    case SS2D_F32: return ts_bwd_run<float>(params, q, st);
    case SS2D_F16: return ts_bwd_run<f16_t>(params, q, st);
    default: return ts_bwd_run<bf16_t>(params, q, st);
    }
}
