// The gradients' kernels of bf16 (token_scan_bwd.h), in a source of their own: they take a minute to compile.
#include "token_scan_bwd.h"

namespace ss2d {
template int ts_bwd_run<bf16_t>(const ss2d_token_scan_bwd_params *p, const TsBwdArgs &q, hipStream_t st);
}  // namespace ss2d
