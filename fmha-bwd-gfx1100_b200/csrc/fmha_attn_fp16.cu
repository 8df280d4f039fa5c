// The fp16 attention entries of libfmha_bwd_fp16.so (include/fmha_bwd.h).
#include "fmha_attn_launch.cuh"

#define FMHA_API __attribute__((visibility("default")))

using fmha_sm100::AttnOp;

extern "C" {

FMHA_API int fmha_cross_fp16_fwd(const fmha_attn_t* args, fmha_stream_t stream) {
  return fmha_sm100::run_attn<__half>(args, AttnOp::kCrossFwd, stream);
}

FMHA_API int fmha_cross_fp16_bwd(const fmha_attn_t* args, fmha_stream_t stream) {
  return fmha_sm100::run_attn<__half>(args, AttnOp::kCrossBwd, stream);
}

FMHA_API int fmha_prefix_fp16_attn(const fmha_attn_t* args, fmha_stream_t stream) {
  return fmha_sm100::run_attn<__half>(args, AttnOp::kPrefix, stream);
}

FMHA_API int fmha_attn_workspace(const fmha_attn_t* args, int op, uint64_t* bytes) {
  using namespace fmha_sm100;
  if (!args || !bytes) return set_error(kErrInvalidArgument, "null argument");
  if (op < FMHA_ATTN_CROSS_FWD || op > FMHA_ATTN_PREFIX) return set_error(kErrInvalidArgument, "unknown operation %d", op);
  return attn_workspace(*args, static_cast<AttnOp>(op), bytes);
}

}  // extern "C"
