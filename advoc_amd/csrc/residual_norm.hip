// C entry points of the residual norm: argument checks and the hand-over to residual_norm_fwd.hip / residual_norm_bwd.hip.
#include "residual_norm.h"

namespace advoc {
bool launch_norm_forward(const NormArgs& a, int dtype, int res_dtype, hipStream_t stream);
int64_t norm_backward_workspace(const NormArgs& a, float* const (&out)[5]);
int clear_norm_sums(int cols, float* const (&out)[5], hipStream_t stream);
int launch_norm_backward(NormArgs a, int dtype, int res_dtype, float* const (&out)[5], int accumulate, void* workspace,
                         int64_t workspace_bytes, hipStream_t stream);
}  // namespace advoc

namespace {

bool norm_kind_ok(int k) { return k == ADVOC_NORM_NONE || k == ADVOC_NORM_RMS || k == ADVOC_NORM_LAYER; }

bool pitch_ok(const advoc_rows& t, const advoc_residual_norm& d) { return !t.p || d.rows <= 1 || t.pitch >= d.cols; }

// what both directions ask of a descriptor
int check(const advoc_residual_norm& d) {
  if (d.rows < 0 || d.cols <= 0) return ADVOC_ERR_BAD_SHAPE;
  if (!(d.eps > 0.f) || !(d.keep_prob > 0.f && d.keep_prob <= 1.f)) return ADVOC_ERR_BAD_SHAPE;
  if (!norm_kind_ok(d.norm_post) || !norm_kind_ok(d.norm_pre)) return ADVOC_ERR_UNSUPPORTED;
  if (d.gate_act != ADVOC_GATE_NONE && d.gate_act != ADVOC_GATE_SIGMOID) return ADVOC_ERR_UNSUPPORTED;
  if (!advoc::dtype_ok(d.dtype) || (d.res_dtype != d.dtype && d.res_dtype != ADVOC_F32)) return ADVOC_ERR_UNSUPPORTED;
  if (d.cols > ADVOC_NORM_MAX_COLS || d.rows > 0x7fffffffLL || (d.offset & 3)) return ADVOC_ERR_UNSUPPORTED;
  if (d.gate.p && (d.gate_group < 1 || d.rows % d.gate_group)) return ADVOC_ERR_BAD_SHAPE;
  if (d.rows > 0 && !d.h.p && (d.norm_post != ADVOC_NORM_NONE || d.gate.p || d.scale)) return ADVOC_ERR_BAD_SHAPE;
  if (d.rows > 0 && !d.h.p && d.norm_pre == ADVOC_NORM_NONE) return ADVOC_ERR_BAD_SHAPE;      // nothing to compute
  if (d.gate.p && d.rows > d.gate_group && d.gate.pitch < d.cols) return ADVOC_ERR_BAD_SHAPE;
  if (!pitch_ok(d.h, d) || !pitch_ok(d.x, d) || !pitch_ok(d.r, d) || !pitch_ok(d.z, d)) return ADVOC_ERR_BAD_SHAPE;
  return ADVOC_OK;
}

advoc::NormArgs device_args(const advoc_residual_norm& d) {
  advoc::NormArgs a = {};
  a.rows = d.rows;
  a.cols = d.cols;
  a.post = d.norm_post;
  a.pre = d.norm_pre;
  a.act = d.gate_act;
  a.gate_group = d.gate.p ? d.gate_group : 1;
  const bool post = d.norm_post != ADVOC_NORM_NONE, pre = d.norm_pre != ADVOC_NORM_NONE;
  a.w_post = post ? d.w_post : nullptr;      // the identity has neither weight nor bias
  a.b_post = post ? d.b_post : nullptr;
  a.scale = d.scale;
  a.w_pre = pre ? d.w_pre : nullptr;
  a.b_pre = pre ? d.b_pre : nullptr;
  a.alpha = d.alpha;
  a.eps = d.eps;
  a.inv_cols = (float)(1.0 / d.cols);
  a.key = advoc::make_drop_key(d.keep_prob, d.seed, d.offset, d.seed_dev);
  a.h = d.h.p;
  a.h_pitch = d.h.pitch;
  a.gate = d.gate.p;
  a.gate_pitch = d.gate.pitch;
  a.stats = reinterpret_cast<float4*>(d.stats);
  return a;
}

// the backward pass's view of a descriptor; `out`: the parameter gradients wanted
int backward_args(const advoc_residual_norm& d, advoc::NormArgs& a, float* (&out)[5]) {
  const int rc = check(d);
  if (rc != ADVOC_OK) return rc;
  if (!pitch_ok(d.dz, d) || !pitch_ok(d.dr, d) || !pitch_ok(d.dh, d) || !pitch_ok(d.dx, d)) return ADVOC_ERR_BAD_SHAPE;
  if (d.dgate.p && d.gate.p && d.rows > d.gate_group && d.dgate.pitch < d.cols) return ADVOC_ERR_BAD_SHAPE;
  a = device_args(d);
  a.x = d.r.p;
  a.x_pitch = d.r.pitch;
  a.dz = d.dz.p;
  a.dz_pitch = d.dz.pitch;
  a.dr = d.dr.p;
  a.dr_pitch = d.dr.pitch;
  a.dh = d.dh.p;
  a.dh_pitch = d.dh.pitch;
  a.dx = d.dx.p;
  a.dx_pitch = d.dx.pitch;
  a.dgate = d.gate.p ? d.dgate.p : nullptr;
  a.dgate_pitch = d.dgate.pitch;
  const bool post = d.norm_post != ADVOC_NORM_NONE, pre = d.norm_pre != ADVOC_NORM_NONE;
  out[0] = post ? d.dw_post : nullptr;
  out[1] = post ? d.db_post : nullptr;
  out[2] = d.h.p ? d.dscale : nullptr;
  out[3] = pre ? d.dw_pre : nullptr;
  out[4] = pre ? d.db_pre : nullptr;
  return ADVOC_OK;
}

}  // namespace

extern "C" int advoc_residual_norm_forward(const advoc_residual_norm* desc, advoc_stream_t stream) {
  if (!desc) return ADVOC_ERR_NULL;
  const advoc_residual_norm& d = *desc;
  const int rc = check(d);
  if (rc != ADVOC_OK) return rc;
  if (d.rows == 0) return ADVOC_OK;
  if (!d.x.p || (d.h.p && !d.r.p) || (d.norm_pre != ADVOC_NORM_NONE && !d.z.p)) return ADVOC_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(d.stats) & 15) return ADVOC_ERR_UNSUPPORTED;
  advoc::NormArgs a = device_args(d);
  a.x = d.x.p;
  a.x_pitch = d.x.pitch;
  a.r = d.r.p;
  a.r_pitch = d.r.pitch;
  a.z = d.z.p;
  a.z_pitch = d.z.pitch;
  ADVOC_CLEAR_LAUNCH_ERROR();
  if (!advoc::launch_norm_forward(a, d.dtype, d.res_dtype, advoc::as_stream(stream))) return ADVOC_ERR_UNSUPPORTED;
  ADVOC_RETURN_IF_LAUNCH_FAILED();
  return ADVOC_OK;
}

extern "C" int64_t advoc_residual_norm_workspace_bytes(const advoc_residual_norm* desc) {
  advoc::NormArgs a;
  float* out[5];
  if (!desc || desc->rows == 0 || backward_args(*desc, a, out) != ADVOC_OK) return 0;
  return advoc::norm_backward_workspace(a, out);
}

extern "C" int advoc_residual_norm_backward(const advoc_residual_norm* desc, advoc_stream_t stream) {
  if (!desc) return ADVOC_ERR_NULL;
  const advoc_residual_norm& d = *desc;
  advoc::NormArgs a;
  float* out[5];
  const int rc = backward_args(d, a, out);
  if (rc != ADVOC_OK) return rc;
  if (d.rows == 0) {
    out[2] = d.dscale;                         // (a tensor of no rows has no address: h may be there all the same)
    return d.accumulate ? ADVOC_OK : advoc::clear_norm_sums(d.cols, out, advoc::as_stream(stream));
  }
  const bool post = d.norm_post != ADVOC_NORM_NONE, pre = d.norm_pre != ADVOC_NORM_NONE;
  if ((pre && (!d.dz.p || !d.r.p)) || (!pre && !d.dr.p) || ((pre || post) && !d.stats)) return ADVOC_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(d.stats) & 15) return ADVOC_ERR_UNSUPPORTED;
  if (d.workspace_bytes > 0 && !d.workspace) return ADVOC_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(d.workspace) & 3) return ADVOC_ERR_UNSUPPORTED;
  return advoc::launch_norm_backward(a, d.dtype, d.res_dtype, out, d.accumulate, d.workspace,
                                     d.workspace ? d.workspace_bytes : 0, advoc::as_stream(stream));
}
