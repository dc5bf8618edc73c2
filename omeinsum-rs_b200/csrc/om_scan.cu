// Gated linear recurrence h_t = a_t h_{t-1} + b_t and its backward pass.
#include <algorithm>

#include "om_convert.cuh"

namespace om {
namespace {

struct ScanArgs {
  int64_t D, T, B;
  const void* gate;
  int64_t gd, gt, gb;
  const void* x;
  int64_t xd, xt, xb;
  const void* h0;
  const int32_t* lengths;
  void* h;
  int64_t hd, ht, hb;
  void* h_last;
  // backward only
  const void* dh;
  int64_t ed, et, eb;
  const void* dh_last;
  void* dgate;
  int64_t pd, pt, pb;
  void* dx;
  int64_t qd, qt, qb;
  void* dh0;
};

// a = sigmoid(g) and 1 - a without cancellation on either side
template <typename S>
__device__ __forceinline__ void sigmoid_pair(S g, S* a, S* keep) {
  const S e = exp(-fabs(g));
  const S r = S(1) / (S(1) + e);
  *a = g >= 0 ? r : e * r;
  *keep = g >= 0 ? e * r : r;
  if (g != g) *a = *keep = g;
}

// One thread per channel, step by step.
template <typename T, bool SIG>
__global__ void scan_forward(ScanArgs p) {
  using S = typename Elem<T>::State;
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= p.D * p.B) return;
  const int64_t d = i % p.D, b = i / p.D;
  int64_t len = p.T;
  if (p.lengths) len = min(max((int64_t)p.lengths[b], (int64_t)0), p.T);
  const T* g = (const T*)p.gate + d * p.gd + b * p.gb;
  const T* x = (const T*)p.x + d * p.xd + b * p.xb;
  T* h = (T*)p.h + d * p.hd + b * p.hb;
  S s = p.h0 ? ((const S*)p.h0)[i] : S(0);
  for (int64_t t = 0; t < len; ++t) {
    S a = Elem<T>::load(g[t * p.gt]), v = Elem<T>::load(x[t * p.xt]);
    if constexpr (SIG) {
      S keep;
      sigmoid_pair(a, &a, &keep);
      v *= keep;
    }
    s = a * s + v;
    h[t * p.ht] = Elem<T>::store(s);
  }
  for (int64_t t = len; t < p.T; ++t) h[t * p.ht] = Elem<T>::store(S(0));
  if (p.h_last) ((S*)p.h_last)[i] = s;
}

template <typename T, bool SIG>
__global__ void scan_backward(ScanArgs p) {
  using S = typename Elem<T>::State;
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= p.D * p.B) return;
  const int64_t d = i % p.D, b = i / p.D;
  int64_t len = p.T;
  if (p.lengths) len = min(max((int64_t)p.lengths[b], (int64_t)0), p.T);
  const T* g = (const T*)p.gate + d * p.gd + b * p.gb;
  const T* x = (const T*)p.x + d * p.xd + b * p.xb;
  const T* h = (const T*)p.h + d * p.hd + b * p.hb;
  const T* e = (const T*)p.dh + d * p.ed + b * p.eb;
  T* dg = (T*)p.dgate + d * p.pd + b * p.pb;
  T* dx = (T*)p.dx + d * p.qd + b * p.qb;
  const S start = p.h0 ? ((const S*)p.h0)[i] : S(0);
  S carry = p.dh_last ? ((const S*)p.dh_last)[i] : S(0);  // a_{t+1} G_{t+1}
  for (int64_t t = p.T - 1; t >= len; --t) {
    dg[t * p.pt] = Elem<T>::store(S(0));
    dx[t * p.qt] = Elem<T>::store(S(0));
  }
  for (int64_t t = len - 1; t >= 0; --t) {
    S a = Elem<T>::load(g[t * p.gt]);
    const S total = Elem<T>::load(e[t * p.et]) + carry;
    const S before = t ? (S)Elem<T>::load(h[(t - 1) * p.ht]) : start;
    S sx = total, sg = total * before;
    if constexpr (SIG) {
      S keep;
      sigmoid_pair(a, &a, &keep);
      sx = total * keep;
      sg = total * (before - Elem<T>::load(x[t * p.xt])) * (a * keep);
    }
    dx[t * p.qt] = Elem<T>::store(sx);
    dg[t * p.pt] = Elem<T>::store(sg);
    carry = a * total;
  }
  if (p.dh0) ((S*)p.dh0)[i] = carry;
}

template <typename T, bool SIG>
int launch_scan(om_backend* be, const ScanArgs& p, bool backward) {
  const int64_t n = p.D * p.B;
  const int64_t blocks = (n + 127) / 128;
  if (blocks > 0x7fffffff) return set_error(OM_ERR_INVALID, "gated_scan: too many channels");
  ProfScope prof(be, backward ? "gated_scan_backward" : "gated_scan");
  if (backward)
    scan_backward<T, SIG><<<(unsigned)blocks, 128, 0, be->stream>>>(p);
  else
    scan_forward<T, SIG><<<(unsigned)blocks, 128, 0, be->stream>>>(p);
  note_launch();
  return check_cuda(cudaGetLastError(), "gated_scan launch");
}

template <typename T>
int launch_scan_kind(om_backend* be, om_gate kind, const ScanArgs& p, bool backward) {
  return kind == OM_GATE_SIGMOID ? launch_scan<T, true>(be, p, backward)
                                 : launch_scan<T, false>(be, p, backward);
}

int dispatch_scan(om_backend* be, om_gate kind, om_dtype dtype, const ScanArgs& p, bool backward) {
  DeviceGuard guard(be->device);
  OM_CUDA(guard.status, "gated_scan: device");
  switch (dtype) {
    case OM_F32: return launch_scan_kind<float>(be, kind, p, backward);
    case OM_F64: return launch_scan_kind<double>(be, kind, p, backward);
    case OM_BF16: return launch_scan_kind<__nv_bfloat16>(be, kind, p, backward);
    case OM_F16: return launch_scan_kind<__half>(be, kind, p, backward);
    default: return set_error(OM_ERR_UNSUPPORTED, "gated_scan: dtype must be f32, f64, bf16 or f16");
  }
}

int check_scan(const char* who, om_backend* be, om_gate kind, om_dtype dtype, const int64_t* shape) {
  const std::string w(who);
  if (!be || !shape) return set_error(OM_ERR_INVALID, w + ": null argument");
  if (kind != OM_GATE_LINEAR && kind != OM_GATE_SIGMOID)
    return set_error(OM_ERR_INVALID, w + ": unknown gate kind");
  if (dtype != OM_F32 && dtype != OM_F64 && !is_half(dtype))
    return set_error(OM_ERR_UNSUPPORTED, w + ": dtype must be f32, f64, bf16 or f16");
  for (int k = 0; k < 3; ++k)
    if (shape[k] < 0) return set_error(OM_ERR_SHAPE, w + ": negative extent");
  return OM_OK;
}

}  // namespace
}  // namespace om

using namespace om;

extern "C" int om_b200_gated_scan(om_backend* be, om_gate kind, om_dtype dtype,
                                  const int64_t* shape, const void* gate,
                                  const int64_t* strides_gate, const void* x,
                                  const int64_t* strides_x, const void* h0, const int32_t* lengths,
                                  void* h, const int64_t* strides_h, void* h_last) {
  OM_TRY(check_scan("om_b200_gated_scan", be, kind, dtype, shape));
  const bool steps = shape[0] && shape[1] && shape[2];
  if (steps && (!gate || !x || !h || !strides_gate || !strides_x || !strides_h))
    return set_error(OM_ERR_INVALID, "om_b200_gated_scan: null argument");
  if (shape[0] == 0 || shape[2] == 0) return OM_OK;
  ScanArgs p{};
  p.D = shape[0], p.T = shape[1], p.B = shape[2];
  if (steps) {
    p.gate = gate, p.gd = strides_gate[0], p.gt = strides_gate[1], p.gb = strides_gate[2];
    p.x = x, p.xd = strides_x[0], p.xt = strides_x[1], p.xb = strides_x[2];
    p.h = h, p.hd = strides_h[0], p.ht = strides_h[1], p.hb = strides_h[2];
  }
  p.h0 = h0, p.lengths = lengths, p.h_last = h_last;
  return dispatch_scan(be, kind, dtype, p, false);
}

extern "C" int om_b200_gated_scan_backward(
    om_backend* be, om_gate kind, om_dtype dtype, const int64_t* shape, const void* gate,
    const int64_t* strides_gate, const void* x, const int64_t* strides_x, const void* h,
    const int64_t* strides_h, const void* h0, const int32_t* lengths, const void* dh,
    const int64_t* strides_dh, const void* dh_last, void* dgate, const int64_t* strides_dgate,
    void* dx, const int64_t* strides_dx, void* dh0) {
  OM_TRY(check_scan("om_b200_gated_scan_backward", be, kind, dtype, shape));
  const bool steps = shape[0] && shape[1] && shape[2];
  const bool need_x = kind == OM_GATE_SIGMOID;
  if (steps && (!gate || !h || !dh || !dgate || !dx || !strides_gate || !strides_h || !strides_dh ||
                !strides_dgate || !strides_dx || (need_x && (!x || !strides_x))))
    return set_error(OM_ERR_INVALID, "om_b200_gated_scan_backward: null argument");
  if (shape[0] == 0 || shape[2] == 0) return OM_OK;
  ScanArgs p{};
  p.D = shape[0], p.T = shape[1], p.B = shape[2];
  if (steps) {
    p.gate = gate, p.gd = strides_gate[0], p.gt = strides_gate[1], p.gb = strides_gate[2];
    if (need_x) p.x = x, p.xd = strides_x[0], p.xt = strides_x[1], p.xb = strides_x[2];
    p.h = (void*)h, p.hd = strides_h[0], p.ht = strides_h[1], p.hb = strides_h[2];
    p.dh = dh, p.ed = strides_dh[0], p.et = strides_dh[1], p.eb = strides_dh[2];
    p.dgate = dgate, p.pd = strides_dgate[0], p.pt = strides_dgate[1], p.pb = strides_dgate[2];
    p.dx = dx, p.qd = strides_dx[0], p.qt = strides_dx[1], p.qb = strides_dx[2];
  }
  p.h0 = h0, p.lengths = lengths, p.dh_last = dh_last, p.dh0 = dh0;
  return dispatch_scan(be, kind, dtype, p, true);
}
