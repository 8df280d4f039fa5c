// Host side shared by the attention entries (cross attention to an encoder's
// states, its backward, and attention behind a shared prefix): argument
// checks and the parameter block that the kernels take.
#pragma once

#include "../../include/fmha_bwd.h"
#include "fmha_bwd_launch.cuh"

namespace fmha_sm100 {

// A strided [batch][heads][rows][D] tensor on the device (strides in
// elements, unit stride along D).
template <typename T>
struct View {
  T* p;
  int64_t sb, sh, sr;
  __host__ __device__ __forceinline__ T* at(int b, int h, int64_t row) const {
    return p + b * sb + h * sh + row * sr;
  }
};

template <typename T>
View<T> view_of(const fmha_tensor_t& t) {
  return View<T>{static_cast<T*>(t.ptr), t.batch, t.head, t.row};
}

// One tensor's pointer and strides. Axes of size 1 are never stepped along,
// so their stride (which callers may leave at anything) is set to `row_size`.
inline int check_tensor(fmha_tensor_t& t, const char* name, int batch, int heads, int rows, int D, bool written) {
  if (!t.ptr) return set_error(kErrInvalidArgument, "%s: null pointer", name);
  if (!aligned16(t.ptr)) return set_error(kErrMisaligned, "%s must be 16-byte aligned", name);
  if (batch == 1) t.batch = D;
  if (heads == 1) t.head = D;
  if (rows == 1) t.row = D;
  const int64_t limit = int64_t(1) << 38;  // tensor maps take strides below 2^40 bytes
  for (int64_t s : {t.batch, t.head, t.row}) {
    if (s <= 0 || s >= limit)
      return set_error(kErrInvalidArgument, "%s: stride %lld outside (0, 2^38)", name, static_cast<long long>(s));
    if (s % 8 != 0)
      return set_error(kErrMisaligned, "%s: stride %lld is not a multiple of 8 elements", name,
                       static_cast<long long>(s));
  }
  if (rows > 1 && t.row < D)
    return set_error(kErrInvalidArgument, "%s: rows overlap (row stride %lld, K_dim %d)", name,
                     static_cast<long long>(t.row), D);
  if (written) {
    // outputs must not overlap themselves: along the axes sorted by stride,
    // each stride steps over everything the smaller ones span
    int64_t st[3] = {t.batch, t.head, t.row};
    int n[3] = {batch, heads, rows};
    int64_t span = D;
    for (int i = 0; i < 3; ++i) {
      int best = -1;
      for (int j = 0; j < 3; ++j)
        if (n[j] > 1 && (best < 0 || st[j] < st[best])) best = j;
      if (best < 0) break;
      if (st[best] < span) return set_error(kErrInvalidArgument, "%s: overlapping strides in an output", name);
      span += st[best] * (n[best] - 1);
      n[best] = 1;
    }
  }
  return kOk;
}

enum class AttnOp : int { kCrossFwd = FMHA_ATTN_CROSS_FWD, kCrossBwd = FMHA_ATTN_CROSS_BWD, kPrefix = FMHA_ATTN_PREFIX };

// Sizes only: what fmha_attn_workspace looks at.
inline int check_attn_sizes(const fmha_attn_t& a, AttnOp op) {
  if (a.batch <= 0 || a.q_heads <= 0 || a.kv_heads <= 0 || a.M <= 0 || a.N <= 0)
    return set_error(kErrInvalidArgument, "sizes must be positive (batch=%d q_heads=%d kv_heads=%d M=%d N=%d)", a.batch,
                     a.q_heads, a.kv_heads, a.M, a.N);
  if (a.K_dim != 64 && a.K_dim != 128)
    return set_error(kErrInvalidArgument, "K_dim=%d unsupported (64 or 128)", a.K_dim);
  if (a.q_heads % a.kv_heads != 0)
    return set_error(kErrInvalidArgument, "q_heads=%d is not a multiple of kv_heads=%d", a.q_heads, a.kv_heads);
  if (static_cast<int64_t>(a.batch) * a.q_heads * a.M > (int64_t(1) << 30))
    return set_error(kErrInvalidArgument, "batch * q_heads * M exceeds 2^30 rows");
  if (static_cast<int64_t>(a.batch) * a.kv_heads * ((static_cast<int64_t>(a.N) + 127) / 128) > (int64_t(1) << 30))
    return set_error(kErrInvalidArgument, "batch * kv_heads * N / 128 exceeds 2^30 tiles");
  if (a.M > (1 << 30) || a.N > (1 << 30)) return set_error(kErrInvalidArgument, "M and N must be at most 2^30");
  // the backward counts steps of 128 rows by 128 keys, a kv head's packed rows at a time
  if (op == AttnOp::kCrossBwd) {
    const double tiles = static_cast<double>(a.q_heads / a.kv_heads) * ((static_cast<double>(a.M) + 127) / 128);
    if (tiles * a.batch * a.kv_heads * ((static_cast<double>(a.N) + 127) / 128) > 1073741824.0)
      return set_error(kErrInvalidArgument, "more than 2^30 tiles of 128 rows by 128 keys");
  }
  if (op == AttnOp::kPrefix) {
    if (a.prefixes <= 0 || a.N_prefix <= 0 || a.N_prefix > (1 << 30))
      return set_error(kErrInvalidArgument, "prefixes=%d and N_prefix=%d must be positive", a.prefixes, a.N_prefix);
    if (a.batch % a.prefixes != 0)
      return set_error(kErrInvalidArgument, "batch=%d is not a multiple of prefixes=%d", a.batch, a.prefixes);
  }
  return kOk;
}

// All arguments; strides of single-row axes are normalised in `a`.
inline int check_attn(fmha_attn_t& a, AttnOp op) {
  int rc = check_attn_sizes(a, op);
  if (rc != kOk) return rc;
  auto q = [&](fmha_tensor_t& t, const char* n, bool w) { return check_tensor(t, n, a.batch, a.q_heads, a.M, a.K_dim, w); };
  auto k = [&](fmha_tensor_t& t, const char* n, bool w) { return check_tensor(t, n, a.batch, a.kv_heads, a.N, a.K_dim, w); };
  const bool bwd = op == AttnOp::kCrossBwd;
  if ((rc = q(a.Q, "Q", false)) || (rc = k(a.K, "K", false)) || (rc = k(a.V, "V", false)) || (rc = q(a.O, "O", !bwd)))
    return rc;
  if (bwd && ((rc = q(a.dO, "dO", false)) || (rc = q(a.dQ, "dQ", true)) || (rc = k(a.dK, "dK", true)) ||
              (rc = k(a.dV, "dV", true))))
    return rc;
  if (op == AttnOp::kPrefix) {
    if ((rc = check_tensor(a.Kp, "Kp", a.prefixes, a.kv_heads, a.N_prefix, a.K_dim, false)) ||
        (rc = check_tensor(a.Vp, "Vp", a.prefixes, a.kv_heads, a.N_prefix, a.K_dim, false)))
      return rc;
    if ((reinterpret_cast<uintptr_t>(a.prefix_lens) & 3u) != 0)
      return set_error(kErrMisaligned, "prefix_lens must be 4-byte aligned");
  }
  const void* read[] = {a.Q.ptr, a.K.ptr, a.V.ptr, bwd ? a.O.ptr : nullptr, bwd ? a.dO.ptr : nullptr,
                        op == AttnOp::kPrefix ? a.Kp.ptr : nullptr, op == AttnOp::kPrefix ? a.Vp.ptr : nullptr};
  const void* written[] = {bwd ? a.dQ.ptr : a.O.ptr, bwd ? a.dK.ptr : a.LSE, bwd ? a.dV.ptr : nullptr};
  for (const void* const& w : written) {
    for (const void* r : read)
      if (r && r == w) return set_error(kErrInvalidArgument, "an output lies over an input");
    for (const void* const& v : written)
      if (&v != &w && v && v == w) return set_error(kErrInvalidArgument, "an output lies over another");
  }
  if (!a.LSE) return set_error(kErrInvalidArgument, "null LSE argument");
  if ((reinterpret_cast<uintptr_t>(a.LSE) & 3u) != 0) return set_error(kErrMisaligned, "LSE must be 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(a.kv_lens) & 3u) != 0)
    return set_error(kErrMisaligned, "kv_lens must be 4-byte aligned");
  if (!(a.softmax_scale > 0.f) || !(a.softmax_scale < 3.0e38f))
    return set_error(kErrInvalidArgument, "softmax_scale must be positive and finite");
  return kOk;
}

// The current device, which has to be an sm_100 one, and its SM count.
inline int attn_device(int& device, int& sms) {
  if (cudaGetDevice(&device) != cudaSuccess) {
    cudaGetLastError();
    return set_error(kErrLaunch, "no current CUDA device");
  }
  struct Seen {
    std::atomic<int> sms{0};
  };
  static Seen seen[64];
  if (device < 64 && (sms = seen[device].sms.load()) > 0) return kOk;
  int major = 0, minor = 0;
  cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device);
  if (major != 10 || minor != 0)
    return set_error(kErrUnsupportedDevice, "device %d is sm_%d%d; this library needs sm_100", device, major, minor);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (sms <= 0) sms = 148;
  if (device < 64) seen[device].sms.store(sms);
  return kOk;
}

// Rows of a length array that count, for one batch entry.
__device__ __forceinline__ int valid_rows(const int* lens, int b, int rows) {
  if (!lens) return rows;
  const int n = __ldg(lens + b);
  return n < 0 ? 0 : (n > rows ? rows : n);
}

}  // namespace fmha_sm100
