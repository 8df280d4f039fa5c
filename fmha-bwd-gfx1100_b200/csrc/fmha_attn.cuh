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
  const double most = static_cast<double>(t.batch) * (batch - 1) + static_cast<double>(t.head) * (heads - 1) +
                      static_cast<double>(t.row) * (rows - 1);
  if (most > 140737488355328.0)  // 2^47 elements are all the addresses there are
    return set_error(kErrInvalidArgument, "%s: strides reach past any memory", name);
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

// The bytes of a strided tensor or an array: `run` consecutive ones at every
// combination of steps along up to three axes, the longest steps first.
struct Region {
  uintptr_t at = 0;
  int axes = 0;
  int64_t n[3] = {1, 1, 1}, step[3] = {0, 0, 0};
  int64_t span[4] = {0, 0, 0, 0};  // bytes from the first to behind the last, of axes i and on
};
inline Region region_of(const void* p, int64_t bytes) {
  Region r;
  r.at = reinterpret_cast<uintptr_t>(p);
  r.span[0] = p ? bytes : 0;
  return r;
}
inline Region region_of(const fmha_tensor_t& t, int batch, int heads, int rows, int D) {
  Region r;
  r.at = reinterpret_cast<uintptr_t>(t.ptr);
  int64_t step[3] = {t.batch, t.head, t.row};
  int n[3] = {batch, heads, rows};
  for (int i = 0; i < 3; ++i) {
    int best = -1;
    for (int j = 0; j < 3; ++j)
      if (n[j] > 1 && (best < 0 || step[j] > step[best])) best = j;
    if (best < 0) break;
    r.n[r.axes] = n[best];
    r.step[r.axes++] = 2 * step[best];
    n[best] = 1;
  }
  r.span[r.axes] = 2 * D;
  for (int i = r.axes - 1; i >= 0; --i) r.span[i] = r.span[i + 1] + r.step[i] * (r.n[i] - 1);
  return r;
}

// Whether two regions share a byte, `off` from a's first to b's first, of axes
// ia and ib on. Along the longest step only the places are followed at which
// what is left of the two can meet, of steps that both have their difference
// alone, so that tensors interleaved in one buffer take a few calls. Those that
// take more than `budget` count as meeting.
inline bool regions_meet(const Region& a, int ia, const Region& b, int ib, int64_t off, int& budget) {
  if (off >= a.span[ia] || -off >= b.span[ib]) return false;
  if (ia == a.axes && ib == b.axes) return true;
  if (--budget < 0) return true;
  const int64_t sa = ia < a.axes ? a.step[ia] : 0, sb = ib < b.axes ? b.step[ib] : 0, s = std::max(sa, sb);
  const int na = sa == s ? ia + 1 : ia, nb = sb == s ? ib + 1 : ib;
  // off + k s for the k with -b.span < off + k s < a.span
  const int64_t least = sa == s ? 1 - a.n[ia] : 0, most = sb == s ? b.n[ib] - 1 : 0;
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0 ? 1 : 0); };
  const int64_t lo = std::max(least, floor_div(-b.span[nb] - off, s) + 1);
  const int64_t hi = std::min(most, floor_div(a.span[na] - off - 1, s));
  for (int64_t k = lo; k <= hi; ++k)
    if (regions_meet(a, na, b, nb, off + k * s, budget)) return true;
  return false;
}
inline bool regions_meet(const Region& a, const Region& b) {
  if (a.span[0] == 0 || b.span[0] == 0) return false;
  int budget = 1 << 17;
  return regions_meet(a, 0, b, 0, static_cast<int64_t>(b.at - a.at), budget);
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

// What a call reads and writes, its workspace apart.
struct AttnRegions {
  Region in[9], out[3];
  int read = 0, written = 0;
  AttnRegions(const fmha_attn_t& a, AttnOp op) {
    auto q = [&](const fmha_tensor_t& t) { return region_of(t, a.batch, a.q_heads, a.M, a.K_dim); };
    auto k = [&](const fmha_tensor_t& t) { return region_of(t, a.batch, a.kv_heads, a.N, a.K_dim); };
    auto kp = [&](const fmha_tensor_t& t) { return region_of(t, a.prefixes, a.kv_heads, a.N_prefix, a.K_dim); };
    const Region lse = region_of(a.LSE, static_cast<int64_t>(a.batch) * a.q_heads * a.M * 4);
    in[read++] = q(a.Q);
    in[read++] = k(a.K);
    in[read++] = k(a.V);
    in[read++] = region_of(a.kv_lens, static_cast<int64_t>(a.batch) * 4);
    if (op == AttnOp::kCrossBwd) {
      in[read++] = q(a.O);
      in[read++] = q(a.dO);
      in[read++] = lse;
      out[written++] = q(a.dQ);
      out[written++] = k(a.dK);
      out[written++] = k(a.dV);
    } else {
      out[written++] = q(a.O);
      out[written++] = lse;
    }
    if (op == AttnOp::kPrefix) {
      in[read++] = kp(a.Kp);
      in[read++] = kp(a.Vp);
      in[read++] = region_of(a.prefix_lens, static_cast<int64_t>(a.prefixes) * 4);
    }
  }
};

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
  if (!a.LSE) return set_error(kErrInvalidArgument, "null LSE argument");
  if ((reinterpret_cast<uintptr_t>(a.LSE) & 3u) != 0) return set_error(kErrMisaligned, "LSE must be 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(a.kv_lens) & 3u) != 0)
    return set_error(kErrMisaligned, "kv_lens must be 4-byte aligned");
  if (!(a.softmax_scale > 0.f) || !(a.softmax_scale < 3.0e38f))
    return set_error(kErrInvalidArgument, "softmax_scale must be positive and finite");
  AttnRegions all(a, op);
  for (int w = 0; w < all.written; ++w) {
    for (int r = 0; r < all.read; ++r)
      if (regions_meet(all.out[w], all.in[r])) return set_error(kErrInvalidArgument, "an output lies over an input");
    for (int v = 0; v < w; ++v)
      if (regions_meet(all.out[w], all.out[v])) return set_error(kErrInvalidArgument, "an output lies over another");
  }
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
