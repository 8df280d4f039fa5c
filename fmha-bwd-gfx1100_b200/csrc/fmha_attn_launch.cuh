// Host side of the attention entries: workspace, tensor maps and launches.
#pragma once

#include "fmha_attn_bwd.cuh"
#include "fmha_attn_decode.cuh"

namespace fmha_sm100 {

// 4-D map over a strided [batch][heads][rows][D] tensor: boxes of 64 columns,
// 128-byte swizzle, zero fill out of bounds.
inline bool encode_map4(CUtensorMap* map, bool bf16, const fmha_tensor_t& t, int D, int rows, int heads, int batch,
                        int box_rows, int box_heads, int box_batch) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(batch)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(t.row) * 2, static_cast<cuuint64_t>(t.head) * 2,
                                 static_cast<cuuint64_t>(t.batch) * 2};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(kBoxCols), static_cast<cuuint32_t>(box_rows),
                             static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_batch)};
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  return encode_fn()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, t.ptr, dims,
                     strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The status slot of `device`. Its allocation on the first call is allowed
// while a stream of this thread is being captured.
inline KernelStatus* attn_status(int device) {
  std::lock_guard<std::mutex> g(ws_mutex());
  DeviceWorkspace& w = ws_map()[device];
  if (!w.host_status) {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    const bool ok = ensure_status_slot(device, w);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (!ok) return nullptr;
  }
  return w.host_status_dev;
}

// Sets a kernel's shared-memory limit, once for each device.
template <auto kKernel>
void allow_smem(int bytes, int device) {
  static std::atomic<bool> done[64];
  if (device < 64 && done[device].load()) return;
  cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (device < 64) done[device].store(true);
}

// The SM count that workspace sizes go by: a call on a device with more SMs
// than this would split finer than its workspace allows, so plans use it too.
constexpr int kPlanSms = 148;

// How a forward over `B` key batches divides its work.
struct FwdPlan {
  RowPack rows;
  int pairs, splits, items;
  int64_t all_rows;
  uint64_t ws_bytes;
};

// Parts of the keys: with fewer items than SMs, as many parts as still leave
// each two key tiles, so that the loads of one item spread over idle SMs.
inline FwdPlan plan_fwd(int M, int G, int S, int B, int Hkv, int N, int D, int sms, bool partial) {
  FwdPlan f;
  f.rows = pack_rows(M, G, S);
  f.pairs = (f.rows.tiles + 1) / 2;
  const int64_t base = static_cast<int64_t>(f.pairs) * B * Hkv;
  const int nt = (N + kTile - 1) / kTile;
  f.splits = 1;
  if (base < sms) f.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sms / base, nt / 2)));
  f.items = static_cast<int>(base * f.splits);
  static_assert(kPlanSms <= kMostParts, "parts that attn_decode_kernel joins");
  f.all_rows = static_cast<int64_t>(B) * S * Hkv * G * M;
  f.ws_bytes = partial || f.splits > 1 ? static_cast<uint64_t>(f.splits) * f.all_rows * (D + 1) * 4 : 0;
  return f;
}

template <typename T>
int enqueue_fwd(const fmha_attn_t& a, const FwdPlan& f, const fmha_tensor_t& K, const fmha_tensor_t& V, int B, int N,
                const int* lens, bool partial, int device, int sms, cudaStream_t stream) {
  constexpr bool kBF16 = Elem<T>::kBF16;
  if (!encode_fn()) return set_error(kErrNoDriver, "cuTensorMapEncodeTiled is unavailable");
  KernelStatus* st = attn_status(device);
  if (!st) return kErrOutOfMemory;
  CUtensorMap mQ, mK, mV;
  if (!encode_map4(&mQ, kBF16, a.Q, a.K_dim, a.M, a.q_heads, a.batch, f.rows.Mt, f.rows.Gt, f.rows.St) ||
      !encode_map4(&mK, kBF16, K, a.K_dim, N, a.kv_heads, B, kTile, 1, 1) ||
      !encode_map4(&mV, kBF16, V, a.K_dim, N, a.kv_heads, B, kTile, 1, 1))
    return set_error(kErrInvalidArgument, "tensor map encoding failed");
  FwdParams<T> p;
  p.rows = f.rows;
  p.B = B;
  p.Hkv = a.kv_heads;
  p.N = N;
  p.lens = lens;
  p.splits = f.splits;
  p.pairs = f.pairs;
  p.items = f.items;
  p.O = view_of<T>(a.O);
  p.LSE = a.LSE;
  p.partial = partial || f.splits > 1;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_lse = p.part_o + static_cast<int64_t>(f.splits) * f.all_rows * a.K_dim;
  p.scale = a.softmax_scale;
  p.status = st;
  p.timeout_ns = effective_timeout_ns();
  const unsigned grid = static_cast<unsigned>(std::min(f.items, sms));
  auto go = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    using Cfg = FwdCfg<D>;
    allow_smem<attn_fwd_kernel<T, D>>(Cfg::kSmemBytes, device);
    attn_fwd_kernel<T, D><<<grid, Cfg::kThreads, Cfg::kSmemBytes, stream>>>(mQ, mK, mV, p);
    if (f.splits > 1 && !partial) {
      const int64_t threads = f.all_rows * (D / 4);
      attn_join_kernel<T, D><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, stream>>>(
          p.part_o, p.part_lse, f.splits, f.all_rows, p.O, p.LSE, a.q_heads, a.M);
    }
  };
  if (a.K_dim == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 64>{});
  return kOk;
}

// How few-row attention divides its work: 8 or 16 rows a block, and either a
// cluster of `splits` blocks to a kv head's keys or, `blocks` > 0, that many
// blocks to equal runs of the whole batch (see DecodeParams).
struct DecodePlan {
  int R, row_tiles, splits, blocks, side, sub;
  int64_t tasks;
  uint64_t ws_bytes;
};

// Stream: evens out lengths and reads at 6.1 TB/s, but costs a second launch
// and some 15 us in all to fill, drain and join, so from kStreamBytes of keys
// and values on. Clusters read at 4.9 (D = 128) and 6.5 TB/s (D = 64) at 7 us:
// at 64 columns they stay ahead (71 against 79 us for 64 x 1500 keys of 16
// heads) until the lengths can differ much (kStreamKeys); at 128 columns 16 x
// 4000 keys of 8 heads take 63 us in clusters and 51 us streamed. Blocks of a
// cluster: of 1 to 16 a tile of rows, the number with the least estimated time:
// waves of blocks times a block's steps of 64 keys plus its fixed costs, which
// measure like kDecodeFixed such steps. `parts`: the caller's parts join in the
// cluster's launch.
constexpr int kDecodeFixed = 4, kStreamKeys = 8192;
constexpr int64_t kStreamBytes = 96ll << 20;
inline DecodePlan plan_decode(int M, int G, int B, int Hkv, int N, int D, bool parts) {
  DecodePlan d;
  const int64_t rows = static_cast<int64_t>(G) * M;
  d.R = rows <= 8 ? 1 : 2;
  d.row_tiles = static_cast<int>((rows + 8 * d.R - 1) / (8 * d.R));
  d.tasks = static_cast<int64_t>(B) * Hkv * d.row_tiles;
  d.splits = d.side = d.sub = 1;
  d.blocks = 0;
  d.ws_bytes = 0;
  const int64_t tiles = (static_cast<int64_t>(N) + 15) / 16;
  if (!parts && d.tasks * N * D * 4 >= kStreamBytes && (D == 128 || N >= kStreamKeys) && d.tasks * tiles < (1ll << 30)) {
    const int warps = D == 128 ? (d.R == 1 ? StreamCfg<128, 1>::kWarps : StreamCfg<128, 2>::kWarps)
                               : (d.R == 1 ? StreamCfg<64, 1>::kWarps : StreamCfg<64, 2>::kWarps);
    // as many items side by side as leave the fewest warps without one
    const int items = Hkv * d.row_tiles;
    int best = warps;
    for (int side = warps; side >= 1; --side) {
      if (warps % side != 0) continue;
      const int idle = (items + side - 1) / side * side - items;
      const int64_t spent = static_cast<int64_t>(items + idle) * ((tiles + warps / side - 1) / (warps / side)) * (warps / side);
      const int64_t least = static_cast<int64_t>((items + best - 1) / best * best) *
                            ((tiles + warps / best - 1) / (warps / best)) * (warps / best);
      if (spent < least) best = side;
    }
    d.side = best;
    d.sub = warps / best;
    d.blocks = kPlanSms;
    d.ws_bytes = 2ull * d.blocks * d.side * 8 * d.R * (D * 4 + 8);
    return d;
  }
  const int64_t steps = (static_cast<int64_t>(N) + 63) / 64;
  const int64_t slots = decode_blocks(D, d.R) * kPlanSms;
  int64_t best = 0;
  for (int s = 1; s <= kMostSplits && s <= steps; s *= 2) {
    const int64_t cost = (d.tasks * s + slots - 1) / slots * ((steps + s - 1) / s + kDecodeFixed);
    if (s == 1 || cost < best) {
      best = cost;
      d.splits = s;
    }
  }
  return d;
}
inline DecodePlan plan_decode(const fmha_attn_t& a, bool parts) {
  return plan_decode(a.M, a.q_heads / a.kv_heads, a.batch, a.kv_heads, a.N, a.K_dim, parts);
}

// Up to this many query rows a kv head go through attn_decode_kernel.
constexpr int kDecodeRows = 16;
inline bool is_decode(const fmha_attn_t& a) {
  return static_cast<int64_t>(a.M) * (a.q_heads / a.kv_heads) <= kDecodeRows;
}

// `parts` > 0: joins that many parts of every row in the workspace, which the
// launch before this one on the stream writes; token m then reads its entry's
// keys up to itself.
template <typename T>
int enqueue_decode(const fmha_attn_t& a, bool prefix, int parts, int64_t all_rows, int device, cudaStream_t stream) {
  const int G = a.q_heads / a.kv_heads;
  const DecodePlan d = plan_decode(a, prefix);
  DecodeParams<T> p;
  p.Q = view_of<T>(a.Q);
  p.K = view_of<T>(a.K);
  p.V = view_of<T>(a.V);
  p.O = view_of<T>(a.O);
  p.LSE = a.LSE;
  p.lens = a.kv_lens;
  p.B = a.batch;
  p.Hkv = a.kv_heads;
  p.G = G;
  p.M = a.M;
  p.N = a.N;
  p.row_tiles = d.row_tiles;
  p.splits = d.splits;
  p.causal = prefix;
  p.scale = a.softmax_scale;
  p.parts = parts;
  p.all_rows = all_rows;
  p.part_o = parts > 0 ? static_cast<const float*>(a.workspace) : nullptr;
  p.part_lse = parts > 0 ? p.part_o + parts * all_rows * a.K_dim : nullptr;
  CUtensorMap mK, mV;
  if (d.blocks > 0) {
    if (!encode_fn()) return set_error(kErrNoDriver, "cuTensorMapEncodeTiled is unavailable");
    p.status = attn_status(device);
    if (!p.status) return kErrOutOfMemory;
    p.timeout_ns = effective_timeout_ns();
    constexpr bool kBF16 = Elem<T>::kBF16;
    if (!encode_map4(&mK, kBF16, a.K, a.K_dim, a.N, a.kv_heads, a.batch, 16, 1, 1) ||
        !encode_map4(&mV, kBF16, a.V, a.K_dim, a.N, a.kv_heads, a.batch, 16, 1, 1))
      return set_error(kErrInvalidArgument, "tensor map encoding failed");
  }
  p.blocks = d.blocks;
  p.side = d.side;
  p.sub = d.sub;
  p.run_o = static_cast<float*>(a.workspace);
  p.run_ml = reinterpret_cast<float2*>(p.run_o + 2ll * d.blocks * d.side * 8 * d.R * a.K_dim);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(d.tasks * d.splits));
  cfg.blockDim = dim3(32 * kDecodeWarps);
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  if (d.splits > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = d.splits;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (parts > 0) {  // starts while the parts are still being written
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = at;
  auto go = [&](auto dim, auto r) {
    constexpr int D = decltype(dim)::value, R = decltype(r)::value;
    if (d.blocks > 0) {
      using Cfg = StreamCfg<D, R>;
      allow_smem<attn_decode_stream_kernel<T, D, R>>(Cfg::kSmemBytes, device);
      attn_decode_stream_kernel<T, D, R><<<d.blocks, 32 * Cfg::kWarps, Cfg::kSmemBytes, stream>>>(mK, mV, p);
      cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(a.batch) * a.q_heads * a.M));
      cfg.blockDim = dim3(D);
      at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.numAttrs = 1;
      return cudaLaunchKernelEx(&cfg, attn_decode_join_kernel<T, D, R>, p);
    }
    constexpr auto kernel = attn_decode_kernel<T, D, R>;
    static std::atomic<bool> done[64];
    if (device >= 64 || !done[device].load()) {
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (device < 64) done[device].store(true);
    }
    return cudaLaunchKernelEx(&cfg, kernel, p);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  using R1 = std::integral_constant<int, 1>;
  using R2 = std::integral_constant<int, 2>;
  const cudaError_t e = a.K_dim == 128 ? (d.R == 1 ? go(D128{}, R1{}) : go(D128{}, R2{}))
                                       : (d.R == 1 ? go(D64{}, R1{}) : go(D64{}, R2{}));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(kErrLaunch, "launch failed: %s", cudaGetErrorString(e));
  }
  return kOk;
}

inline FwdPlan cross_plan(const fmha_attn_t& a) {
  return plan_fwd(a.M, a.q_heads / a.kv_heads, 1, a.batch, a.kv_heads, a.N, a.K_dim, kPlanSms, false);
}

inline FwdPlan prefix_plan(const fmha_attn_t& a) {
  return plan_fwd(a.M, a.q_heads / a.kv_heads, a.batch / a.prefixes, a.prefixes, a.kv_heads, a.N_prefix, a.K_dim,
                  kPlanSms, true);
}

// How a backward divides its work, and its workspace: packed LSE and D, the
// amplitudes (fp16), and two partial-sum slots for each CTA of both kernels.
struct BwdPlan {
  RowPack rows;
  int pairs, grid_q, grid_k, delta_blocks;
  bool join;  // some item may fall to several CTAs
  int64_t packed_rows, slot_floats;
  uint64_t ws_bytes;
};

inline BwdPlan plan_bwd(const fmha_attn_t& a) {
  BwdPlan f;
  f.rows = pack_rows(a.M, a.q_heads / a.kv_heads, 1, true);
  f.pairs = (f.rows.tiles + 1) / 2;
  const int64_t heads = static_cast<int64_t>(a.batch) * a.kv_heads;
  const int64_t nt = (a.N + kTile - 1) / kTile;
  f.grid_q = static_cast<int>(std::min<int64_t>(kPlanSms, heads * f.pairs * nt));
  f.grid_k = static_cast<int>(std::min<int64_t>(kPlanSms, heads * f.rows.tiles * nt));
  f.join = a.kv_lens != nullptr ||
           bwd_by_steps((heads * f.pairs + f.grid_q - 1) / f.grid_q * nt, heads * f.pairs * nt, f.grid_q) ||
           bwd_by_steps((heads * nt + f.grid_k - 1) / f.grid_k * f.rows.tiles, heads * nt * f.rows.tiles, f.grid_k);
  f.packed_rows = heads * f.rows.tiles * kTile;
  f.delta_blocks = static_cast<int>(std::min<int64_t>(6 * kPlanSms, heads * std::max<int64_t>(f.rows.tiles, nt)));
  f.slot_floats = 2 * static_cast<int64_t>(kTile) * a.K_dim;
  f.ws_bytes = 4 * static_cast<uint64_t>(2 * f.packed_rows + 2 * ((f.delta_blocks + 1) / 2 * 2) +
                                         2 * (f.grid_q + f.grid_k) * f.slot_floats);
  return f;
}

template <typename T>
int enqueue_bwd(const fmha_attn_t& a, int device, cudaStream_t stream) {
  constexpr bool kBF16 = Elem<T>::kBF16;
  if (!encode_fn()) return set_error(kErrNoDriver, "cuTensorMapEncodeTiled is unavailable");
  KernelStatus* st = attn_status(device);
  if (!st) return kErrOutOfMemory;
  const BwdPlan f = plan_bwd(a);
  CUtensorMap mQ, mK, mV, mdO;
  if (!encode_map4(&mQ, kBF16, a.Q, a.K_dim, a.M, a.q_heads, a.batch, f.rows.Mt, f.rows.Gt, 1) ||
      !encode_map4(&mdO, kBF16, a.dO, a.K_dim, a.M, a.q_heads, a.batch, f.rows.Mt, f.rows.Gt, 1) ||
      !encode_map4(&mK, kBF16, a.K, a.K_dim, a.N, a.kv_heads, a.batch, kTile, 1, 1) ||
      !encode_map4(&mV, kBF16, a.V, a.K_dim, a.N, a.kv_heads, a.batch, kTile, 1, 1))
    return set_error(kErrInvalidArgument, "tensor map encoding failed");
  float* nlse2 = static_cast<float*>(a.workspace);
  float* ndelta = nlse2 + f.packed_rows;
  float2* amax = reinterpret_cast<float2*>(ndelta + f.packed_rows);
  BwdParams<T> q;
  q.rows = f.rows;
  q.B = a.batch;
  q.Hkv = a.kv_heads;
  q.N = a.N;
  q.pairs = f.pairs;
  q.lens = a.kv_lens;
  q.dQ = view_of<T>(a.dQ);
  q.dK = view_of<T>(a.dK);
  q.dV = view_of<T>(a.dV);
  q.nlse2 = nlse2;
  q.ndelta = ndelta;
  q.amax = amax;
  q.amax_count = f.delta_blocks;
  q.part = reinterpret_cast<float*>(amax + (f.delta_blocks + 1) / 2 * 2);
  q.scale = a.softmax_scale;
  q.status = st;
  q.timeout_ns = effective_timeout_ns();
  BwdParams<T> k = q;
  k.part = q.part + 2 * f.grid_q * f.slot_floats;
  auto go = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    allow_smem<attn_dq_kernel<T, D>>(DqCfg2<D>::kSmemBytes, device);
    allow_smem<attn_dkv_kernel<T, D>>(DkvCfg2<D>::kSmemBytes, device);
    attn_delta_kernel<T, D><<<f.delta_blocks, 256, 0, stream>>>(view_of<T>(a.dO), view_of<T>(a.O), view_of<T>(a.V),
                                                               a.LSE, q, nlse2, ndelta, amax);
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(f.grid_q);
    cfg.blockDim = dim3(kBwdThreads);
    cfg.dynamicSmemBytes = DqCfg2<D>::kSmemBytes;
    cudaError_t e = cudaLaunchKernelEx(&cfg, attn_dq_kernel<T, D>, mQ, mK, mV, mdO, q);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(f.grid_k);
    cfg.dynamicSmemBytes = DkvCfg2<D>::kSmemBytes;
    e = cudaLaunchKernelEx(&cfg, attn_dkv_kernel<T, D>, mQ, mK, mV, mdO, k);
    const int marks = std::max(f.grid_q, f.grid_k) - 1;
    if (e == cudaSuccess && f.join && marks > 0)
      attn_bwd_join_kernel<T, D><<<dim3(kJoinBlocks, marks, 2), 256, 0, stream>>>(q, k, f.grid_q, f.grid_k);
    return e;
  };
  const cudaError_t e =
      a.K_dim == 128 ? go(std::integral_constant<int, 128>{}) : go(std::integral_constant<int, 64>{});
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(kErrLaunch, "launch failed: %s", cudaGetErrorString(e));
  }
  return kOk;
}

inline int attn_workspace(const fmha_attn_t& a, AttnOp op, uint64_t* bytes) {
  const int rc = check_attn_sizes(a, op);
  if (rc != kOk) return rc;
  *bytes = 0;
  if (op == AttnOp::kCrossFwd) *bytes = is_decode(a) ? plan_decode(a, false).ws_bytes : cross_plan(a).ws_bytes;
  if (op == AttnOp::kPrefix) *bytes = prefix_plan(a).ws_bytes;
  if (op == AttnOp::kCrossBwd) *bytes = plan_bwd(a).ws_bytes;
  return kOk;
}

template <typename T>
int run_attn(const fmha_attn_t* args, AttnOp op, cudaStream_t stream) {
  if (!args) return set_error(kErrInvalidArgument, "null arguments");
  fmha_attn_t a = *args;
  int rc = check_attn(a, op);
  if (rc != kOk) return rc;
  uint64_t need = 0;
  if ((rc = attn_workspace(a, op, &need)) != kOk) return rc;
  if (need > 0 && (!a.workspace || a.workspace_bytes < need))
    return set_error(kErrInvalidArgument, "workspace of %llu bytes, %llu needed",
                     static_cast<unsigned long long>(a.workspace ? a.workspace_bytes : 0),
                     static_cast<unsigned long long>(need));
  if (need > 0 && !aligned16(a.workspace)) return set_error(kErrMisaligned, "workspace must be 16-byte aligned");
  int device = 0, sms = 0;
  if ((rc = attn_device(device, sms)) != kOk) return rc;
  if (op == AttnOp::kCrossFwd && is_decode(a)) {
    rc = enqueue_decode<T>(a, false, 0, 0, device, stream);
  } else if (op == AttnOp::kPrefix) {
    const FwdPlan f = prefix_plan(a);
    rc = enqueue_fwd<T>(a, f, a.Kp, a.Vp, a.prefixes, a.N_prefix, a.prefix_lens, true, device, sms, stream);
    if (rc == kOk) rc = enqueue_decode<T>(a, true, f.splits, f.all_rows, device, stream);
  } else if (op == AttnOp::kCrossFwd) {
    rc = enqueue_fwd<T>(a, cross_plan(a), a.K, a.V, a.batch, a.N, a.kv_lens, false, device, sms, stream);
  } else {
    rc = enqueue_bwd<T>(a, device, stream);
  }
  if (rc != kOk) return rc;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(kErrLaunch, "launch failed: %s", cudaGetErrorString(e));
  return set_error(kOk, "");
}

}  // namespace fmha_sm100
