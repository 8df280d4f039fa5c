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

// Shared memory's share of an SM for `kernel`, in percent, set once. Without a
// word on it, a kernel that follows one with 227 KB of shared memory before its
// SMs are idle runs with what that left of L1, in which too few loads find room
// (64 entries behind 8192 keys: 52.4 against 41.4 us).
template <auto kernel>
void share_smem(int percent, int device) {
  static std::atomic<bool> done[64];
  if (device < 64 && done[device].load()) return;
  cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, percent);
  if (device < 64) done[device].store(true);
}

// The SM count that workspace sizes go by: a call on a device with more SMs
// than this would split finer than its workspace allows, so plans use it too.
constexpr int kPlanSms = 148;

inline int launched(cudaError_t e) {
  if (e == cudaSuccess) return kOk;
  cudaGetLastError();
  return set_error(kErrLaunch, "launch failed: %s", cudaGetErrorString(e));
}

// Launches `kernel`; with `early`, as soon as the launch before it on the
// stream lets it (griddepcontrol), which it then waits for itself.
template <typename... P, typename... A>
cudaError_t launch_after(bool early, void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t stream,
                         const A&... args) {
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &at;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// How a forward over `B` key batches divides its work.
struct FwdPlan {
  RowPack rows;
  int pairs, splits, items;
  int64_t all_rows;
  uint64_t ws_bytes;
};

// Parts of the keys, so that one item's chain of key tiles is worked off by
// several SMs. With fewer items than `want`, as many as still leave each two
// key tiles (four above 32 parts: 19 against 22 us with 62 for 125 tiles). If a
// join comes for their sake only, that has to be worth some 5 us, about five
// tiles (24 heads of 512 x 512, d 128: 14.5 us whole, 20.5 in 3 parts; 16 of 77
// x 1000, d 64: 15.9 and 10.7 in 4). `partial`: it comes anyway, and small
// calls get a part for each tile.
inline FwdPlan plan_fwd(int M, int G, int S, int B, int Hkv, int N, int D, int want, bool partial) {
  FwdPlan f;
  f.rows = pack_rows(M, G, S);
  f.pairs = (f.rows.tiles + 1) / 2;
  const int64_t base = static_cast<int64_t>(f.pairs) * B * Hkv;
  const int nt = (N + kTile - 1) / kTile;
  f.splits = 1;
  if (base < want) {
    const int most = partial && nt < 16 ? nt : std::min((nt + 1) / 2, std::max(32, nt / 4));
    f.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want / base, most)));
    if (!partial && nt - (nt + f.splits - 1) / f.splits < 5) f.splits = 1;
  }
  f.items = static_cast<int>(base * f.splits);
  f.all_rows = static_cast<int64_t>(B) * S * Hkv * G * M;
  f.ws_bytes = partial || f.splits > 1 ? static_cast<uint64_t>(f.splits) * f.all_rows * (D + 1) * 4 : 0;
  return f;
}

template <typename T>
int enqueue_fwd(const fmha_attn_t& a, const FwdPlan& f, const fmha_tensor_t& K, const fmha_tensor_t& V, int B, int N,
                const int* lens, float* part_o, float* part_lse, bool own, int device, int sms, cudaStream_t stream) {
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
  p.V = view_of<T>(V);
  p.O = view_of<T>(a.O);
  p.LSE = a.LSE;
  p.partial = part_o != nullptr;
  p.in_turn = p.partial && f.items <= sms;
  p.part_o = part_o;
  p.part_lse = part_lse;
  p.scale = a.softmax_scale;
  p.status = st;
  p.timeout_ns = effective_timeout_ns();
  const unsigned grid = static_cast<unsigned>(std::min(f.items, sms));
  auto go = [&](auto dim, auto kind) {
    constexpr int D = decltype(dim)::value;
    constexpr bool kOwn = decltype(kind)::value;
    using Cfg = FwdCfg<D>;
    allow_smem<attn_fwd_kernel<T, D, kOwn>>(Cfg::kSmemBytes, device);
    return launch_after(kOwn, attn_fwd_kernel<T, D, kOwn>, dim3(grid), Cfg::kThreads, Cfg::kSmemBytes, stream, mQ, mK, mV,
                        p);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  return launched(a.K_dim == 128 ? (own ? go(D128{}, std::true_type{}) : go(D128{}, std::false_type{}))
                                 : (own ? go(D64{}, std::true_type{}) : go(D64{}, std::false_type{})));
}

// O and LSE from `parts` parts of every row, behind the launches that write
// them. Launched `early` behind one whose blocks all run at once: otherwise its
// blocks would take the place of some that have work (64 entries behind 8192
// keys: 54.1 against 51.8 us).
template <typename T>
int enqueue_join(const fmha_attn_t& a, const float* part_o, const float* part_lse, int parts, int64_t rows, bool early,
                 int device, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((rows * (a.K_dim / 4) + 255) / 256));
  auto go = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    return launch_after(early, attn_join_kernel<T, D>, grid, 256, 0, stream, part_o, part_lse, parts, rows, view_of<T>(a.O),
                        a.LSE, a.q_heads, a.M);
  };
  return launched(a.K_dim == 128 ? go(std::integral_constant<int, 128>{}) : go(std::integral_constant<int, 64>{}));
}

// How few-row attention divides its work: 8 or 16 rows a block, and either a
// cluster of `splits` blocks to a kv head's keys or, `blocks` > 0, that many
// blocks to equal runs of the whole batch (see DecodeParams).
struct DecodePlan {
  int R, splits, blocks, side, sub;
  int64_t tasks;
  uint64_t ws_bytes;
};

// Stream: evens out lengths and reads at 6.1 TB/s, but costs a second launch
// and some 15 us in all to fill, drain and join. A block to a kv head needs
// enough of them: 512 (64 entries of 8 heads of 128, up to 512 keys) take
// 19 us, 34 streamed; 1024 of 1500 keys of 64 columns 72 and 79 us. With fewer
// than the GPU holds at a time, clusters divide the keys (some 9 ns a block for
// the launch): 16 x 4000 keys of 8 heads of 128 take 63 us that way, 51
// streamed. So streamed are calls of kStreamBytes of keys and values whose kv
// heads do not fill the GPU, or whose lengths can differ much (kStreamKeys). `part`: the output goes to a join anyway, behind a prefix.
constexpr int kStreamKeys = 8192;
constexpr int64_t kStreamBytes = 96ll << 20;
inline DecodePlan plan_decode(int M, int G, int B, int Hkv, int N, int D, bool part) {
  DecodePlan d;
  d.R = static_cast<int64_t>(G) * M <= 8 ? 1 : 2;
  d.tasks = static_cast<int64_t>(B) * Hkv;
  d.splits = d.side = d.sub = 1;
  d.blocks = 0;
  d.ws_bytes = 0;
  const int64_t tiles = (static_cast<int64_t>(N) + 15) / 16;
  const int64_t slots = decode_blocks(D, d.R) * kPlanSms;
  if (!part && d.tasks * N * D * 4 >= kStreamBytes && (d.tasks < slots || N >= kStreamKeys) && d.tasks * tiles < (1ll << 30)) {
    const int warps = D == 128 ? (d.R == 1 ? StreamCfg<128, 1>::kWarps : StreamCfg<128, 2>::kWarps)
                               : (d.R == 1 ? StreamCfg<64, 1>::kWarps : StreamCfg<64, 2>::kWarps);
    // as many heads side by side as leave the fewest warps without one
    int best = warps;
    for (int side = warps; side >= 1; --side) {
      if (warps % side != 0) continue;
      const int64_t spent = static_cast<int64_t>((Hkv + side - 1) / side * side) *
                            ((tiles + warps / side - 1) / (warps / side)) * (warps / side);
      const int64_t least = static_cast<int64_t>((Hkv + best - 1) / best * best) *
                            ((tiles + warps / best - 1) / (warps / best)) * (warps / best);
      if (spent < least) best = side;
    }
    d.side = best;
    d.sub = warps / best;
    d.blocks = kPlanSms;
    d.ws_bytes = 2ull * d.blocks * d.side * 8 * d.R * (D * 4 + 8);
    return d;
  }
  while (d.splits < kMostSplits && 2 * d.splits * d.tasks <= slots && 64ll * 2 * d.splits <= N) d.splits *= 2;
  return d;
}
inline DecodePlan plan_decode(const fmha_attn_t& a, bool part) {
  return plan_decode(a.M, a.q_heads / a.kv_heads, a.batch, a.kv_heads, a.N, a.K_dim, part);
}

// Up to this many query rows a kv head go through attn_decode_kernel.
constexpr int kDecodeRows = 16;
inline bool is_decode(const fmha_attn_t& a) {
  return static_cast<int64_t>(a.M) * (a.q_heads / a.kv_heads) <= kDecodeRows;
}

// Behind a prefix: whether one launch of attn_decode_kernel reads the prefix for
// each entry anew, instead of parts and their join. It does for kTogetherBytes
// of keys and values in all, read so (4 entries of 16 heads behind 1000 keys: 8.2
// and 11.2 us; 8 of 8 heads behind 4 prefixes of 1000, 34 MB: 11 and 17; but 8
// behind 2000, 66 MB: 15 and 13), unless they are few long caches, for which a
// cluster is too little (kTogetherKeys: 23 us either way for one of 20000); and
// for prefixes of one entry each, if there are many (64 caches of 8192 + 512
// keys: 56 and 79 us).
constexpr int64_t kTogetherBytes = 48ll << 20, kTogetherKeys = 20480, kTogetherTasks = 32;
inline bool prefix_together(const fmha_attn_t& a) {
  if (!is_decode(a)) return false;
  const int64_t tasks = static_cast<int64_t>(a.batch) * a.kv_heads, keys = static_cast<int64_t>(a.N_prefix) + a.N;
  if (a.prefixes == a.batch && tasks >= kTogetherTasks) return keys < (1 << 30);
  return keys <= kTogetherKeys && tasks * keys * a.K_dim * 4 <= kTogetherBytes;
}

// kPrefix: token m reads its entry's keys up to itself, and with part_o and
// part_lse O and LSE go there as a part, else the prefix's keys come along.
template <typename T>
int enqueue_decode(const fmha_attn_t& a, AttnOp op, float* part_o, float* part_lse, int device, cudaStream_t stream) {
  const int G = a.q_heads / a.kv_heads;
  const bool behind = op == AttnOp::kPrefix && !part_o;
  const DecodePlan d = behind ? plan_decode(a.M, G, a.batch, a.kv_heads, a.N_prefix + a.N, a.K_dim, true)
                              : plan_decode(a, op == AttnOp::kPrefix);
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
  p.splits = d.splits;
  p.causal = op == AttnOp::kPrefix;
  p.d16 = a.K_dim / 16;
  p.scale = a.softmax_scale;
  p.part_o = part_o;
  p.part_lse = part_lse;
  p.Kp = view_of<T>(a.Kp);
  p.Vp = view_of<T>(a.Vp);
  p.prefix_lens = a.prefix_lens;
  p.share = behind ? a.batch / a.prefixes : 1;
  p.Np = a.N_prefix;
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
  auto go = [&](auto dim, auto r, auto kind) {
    constexpr int D = decltype(dim)::value, R = decltype(r)::value;
    if (d.blocks > 0) {
      using Cfg = StreamCfg<D, R>;
      allow_smem<attn_decode_stream_kernel<T, D, R>>(Cfg::kSmemBytes, device);
      const cudaError_t e = launch_after(false, attn_decode_stream_kernel<T, D, R>, dim3(d.blocks), 32 * Cfg::kWarps,
                                         Cfg::kSmemBytes, stream, mK, mV, p);
      if (e != cudaSuccess) return e;
      const int64_t rows = static_cast<int64_t>(a.batch) * a.q_heads * a.M;
      return launch_after(true, attn_decode_join_kernel<T, D, R>, dim3(static_cast<unsigned>(rows)), D, 0, stream, p);
    }
    const dim3 grid(static_cast<unsigned>(d.tasks * d.splits));
    // the blocks' sums, and 2 KB each for what is small or reserved
    constexpr int kShare = decode_blocks(D, R) * (kDecodeWarps * 8 * R * D * 4 + 2048) * 100 / (228 * 1024) + 1;
    constexpr bool kBehind = decltype(kind)::value;
    constexpr auto kernel = attn_decode_kernel<T, D, R, kBehind>;
    share_smem<kernel>(kShare, device);
    if (d.splits == 1) return launch_after(part_o != nullptr, kernel, grid, 32 * kDecodeWarps, 0, stream, p);
    static std::atomic<bool> done[64];
    if (device >= 64 || !done[device].load()) {
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (device < 64) done[device].store(true);
    }
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = d.splits;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(32 * kDecodeWarps);
    cfg.stream = stream;
    cfg.attrs = at;
    cfg.numAttrs = part_o ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  using R1 = std::integral_constant<int, 1>;
  using R2 = std::integral_constant<int, 2>;
  auto with = [&](auto kind) {
    return a.K_dim == 128 ? (d.R == 1 ? go(D128{}, R1{}, kind) : go(D128{}, R2{}, kind))
                          : (d.R == 1 ? go(D64{}, R1{}, kind) : go(D64{}, R2{}, kind));
  };
  return launched(behind ? with(std::true_type{}) : with(std::false_type{}));
}

inline FwdPlan cross_plan(const fmha_attn_t& a) {
  return plan_fwd(a.M, a.q_heads / a.kv_heads, 1, a.batch, a.kv_heads, a.N, a.K_dim, kPlanSms, false);
}
// Parts of the prefix: twice as many with several, which can differ in length.
inline FwdPlan prefix_plan(const fmha_attn_t& a) {
  return plan_fwd(a.M, a.q_heads / a.kv_heads, a.batch / a.prefixes, a.prefixes, a.kv_heads, a.N_prefix, a.K_dim,
                  a.prefixes > 1 ? 2 * kPlanSms : kPlanSms, true);
}
// Behind a prefix: the entries' own keys, where they have too many rows for
// attn_decode_kernel.
inline FwdPlan own_plan(const fmha_attn_t& a) {
  return plan_fwd(a.M, a.q_heads / a.kv_heads, 1, a.batch, a.kv_heads, a.N, a.K_dim, kPlanSms, true);
}

// How a backward divides its work, and its workspace: packed LSE and D, the
// tiles' magnitudes (fp16), and two partial-sum slots for each CTA of both kernels.
struct BwdPlan {
  RowPack rows;
  int pairs, grid_q, grid_k, delta_blocks;
  bool join;  // some item may fall to several CTAs
  int64_t packed_rows, row_tiles, key_tiles, slot_floats;
  uint64_t ws_bytes;
};

// Small calls (up to kBesideSteps key-major steps an SM) run the two kernels
// beside each other, on up to kBesideQ of the SMs and the others, about as their
// steps cost, instead of one after the other with more parts or gaps at the end
// of each (32 heads over 4, 300 x 900, d 128: 67 to 46 us; 24 heads of 1024 x
// 1024: 56 us one after the other, 58 beside).
constexpr int kBesideQ = 60, kBesideSteps = 8;
inline BwdPlan plan_bwd(const fmha_attn_t& a) {
  BwdPlan f;
  f.rows = pack_rows(a.M, a.q_heads / a.kv_heads, 1, true);
  f.pairs = (f.rows.tiles + 1) / 2;
  const int64_t heads = static_cast<int64_t>(a.batch) * a.kv_heads;
  const int64_t nt = (a.N + kTile - 1) / kTile;
  f.grid_q = static_cast<int>(std::min<int64_t>(kPlanSms, heads * f.pairs * nt));
  f.grid_k = static_cast<int>(std::min<int64_t>(kPlanSms, heads * f.rows.tiles * nt));
  if (heads * nt * f.rows.tiles <= kBesideSteps * kPlanSms) {
    const int64_t items = heads * f.pairs;
    const int busy = bwd_by_steps((items + kPlanSms - 1) / kPlanSms * nt, items * nt, kPlanSms)
                         ? bwd_parts(items * nt, kPlanSms, true)
                         : static_cast<int>(std::min<int64_t>(items, kPlanSms));
    f.grid_q = std::min(f.grid_q, std::min(busy, kBesideQ));
    f.grid_k = std::min(f.grid_k, kPlanSms - f.grid_q);
  }
  // steps of the busiest CTA with whole items, no fewer than with any lengths
  const int64_t whole_q = (heads * f.pairs + f.grid_q - 1) / f.grid_q * nt;
  const int64_t whole_k = (heads * nt + f.grid_k - 1) / f.grid_k * f.rows.tiles;
  f.join = a.kv_lens ? bwd_by_steps(std::max(whole_q, whole_k), 1, kPlanSms)
                     : bwd_by_steps(whole_q, heads * f.pairs * nt, f.grid_q) ||
                           bwd_by_steps(whole_k, heads * nt * f.rows.tiles, f.grid_k);
  f.row_tiles = heads * f.rows.tiles;
  f.key_tiles = heads * nt;
  f.packed_rows = f.row_tiles * kTile;
  f.delta_blocks = static_cast<int>(std::min<int64_t>(6 * kPlanSms, heads * std::max<int64_t>(f.rows.tiles, nt)));
  f.slot_floats = 2 * static_cast<int64_t>(kTile) * a.K_dim;
  f.ws_bytes = 4 * static_cast<uint64_t>(2 * f.packed_rows + (f.row_tiles + f.key_tiles + 3) / 4 * 4 +
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
  float* top_do = ndelta + f.packed_rows;
  float* top_v = top_do + f.row_tiles;
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
  q.top_do = top_do;
  q.top_v = top_v;
  q.part = top_do + (f.row_tiles + f.key_tiles + 3) / 4 * 4;
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
                                                               a.LSE, q, nlse2, ndelta, top_do, top_v);
    cudaError_t e = launch_after(true, attn_dq_kernel<T, D>, dim3(f.grid_q), kBwdThreads, DqCfg2<D>::kSmemBytes, stream, mQ,
                                 mK, mV, mdO, q);
    if (e == cudaSuccess)
      e = launch_after(true, attn_dkv_kernel<T, D>, dim3(f.grid_k), kBwdThreads, DkvCfg2<D>::kSmemBytes, stream, mQ, mK, mV,
                       mdO, k);
    const int marks = std::max(f.grid_q, f.grid_k) - 1;
    if (e == cudaSuccess && f.join && marks > 0)
      attn_bwd_join_kernel<T, D><<<dim3(kJoinBlocks, marks, 2), 256, 0, stream>>>(q, k, f.grid_q, f.grid_k);
    return e;
  };
  return launched(a.K_dim == 128 ? go(std::integral_constant<int, 128>{}) : go(std::integral_constant<int, 64>{}));
}

inline int attn_workspace(const fmha_attn_t& a, AttnOp op, uint64_t* bytes) {
  const int rc = check_attn_sizes(a, op);
  if (rc != kOk) return rc;
  *bytes = 0;
  if (op == AttnOp::kCrossFwd) *bytes = is_decode(a) ? plan_decode(a, false).ws_bytes : cross_plan(a).ws_bytes;
  if (op == AttnOp::kPrefix && !prefix_together(a)) {
    const FwdPlan f = prefix_plan(a);
    const int parts = f.splits + (is_decode(a) ? 1 : own_plan(a).splits);
    *bytes = static_cast<uint64_t>(parts) * f.all_rows * (a.K_dim + 1) * 4;
  }
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
  if (need > 0) {
    const AttnRegions all(a, op);
    const Region ws = region_of(a.workspace, static_cast<int64_t>(need));
    for (int i = 0; i < all.read + all.written; ++i)
      if (regions_meet(ws, i < all.read ? all.in[i] : all.out[i - all.read]))
        return set_error(kErrInvalidArgument, "the workspace lies over a tensor");
  }
  int device = 0, sms = 0;
  if ((rc = attn_device(device, sms)) != kOk) return rc;
  if (op == AttnOp::kCrossFwd ? is_decode(a) : op == AttnOp::kPrefix && prefix_together(a)) {
    rc = enqueue_decode<T>(a, op, nullptr, nullptr, device, stream);
  } else if (op == AttnOp::kCrossFwd) {
    const FwdPlan f = cross_plan(a);
    float* part_o = f.splits > 1 ? static_cast<float*>(a.workspace) : nullptr;
    float* part_lse = f.splits > 1 ? part_o + f.splits * f.all_rows * a.K_dim : nullptr;
    rc = enqueue_fwd<T>(a, f, a.K, a.V, a.batch, a.N, a.kv_lens, part_o, part_lse, false, device, sms, stream);
    if (rc == kOk && f.splits > 1) rc = enqueue_join<T>(a, part_o, part_lse, f.splits, f.all_rows, true, device, stream);
  } else if (op == AttnOp::kPrefix) {
    // parts of the prefix, parts of the entries' own keys, and their join; the
    // second launch needs nothing of the first, and the third waits for both
    const FwdPlan f = prefix_plan(a), g = own_plan(a);
    const int parts = f.splits + (is_decode(a) ? 1 : g.splits);
    float* part_o = static_cast<float*>(a.workspace);
    float* part_lse = part_o + parts * f.all_rows * a.K_dim;
    float* own_o = part_o + f.splits * f.all_rows * a.K_dim;
    float* own_lse = part_lse + f.splits * f.all_rows;
    rc = enqueue_fwd<T>(a, f, a.Kp, a.Vp, a.prefixes, a.N_prefix, a.prefix_lens, part_o, part_lse, false, device, sms,
                        stream);
    if (rc == kOk)
      rc = is_decode(a) ? enqueue_decode<T>(a, op, own_o, own_lse, device, stream)
                        : enqueue_fwd<T>(a, g, a.K, a.V, a.batch, a.N, a.kv_lens, own_o, own_lse, true, device, sms, stream);
    const DecodePlan d = plan_decode(a, true);
    if (rc == kOk)
      rc = enqueue_join<T>(a, part_o, part_lse, parts, f.all_rows, is_decode(a) && d.tasks * d.splits <= sms, device, stream);
  } else {
    rc = enqueue_bwd<T>(a, device, stream);
  }
  if (rc != kOk) return rc;
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(kErrLaunch, "launch failed: %s", cudaGetErrorString(e));
  return set_error(kOk, "");
}

}  // namespace fmha_sm100
