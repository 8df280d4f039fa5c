// Attention of a few query rows (single tokens): every key and value is read
// once, in the pieces that the tensor core's fragments are made of.
//
// The floor is the bytes of K and V, so the kernels are built around loads in
// flight (a plain read needs some 130 KB an SM on its way for 6.5 TB/s here).
// The products are transposed, keys and value columns on the 16-row side of
// mma.m16n8k16 and the query rows on its 8-column side (R = 1: up to 8 rows of
// a kv head, R = 2: up to 16):
//
//   S^T [16 keys x 8 rows]   = K [16 x D] Q^T
//   O^T [16 columns x 8 rows] += V^T [16 x 16 keys] P^T
//
// A contraction may run over its index in any order as long as both operands
// use the same one, and the rows of a product may come out in any order. So
// each thread takes its K fragment as 16-byte pieces of a key's row (the
// order of the D columns within a 32-column block is a permutation of the
// fragment's, Q is loaded in the same one), and its V fragment as 16-byte
// pieces of four keys' rows, paired key by key with byte permutes; a thread
// then holds 8 neighbouring columns of O for two rows. P^T is turned from
// accumulator to operand layout by movmatrix. The rows' references m move only
// when some row's maximum is over 2^8 times its own (see attn_fwd_kernel; the
// same bias in fp16).
//
// Two kernels share this:
//   * attn_decode_kernel: a block to a kv head's rows (16 at most); with few of
//     those, a cluster of blocks splits the keys and meets in each other's
//     shared memory. One launch, no workspace; pieces go straight to registers,
//     one tile ahead. Behind a shared prefix it takes the prefix's keys along
//     (few of them), or leaves its O and LSE as one part more for
//     attn_join_kernel.
//   * attn_decode_stream_kernel, for long caches: every block takes an equal run
//     of the keys of the whole batch, counted on the device from the lengths,
//     its warps side by side in neighbouring heads: those lie together in a
//     [token][head] cache, whose 128-byte rows otherwise come one to a DRAM page
//     (4.3 instead of 6.1 TB/s). Each warp keeps a ring of 16-key tiles on its
//     way into shared memory by TMA, across the entries that the run passes.
//     Heads whose keys fall to several blocks leave fp32 sums for
//     attn_decode_join_kernel.
// Both add up in a fixed order: the same bits each time.
#pragma once

#include "fmha_attn_fwd.cuh"

namespace fmha_sm100 {

__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <bool kBF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (kBF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8x8 matrix of 16-bit elements held by a warp (thread t:
// row t / 4, columns 2 (t % 4) + {0, 1}).
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// An address in the same place of another block's shared memory.
__device__ __forceinline__ float load_cluster(const float* local, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 load_cluster4(const float* local, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T>
struct DecodeParams {
  View<T> Q, K, V, O;
  float* LSE;
  const int* lens;  // [B] or null
  int B, Hkv, G, M, N;
  int splits;       // blocks (a cluster) that share a kv head's keys
  int d16;          // D / 16
  bool causal;      // token m reads lens - (M - 1 - m) keys
  float scale;
  float* part_o;    // null, or where O and LSE go as a part: [row][D], normalised, and
  float* part_lse;  // [row]
  View<T> Kp, Vp;         // kBehind: the keys that `share` entries have before their own,
  const int* prefix_lens; // [B / share] or null
  int share, Np;
  int blocks;         // stream: blocks,
  int side;           // items (kv heads) that a block has side by side,
  int sub;            // warps to an item (side * sub warps a block)
  float* run_o;       // [2 * blocks][side][8 R rows][D] and
  float2* run_ml;     // [2 * blocks][side][8 R rows] partial sums
  KernelStatus* status;
  uint64_t timeout_ns;
};

// A warp's share of a kv head's rows: Q, the sums and what they refer to.
template <typename T, int D, int R>
struct DecodeWarp {
  static constexpr bool kB = Elem<T>::kBF16;
  static constexpr float kBias = kB ? 0.f : 6.f;
  uint4 qf[R][D / 32];
  float o[R][D / 16][4];
  float m[R][2], l[R][2];

  // Q of rows g (+ 8), in K's order of columns; no sums yet
  __device__ __forceinline__ void begin(const DecodeParams<T>& p, int b, int hk) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = 8 * r + g;
      const T* at = p.Q.at(b, hk * p.G + row / p.M, row % p.M) + 8 * t;
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
        qf[r][c] = row < p.G * p.M ? *reinterpret_cast<const uint4*>(at + 32 * c) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[r][c][x] = 0.f;
      m[r][0] = m[r][1] = kNoMax;
      l[r][0] = l[r][1] = 0.f;
    }
  }
  // S^T of 16 keys; k(x, c): the piece of key g + 8 x at column 32 c + 8 t
  template <typename F>
  __device__ __forceinline__ void scores(float (&s)[R][4], F&& k) {
    float s2[R][4];  // two chains of sums: half the latency
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[r][x] = s2[r][x] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint4 k0 = k(0, c), k1 = k(1, c);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        mma_16816<kB>(s[r], k0.x, k1.x, k0.y, k1.y, qf[r][c].x, qf[r][c].y);
        mma_16816<kB>(s2[r], k0.z, k1.z, k0.w, k1.w, qf[r][c].z, qf[r][c].w);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[r][x] += s2[r][x];
  }
  // Weights of keys key0 + g (s[r][0], [1] for rows 2t, 2t + 1) and key0 + g + 8
  // ([2], [3]), each row's keys ending at limit; P^T in operand layout.
  __device__ __forceinline__ void weights(float (&s)[R][4], uint32_t (&pt)[R][2], int key0, const int (&limit)[R][2],
                                          float sl2) {
    const int g = (threadIdx.x & 31) >> 2;
    bool move = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int x = 0; x < 4; ++x) s[r][x] = key0 + g + 8 * (x >> 1) < limit[r][x & 1] ? s[r][x] * sl2 : -INFINITY;
      move |= fmaxf(s[r][0], s[r][2]) > m[r][0] + (8.f + kBias) || fmaxf(s[r][1], s[r][3]) > m[r][1] + (8.f + kBias);
    }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float top = fmaxf(s[r][x], s[r][x + 2]);
#pragma unroll
          for (int y = 4; y < 32; y <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, y));
          const float to = fmaxf(top - kBias, m[r][x]);
          const float f = ex2_approx(m[r][x] - to);
          m[r][x] = to;
          l[r][x] *= f;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            o[r][c][x] *= f;
            o[r][c][x + 2] *= f;
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[r][x] = ex2_approx(s[r][x] - m[r][x & 1]);
        l[r][x & 1] += s[r][x];
      }
      pt[r][0] = transpose_8x8(Elem<T>::pack(s[r][0], s[r][1]));
      pt[r][1] = transpose_8x8(Elem<T>::pack(s[r][2], s[r][3]));
    }
  }
  // O^T += V^T P^T; v(x, c): the piece of key 2t + x % 2 + 8 (x / 2) at column 64 c + 8 g
  template <typename F>
  __device__ __forceinline__ void values(const uint32_t (&pt)[R][2], F&& v) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 f[4] = {v(0, c), v(1, c), v(2, c), v(3, c)};
      const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&f[0]);
      const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&f[1]);
      const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&f[2]);
      const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&f[3]);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t a0 = __byte_perm(v0[x], v1[x], 0x5410), a1 = __byte_perm(v0[x], v1[x], 0x7632);
        const uint32_t a2 = __byte_perm(v2[x], v3[x], 0x5410), a3 = __byte_perm(v2[x], v3[x], 0x7632);
#pragma unroll
        for (int r = 0; r < R; ++r) mma_16816<kB>(o[r][4 * c + x], a0, a1, a2, a3, pt[r][0], pt[r][1]);
      }
    }
  }
  // The rows' sums over the warp, in every lane of the row's column.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 4; y < 32; y <<= 1) l[r][x] += __shfl_xor_sync(0xffffffffu, l[r][x], y);
  }
  // 8 columns 64 c + 8 g of row 8 r + 2t + x
  __device__ __forceinline__ void columns(int r, int x, int c, float f, float4& a, float4& b) const {
    a = make_float4(f * o[r][4 * c][x], f * o[r][4 * c][x + 2], f * o[r][4 * c + 1][x], f * o[r][4 * c + 1][x + 2]);
    b = make_float4(f * o[r][4 * c + 2][x], f * o[r][4 * c + 2][x + 2], f * o[r][4 * c + 3][x], f * o[r][4 * c + 3][x + 2]);
  }
};

__device__ __forceinline__ void add_weighted(float4& acc, float w, const float4& v) {
  acc.x = fmaf(w, v.x, acc.x);
  acc.y = fmaf(w, v.y, acc.y);
  acc.z = fmaf(w, v.z, acc.z);
  acc.w = fmaf(w, v.w, acc.w);
}

// The infinities and NaN that 4 columns of `count` rows of V hold (every weight
// is above 0), into a row's sums: see hide_odd.
template <typename T>
__device__ __forceinline__ void add_odd4(const T* v, int64_t stride, int count, float4& acc) {
#pragma unroll 1
  for (int k = 0; k < count; ++k) {
    const uint2 all = *reinterpret_cast<const uint2*>(v + k * stride);
    uint2 rest = all;
    drop_odd<T>(rest.x);
    drop_odd<T>(rest.y);
    const float2 a = Elem<T>::unpack(all.x ^ rest.x), b = Elem<T>::unpack(all.y ^ rest.y);
    acc.x += a.x;
    acc.y += a.y;
    acc.z += b.x;
    acc.w += b.y;
  }
}

// 4 columns of O (and, with the first, LSE) of packed row q of a kv head, from
// their sum at the reference m. A sum of 0 has no key behind it; NaN stays.
template <typename T>
__device__ __forceinline__ void decode_output(const DecodeParams<T>& p, int b, int hk, int q, int c, float m, float sum,
                                              const float4& acc) {
  const int head = hk * p.G + q / p.M, tok = q % p.M;
  const int64_t row = (static_cast<int64_t>(b) * p.Hkv * p.G + head) * p.M + tok;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (p.part_o)
    reinterpret_cast<float4*>(p.part_o + row * (16 * p.d16))[c] = make_float4(inv * acc.x, inv * acc.y, inv * acc.z, inv * acc.w);
  else
    *reinterpret_cast<uint2*>(p.O.at(b, head, tok) + 4 * c) =
        make_uint2(Elem<T>::pack(inv * acc.x, inv * acc.y), Elem<T>::pack(inv * acc.z, inv * acc.w));
  if (c == 0) (p.part_o ? p.part_lse : p.LSE)[row] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
}

// ------------------------------------------------------------------- clusters
constexpr int kMostSplits = 16, kDecodeWarps = 4;
// Blocks that an SM holds at a time.
__host__ __device__ constexpr int decode_blocks(int D, int R) { return D == 128 ? (R == 1 ? 3 : 2) : (R == 1 ? 5 : 4); }

// 64 x 16 heads, 1500 keys of 64: 72 to 75 us, 5.2 to 5.5 TB/s; 8 kv heads of 4096 keys of
// 128 in clusters of 16: 12 us, bound by latency (lengths, first keys, Q, the
// exchange).
// kBehind: over a shared prefix's keys and an entry's own in one go.
template <typename T, int D, int R, bool kBehind>
__global__ void __launch_bounds__(32 * kDecodeWarps, decode_blocks(D, R) - (kBehind && D == 64))
    attn_decode_kernel(const __grid_constant__ DecodeParams<T> p) {
  constexpr int kRows = 8 * R, W = kDecodeWarps, kThreads = 32 * W;
  if (p.part_o) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ __align__(16) float sum_o[W][kRows][D];
  __shared__ float warp_m[W][kRows], warp_l[W][kRows], block_m[kRows], block_l[kRows];
  __shared__ float weight[kMostSplits][kRows], total[kRows], top_of[kRows], block_odd;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % p.splits;
  const int u = blockIdx.x / p.splits;
  const int hk = u % p.Hkv, b = u / p.Hkv;
  const int rows = p.G * p.M;
  const int n = valid_rows(p.lens, b, p.N);
  const int bp = kBehind ? b / p.share : 0, np = kBehind ? valid_rows(p.prefix_lens, bp, p.Np) : 0;
  const int ahead = (np + 15) / 16;  // tiles of the prefix
  const int tiles = ahead + (n + 15) / 16;
  const int lo = static_cast<int>(static_cast<int64_t>(tiles) * split / p.splits);
  const int hi = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / p.splits);

  uint4 kf[2][D / 32], vf[4][D / 64];
  auto load_k = [&](int i) {
    const bool own = !kBehind || i >= ahead;
    const int from = 16 * (own ? i - ahead : i), most = own ? n : np;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int key = from + g + 8 * x;
      const T* at = (own ? p.K.at(b, hk, key) : p.Kp.at(bp, hk, key)) + 8 * t;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) kf[x][c] = key < most ? load_stream(at + 32 * c) : make_uint4(0, 0, 0, 0);
    }
  };
  auto load_v = [&](int i) {
    const bool own = !kBehind || i >= ahead;
    const int from = 16 * (own ? i - ahead : i), most = own ? n : np;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int key = from + 2 * t + (x & 1) + 8 * (x >> 1);
      const T* at = (own ? p.V.at(b, hk, key) : p.Vp.at(bp, hk, key)) + 8 * g;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) vf[x][c] = key < most ? load_stream(at + 64 * c) : make_uint4(0, 0, 0, 0);
    }
  };
  int i = lo + warp;
  if (i < hi) {
    load_k(i);
    load_v(i);
  }
  DecodeWarp<T, D, R> w;
  w.begin(p, b, hk);
  int limit[R][2];  // keys that rows 2t and 2t + 1 may read
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int x = 0; x < 2; ++x)
      limit[r][x] = p.causal ? n - (p.M - 1 - (8 * r + 2 * t + x) % p.M) : n;
  const float sl2 = p.scale * kLog2e;
  // own keys that every token reads; what infinities and NaN V holds behind them
  // is left out, and added to the tokens that do read it at the end
  const int shown = p.causal ? max(0, n - (p.M - 1)) : n;
  int odd = 0;
  for (; i < hi; i += W) {
    float s[R][4];
    uint32_t pt[R][2];
    w.scores(s, [&](int x, int c) { return kf[x][c]; });
    const bool more = i + W < hi;
    if (more) load_k(i + W);
    if (!kBehind || i >= ahead) {
      w.weights(s, pt, 16 * (i - ahead), limit, sl2);
    } else {
      int all[R][2];
#pragma unroll
      for (int r = 0; r < R; ++r) all[r][0] = all[r][1] = np;
      w.weights(s, pt, 16 * i, all, sl2);
    }
    if (shown < n && 16 * (i - ahead) + 16 > shown) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          if (16 * (i - ahead) + 2 * t + (x & 1) + 8 * (x >> 1) >= shown && drop_odd<T>(vf[x][c])) odd = 1;
    }
    w.values(pt, [&](int x, int c) { return vf[x][c]; });
    if (more) load_v(i + W);
  }

  // ---- the warps' sums
  w.finish();
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (g == 0) {
        warp_m[warp][8 * r + 2 * t + x] = w.m[r][x];
        warp_l[warp][8 * r + 2 * t + x] = w.l[r][x];
      }
  odd = __syncthreads_or(odd);
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = 8 * r + 2 * t + x;
      float top = warp_m[0][row];
#pragma unroll
      for (int y = 1; y < W; ++y) top = fmaxf(top, warp_m[y][row]);
      if (row < rows) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          float4* at = reinterpret_cast<float4*>(&sum_o[warp][row][64 * c + 8 * g]);
          w.columns(r, x, c, ex2_approx(w.m[r][x] - top), at[0], at[1]);
        }
      }
      if (warp == 0 && g == 0) {
        float sum = 0.f;
#pragma unroll
        for (int y = 0; y < W; ++y) sum = fmaf(ex2_approx(warp_m[y][row] - top), warp_l[y][row], sum);
        block_m[row] = top;
        block_l[row] = sum;
      }
    }
  }
  __syncthreads();
  auto sum4 = [&](int row, int c) {
    float4 a = *reinterpret_cast<float4*>(&sum_o[0][row][4 * c]);
#pragma unroll
    for (int y = 1; y < W; ++y) add_weighted(a, 1.f, *reinterpret_cast<float4*>(&sum_o[y][row][4 * c]));
    return a;
  };
  if (p.splits > 1) {
    for (int e = threadIdx.x; e < rows * (D / 4); e += kThreads)
      *reinterpret_cast<float4*>(&sum_o[0][e / (D / 4)][4 * (e % (D / 4))]) = sum4(e / (D / 4), e % (D / 4));
    if (threadIdx.x == 0) block_odd = odd ? 1.f : 0.f;
    cluster_sync();
    // the blocks' references and sums, each read by a thread of its own
    for (int e = threadIdx.x; e < p.splits * kRows; e += kThreads)
      weight[e / kRows][e % kRows] = load_cluster(&block_m[e % kRows], e / kRows);
    odd = __syncthreads_or(shown < n && threadIdx.x < p.splits && load_cluster(&block_odd, threadIdx.x) != 0.f);
    if (threadIdx.x < kRows) {
      float top = kNoMax;
      for (int y = 0; y < p.splits; ++y) top = fmaxf(top, weight[y][threadIdx.x]);
      top_of[threadIdx.x] = top;
      float sum = 0.f;
#pragma unroll 4
      for (int y = 0; y < p.splits; ++y) {
        const float f = ex2_approx(weight[y][threadIdx.x] - top);
        weight[y][threadIdx.x] = f;
        sum = fmaf(f, load_cluster(&block_l[threadIdx.x], y), sum);
      }
      total[threadIdx.x] = sum;
    }
    __syncthreads();
  }
  // ---- the blocks' sums: each block finishes a share
  for (int e = threadIdx.x * p.splits + split; e < rows * (D / 4); e += p.splits * kThreads) {
    const int row = e / (D / 4), c = e % (D / 4);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.splits == 1) {
      acc = sum4(row, c);
    } else {
#pragma unroll 4
      for (int y = 0; y < p.splits; ++y) add_weighted(acc, weight[y][row], load_cluster4(&sum_o[0][row][4 * c], y));
    }
    if (odd) add_odd4(p.V.at(b, hk, shown) + 4 * c, p.V.sr, n - (p.M - 1) + row % p.M - shown, acc);
    decode_output(p, b, hk, row, c, p.splits == 1 ? block_m[row] : top_of[row], p.splits == 1 ? block_l[row] : total[row],
                  acc);
  }
  if (p.splits > 1) cluster_sync();  // no block leaves while its sums are read
  // behind a prefix: the launch before this one, for the join
  if (p.part_o) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// --------------------------------------------------------------------- stream
// The batch as one line of steps: entries in order, in each the groups of
// `side` items, in each the steps of `sub` 16-key tiles. All lanes of a warp
// hold the same numbers. The host keeps the line under 2^31.
template <typename T>
struct DecodeLine {
  const DecodeParams<T>& p;
  int groups, total, each, more;  // groups of an entry, steps, steps of a block, blocks with one more

  __device__ __forceinline__ int steps_of(int b) const {
    return ((valid_rows(p.lens, b, p.N) + 15) / 16 + p.sub - 1) / p.sub;
  }
  __device__ DecodeLine(const DecodeParams<T>& params) : p(params) {
    groups = (p.Hkv + p.side - 1) / p.side;
    total = before_entry(p.B);
    each = total / p.blocks;
    more = total % p.blocks;
  }
  // Steps of the entries before b.
  __device__ int before_entry(int b) const {
    if (!p.lens) return steps_of(0) * b * groups;
    int sum = 0;
    for (int e = threadIdx.x & 31; e < b; e += 32) sum += steps_of(e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum * groups;
  }
  // The first step of block c, and the block that has step `pos`.
  __device__ __forceinline__ int mark(int c) const { return c * each + min(c, more); }
  __device__ __forceinline__ int block_of(int pos) const {
    return pos < more * (each + 1) ? pos / (each + 1) : more + (pos - more * (each + 1)) / each;
  }
};

// A warp's place in the line: step j of `steps` (n keys) of its item in group
// `group` of entry b.
template <typename T>
struct DecodeCursor {
  const DecodeLine<T>& line;
  int left;  // steps of the run from here on
  int b, group, j, steps, n;
  __device__ __forceinline__ void entry() {
    n = valid_rows(line.p.lens, b, line.p.N);
    steps = line.steps_of(b);
  }
  __device__ DecodeCursor(const DecodeLine<T>& l, int pos, int end) : line(l), left(end - pos) {
    b = group = j = steps = n = 0;
    if (left <= 0) return;
    if (!line.p.lens) {
      b = pos / (line.steps_of(0) * line.groups);
      pos -= b * line.steps_of(0) * line.groups;
    } else {
      // the first entry whose end is past pos, 32 at a time
      const int lane = threadIdx.x & 31;
      for (;; b += 32) {
        const int own = b + lane < line.p.B ? line.steps_of(b + lane) * line.groups : 0;
        int upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const unsigned past = __ballot_sync(0xffffffffu, upto > pos);
        if (past) {
          const int first = __ffs(past) - 1;
          pos -= __shfl_sync(0xffffffffu, upto - own, first);
          b += first;
          break;
        }
        pos -= __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    entry();
    group = pos / steps;
    j = pos % steps;
  }
  // One step on; true if it opens another group.
  __device__ __forceinline__ bool step() {
    --left;
    if (++j < steps) return false;
    j = 0;
    if (++group == line.groups) {
      group = 0;
      do {
        ++b;
        if (left > 0) entry();
      } while (left > 0 && steps == 0);
    }
    return true;
  }
};

// Up to 192 KB on their way in an SM; more warps rather than longer rings, as a
// warp's own latencies are what it waits for otherwise. (Rings filled by
// cp.async cost 110 of 300 instructions a tile: 98 us for 64 x 1500 keys of 16
// heads of 64.)
template <int D, int R>
struct StreamCfg {
  static constexpr int kWarps = D == 64 ? 16 : (R == 1 ? 12 : 8);  // of a block, one block an SM
  static constexpr int kStages = D == 64 && R == 1 ? 3 : 2;
  static constexpr int kBox = 16 * 128;                            // 16 keys x 64 columns, 128-byte swizzle
  static constexpr int kStageBytes = 2 * (D / 64) * kBox;          // K, V
  static constexpr int kSumBytes = 8 * R * (D + 2) * 4;            // a warp's sums, references, row sums
  static constexpr int kOffSum = kWarps * kStages * kStageBytes;   // of one warp of each item
  static constexpr int kOffBar = kOffSum + kWarps / 2 * kSumBytes;
  static constexpr int kSmemBytes = kOffBar + 512;
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

// 4 entries of 8 kv heads, 4096 to 32768 keys of 128: 48 to 53 us without the
// join, 5.4 to 5.9 TB/s; blocks of equal work end 38 to 48 us after the start.
template <typename T, int D, int R>
__global__ void __launch_bounds__(32 * StreamCfg<D, R>::kWarps, 1)
    attn_decode_stream_kernel(const __grid_constant__ CUtensorMap tm_K, const __grid_constant__ CUtensorMap tm_V,
                              const __grid_constant__ DecodeParams<T> p) {
  using Cfg = StreamCfg<D, R>;
  constexpr int kRows = 8 * R, S = Cfg::kStages, kV = (D / 64) * Cfg::kBox;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // never, short of a toolchain that drops the alignment
    if (threadIdx.x == 0) publish_failure(1 + 500, p.status);
    return;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int place = warp % p.side, part = warp / p.side;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar) + warp * S;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Cfg::kOffBar + 8 * Cfg::kWarps * S);
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_K);
    tma_prefetch_desc(&tm_V);
    *abort_flag = 0;
  }
  if (lane == 0) {
    for (int x = 0; x < S; ++x) mbar_init(&bar[x], 1);
    fence_mbar_init();
  }
  __syncthreads();
  WaitCtx ctx{abort_flag, p.timeout_ns};
  const DecodeLine<T> line(p);
  DecodeCursor<T> at(line, line.mark(blockIdx.x), line.mark(blockIdx.x + 1));
  DecodeCursor<T> ahead = at;
  uint8_t* own = smem + warp * (S * Cfg::kStageBytes);
  const uint64_t policy = l2_policy_evict_first();
  int loads = 0;
  auto load = [&](int stage) {  // the next step that has a tile for this warp; all lanes walk, one loads
    for (bool found = false; ahead.left > 0 && !found; ahead.step()) {
      const int hk = ahead.group * p.side + place, i = ahead.j * p.sub + part;
      found = hk < p.Hkv && 16 * i < ahead.n;
      if (found && lane == 0) {
        uint8_t* dst = own + stage * Cfg::kStageBytes;
        mbar_arrive_expect_tx(&bar[stage], Cfg::kStageBytes);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          tma_load_4d(dst + c * Cfg::kBox, &tm_K, &bar[stage], 64 * c, 16 * i, hk, ahead.b, policy);
          tma_load_4d(dst + kV + c * Cfg::kBox, &tm_V, &bar[stage], 64 * c, 16 * i, hk, ahead.b, policy);
        }
      }
      if (found) ++loads;
    }
  };
#pragma unroll 1
  for (int x = 0; x < S; ++x) load(x);
  DecodeWarp<T, D, R> w;
  const float sl2 = p.scale * kLog2e;
  int stage = 0, turn = 0, slot = 2 * blockIdx.x, done = 0;
  bool whole = at.j == 0;  // the group's keys from the first on, in this block
  bool fresh = true, ok = true;
  while (at.left > 0) {
    const int b = at.b, hk = at.group * p.side + place, i = at.j * p.sub + part, n = at.n;
    const bool mine = hk < p.Hkv;
    if (fresh && mine) w.begin(p, b, hk);
    fresh = false;
    const bool last = at.j + 1 == at.steps;
    const bool opens = at.step();
    // (after a wait that gave up, a warp still walks to the block's barriers)
    if (mine && 16 * i < n && ok) ok = __all_sync(0xffffffffu, mbar_wait(&bar[stage], turn, ctx, 501));
    if (mine && 16 * i < n && ok) {
    uint8_t* src = own + stage * Cfg::kStageBytes;
    const int left = n - 16 * i;
    if (left < 16) {  // V behind the last key may hold anything
      for (int x = lane; x < (16 - left) * (D / 8); x += 32) {
        const int row = left + x / (D / 8), c = x % (D / 8);
        *reinterpret_cast<uint4*>(src + kV + (c >> 3) * Cfg::kBox + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
            make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();  // the next copy into this stage comes behind these stores
      __syncwarp();
    }
    // 16 bytes at column 8 `chunk` of a key's row
    auto piece = [&](const uint8_t* tile, int row, int chunk) {
      return *reinterpret_cast<const uint4*>(tile + (chunk >> 3) * Cfg::kBox + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
    };
    float s[R][4];
    uint32_t pt[R][2];
    int limit[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) limit[r][0] = limit[r][1] = n;
    w.scores(s, [&](int x, int c) { return piece(src, g + 8 * x, 4 * c + t); });
    w.weights(s, pt, 16 * i, limit, sl2);
    w.values(pt, [&](int x, int c) { return piece(src + kV, 2 * t + (x & 1) + 8 * (x >> 1), 8 * c + g); });
    __syncwarp();
    load(stage);
    ++done;
    if (++stage == S) {
      stage = 0;
      turn ^= 1;
    }
    }
    if (!opens && at.left > 0) continue;
    // ---- the end of the group or the run: the first warp of each item gathers
    // the others' sums, in order
    if (mine) w.finish();
    float* sums = reinterpret_cast<float*>(smem + Cfg::kOffSum + place * Cfg::kSumBytes);
#pragma unroll 1
    for (int y = 1; y < p.sub; ++y) {
      if (mine && part == y) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int row = 8 * r + 2 * t + x;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              float4* o4 = reinterpret_cast<float4*>(sums + row * D + 64 * c + 8 * g);
              w.columns(r, x, c, 1.f, o4[0], o4[1]);
            }
            if (g == 0) {
              sums[kRows * D + row] = w.m[r][x];
              sums[kRows * (D + 1) + row] = w.l[r][x];
            }
          }
      }
      __syncthreads();
      if (mine && part == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int row = 8 * r + 2 * t + x;
            const float m = sums[kRows * D + row], top = fmaxf(m, w.m[r][x]);
            const float f = ex2_approx(w.m[r][x] - top), h = ex2_approx(m - top);
            w.m[r][x] = top;
            w.l[r][x] = fmaf(h, sums[kRows * (D + 1) + row], f * w.l[r][x]);
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                float& o = w.o[r][4 * c + e / 2][x + 2 * (e & 1)];
                o = fmaf(h, sums[row * D + 64 * c + 8 * g + e], f * o);
              }
          }
      }
      __syncthreads();
    }
    if (mine && part == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = 8 * r + 2 * t + x;
          if (row >= p.G * p.M) continue;
          const float2 ml = make_float2(w.m[r][x], w.l[r][x]);
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            float4 a, d;
            w.columns(r, x, c, 1.f, a, d);
            const int col4 = 16 * c + 2 * g;
            if (whole && last) {
              decode_output(p, b, hk, row, col4, ml.x, ml.y, a);
              decode_output(p, b, hk, row, col4 + 1, ml.x, ml.y, d);
            } else {
              const int64_t to = (static_cast<int64_t>(slot) * p.side + place) * kRows + row;
              reinterpret_cast<float4*>(p.run_o + to * D)[col4] = a;
              reinterpret_cast<float4*>(p.run_o + to * D)[col4 + 1] = d;
              if (col4 == 0) p.run_ml[to] = ml;
            }
          }
        }
      }
      __syncwarp();
    }
    whole = true;
    slot = 2 * blockIdx.x + 1;  // a block's later partial group is its last
    fresh = true;
  }
  if (lane == 0 && *abort_flag)  // every copy in flight ends before the block does
    for (int x = done; x < loads; ++x) mbar_wait_drain(&bar[x % S], (x / S) & 1, p.timeout_ns);
  __syncthreads();
  if (threadIdx.x == 0) publish_failure(*abort_flag, p.status);
}

// Joins the partial sums of one row (a block each; a thread takes 4 columns,
// over a quarter of the sums), if its keys fell to several blocks. 5 us behind
// its launch for 256 rows of some 18 sums, bound by the latency of lengths,
// references and sums in turn.
template <typename T, int D, int R>
__global__ void __launch_bounds__(D) attn_decode_join_kernel(const __grid_constant__ DecodeParams<T> p) {
  constexpr int kRows = 8 * R, kMost = 256;
  __shared__ float4 part[4][D / 4];
  __shared__ float weight[kMost], mass[kMost], reduce[2][D / 32];
  const int rows = p.G * p.M, q = blockIdx.x % rows;
  const int hk = blockIdx.x / rows % p.Hkv, b = blockIdx.x / rows / p.Hkv;
  const DecodeLine<T> line(p);
  const int steps = line.steps_of(b);
  const int c = threadIdx.x % (D / 4), quarter = threadIdx.x / (D / 4);
  if (steps == 0) {  // an entry without keys: O = 0, LSE = -inf
    if (quarter == 0) decode_output(p, b, hk, q, c, 0.f, 0.f, make_float4(0.f, 0.f, 0.f, 0.f));
    asm volatile("griddepcontrol.wait;" ::: "memory");  // never done before the launch before it
    return;
  }
  const int start = line.before_entry(b) + hk / p.side * steps;
  const int c0 = line.block_of(start), c1 = line.block_of(start + steps - 1);
  const int count = c1 - c0 + 1;
  const int skip = line.mark(c0) < start ? 1 : 0;  // a block that begins in the group has it in its first slot
  auto at = [&](int k) {  // the sum of block c0 + k
    return ((2ll * (c0 + k) + (k == 0 ? skip : 0)) * p.side + hk % p.side) * kRows + q;
  };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (count == 1) return;
  float top = kNoMax, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  // kMost sums at a time: references and sums first, a thread each, then O
  for (int from = 0; from < count; from += kMost) {
    const int here = min(kMost, count - from);
    float most = top;
    for (int k = threadIdx.x; k < here; k += D) {
      const float2 ml = __ldcg(p.run_ml + at(from + k));
      weight[k] = ml.x;
      mass[k] = ml.y;
      most = fmaxf(most, weight[k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (threadIdx.x % 32 == 0) reduce[0][threadIdx.x / 32] = most;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < D / 32; ++x) most = fmaxf(most, reduce[0][x]);
    const float keep = ex2_approx(top - most);
    top = most;
    sum *= keep;
    acc = make_float4(keep * acc.x, keep * acc.y, keep * acc.z, keep * acc.w);
    float mine = 0.f;
    for (int k = threadIdx.x; k < here; k += D) {
      weight[k] = ex2_approx(weight[k] - top);
      mine = fmaf(weight[k], mass[k], mine);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (threadIdx.x % 32 == 0) reduce[1][threadIdx.x / 32] = mine;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < D / 32; ++x) sum += reduce[1][x];
    const int hi = here * (quarter + 1) / 4;
#pragma unroll 8
    for (int k = here * quarter / 4; k < hi; ++k)
      add_weighted(acc, weight[k], __ldcg(reinterpret_cast<const float4*>(p.run_o + at(from + k) * D) + c));
    __syncthreads();
  }
  part[quarter][c] = acc;
  __syncthreads();
  if (quarter > 0) return;
#pragma unroll
  for (int k = 1; k < 4; ++k) add_weighted(acc, 1.f, part[k][c]);
  decode_output(p, b, hk, q, c, top, sum, acc);
}

}  // namespace fmha_sm100
