// Attention of a few query rows (single tokens): every key and value is read
// once, from global memory straight into tensor-core fragments.
//
// The floor is the bytes of K and V, so the kernel is built around loads in
// flight and has no shared-memory stage. The products are transposed, keys
// and value columns on the 16-row side of mma.m16n8k16 and the query rows on
// its 8-column side (R = 1: up to 8 rows of a kv head, R = 2: up to 16):
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
// accumulator to operand layout by movmatrix.
//
// A warp takes every fourth tile of 16 keys of its block, K and V of the next
// tile on their way while it computes. The rows' references m move only when
// some row's maximum is over 2^8 times its own (see attn_fwd_kernel; the same
// bias in fp16). The four warps' sums meet in shared memory, the blocks that
// split one kv head's keys form a cluster and meet in each other's shared
// memory, in a fixed order: one launch, no workspace, the same bits each time.
//
// With `parts`, O and LSE of other keys (a shared prefix) join at the end.
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
  int row_tiles;    // tiles of 8 R query rows of a kv head
  int splits;       // blocks (a cluster) that share a tile's keys
  bool causal;      // token m reads lens - (M - 1 - m) keys
  float scale;
  const float* part_o;  // null, or [parts][row][D] and [parts][row] to join
  const float* part_lse;
  int parts;
  int64_t all_rows;
};

constexpr int kDecodeWarps = 4;
constexpr float kNoMax = -3.0e38f;  // the reference of a row before its first key

template <typename T, int D, int R>
__global__ void __launch_bounds__(32 * kDecodeWarps)
    attn_decode_kernel(const __grid_constant__ DecodeParams<T> p) {
  constexpr bool kB = Elem<T>::kBF16;
  constexpr float kBias = kB ? 0.f : 6.f;
  constexpr int kRows = 8 * R;
  __shared__ __align__(16) float sum_o[kDecodeWarps][kRows][D];
  __shared__ float warp_m[kDecodeWarps][kRows], warp_l[kDecodeWarps][kRows];
  __shared__ float block_m[kRows], block_l[kRows];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % p.splits;
  int u = blockIdx.x / p.splits;
  const int tile = u % p.row_tiles;
  u /= p.row_tiles;
  const int hk = u % p.Hkv, b = u / p.Hkv;
  const int rows = p.G * p.M, row0 = tile * kRows;
  const int n = valid_rows(p.lens, b, p.N);
  const int tiles = (n + 15) / 16;
  const int lo = static_cast<int>(static_cast<int64_t>(tiles) * split / p.splits);
  const int hi = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / p.splits);

  // this thread's pieces: K rows g and g + 8 of a tile, 16 bytes at column
  // 8 t of each 32; V rows 2t, 2t + 1, 2t + 8, 2t + 9, 16 bytes at column 8 g
  // of each 64
  uint4 kf[2][D / 32], vf[4][D / 64];
  auto load_k = [&](int i) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int key = 16 * i + g + 8 * x;
      const T* at = p.K.at(b, hk, key) + 8 * t;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) kf[x][c] = key < n ? load_stream(at + 32 * c) : make_uint4(0, 0, 0, 0);
    }
  };
  auto load_v = [&](int i) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int key = 16 * i + 2 * t + (x & 1) + 8 * (x >> 1);
      const T* at = p.V.at(b, hk, key) + 8 * g;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) vf[x][c] = key < n ? load_stream(at + 64 * c) : make_uint4(0, 0, 0, 0);
    }
  };
  int i = lo + warp;
  if (i < hi) {
    load_k(i);
    load_v(i);
  }
  // Q of row g (+ 8 of the second half), in K's order of columns
  uint4 qf[R][D / 32];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + 8 * r + g;
    const T* at = p.Q.at(b, hk * p.G + row / p.M, row % p.M) + 8 * t;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
      qf[r][c] = row < rows ? *reinterpret_cast<const uint4*>(at + 32 * c) : make_uint4(0, 0, 0, 0);
  }
  // keys that rows 2t and 2t + 1 may read
  int limit[R][2];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int x = 0; x < 2; ++x)
      limit[r][x] = p.causal ? n - (p.M - 1 - (row0 + 8 * r + 2 * t + x) % p.M) : n;

  float o[R][D / 16][4];
  float m[R][2], l[R][2];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[r][c][x] = 0.f;
    m[r][0] = m[r][1] = kNoMax;
    l[r][0] = l[r][1] = 0.f;
  }
  const float sl2 = p.scale * kLog2e;

  for (; i < hi; i += kDecodeWarps) {
    float s[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        mma_16816<kB>(s[r], kf[0][c].x, kf[1][c].x, kf[0][c].y, kf[1][c].y, qf[r][c].x, qf[r][c].y);
        mma_16816<kB>(s[r], kf[0][c].z, kf[1][c].z, kf[0][c].w, kf[1][c].w, qf[r][c].z, qf[r][c].w);
      }
    }
    const bool more = i + kDecodeWarps < hi;
    if (more) load_k(i + kDecodeWarps);
    // s[r][0], [1]: key 16 i + g, rows 2t and 2t + 1; [2], [3]: key + 8
    bool move = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int key = 16 * i + g + 8 * (x >> 1);
        s[r][x] = key < limit[r][x & 1] ? s[r][x] * sl2 : -INFINITY;
      }
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
    uint32_t pt[R][2];
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
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vf[0][c]);
      const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vf[1][c]);
      const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vf[2][c]);
      const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vf[3][c]);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t a0 = __byte_perm(v0[x], v1[x], 0x5410), a1 = __byte_perm(v0[x], v1[x], 0x7632);
        const uint32_t a2 = __byte_perm(v2[x], v3[x], 0x5410), a3 = __byte_perm(v2[x], v3[x], 0x7632);
#pragma unroll
        for (int r = 0; r < R; ++r) mma_16816<kB>(o[r][4 * c + x], a0, a1, a2, a3, pt[r][0], pt[r][1]);
      }
    }
    if (more) load_v(i + kDecodeWarps);
  }

  // ---- the warps' sums: o[r][4c + x][y] is column 64c + 8g + 2x + y / 2 of
  // row 8r + 2t + y % 2
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int y = 4; y < 32; y <<= 1) l[r][x] += __shfl_xor_sync(0xffffffffu, l[r][x], y);
      if (g == 0) {
        warp_m[warp][8 * r + 2 * t + x] = m[r][x];
        warp_l[warp][8 * r + 2 * t + x] = l[r][x];
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = 8 * r + 2 * t + x;
      float top = warp_m[0][row];
#pragma unroll
      for (int w = 1; w < kDecodeWarps; ++w) top = fmaxf(top, warp_m[w][row]);
      const float f = ex2_approx(m[r][x] - top);
      if (row0 + row < rows) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          float* at = &sum_o[warp][row][64 * c + 8 * g];
          *reinterpret_cast<float4*>(at) = make_float4(f * o[r][4 * c][x], f * o[r][4 * c][x + 2], f * o[r][4 * c + 1][x],
                                                       f * o[r][4 * c + 1][x + 2]);
          *reinterpret_cast<float4*>(at + 4) =
              make_float4(f * o[r][4 * c + 2][x], f * o[r][4 * c + 2][x + 2], f * o[r][4 * c + 3][x],
                          f * o[r][4 * c + 3][x + 2]);
        }
      }
      if (warp == 0 && g == 0) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) sum = fmaf(ex2_approx(warp_m[w][row] - top), warp_l[w][row], sum);
        block_m[row] = top;
        block_l[row] = sum;
      }
    }
  }
  __syncthreads();
  const int real = min(kRows, rows - row0);
  if (p.splits > 1) {
    for (int e = threadIdx.x; e < real * (D / 4); e += 32 * kDecodeWarps) {
      const int row = e / (D / 4), c = e % (D / 4);
      float4 a = *reinterpret_cast<float4*>(&sum_o[0][row][4 * c]);
#pragma unroll
      for (int w = 1; w < kDecodeWarps; ++w) {
        const float4 v = *reinterpret_cast<float4*>(&sum_o[w][row][4 * c]);
        a.x += v.x;
        a.y += v.y;
        a.z += v.z;
        a.w += v.w;
      }
      *reinterpret_cast<float4*>(&sum_o[0][row][4 * c]) = a;
    }
    cluster_sync();
  }
  if (p.part_o) asm volatile("griddepcontrol.wait;" ::: "memory");  // the launch that wrote the parts
  // ---- the blocks' sums, and the parts: each block finishes a share
  for (int e = split * 32 * kDecodeWarps + threadIdx.x; e < real * (D / 4); e += p.splits * 32 * kDecodeWarps) {
    const int row = e / (D / 4), c = e % (D / 4);
    const int q = row0 + row, head = hk * p.G + q / p.M, tok = q % p.M;
    const int64_t id = (static_cast<int64_t>(b) * p.Hkv * p.G + head) * p.M + tok;
    float top = block_m[row];
    for (int k = 0; k < p.splits; ++k)
      if (k != split) top = fmaxf(top, load_cluster(&block_m[row], k));
    for (int k = 0; k < p.parts; ++k) top = fmaxf(top, p.part_lse[k * p.all_rows + id] * kLog2e);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float w, float4 v) {
      acc.x = fmaf(w, v.x, acc.x);
      acc.y = fmaf(w, v.y, acc.y);
      acc.z = fmaf(w, v.z, acc.z);
      acc.w = fmaf(w, v.w, acc.w);
    };
    if (p.splits == 1) {
      const float w = ex2_approx(block_m[row] - top);
      sum = w * block_l[row];
#pragma unroll
      for (int k = 0; k < kDecodeWarps; ++k) add(w, *reinterpret_cast<float4*>(&sum_o[k][row][4 * c]));
    } else {
      for (int k = 0; k < p.splits; ++k) {
        const float w = ex2_approx(load_cluster(&block_m[row], k) - top);
        sum = fmaf(w, load_cluster(&block_l[row], k), sum);
        add(w, load_cluster4(&sum_o[0][row][4 * c], k));
      }
    }
    for (int k = 0; k < p.parts; ++k) {
      // a part is normalised: its sum is 1 at the reference LSE log2e
      const float w = ex2_approx(fmaf(p.part_lse[k * p.all_rows + id], kLog2e, -top));
      sum += w;
      add(w, reinterpret_cast<const float4*>(p.part_o + (k * p.all_rows + id) * D)[c]);
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // NaN stays
    *reinterpret_cast<uint2*>(p.O.at(b, head, tok) + 4 * c) =
        make_uint2(Elem<T>::pack(inv * acc.x, inv * acc.y), Elem<T>::pack(inv * acc.z, inv * acc.w));
    if (c == 0) p.LSE[id] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  }
  if (p.splits > 1) cluster_sync();  // no block leaves while its sums are read
}

}  // namespace fmha_sm100
