// Backward of attention on the tensor cores, from O and LSE, with the weights
// P = exp(S - LSE) rebuilt on chip:
//
//   D = rowsum(dO * O),  dP = dO V^T,  dS = P (dP - D),
//   dQ = scale dS K,  dK = scale sum dS^T Q,  dV = sum P^T dO
//
// Launches: attn_delta_kernel (D, and LSE in powers of two, per packed row),
// attn_dq_kernel (query-major: three products a tile pair), attn_dkv_kernel
// (key-major: four), attn_bwd_join_kernel. Two kernels with S and dP formed
// in both cost 14 M N d operations where one would do with 10, but one would
// have to add dQ up across key tiles by atomics, in no fixed order.
//
// Rows are packed into tiles of 128 as in the forward (RowPack), so that the
// short query rows of all heads of a kv head share a tile; the rows of a box
// that hold no row have LSE = +inf, hence P = 0.
//
// Work is divided by steps (one key tile for one pair of row tiles; one row
// tile for one key tile), counted on the device from the lengths. If whole
// items leave the SMs uneven, each CTA takes an equal run of steps instead;
// an item that falls to several CTAs leaves fp32 sums for the join, which adds
// them in order.
//
// P and dS are rounded to 16 bits for the tensor cores, after dS was formed
// from the fp32 P. In fp16, P is held times 2^10 and dS times 2^e with e from
// the largest |dO| and |V|, so that 2 d |dO| |V| 2^e <= 65504: dS cannot
// overflow, and gradients of any size keep fp16's precision.
#pragma once

#include "fmha_attn_fwd.cuh"

namespace fmha_sm100 {

template <typename T>
struct BwdParams {
  RowPack rows;       // S = 1, Gt divides G
  int B, Hkv, N, pairs;
  const int* lens;
  View<T> dQ, dK, dV;
  const float* lse2;  // [B * Hkv * tiles * 128] LSE log2e, packed rows
  const float* delta; // the same rows' D
  const float2* amax; // [blocks of attn_delta_kernel]: largest |dO|, |V| (fp16 only)
  int amax_count;
  float* part;        // [2 * grid][2][128][D] partial sums
  float scale;
  KernelStatus* status;
  uint64_t timeout_ns;
};

// ------------------------------------------------------------------- schedule
// Steps of an item are consecutive; the items of a batch entry follow one
// another, entries in order. `q_major`: items are (kv head, tile pair) with a
// step for each key tile; else (kv head, key tile) with a step for each row
// tile.
struct BwdUnit {
  int b, hk, idx;  // idx: tile pair, or key tile
  int lo, hi;      // steps of the item
  int len;         // its steps in all
  int slot;        // partial-sum slot, or -1 for a whole item
  int n;           // valid keys of the entry
};

// Steps that a division by steps has to save, as its partial sums cost about
// as much, and the least number of steps of a CTA under it.
constexpr int kBwdSpare = 8, kBwdLeast = 4;
__host__ __device__ inline bool bwd_by_steps(int64_t items, int64_t most, int64_t total, int64_t grid) {
  return (items + grid - 1) / grid * most > (total + grid - 1) / grid + kBwdSpare;
}
__host__ __device__ inline int bwd_parts(int64_t total, int grid) {
  const int64_t most = (total + kBwdLeast - 1) / kBwdLeast;
  return most < grid ? (most > 0 ? static_cast<int>(most) : 1) : grid;
}

template <typename T, bool kQMajor>
struct BwdSchedule {
  const BwdParams<T>& p;
  int grid, parts, cta;  // parts: the CTAs that a division by steps uses
  int64_t total, items;
  bool by_steps;
  int64_t pos, end;  // steps, or items
  int b;             // the entry that the walk has reached, and what lies before it
  int64_t before;
  int first_unit;

  __device__ __forceinline__ int key_tiles(int e) const {
    return (valid_rows(p.lens, e, p.N) + kTile - 1) / kTile;
  }
  __device__ __forceinline__ int64_t items_of(int nt) const {
    return kQMajor ? (nt > 0 ? static_cast<int64_t>(p.Hkv) * p.pairs : 0) : static_cast<int64_t>(p.Hkv) * nt;
  }
  __device__ __forceinline__ int len_of(int nt) const { return kQMajor ? nt : p.rows.tiles; }
  __device__ __forceinline__ int64_t mark(int c) const { return c < parts ? total * c / parts : total; }

  __device__ BwdSchedule(const BwdParams<T>& params, int g, int c) : p(params), grid(g), cta(c) {
    total = items = 0;
    int most = 0;
    if (!p.lens) {
      most = key_tiles(0);
      items = items_of(most) * p.B;
      total = items * len_of(most);
    } else {
      for (int e = 0; e < p.B; ++e) {
        const int nt = key_tiles(e);
        most = max(most, nt);
        items += items_of(nt);
        total += items_of(nt) * len_of(nt);
      }
    }
    by_steps = bwd_by_steps(items, len_of(most), total, grid);
    parts = bwd_parts(total, grid);
    pos = by_steps ? mark(c) : c;
    end = by_steps ? mark(c + 1) : items;
    b = 0;
    before = 0;
    first_unit = 1;
  }
  // The next unit of this CTA; false when there is none.
  __device__ bool next(BwdUnit& u) {
    if (pos >= end) return false;
    int nt;
    for (;; ++b) {
      nt = key_tiles(b);
      const int64_t n = by_steps ? items_of(nt) * len_of(nt) : items_of(nt);
      if (pos < before + n) break;
      before += n;
    }
    u.b = b;
    u.n = valid_rows(p.lens, b, p.N);
    u.len = len_of(nt);
    int64_t item = pos - before;
    u.lo = 0;
    u.hi = u.len;
    u.slot = -1;
    if (by_steps) {
      u.lo = static_cast<int>(item % u.len);
      item /= u.len;
      u.hi = static_cast<int>(min(static_cast<int64_t>(u.len), u.lo + (end - pos)));
      if (u.hi - u.lo < u.len) u.slot = 2 * cta + 1 - first_unit;
      pos += u.hi - u.lo;
    } else {
      pos += grid;
    }
    first_unit = 0;
    const int per = kQMajor ? p.pairs : nt;
    u.hk = static_cast<int>(item / per);
    u.idx = static_cast<int>(item % per);
    return true;
  }
};

// The power of two by which fp16 holds dS (see the top), 0 for bf16.
template <typename T, int D>
__device__ __forceinline__ int ds_exponent(const BwdParams<T>& p, int lane) {
  if (Elem<T>::kBF16) return 0;
  float2 a = make_float2(0.f, 0.f);
  for (int i = lane; i < p.amax_count; i += 32) {
    const float2 v = __ldcg(p.amax + i);
    a.x = fmaxf(a.x, v.x);
    a.y = fmaxf(a.y, v.y);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.x = fmaxf(a.x, __shfl_xor_sync(0xffffffffu, a.x, o));
    a.y = fmaxf(a.y, __shfl_xor_sync(0xffffffffu, a.y, o));
  }
  // exponents e with x < 2^e; a zero, infinity or NaN leaves dS as it is
  if (!(a.x > 0.f && a.x < INFINITY && a.y > 0.f && a.y < INFINITY)) return 0;
  const int ex = static_cast<int>(__float_as_uint(a.x) >> 23) - 126, ey = static_cast<int>(__float_as_uint(a.y) >> 23) - 126;
  const int e = 15 - (D == 128 ? 8 : 7) - ex - ey;  // 2 d 2^ex 2^ey 2^e = 2^15
  return e < -40 ? -40 : (e > 60 ? 60 : e);
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// ==================================================================== delta
// Per packed row: lse2 = LSE log2e (0 for a row without keys, +inf where the
// tile holds no row) and D, D / 8 threads a row. In fp16 also the largest |dO|
// and valid |V| that the block saw.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    attn_delta_kernel(View<T> dO, View<T> O, View<T> V, const float* __restrict__ LSE, BwdParams<T> p,
                      float* __restrict__ lse2, float* __restrict__ delta, float2* __restrict__ amax) {
  constexpr int kPer = D / 8;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int chunk = threadIdx.x % kPer;
  const int64_t rows = static_cast<int64_t>(p.B) * p.Hkv * p.rows.tiles * kTile;
  float top_do = 0.f, top_v = 0.f;
  auto widest = [](float top, const uint32_t (&w)[4]) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float2 v = Elem<T>::unpack(w[x]);
      top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
    }
    return top;
  };
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (256 / kPer) + threadIdx.x / kPer; i < rows;
       i += static_cast<int64_t>(gridDim.x) * (256 / kPer)) {
    const int r = static_cast<int>(i % kTile);
    const int64_t u = i / kTile;
    const int tile = static_cast<int>(u % p.rows.tiles);
    const int64_t bh = u / p.rows.tiles;
    const int hk = static_cast<int>(bh % p.Hkv), b = static_cast<int>(bh / p.Hkv);
    int m, g, s;
    const bool real = p.rows.row(tile, r, m, g, s);
    float acc = 0.f;
    if (real) {
      const uint4 x = *(reinterpret_cast<const uint4*>(dO.at(b, hk * p.rows.G + g, m)) + chunk);
      const uint4 y = *(reinterpret_cast<const uint4*>(O.at(b, hk * p.rows.G + g, m)) + chunk);
      const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float2 a = Elem<T>::unpack(xw[t]), c = Elem<T>::unpack(yw[t]);
        acc = fmaf(a.x, c.x, acc);
        acc = fmaf(a.y, c.y, acc);
      }
      if (!Elem<T>::kBF16) top_do = widest(top_do, xw);
    }
#pragma unroll
    for (int o = kPer / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o, kPer);
    if (chunk == 0) {
      float l = INFINITY;
      if (real) {
        l = LSE[(static_cast<int64_t>(b) * p.Hkv * p.rows.G + hk * p.rows.G + g) * p.rows.M + m];
        l = l == -INFINITY ? 0.f : l * kLog2e;
      }
      lse2[i] = l;
      delta[i] = acc;
    }
  }
  if (!Elem<T>::kBF16) {
    const int64_t keys = static_cast<int64_t>(p.B) * p.Hkv * p.N;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * (256 / kPer) + threadIdx.x / kPer; i < keys;
         i += static_cast<int64_t>(gridDim.x) * (256 / kPer)) {
      const int key = static_cast<int>(i % p.N);
      const int64_t bh = i / p.N;
      const int hk = static_cast<int>(bh % p.Hkv), b = static_cast<int>(bh / p.Hkv);
      if (key < valid_rows(p.lens, b, p.N)) {
        const uint4 x = *(reinterpret_cast<const uint4*>(V.at(b, hk, key)) + chunk);
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
        top_v = widest(top_v, xw);
      }
    }
    __shared__ float2 tops[8];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      top_do = fmaxf(top_do, __shfl_xor_sync(0xffffffffu, top_do, o));
      top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, o));
    }
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = make_float2(top_do, top_v);
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) {
        top_do = fmaxf(top_do, tops[w].x);
        top_v = fmaxf(top_v, tops[w].y);
      }
      amax[blockIdx.x] = make_float2(top_do, top_v);
    }
  }
}

// Zeroes rows [from, rows) of each head of a tensor, by the given threads.
template <typename T, int D>
__device__ __forceinline__ void zero_rows(const View<T>& v, int b, int heads, int from, int rows, int64_t thread,
                                          int64_t threads) {
  const int64_t per = static_cast<int64_t>(rows - from) * (D / 8);
  for (int64_t i = thread; i < per * heads; i += threads) {
    const int h = static_cast<int>(i / per);
    const int64_t w = i % per;
    *(reinterpret_cast<uint4*>(v.at(b, h, from + w / (D / 8))) + w % (D / 8)) = make_uint4(0, 0, 0, 0);
  }
}

// One row's 32 columns: 16-bit, scaled, or fp32 into a partial-sum slot.
__device__ __forceinline__ void store_part_32(float* out, const uint32_t (&v)[32]) {
#pragma unroll
  for (int y = 0; y < 8; ++y)
    reinterpret_cast<uint4*>(out)[y] = make_uint4(v[4 * y], v[4 * y + 1], v[4 * y + 2], v[4 * y + 3]);
}

// ======================================================================= dq
// One CTA walks units (two row tiles, a run of key tiles). Per tile and step:
//   S = Q K^T -> TMEM R;  the tile's warpgroup (thread = row) takes S into
//   registers and frees R;  dP = dO V^T -> R while it forms P;
//   dS (16-bit) -> R;  dQ += dS K (A from TMEM)
// and the tensor core works on the other tile in between.
//
// Shared memory (D = 128): Q, dO of both tiles 128 KB, K x2, V x1 = 224 KB.
// TMEM: R_t [128 t, +128), dQ_t [256 + D t, +D).
template <int D>
struct DqCfg2 {
  static constexpr int kTileBytes = (D / kBoxCols) * kBoxBytes;
  static constexpr int kSK = D == 128 ? 2 : 4, kSV = D == 128 ? 1 : 4;
  static constexpr int kOffQ = 0, kOffdO = 2 * kTileBytes;
  static constexpr int kOffK = 4 * kTileBytes, kOffV = kOffK + kSK * kTileBytes;
  static constexpr int kOffBar = kOffV + kSV * kTileBytes;
  static constexpr int kSmemBytes = kOffBar + 512;
  static constexpr int kThreads = 384;
  // 2 * 128 * 208 + 128 * 80 of the launch's 384 * 168 registers
  static constexpr int kComputeRegs = 208, kOtherRegs = 80;
  static_assert(2 * kComputeRegs + kOtherRegs <= 3 * 168, "register split");
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

enum DqBar2 : int {
  kBqQFull0 = 0,    // + tile: Q and dO
  kBqQEmpty0 = 2,   // + tile: the unit's last dP of the tile is done
  kBqKFull0 = 4,    // + slot (up to 4)
  kBqKEmpty0 = 8,
  kBqVFull0 = 12,
  kBqVEmpty0 = 16,
  kBqSFull0 = 20,   // + tile
  kBqSRead0 = 22,   // + tile: S is in registers (4 warps)
  kBqXFull0 = 24,   // + tile: dP
  kBqDSFull0 = 26,  // + tile: dS written (4 warps)
  kBqAcc0 = 28,     // + tile: the unit's dQ is complete
  kBqAccEmpty0 = 30,// + tile: and read (4 warps)
  kBqDrain = 32,
  kNumBqBars = 33,
};

template <typename T, int D>
__global__ void __launch_bounds__(DqCfg2<D>::kThreads, 1)
    attn_dq_kernel(const __grid_constant__ CUtensorMap tm_Q, const __grid_constant__ CUtensorMap tm_K,
                   const __grid_constant__ CUtensorMap tm_V, const __grid_constant__ CUtensorMap tm_dO,
                   const __grid_constant__ BwdParams<T> p) {
  using Cfg = DqCfg2<D>;
  constexpr bool kB = Elem<T>::kBF16;
  constexpr int SK = Cfg::kSK, SV = Cfg::kSV;
  constexpr int kPBias = kB ? 0 : 10;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // never, short of a toolchain that drops the alignment
    if (threadIdx.x == 0) publish_failure(1 + 300, p.status);
    return;
  }
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kNumBqBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bar[kBqQFull0 + t], 1);
      mbar_init(&bar[kBqQEmpty0 + t], 1);
      mbar_init(&bar[kBqSFull0 + t], 1);
      mbar_init(&bar[kBqSRead0 + t], 4);
      mbar_init(&bar[kBqXFull0 + t], 1);
      mbar_init(&bar[kBqDSFull0 + t], 4);
      mbar_init(&bar[kBqAcc0 + t], 1);
      mbar_init(&bar[kBqAccEmpty0 + t], 4);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&bar[kBqKFull0 + s], 1);
      mbar_init(&bar[kBqKEmpty0 + s], 1);
      mbar_init(&bar[kBqVFull0 + s], 1);
      mbar_init(&bar[kBqVEmpty0 + s], 1);
    }
    mbar_init(&bar[kBqDrain], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  WaitCtx ctx{abort_flag, p.timeout_ns};
  // lse2, delta and the exponents come from the launch before; the launch after needs only those
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int q_tiles = p.rows.tiles;

  if (warp >= 8) {
    regs_lower<Cfg::kOtherRegs>();
    if (warp == 8 && lane == 0) {
      // ---- TMA producer
      tma_prefetch_desc(&tm_Q);
      tma_prefetch_desc(&tm_K);
      tma_prefetch_desc(&tm_V);
      tma_prefetch_desc(&tm_dO);
      const uint64_t pol_q = l2_policy_evict_first(), pol_kv = l2_policy_evict_last();
      const uint32_t q_bytes = static_cast<uint32_t>(p.rows.Mt * p.rows.Gt) * 128u * (D / kBoxCols);
      int nq[2] = {0, 0}, nk = 0, nv = 0;
      bool ok = true;
      auto load_q = [&](const BwdUnit& u, int t) {
        if (nq[t] > 0 && !mbar_wait(&bar[kBqQEmpty0 + t], (nq[t] - 1) & 1, ctx, 301)) return false;
        const int tile = 2 * u.idx + t;
        const int m0 = tile % p.rows.nm * p.rows.Mt, h0 = u.hk * p.rows.G + tile / p.rows.nm * p.rows.Gt;
        mbar_arrive_expect_tx(&bar[kBqQFull0 + t], 2 * q_bytes);
#pragma unroll
        for (int x = 0; x < D / kBoxCols; ++x) {
          tma_load_4d(smem + Cfg::kOffQ + t * Cfg::kTileBytes + x * kBoxBytes, &tm_Q, &bar[kBqQFull0 + t], x * kBoxCols,
                      m0, h0, u.b, pol_q);
          tma_load_4d(smem + Cfg::kOffdO + t * Cfg::kTileBytes + x * kBoxBytes, &tm_dO, &bar[kBqQFull0 + t], x * kBoxCols,
                      m0, h0, u.b, pol_q);
        }
        ++nq[t];
        return true;
      };
      auto load_kv = [&](const CUtensorMap* tm, const BwdUnit& u, int j, int full, int empty, int off, int slots, int& n) {
        const int s = n % slots;
        if (n >= slots && !mbar_wait(&bar[empty + s], ((n / slots) - 1) & 1, ctx, 302)) return false;
        mbar_arrive_expect_tx(&bar[full + s], Cfg::kTileBytes);
#pragma unroll
        for (int x = 0; x < D / kBoxCols; ++x)
          tma_load_4d(smem + off + s * Cfg::kTileBytes + x * kBoxBytes, tm, &bar[full + s], x * kBoxCols, j * kTile, u.hk,
                      u.b, pol_kv);
        ++n;
        return true;
      };
      BwdSchedule<T, true> sched(p, gridDim.x, blockIdx.x);
      BwdUnit u;
      while (ok && sched.next(u)) {
        const bool two = 2 * u.idx + 1 < q_tiles;
        ok = load_q(u, 0) && load_kv(&tm_K, u, u.lo, kBqKFull0, kBqKEmpty0, Cfg::kOffK, SK, nk) &&
             (!two || load_q(u, 1));
        for (int j = u.lo; j < u.hi && ok; ++j)
          ok = load_kv(&tm_V, u, j, kBqVFull0, kBqVEmpty0, Cfg::kOffV, SV, nv) &&
               (j + 1 == u.hi || load_kv(&tm_K, u, j + 1, kBqKFull0, kBqKEmpty0, Cfg::kOffK, SK, nk));
      }
      if (*abort_flag) {
        for (int t = 0; t < 2; ++t)
          if (nq[t] > 0) mbar_wait_drain(&bar[kBqQFull0 + t], (nq[t] - 1) & 1, p.timeout_ns);
        for (int i = (nk > SK ? nk - SK : 0); i < nk; ++i)
          mbar_wait_drain(&bar[kBqKFull0 + i % SK], (i / SK) & 1, p.timeout_ns);
        for (int i = (nv > SV ? nv - SV : 0); i < nv; ++i)
          mbar_wait_drain(&bar[kBqVFull0 + i % SV], (i / SV) & 1, p.timeout_ns);
      }
    } else if (warp == 9) {
      // ---- MMA: lane 0 issues, per step: dP0, [dQ1 of the step before, S1],
      // dP1, [dQ0, S0 of the next step], so that each warpgroup forms P and dS
      // while the tensor core works on the other tile. The whole warp clears
      // the K rows between the last valid key and the next multiple of 16,
      // which dQ would multiply by dS = 0 whatever they hold.
      constexpr uint32_t id_S = make_idesc_f16<kB>(kTile, kTile, false, false);
      constexpr uint32_t id_A = make_idesc_f16<kB>(kTile, D, false, true);
      const uint32_t sQ = smem_u32(smem + Cfg::kOffQ), sdO = smem_u32(smem + Cfg::kOffdO);
      const uint32_t sK = smem_u32(smem + Cfg::kOffK), sV = smem_u32(smem + Cfg::kOffV);
      struct Step {
        int j, lo, hi, n, g;  // key tile, the unit's, valid keys, count of steps before
        bool two;
      };
      BwdSchedule<T, true> sched(p, gridDim.x, blockIdx.x);
      BwdUnit u;
      auto open = [&](Step& s, int g) {
        if (!sched.next(u)) return false;
        s = Step{u.lo, u.lo, u.hi, u.n, g, 2 * u.idx + 1 < q_tiles};
        return true;
      };
      int nq[2] = {0, 0}, ns[2] = {0, 0}, nd[2] = {0, 0}, na[2] = {0, 0};
      bool ok = true;
      auto product = [&](uint32_t d, uint32_t a, uint32_t b) {  // A, B K-major over D
        const uint64_t da = make_sw128_desc(a, 16, 1024), db = make_sw128_desc(b, 16, 1024);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k >> 2) * kBoxBytes + (k & 3) * 32;
          umma_f16_ss(d, desc_advance(da, off), desc_advance(db, off), id_S, k > 0 ? 1u : 0u);
        }
      };
      // lane 0: S of tile t (K has landed)
      auto do_s = [&](const Step& s, int t) {
        if (s.j == s.lo) {
          if (!mbar_wait(&bar[kBqQFull0 + t], nq[t] & 1, ctx, 311)) return false;
          ++nq[t];
        }
        tc_fence_after();
        product(tmem + 128 * t, sQ + t * Cfg::kTileBytes, sK + (s.g % SK) * Cfg::kTileBytes);
        umma_commit(&bar[kBqSFull0 + t]);
        return true;
      };
      auto do_dp = [&](const Step& s, int t) {
        if (t == 0 && !mbar_wait(&bar[kBqVFull0 + s.g % SV], (s.g / SV) & 1, ctx, 312)) return false;
        if (!mbar_wait(&bar[kBqSRead0 + t], ns[t] & 1, ctx, 313)) return false;
        ++ns[t];
        tc_fence_after();
        product(tmem + 128 * t, sdO + t * Cfg::kTileBytes, sV + (s.g % SV) * Cfg::kTileBytes);
        umma_commit(&bar[kBqXFull0 + t]);
        if (t == 1 || !s.two) umma_commit(&bar[kBqVEmpty0 + s.g % SV]);
        if (s.j + 1 == s.hi) umma_commit(&bar[kBqQEmpty0 + t]);
        return true;
      };
      auto do_dq = [&](const Step& s, int t) {
        if (s.j == s.lo) {
          if (na[t] > 0 && !mbar_wait(&bar[kBqAccEmpty0 + t], (na[t] - 1) & 1, ctx, 314)) return false;
          ++na[t];
        }
        if (!mbar_wait(&bar[kBqDSFull0 + t], nd[t] & 1, ctx, 315)) return false;
        ++nd[t];
        tc_fence_after();
        const int left = s.n - s.j * kTile, steps = left >= kTile ? kTile / 16 : (left + 15) / 16;
        const uint64_t dk = make_sw128_desc(sK + (s.g % SK) * Cfg::kTileBytes, kBoxBytes, 1024);
        const uint32_t keep = s.j > s.lo ? 1u : 0u;
        for (int k = 0; k < steps; ++k)
          umma_f16_ts(tmem + 256 + D * t, tmem + 128 * t + k * 8, desc_advance(dk, k * 2048), id_A, k > 0 ? 1u : keep);
        if (t == 1 || !s.two) umma_commit(&bar[kBqKEmpty0 + s.g % SK]);
        if (s.j + 1 == s.hi) umma_commit(&bar[kBqAcc0 + t]);
        return true;
      };
      // whole warp: K of step s has landed and its rows behind the last key are zero
      auto have_k = [&](const Step& s) {
        bool good = true;
        if (lane == 0) good = mbar_wait(&bar[kBqKFull0 + s.g % SK], (s.g / SK) & 1, ctx, 310);
        const int left = s.n - s.j * kTile;
        if (left < kTile && (left & 15) != 0) {
          good = __shfl_sync(0xffffffffu, good, 0);
          if (good) {
            uint8_t* k = smem + Cfg::kOffK + (s.g % SK) * Cfg::kTileBytes;
            const int rows = 16 - (left & 15);
            for (int i = lane; i < rows * (D / 8); i += 32) {
              const int row = left + i / (D / 8), c = i % (D / 8);
              *reinterpret_cast<uint4*>(k + (c >> 3) * kBoxBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
                  make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
          __syncwarp();
        }
        return good;
      };
      Step cur, nxt, prev;
      bool has = open(cur, 0), has_prev = false;
      if (has) {
        ok = have_k(cur);
        if (lane == 0 && ok) ok = do_s(cur, 0);
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      while (has && ok) {
        // prev: the step before, whose dQ1 is still to come
        if (lane == 0) {
          ok = do_dp(cur, 0);
          if (ok && has_prev && prev.two) ok = do_dq(prev, 1);
          if (ok && cur.two) ok = do_s(cur, 1) && do_dp(cur, 1);
          if (ok) ok = do_dq(cur, 0);
        }
        nxt = cur;
        ++nxt.j;
        ++nxt.g;
        bool more = true;
        if (nxt.j == nxt.hi) more = open(nxt, nxt.g);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (ok && more) {
          ok = have_k(nxt);
          if (lane == 0 && ok) ok = do_s(nxt, 0);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        prev = cur;
        has_prev = true;
        cur = nxt;
        has = more;
      }
      if (lane == 0 && ok && has_prev && prev.two) ok = do_dq(prev, 1);
      if (!ok && lane == 0) {
        umma_commit(&bar[kBqDrain]);
        mbar_wait_drain(&bar[kBqDrain], 0, p.timeout_ns);
      }
      __syncwarp();
    } else if (warp >= 10) {
      // ---- entries without keys: dQ = 0
      const int64_t thread = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x - 320, threads = 64ll * gridDim.x;
      if (p.lens)
        for (int b = 0; b < p.B; ++b)
          if (valid_rows(p.lens, b, p.N) == 0)
            zero_rows<T, D>(p.dQ, b, p.Hkv * p.rows.G, 0, p.rows.M, thread, threads);
    }
  } else {
    // ---- P and dS: warpgroup t owns tile t, thread = row (TMEM lane)
    regs_raise<Cfg::kComputeRegs>();
    const int t = warp >> 2, r = threadIdx.x & 127;
    const uint32_t tR = tmem + 128 * t + (static_cast<uint32_t>(r & 96) << 16);
    const uint32_t tA = tmem + 256 + D * t + (static_cast<uint32_t>(r & 96) << 16);
    const float sl2 = p.scale * kLog2e;
    const int ds_exp = ds_exponent<T, D>(p, lane);
    const float ds_mul = pow2(ds_exp - kPBias), out_mul = p.scale * pow2(-ds_exp);
    int ns = 0, na = 0;
    bool ok = true;
    BwdSchedule<T, true> sched(p, gridDim.x, blockIdx.x);
    BwdUnit u;
    while (ok && sched.next(u)) {
      const int tile = 2 * u.idx + t;
      if (tile >= q_tiles) continue;
      const int64_t row = ((static_cast<int64_t>(u.b) * p.Hkv + u.hk) * q_tiles + tile) * kTile + r;
      const float nl = static_cast<float>(kPBias) - __ldcg(p.lse2 + row);
      const float nd = -ds_mul * __ldcg(p.delta + row);
      for (int j = u.lo; j < u.hi; ++j, ++ns) {
        if (!mbar_wait(&bar[kBqSFull0 + t], ns & 1, ctx, 320)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        uint32_t s[128];
        tmem_load_64(tR, *reinterpret_cast<uint32_t(*)[64]>(s));
        tmem_load_64(tR + 64, *reinterpret_cast<uint32_t(*)[64]>(s + 64));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBqSRead0 + t]);
#pragma unroll
        for (int x = 0; x < 128; x += 2) {
          const float2 a = fma_f32x2(make_float2(__uint_as_float(s[x]), __uint_as_float(s[x + 1])),
                                     make_float2(sl2, sl2), make_float2(nl, nl));
          s[x] = __float_as_uint(ex2_approx(a.x));
          s[x + 1] = __float_as_uint(ex2_approx(a.y));
        }
        if (!mbar_wait(&bar[kBqXFull0 + t], ns & 1, ctx, 321)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        const int left = u.n - j * kTile;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t e[32];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t dp[32];
            tmem_load_32(tR + 64 * h + 32 * q, dp);
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const uint32_t* sp = s + 64 * h + 32 * q + 2 * x;
              float2 a = fma_f32x2(make_float2(__uint_as_float(dp[2 * x]), __uint_as_float(dp[2 * x + 1])),
                                   make_float2(ds_mul, ds_mul), make_float2(nd, nd));
              a = mul_f32x2(a, make_float2(__uint_as_float(sp[0]), __uint_as_float(sp[1])));
              if (left < kTile) {  // keys that do not count, whatever K and V held there
                const int col = 64 * h + 32 * q + 2 * x;
                if (col >= left) a.x = 0.f;
                if (col + 1 >= left) a.y = 0.f;
              }
              e[16 * q + x] = Elem<T>::pack(a.x, a.y);
            }
          }
          tmem_store_32(tR + 32 * h, e);
        }
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBqDSFull0 + t]);
      }
      if (!ok) break;
      if (!mbar_wait(&bar[kBqAcc0 + t], na & 1, ctx, 322)) { ok = false; break; }
      ++na;
      __syncwarp();
      tc_fence_after();
      int m, g, sidx;
      const bool real = p.rows.row(tile, r, m, g, sidx);
      uint8_t* out = real ? reinterpret_cast<uint8_t*>(p.dQ.at(u.b, u.hk * p.rows.G + g, m)) : nullptr;
      float* part = p.part + ((static_cast<int64_t>(u.slot) * 2 + t) * kTile + r) * D;
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        uint32_t v[32];
        __syncwarp();
        tmem_load_32(tA + 32 * x, v);
        if (u.slot >= 0) {
          store_part_32(part + 32 * x, v);
        } else {
          uint4 ch[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) ch[y] = pack8<T>(v + 8 * y, out_mul);
          store_rows_anywhere<4>(ch, out ? out + 64 * x : nullptr, lane);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[kBqAccEmpty0 + t]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) publish_failure(*abort_flag, p.status);
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ====================================================================== dkv
// One CTA walks units (a key tile, a run of row tiles); K and V stay, Q and dO
// stream. Keys lie on the TMEM lanes. Per row tile:
//   S^T = K Q^T -> TMEM;  P^T = 2^(S^T scale log2e - lse2), 16-bit, over S^T;
//   dV += P^T dO;  dP^T = V dO^T -> TMEM;  dS^T, 16-bit, over dP^T;  dK += dS^T Q
// issued as dV, S^T of the next tile, dK, dP^T of the next tile: the warps
// form dS^T during dV and S^T, and the next P^T during dK and dP^T.
//
// Shared memory (D = 128): K, V 64 KB, Q x2, dO x2 128 KB, lse2 and delta.
// TMEM: S^T [0, 128), dP^T [128, 256), dV, dK behind. Warps 0-7 form P and dS:
// lane quarter warp % 4, rows 64 c .. 64 c + 63 of the row tile, c = warp / 4;
// the 16-bit halves lie in columns [64 c, 64 c + 32).
template <int D>
struct DkvCfg2 {
  static constexpr int kTileBytes = (D / kBoxCols) * kBoxBytes;
  static constexpr int kOffK = 0, kOffV = kTileBytes;
  static constexpr int kOffQ = 2 * kTileBytes, kOffdO = 4 * kTileBytes;  // two slots each
  static constexpr int kOffL = 6 * kTileBytes;                          // [2 slots][lse2, delta][128]
  static constexpr int kOffBar = kOffL + 2 * 2 * kTile * 4;
  static constexpr int kSmemBytes = kOffBar + 256;
  static constexpr int kThreads = 384;
  static constexpr int kComputeRegs = 208, kOtherRegs = 80;
  static constexpr uint32_t kColS = 0, kColX = 128, kColdV = 256, kColdK = 256 + D;
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

enum DkvBar2 : int {
  kBkKV = 0,
  kBkKVEmpty = 1,
  kBkQFull0 = 2,   // + slot: Q, lse2, delta
  kBkQEmpty0 = 4,
  kBkOFull0 = 6,   // + slot: dO
  kBkOEmpty0 = 8,
  kBkSFull = 10,
  kBkPFull = 11,   // 8 warps
  kBkXFull = 12,
  kBkDSFull = 13,  // 8 warps
  kBkAcc = 14,
  kBkAccEmpty = 15, // 8 warps
  kBkDrain = 16,
  kNumBkBars = 17,
};

template <typename T, int D>
__global__ void __launch_bounds__(DkvCfg2<D>::kThreads, 1)
    attn_dkv_kernel(const __grid_constant__ CUtensorMap tm_Q, const __grid_constant__ CUtensorMap tm_K,
                    const __grid_constant__ CUtensorMap tm_V, const __grid_constant__ CUtensorMap tm_dO,
                    const __grid_constant__ BwdParams<T> p) {
  using Cfg = DkvCfg2<D>;
  constexpr bool kB = Elem<T>::kBF16;
  constexpr int kPBias = kB ? 0 : 10;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // never, short of a toolchain that drops the alignment
    if (threadIdx.x == 0) publish_failure(1 + 400, p.status);
    return;
  }
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kNumBkBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_tiles = p.rows.tiles;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kNumBkBars; ++i)
      mbar_init(&bar[i], i == kBkPFull || i == kBkDSFull || i == kBkAccEmpty ? 8 : 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // rows of the Q and dO slots that no box fills are summed over with P = dS = 0
  const int box_rows = p.rows.Mt * p.rows.Gt;
  if (box_rows < kTile) {
    for (int i = threadIdx.x; i < 4 * Cfg::kTileBytes / 16; i += Cfg::kThreads)
      *reinterpret_cast<uint4*>(smem + Cfg::kOffQ + 16 * i) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  WaitCtx ctx{abort_flag, p.timeout_ns};
  // The launch before (attn_dq_kernel) let this one start after its own wait
  // for attn_delta_kernel, whose rows are thus there; attn_dq_kernel itself is
  // waited for at the end, for the launches after.

  if (warp >= 8) {
    regs_lower<Cfg::kOtherRegs>();
    if (warp == 8 && lane == 0) {
      // ---- TMA producer
      tma_prefetch_desc(&tm_Q);
      tma_prefetch_desc(&tm_K);
      tma_prefetch_desc(&tm_V);
      tma_prefetch_desc(&tm_dO);
      const uint64_t pol_q = l2_policy_evict_last(), pol_kv = l2_policy_evict_first();
      const uint32_t q_bytes = static_cast<uint32_t>(box_rows) * 128u * (D / kBoxCols);
      int nu = 0, n = 0, no = 0;
      bool ok = true;
      BwdSchedule<T, false> sched(p, gridDim.x, blockIdx.x);
      BwdUnit u;
      while (ok && sched.next(u)) {
        if (nu > 0 && !mbar_wait(&bar[kBkKVEmpty], (nu - 1) & 1, ctx, 401)) { ok = false; break; }
        mbar_arrive_expect_tx(&bar[kBkKV], 2 * Cfg::kTileBytes);
#pragma unroll
        for (int x = 0; x < D / kBoxCols; ++x) {
          tma_load_4d(smem + Cfg::kOffK + x * kBoxBytes, &tm_K, &bar[kBkKV], x * kBoxCols, u.idx * kTile, u.hk, u.b, pol_kv);
          tma_load_4d(smem + Cfg::kOffV + x * kBoxBytes, &tm_V, &bar[kBkKV], x * kBoxCols, u.idx * kTile, u.hk, u.b, pol_kv);
        }
        ++nu;
        for (int i = u.lo; i < u.hi; ++i) {
          const int s = n & 1;
          const int m0 = i % p.rows.nm * p.rows.Mt, h0 = u.hk * p.rows.G + i / p.rows.nm * p.rows.Gt;
          const int64_t row = ((static_cast<int64_t>(u.b) * p.Hkv + u.hk) * q_tiles + i) * kTile;
          if (n >= 2 && !mbar_wait(&bar[kBkQEmpty0 + s], ((n >> 1) - 1) & 1, ctx, 402)) { ok = false; break; }
          mbar_arrive_expect_tx(&bar[kBkQFull0 + s], q_bytes + 2 * kTile * 4);
#pragma unroll
          for (int x = 0; x < D / kBoxCols; ++x)
            tma_load_4d(smem + Cfg::kOffQ + s * Cfg::kTileBytes + x * kBoxBytes, &tm_Q, &bar[kBkQFull0 + s], x * kBoxCols,
                        m0, h0, u.b, pol_q);
          bulk_load(smem + Cfg::kOffL + s * 2 * kTile * 4, p.lse2 + row, kTile * 4, &bar[kBkQFull0 + s]);
          bulk_load(smem + Cfg::kOffL + (s * 2 + 1) * kTile * 4, p.delta + row, kTile * 4, &bar[kBkQFull0 + s]);
          ++n;
          if (n > 2 && !mbar_wait(&bar[kBkOEmpty0 + s], (((n - 1) >> 1) - 1) & 1, ctx, 403)) { ok = false; break; }
          mbar_arrive_expect_tx(&bar[kBkOFull0 + s], q_bytes);
#pragma unroll
          for (int x = 0; x < D / kBoxCols; ++x)
            tma_load_4d(smem + Cfg::kOffdO + s * Cfg::kTileBytes + x * kBoxBytes, &tm_dO, &bar[kBkOFull0 + s],
                        x * kBoxCols, m0, h0, u.b, pol_q);
          ++no;
        }
      }
      if (*abort_flag) {
        if (nu > 0) mbar_wait_drain(&bar[kBkKV], (nu - 1) & 1, p.timeout_ns);
        for (int i = (n > 2 ? n - 2 : 0); i < n; ++i)
          mbar_wait_drain(&bar[kBkQFull0 + (i & 1)], (i >> 1) & 1, p.timeout_ns);
        for (int i = (no > 2 ? no - 2 : 0); i < no; ++i)
          mbar_wait_drain(&bar[kBkOFull0 + (i & 1)], (i >> 1) & 1, p.timeout_ns);
      }
    } else if (warp == 9 && lane == 0) {
      // ---- MMA
      constexpr uint32_t id_S = make_idesc_f16<kB>(kTile, kTile, false, false);
      constexpr uint32_t id_A = make_idesc_f16<kB>(kTile, D, false, true);
      const uint32_t sK = smem_u32(smem + Cfg::kOffK), sV = smem_u32(smem + Cfg::kOffV);
      const uint32_t sQ = smem_u32(smem + Cfg::kOffQ), sdO = smem_u32(smem + Cfg::kOffdO);
      auto product = [&](uint32_t d, uint32_t a, uint32_t b) {
        const uint64_t da = make_sw128_desc(a, 16, 1024), db = make_sw128_desc(b, 16, 1024);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k >> 2) * kBoxBytes + (k & 3) * 32;
          umma_f16_ss(d, desc_advance(da, off), desc_advance(db, off), id_S, k > 0 ? 1u : 0u);
        }
      };
      auto accumulate = [&](uint32_t d, uint32_t a, uint32_t b, uint32_t keep) {
        const uint64_t db = make_sw128_desc(b, kBoxBytes, 1024);
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
          umma_f16_ts(d, a + (k >> 2) * 64 + (k & 3) * 8, desc_advance(db, k * 2048), id_A, k > 0 ? 1u : keep);
      };
      BwdSchedule<T, false> sched(p, gridDim.x, blockIdx.x);
      BwdUnit u, w;  // the unit of step n and of the next step
      int n = 0, nu = 0, i = 0;
      bool ok = true, has = sched.next(u);
      auto do_s = [&](int n1, bool opens) {
        if (opens) {
          if (!mbar_wait(&bar[kBkKV], nu & 1, ctx, 410)) return false;
          ++nu;
        }
        if (!mbar_wait(&bar[kBkQFull0 + (n1 & 1)], (n1 >> 1) & 1, ctx, 411)) return false;
        tc_fence_after();
        product(tmem + Cfg::kColS, sK, sQ + (n1 & 1) * Cfg::kTileBytes);
        umma_commit(&bar[kBkSFull]);
        return true;
      };
      auto do_dp = [&](int n1, bool closes) {
        if (!mbar_wait(&bar[kBkOFull0 + (n1 & 1)], (n1 >> 1) & 1, ctx, 412)) return false;
        tc_fence_after();
        product(tmem + Cfg::kColX, sV, sdO + (n1 & 1) * Cfg::kTileBytes);
        umma_commit(&bar[kBkXFull]);
        if (closes) umma_commit(&bar[kBkKVEmpty]);
        return true;
      };
      if (has) {
        i = u.lo;
        ok = do_s(0, true) && do_dp(0, u.lo + 1 == u.hi);
      }
      while (has && ok) {
        w = u;
        int i1 = i + 1;
        bool more = true, opens = false;
        if (i1 == u.hi) {
          more = sched.next(w);
          i1 = w.lo;
          opens = true;
        }
        const uint32_t keep = i > u.lo ? 1u : 0u;
        if (i == u.lo && nu > 1) {
          // the sums of the unit before have been read
          ok = mbar_wait(&bar[kBkAccEmpty], (nu - 2) & 1, ctx, 413);
        }
        ok = ok && mbar_wait(&bar[kBkPFull], n & 1, ctx, 414);
        if (!ok) break;
        tc_fence_after();
        accumulate(tmem + Cfg::kColdV, tmem + Cfg::kColS, sdO + (n & 1) * Cfg::kTileBytes, keep);
        umma_commit(&bar[kBkOEmpty0 + (n & 1)]);
        if (more && !(ok = do_s(n + 1, opens))) break;
        if (!(ok = mbar_wait(&bar[kBkDSFull], n & 1, ctx, 415))) break;
        tc_fence_after();
        accumulate(tmem + Cfg::kColdK, tmem + Cfg::kColX, sQ + (n & 1) * Cfg::kTileBytes, keep);
        umma_commit(&bar[kBkQEmpty0 + (n & 1)]);
        if (i + 1 == u.hi) umma_commit(&bar[kBkAcc]);
        if (more && !(ok = do_dp(n + 1, i1 + 1 == w.hi))) break;
        u = w;
        i = i1;
        has = more;
        ++n;
      }
      if (!ok) {
        umma_commit(&bar[kBkDrain]);
        mbar_wait_drain(&bar[kBkDrain], 0, p.timeout_ns);
      }
    } else if (warp >= 10) {
      // ---- key tiles without a valid key: dK = dV = 0
      const int64_t thread = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x - 320, threads = 64ll * gridDim.x;
      if (p.lens)
        for (int b = 0; b < p.B; ++b) {
          const int from = (valid_rows(p.lens, b, p.N) + kTile - 1) / kTile * kTile;
          if (from < p.N) {
            zero_rows<T, D>(p.dK, b, p.Hkv, from, p.N, thread, threads);
            zero_rows<T, D>(p.dV, b, p.Hkv, from, p.N, thread, threads);
          }
        }
    }
  } else {
    // ---- P^T and dS^T
    regs_raise<Cfg::kComputeRegs>();
    const int c = warp >> 2, r = threadIdx.x & 127;  // r: key within the tile (TMEM lane)
    const uint32_t lanes = static_cast<uint32_t>(r & 96) << 16;
    const uint32_t tS = tmem + Cfg::kColS + 64 * c + lanes, tX = tmem + Cfg::kColX + 64 * c + lanes;
    const float sl2 = p.scale * kLog2e;
    const int ds_exp = ds_exponent<T, D>(p, lane);
    const float ds_mul = pow2(ds_exp - kPBias);
    const float dk_mul = p.scale * pow2(-ds_exp), dv_mul = pow2(-kPBias);
    int n = 0, nu = 0;
    bool ok = true;
    BwdSchedule<T, false> sched(p, gridDim.x, blockIdx.x);
    BwdUnit u;
    while (ok && sched.next(u)) {
      const int key = u.idx * kTile + r;
      const bool valid = key < u.n;
      for (int i = u.lo; i < u.hi; ++i, ++n) {
        const float4* lse = reinterpret_cast<const float4*>(smem + Cfg::kOffL + (n & 1) * 2 * kTile * 4) + 16 * c;
        const float4* del = lse + kTile / 4;
        if (!mbar_wait(&bar[kBkQFull0 + (n & 1)], (n >> 1) & 1, ctx, 420)) { ok = false; break; }
        if (!mbar_wait(&bar[kBkSFull], n & 1, ctx, 421)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        uint32_t s[64], e[32];
        tmem_load_64(tS, s);
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float4 l = lse[x];
          float2 a = fma_f32x2(make_float2(__uint_as_float(s[4 * x]), __uint_as_float(s[4 * x + 1])),
                               make_float2(sl2, sl2), make_float2(kPBias - l.x, kPBias - l.y));
          float2 b = fma_f32x2(make_float2(__uint_as_float(s[4 * x + 2]), __uint_as_float(s[4 * x + 3])),
                               make_float2(sl2, sl2), make_float2(kPBias - l.z, kPBias - l.w));
          a.x = valid ? ex2_approx(a.x) : 0.f;
          a.y = valid ? ex2_approx(a.y) : 0.f;
          b.x = valid ? ex2_approx(b.x) : 0.f;
          b.y = valid ? ex2_approx(b.y) : 0.f;
          s[4 * x] = __float_as_uint(a.x);
          s[4 * x + 1] = __float_as_uint(a.y);
          s[4 * x + 2] = __float_as_uint(b.x);
          s[4 * x + 3] = __float_as_uint(b.y);
          e[2 * x] = Elem<T>::pack(a.x, a.y);
          e[2 * x + 1] = Elem<T>::pack(b.x, b.y);
        }
        tmem_store_32(tS, e);
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBkPFull]);
        if (!mbar_wait(&bar[kBkXFull], n & 1, ctx, 422)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t dp[32];
          tmem_load_32(tX + 32 * q, dp);
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float4 d = del[8 * q + x];
            const uint32_t* sp = s + 32 * q + 4 * x;
            float2 a = add_f32x2(make_float2(__uint_as_float(dp[4 * x]), __uint_as_float(dp[4 * x + 1])),
                                 make_float2(-d.x, -d.y));
            float2 b = add_f32x2(make_float2(__uint_as_float(dp[4 * x + 2]), __uint_as_float(dp[4 * x + 3])),
                                 make_float2(-d.z, -d.w));
            if (!kB) {
              a = mul_f32x2(a, make_float2(ds_mul, ds_mul));
              b = mul_f32x2(b, make_float2(ds_mul, ds_mul));
            }
            a = mul_f32x2(a, make_float2(__uint_as_float(sp[0]), __uint_as_float(sp[1])));
            b = mul_f32x2(b, make_float2(__uint_as_float(sp[2]), __uint_as_float(sp[3])));
            e[16 * q + 2 * x] = Elem<T>::pack(a.x, a.y);
            e[16 * q + 2 * x + 1] = Elem<T>::pack(b.x, b.y);
          }
        }
        if (!valid) {  // V of such a row may hold anything
#pragma unroll
          for (int x = 0; x < 32; ++x) e[x] = 0u;
        }
        tmem_store_32(tX, e);
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBkDSFull]);
      }
      if (!ok) break;
      if (!mbar_wait(&bar[kBkAcc], nu & 1, ctx, 423)) { ok = false; break; }
      ++nu;
      __syncwarp();
      tc_fence_after();
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const uint32_t col = (which == 0 ? Cfg::kColdV : Cfg::kColdK) + c * (D / 2) + lanes;
        const float mul = which == 0 ? dv_mul : dk_mul;
        const View<T>& v = which == 0 ? p.dV : p.dK;
        uint8_t* out = key < p.N ? reinterpret_cast<uint8_t*>(v.at(u.b, u.hk, key) + c * (D / 2)) : nullptr;
        float* part = p.part + ((static_cast<int64_t>(u.slot) * 2 + which) * kTile + r) * D + c * (D / 2);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
          uint32_t a[32];
          __syncwarp();
          tmem_load_32(tmem + col + 32 * x, a);
          if (u.slot >= 0) {
            store_part_32(part + 32 * x, a);
          } else {
            uint4 ch[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) ch[y] = valid ? pack8<T>(a + 8 * y, mul) : make_uint4(0, 0, 0, 0);
            store_rows_anywhere<4>(ch, out ? out + 64 * x : nullptr, lane);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[kBkAccEmpty]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) publish_failure(*abort_flag, p.status);
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ===================================================================== join
// Items that fell to several CTAs: adds their partial sums in CTA order. Block
// (x, c - 1) looks at the boundary before CTA c; the first boundary inside an
// item owns it. One thread per 4 columns of the item's two [128][D] sums.
template <typename T, int D, bool kQMajor>
__device__ void join_item(const BwdParams<T>& p, int grid, int c, int e, int lane) {
  BwdSchedule<T, kQMajor> sched(p, grid, c);
  if (!sched.by_steps || sched.pos >= sched.total) return;
  const int64_t at = sched.pos;
  sched.end = sched.total;  // the whole item around the boundary
  BwdUnit u;
  sched.next(u);
  const int64_t start = at - u.lo, stop = start + u.len;
  if (u.lo == 0 || sched.mark(c - 1) > start) return;
  const int which = e / (kTile * D / 4), row = e / (D / 4) % kTile, col = e % (D / 4);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = c - 1; k < sched.parts && sched.mark(k) < stop; ++k) {
    if (sched.mark(k + 1) <= max(sched.mark(k), start)) continue;  // a CTA without steps in it
    const int slot = 2 * k + (sched.mark(k) >= start ? 0 : 1);
    const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part) + ((static_cast<int64_t>(slot) * 2 + which) * kTile + row) * (D / 4) + col);
    a.x += v.x;
    a.y += v.y;
    a.z += v.z;
    a.w += v.w;
  }
  const int ds_exp = ds_exponent<T, D>(p, lane);
  T* out = nullptr;
  float mul = p.scale * pow2(-ds_exp);
  if (kQMajor) {
    int m, g, s;
    const int tile = 2 * u.idx + which;
    if (tile < p.rows.tiles && p.rows.row(tile, row, m, g, s)) out = p.dQ.at(u.b, u.hk * p.rows.G + g, m);
  } else {
    const int key = u.idx * kTile + row;
    if (which == 0) mul = Elem<T>::kBF16 ? 1.f : pow2(-10);
    if (key < p.N) out = (which == 0 ? p.dV : p.dK).at(u.b, u.hk, key);
    if (key >= u.n) a = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (out)
    *reinterpret_cast<uint2*>(out + 4 * col) =
        make_uint2(Elem<T>::pack(mul * a.x, mul * a.y), Elem<T>::pack(mul * a.z, mul * a.w));
}

template <typename T, int D>
__global__ void __launch_bounds__(256)
    attn_bwd_join_kernel(const __grid_constant__ BwdParams<T> q, const __grid_constant__ BwdParams<T> k, int grid_q,
                         int grid_k) {
  const int e = blockIdx.x * 256 + threadIdx.x, c = blockIdx.y + 1;
  if (c < grid_q) join_item<T, D, true>(q, grid_q, c, e, threadIdx.x & 31);
  if (c < grid_k) join_item<T, D, false>(k, grid_k, c, e, threadIdx.x & 31);
}

}  // namespace fmha_sm100
