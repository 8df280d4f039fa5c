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
  int total, items;      // the host refuses more than 2^31 steps
  bool by_steps;
  int pos, end;          // steps, or items
  int b, before;         // the entry that the walk has reached, and what lies before it
  int first_unit;

  __device__ __forceinline__ int key_tiles(int e) const {
    return (valid_rows(p.lens, e, p.N) + kTile - 1) / kTile;
  }
  __device__ __forceinline__ int items_of(int nt) const { return kQMajor ? (nt > 0 ? p.Hkv * p.pairs : 0) : p.Hkv * nt; }
  __device__ __forceinline__ int len_of(int nt) const { return kQMajor ? nt : p.rows.tiles; }
  __device__ __forceinline__ int mark(int c) const {
    return c < parts ? static_cast<int>(static_cast<int64_t>(total) * c / parts) : total;
  }

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
    b = before = 0;
    first_unit = 1;
  }
  // The next unit of this CTA; false when there is none.
  __device__ bool next(BwdUnit& u) {
    if (pos >= end) return false;
    int nt;
    for (;; ++b) {
      nt = key_tiles(b);
      const int n = by_steps ? items_of(nt) * len_of(nt) : items_of(nt);
      if (pos < before + n) break;
      before += n;
    }
    u.b = b;
    u.n = valid_rows(p.lens, b, p.N);
    u.len = len_of(nt);
    int item = pos - before;
    u.lo = 0;
    u.hi = u.len;
    u.slot = -1;
    if (by_steps) {
      u.lo = item % u.len;
      item /= u.len;
      u.hi = min(u.len, u.lo + (end - pos));
      if (u.hi - u.lo < u.len) u.slot = 2 * cta + 1 - first_unit;
      pos += u.hi - u.lo;
    } else {
      pos += grid;
    }
    first_unit = 0;
    const int per = kQMajor ? p.pairs : nt;
    u.hk = item / per;
    u.idx = item % per;
    return true;
  }
};

template <typename T, bool kQMajor>
__device__ void feed_units(const BwdParams<T>& p, UnitRing* ring, uint64_t* full, uint64_t* empty, const WaitCtx& ctx,
                           int where) {
  BwdSchedule<T, kQMajor> sched(p, gridDim.x, blockIdx.x);
  BwdUnit u{};
  for (int k = 0;; ++k) {
    const bool more = sched.next(u);
    if (!put_unit(ring, full, empty, k, make_int4(u.b, u.hk, u.idx, u.slot), make_int4(u.lo, u.hi, u.n, more ? 1 : 0),
                  ctx, where) || !more)
      return;
  }
}

template <bool kWarp>
__device__ __forceinline__ bool take_unit(const UnitRing* ring, uint64_t* full, uint64_t* empty, int& k, BwdUnit& u,
                                          const WaitCtx& ctx, int where, bool& ok) {
  int4 a, b;
  if (!get_unit<kWarp>(ring, full, empty, k, a, b, ctx, where, ok)) return false;
  u.b = a.x;
  u.hk = a.y;
  u.idx = a.z;
  u.slot = a.w;
  u.lo = b.x;
  u.hi = b.y;
  u.n = b.z;
  return true;
}

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
// tile holds no row) and D. A block takes row tiles one by one, D / 8 threads
// a row, several rows' loads in flight. In fp16 also the largest |dO| and
// valid |V| that the block saw.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    attn_delta_kernel(View<T> dO, View<T> O, View<T> V, const float* __restrict__ LSE, BwdParams<T> p,
                      float* __restrict__ lse2, float* __restrict__ delta, float2* __restrict__ amax) {
  constexpr int kPer = D / 8, kStep = 256 / kPer;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int chunk = threadIdx.x % kPer, r0 = threadIdx.x / kPer;
  const int tiles = p.B * p.Hkv * p.rows.tiles;
  float top_do = 0.f, top_v = 0.f;
  auto widest = [](float top, const uint32_t (&w)[4]) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float2 v = Elem<T>::unpack(w[x]);
      top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
    }
    return top;
  };
  for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
    const int tile = i % p.rows.tiles, bh = i / p.rows.tiles;
    const int hk = bh % p.Hkv, b = bh / p.Hkv;
#pragma unroll 4
    for (int r = r0; r < kTile; r += kStep) {
      int m, g, s;
      const bool real = p.rows.row(tile, r, m, g, s);
      float acc = 0.f;
      if (real) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(dO.at(b, hk * p.rows.G + g, m)) + chunk);
        const uint4 y = __ldg(reinterpret_cast<const uint4*>(O.at(b, hk * p.rows.G + g, m)) + chunk);
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
        const int64_t at = static_cast<int64_t>(i) * kTile + r;
        lse2[at] = l;
        delta[at] = acc;
      }
    }
  }
  if (!Elem<T>::kBF16) {
    const int nt = (p.N + kTile - 1) / kTile, key_tiles = p.B * p.Hkv * nt;
    for (int i = blockIdx.x; i < key_tiles; i += gridDim.x) {
      const int bh = i / nt, hk = bh % p.Hkv, b = bh / p.Hkv;
      const int n = valid_rows(p.lens, b, p.N);
#pragma unroll 4
      for (int r = r0; r < kTile; r += kStep) {
        const int key = i % nt * kTile + r;
        if (key < n) {
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(V.at(b, hk, key)) + chunk);
          const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
          top_v = widest(top_v, xw);
        }
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

// This thread's row of D sums in TMEM, to a partial-sum slot or, scaled, to
// its 16-bit output row (null: none).
template <typename T, int D>
__device__ __forceinline__ void store_sums(uint32_t taddr, uint8_t* out, float mul, float* part, int lane) {
#pragma unroll
  for (int x = 0; x < D / 32; ++x) {
    uint32_t v[32];
    __syncwarp();
    tmem_load_32(taddr + 32 * x, v);
    if (part) {
      store_part_32(part + 32 * x, v);
    } else {
      uint4 ch[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) ch[y] = pack8<T>(v + 8 * y, mul);
      store_rows_anywhere<4>(ch, out ? out + 64 * x : nullptr, lane);
    }
  }
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
  static constexpr int kOffRing = kOffV + kSV * kTileBytes;
  static constexpr int kOffBar = kOffRing + sizeof(UnitRing);
  static constexpr int kSmemBytes = kOffBar + 512;
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};
// Both kernels: warpgroups 0 and 1 form P and dS, 2 stores the sums, 3 holds
// the TMA producer (warp 12), the MMA issuer (13), the scheduler (14) and the
// warp that zeroes what has no keys (15). Registers: 2 * 128 * 184 + 2 * 128 *
// 72, the 512 * 128 of the launch.
constexpr int kBwdThreads = 512, kBwdComputeRegs = 184, kBwdOtherRegs = 72;
static_assert(2 * kBwdComputeRegs + 2 * kBwdOtherRegs == 4 * 128, "register split");
constexpr int kUnitReaders = 14;  // warps 0-13

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
  kBqUnitFull0 = 33,
  kBqUnitEmpty0 = 37,
  kNumBqBars = 41,
};

// dS of one row from P (in `s`) and dP (TMEM), 16 bits each, over dP. Columns
// at and past `left` do not count, whatever K and V held there.
template <typename T, bool kTail>
__device__ __forceinline__ void form_ds(const uint32_t (&s)[128], uint32_t tR, float mul, float nd, int left) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    uint32_t dp[16], e[8];
    tmem_load_16(tR + 16 * q, dp);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int col = 16 * q + 2 * x;
      float2 a = fma_f32x2(make_float2(__uint_as_float(dp[2 * x]), __uint_as_float(dp[2 * x + 1])),
                           make_float2(mul, mul), make_float2(nd, nd));
      a = mul_f32x2(a, make_float2(__uint_as_float(s[col]), __uint_as_float(s[col + 1])));
      if (kTail && col >= left) a.x = 0.f;
      if (kTail && col + 1 >= left) a.y = 0.f;
      e[x] = Elem<T>::pack(a.x, a.y);
    }
    tmem_store_8(tR + 8 * q, e);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
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
  UnitRing* ring = reinterpret_cast<UnitRing*>(smem + Cfg::kOffRing);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kNumBqBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kNumBqBars; ++i) {
      const bool four = (i >= kBqSRead0 && i < kBqXFull0) || (i >= kBqDSFull0 && i < kBqAcc0) ||
                        (i >= kBqAccEmpty0 && i < kBqDrain);
      mbar_init(&bar[i], i >= kBqUnitEmpty0 ? kUnitReaders : (four ? 4 : 1));
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 13) {
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
  uint64_t *unit_full = &bar[kBqUnitFull0], *unit_empty = &bar[kBqUnitEmpty0];
  BwdUnit u;
  int k = 0;
  bool ok = true;

  if (warp >= 12) {
    regs_lower<kBwdOtherRegs>();
    if (warp == 12) {
      // ---- TMA producer (the whole warp walks the units, lane 0 loads)
      if (lane == 0) {
        tma_prefetch_desc(&tm_Q);
        tma_prefetch_desc(&tm_K);
        tma_prefetch_desc(&tm_V);
        tma_prefetch_desc(&tm_dO);
      }
      const uint64_t pol_q = l2_policy_evict_first(), pol_kv = l2_policy_evict_last();
      const uint32_t q_bytes = static_cast<uint32_t>(p.rows.Mt * p.rows.Gt) * 128u * (D / kBoxCols);
      int nq0 = 0, nq1 = 0, nk = 0, nv = 0;
      auto load_q = [&](int t, int& n) {
        if (n > 0 && !mbar_wait(&bar[kBqQEmpty0 + t], (n - 1) & 1, ctx, 301)) return false;
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
        ++n;
        return true;
      };
      auto load_k = [&](int j) {
        const int s = nk % SK;
        if (nk >= SK && !mbar_wait(&bar[kBqKEmpty0 + s], ((nk / SK) - 1) & 1, ctx, 302)) return false;
        mbar_arrive_expect_tx(&bar[kBqKFull0 + s], Cfg::kTileBytes);
#pragma unroll
        for (int x = 0; x < D / kBoxCols; ++x)
          tma_load_4d(smem + Cfg::kOffK + s * Cfg::kTileBytes + x * kBoxBytes, &tm_K, &bar[kBqKFull0 + s], x * kBoxCols,
                      j * kTile, u.hk, u.b, pol_kv);
        ++nk;
        return true;
      };
      auto load_v = [&](int j) {
        const int s = nv % SV;
        if (nv >= SV && !mbar_wait(&bar[kBqVEmpty0 + s], ((nv / SV) - 1) & 1, ctx, 303)) return false;
        mbar_arrive_expect_tx(&bar[kBqVFull0 + s], Cfg::kTileBytes);
#pragma unroll
        for (int x = 0; x < D / kBoxCols; ++x)
          tma_load_4d(smem + Cfg::kOffV + s * Cfg::kTileBytes + x * kBoxBytes, &tm_V, &bar[kBqVFull0 + s], x * kBoxCols,
                      j * kTile, u.hk, u.b, pol_kv);
        ++nv;
        return true;
      };
      while (take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 300, ok)) {
        if (lane == 0) {
          ok = load_q(0, nq0) && load_k(u.lo) && (2 * u.idx + 1 >= q_tiles || load_q(1, nq1));
          for (int j = u.lo; j < u.hi && ok; ++j) ok = load_v(j) && (j + 1 == u.hi || load_k(j + 1));
        }
      }
      if (lane == 0 && *abort_flag) {
        if (nq0 > 0) mbar_wait_drain(&bar[kBqQFull0], (nq0 - 1) & 1, p.timeout_ns);
        if (nq1 > 0) mbar_wait_drain(&bar[kBqQFull0 + 1], (nq1 - 1) & 1, p.timeout_ns);
        for (int i = (nk > SK ? nk - SK : 0); i < nk; ++i)
          mbar_wait_drain(&bar[kBqKFull0 + i % SK], (i / SK) & 1, p.timeout_ns);
        for (int i = (nv > SV ? nv - SV : 0); i < nv; ++i)
          mbar_wait_drain(&bar[kBqVFull0 + i % SV], (i / SV) & 1, p.timeout_ns);
      }
      __syncwarp();
    } else if (warp == 13) {
      // ---- MMA: lane 0 issues, per step: dP0, [dQ1 of the step before, S1],
      // dP1, [dQ0, S0 of the next step], so that each warpgroup forms P and dS
      // while the tensor core works on the other tile. The whole warp clears
      // the K rows between the last valid key and the next multiple of 16,
      // which dQ would multiply by dS = 0 whatever they hold.
      constexpr uint32_t id_S = make_idesc_f16<kB>(kTile, kTile, false, false);
      constexpr uint32_t id_A = make_idesc_f16<kB>(kTile, D, false, true);
      const uint32_t base = smem_u32(smem);
      auto product = [&](uint32_t d, uint32_t a, uint32_t b) {  // A, B K-major over D
        const uint64_t da = make_sw128_desc(a, 16, 1024), db = make_sw128_desc(b, 16, 1024);
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          const uint32_t off = (x >> 2) * kBoxBytes + (x & 3) * 32;
          umma_f16_ss(d, desc_advance(da, off), desc_advance(db, off), id_S, x > 0 ? 1u : 0u);
        }
      };
      int nq = 0, n0 = 0, n1 = 0, a0 = 0, a1 = 0;  // units; steps of tiles 0, 1; units of tiles 0, 1 (sums)
      int nq1 = 0;
      auto do_s = [&](int t, int g, bool opens) {
        if (opens) {
          if (!mbar_wait(&bar[kBqQFull0 + t], (t == 0 ? nq : nq1) & 1, ctx, 311)) return false;
          if (t == 0) ++nq;
          else ++nq1;
        }
        tc_fence_after();
        product(tmem + 128 * t, base + Cfg::kOffQ + t * Cfg::kTileBytes, base + Cfg::kOffK + (g % SK) * Cfg::kTileBytes);
        umma_commit(&bar[kBqSFull0 + t]);
        return true;
      };
      auto do_dp = [&](int t, int n, int g, bool frees_v, bool closes) {
        if (t == 0 && !mbar_wait(&bar[kBqVFull0 + g % SV], (g / SV) & 1, ctx, 312)) return false;
        if (!mbar_wait(&bar[kBqSRead0 + t], n & 1, ctx, 313)) return false;
        tc_fence_after();
        product(tmem + 128 * t, base + Cfg::kOffdO + t * Cfg::kTileBytes, base + Cfg::kOffV + (g % SV) * Cfg::kTileBytes);
        umma_commit(&bar[kBqXFull0 + t]);
        if (frees_v) umma_commit(&bar[kBqVEmpty0 + g % SV]);
        if (closes) umma_commit(&bar[kBqQEmpty0 + t]);
        return true;
      };
      // `steps` of 16 keys; keep: not the unit's first step
      auto do_dq = [&](int t, int n, int& na, int g, int steps, bool keep, bool frees_k, bool closes) {
        if (!keep) {
          if (na > 0 && !mbar_wait(&bar[kBqAccEmpty0 + t], (na - 1) & 1, ctx, 314)) return false;
          ++na;
        }
        if (!mbar_wait(&bar[kBqDSFull0 + t], n & 1, ctx, 315)) return false;
        tc_fence_after();
        const uint64_t dk = make_sw128_desc(base + Cfg::kOffK + (g % SK) * Cfg::kTileBytes, kBoxBytes, 1024);
        const uint32_t tA = tmem + 256 + D * t, tR = tmem + 128 * t;
        if (steps == kTile / 16) {
#pragma unroll
          for (int x = 0; x < kTile / 16; ++x)
            umma_f16_ts(tA, tR + x * 8, desc_advance(dk, x * 2048), id_A, x > 0 || keep ? 1u : 0u);
        } else {
          for (int x = 0; x < steps; ++x)
            umma_f16_ts(tA, tR + x * 8, desc_advance(dk, x * 2048), id_A, x > 0 || keep ? 1u : 0u);
        }
        if (frees_k) umma_commit(&bar[kBqKEmpty0 + g % SK]);
        if (closes) umma_commit(&bar[kBqAcc0 + t]);
        return true;
      };
      // whole warp: K of step g (`left` keys from its tile on) has landed and
      // its rows behind the last key are zero
      auto have_k = [&](int g, int left) {
        bool good = true;
        if (lane == 0) good = mbar_wait(&bar[kBqKFull0 + g % SK], (g / SK) & 1, ctx, 310);
        if (left < kTile && (left & 15) != 0) {
          good = __shfl_sync(0xffffffffu, good, 0);
          if (good) {
            uint8_t* kt = smem + Cfg::kOffK + (g % SK) * Cfg::kTileBytes;
            const int rows = 16 - (left & 15);
            for (int i = lane; i < rows * (D / 8); i += 32) {
              const int row = left + i / (D / 8), c = i % (D / 8);
              *reinterpret_cast<uint4*>(kt + (c >> 3) * kBoxBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
                  make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
          __syncwarp();
        }
        return good;
      };
      bool has = take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 309, ok);
      int g = 0, j = u.lo;
      bool two = 2 * u.idx + 1 < q_tiles;
      // what dQ1 of the step before needs
      bool prev = false, prev_keep = false, prev_closes = false;
      int prev_steps = 0;
      if (has) {
        ok = have_k(0, u.n - j * kTile);
        if (lane == 0 && ok) ok = do_s(0, 0, true);
        ok = __shfl_sync(0xffffffffu, ok, 0);
      }
      while (has && ok) {
        const int left = u.n - j * kTile, steps = left >= kTile ? kTile / 16 : (left + 15) / 16;
        const bool keep = j > u.lo, closes = j + 1 == u.hi;
        if (lane == 0) {
          ok = do_dp(0, n0, g, !two, closes);
          if (ok && prev) ok = do_dq(1, n1 - 1, a1, g - 1, prev_steps, prev_keep, true, prev_closes);
          if (ok && two) ok = do_s(1, g, !keep) && do_dp(1, n1, g, true, closes);
          if (ok) ok = do_dq(0, n0, a0, g, steps, keep, !two, closes);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        prev = two;
        prev_keep = keep;
        prev_closes = closes;
        prev_steps = steps;
        ++n0;
        if (two) ++n1;
        ++g;
        ++j;
        bool opens = false;
        if (ok && closes) {
          has = take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 309, ok);
          j = u.lo;
          two = 2 * u.idx + 1 < q_tiles;
          opens = true;
        }
        if (ok && has) {
          ok = have_k(g, u.n - j * kTile);
          if (lane == 0 && ok) ok = do_s(0, g, opens);
          ok = __shfl_sync(0xffffffffu, ok, 0);
        }
      }
      if (lane == 0) {
        if (ok && prev) ok = do_dq(1, n1 - 1, a1, g - 1, prev_steps, prev_keep, true, prev_closes);
        if (!ok) {
          umma_commit(&bar[kBqDrain]);
          mbar_wait_drain(&bar[kBqDrain], 0, p.timeout_ns);
        }
      }
      __syncwarp();
    } else if (warp == 14) {
      if (lane == 0) feed_units<T, true>(p, ring, unit_full, unit_empty, ctx, 305);
      __syncwarp();
    } else {
      // ---- entries without keys: dQ = 0
      if (p.lens)
        for (int b = 0; b < p.B; ++b)
          if (valid_rows(p.lens, b, p.N) == 0)
            zero_rows<T, D>(p.dQ, b, p.Hkv * p.rows.G, 0, p.rows.M, static_cast<int64_t>(blockIdx.x) * 32 + lane,
                            32ll * gridDim.x);
    }
  } else if (warp < 8) {
    // ---- P and dS: warpgroup t owns tile t, thread = row (TMEM lane)
    regs_raise<kBwdComputeRegs>();
    const int t = warp >> 2, r = threadIdx.x & 127;
    const uint32_t tR = tmem + 128 * t + (static_cast<uint32_t>(r & 96) << 16);
    const float sl2 = p.scale * kLog2e;
    const float ds_mul = pow2(ds_exponent<T, D>(p, lane) - kPBias);
    int ns = 0;
    while (take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 319, ok)) {
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
        if (left >= kTile) form_ds<T, false>(s, tR, ds_mul, nd, left);
        else form_ds<T, true>(s, tR, ds_mul, nd, left);
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBqDSFull0 + t]);
      }
    }
  } else {
    // ---- dQ: thread = row of each tile in turn
    regs_lower<kBwdOtherRegs>();
    const int r = threadIdx.x & 127;
    const float out_mul = p.scale * pow2(-ds_exponent<T, D>(p, lane));
    int na[2] = {0, 0};
    while (take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 329, ok)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int tile = 2 * u.idx + t;
        if (tile >= q_tiles) continue;
        if (!mbar_wait(&bar[kBqAcc0 + t], na[t] & 1, ctx, 330)) { ok = false; break; }
        ++na[t];
        __syncwarp();
        tc_fence_after();
        int m, g, s;
        const bool real = p.rows.row(tile, r, m, g, s);
        uint8_t* out = real ? reinterpret_cast<uint8_t*>(p.dQ.at(u.b, u.hk * p.rows.G + g, m)) : nullptr;
        store_sums<T, D>(tmem + 256 + D * t + (static_cast<uint32_t>(r & 96) << 16), out, out_mul,
                         u.slot < 0 ? nullptr : p.part + ((static_cast<int64_t>(u.slot) * 2 + t) * kTile + r) * D, lane);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBqAccEmpty0 + t]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) publish_failure(*abort_flag, p.status);
  if (warp == 13) {
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
  static constexpr int kOffRing = kOffL + 2 * 2 * kTile * 4;
  static constexpr int kOffBar = kOffRing + sizeof(UnitRing);
  static constexpr int kSmemBytes = kOffBar + 256;
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
  kBkAccEmpty = 15, // 4 warps
  kBkDrain = 16,
  kBkUnitFull0 = 17,
  kBkUnitEmpty0 = 21,
  kNumBkBars = 25,
};

template <typename T, int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
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
  UnitRing* ring = reinterpret_cast<UnitRing*>(smem + Cfg::kOffRing);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kNumBkBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_tiles = p.rows.tiles;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kNumBkBars; ++i)
      mbar_init(&bar[i], i == kBkPFull || i == kBkDSFull ? 8 : (i == kBkAccEmpty ? 4 : (i >= kBkUnitEmpty0 ? kUnitReaders : 1)));
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 13) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // rows of the Q and dO slots that no box fills are summed over with P = dS = 0
  const int box_rows = p.rows.Mt * p.rows.Gt;
  if (box_rows < kTile) {
    for (int i = threadIdx.x; i < 4 * Cfg::kTileBytes / 16; i += kBwdThreads)
      *reinterpret_cast<uint4*>(smem + Cfg::kOffQ + 16 * i) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  WaitCtx ctx{abort_flag, p.timeout_ns};
  uint64_t *unit_full = &bar[kBkUnitFull0], *unit_empty = &bar[kBkUnitEmpty0];
  BwdUnit u;
  int k = 0;
  bool ok = true;
  // The launch before (attn_dq_kernel) let this one start after its own wait
  // for attn_delta_kernel, whose rows are thus there; attn_dq_kernel itself is
  // waited for at the end, for the launches after.

  if (warp >= 12) {
    regs_lower<kBwdOtherRegs>();
    if (warp == 12) {
      // ---- TMA producer
      if (lane == 0) {
        tma_prefetch_desc(&tm_Q);
        tma_prefetch_desc(&tm_K);
        tma_prefetch_desc(&tm_V);
        tma_prefetch_desc(&tm_dO);
      }
      const uint64_t pol_q = l2_policy_evict_last(), pol_kv = l2_policy_evict_first();
      const uint32_t q_bytes = static_cast<uint32_t>(box_rows) * 128u * (D / kBoxCols);
      int nu = 0, n = 0, no = 0;
      while (take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 400, ok)) {
        if (lane == 0) {
          ok = nu == 0 || mbar_wait(&bar[kBkKVEmpty], (nu - 1) & 1, ctx, 401);
          if (ok) {
            mbar_arrive_expect_tx(&bar[kBkKV], 2 * Cfg::kTileBytes);
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x) {
              tma_load_4d(smem + Cfg::kOffK + x * kBoxBytes, &tm_K, &bar[kBkKV], x * kBoxCols, u.idx * kTile, u.hk, u.b,
                          pol_kv);
              tma_load_4d(smem + Cfg::kOffV + x * kBoxBytes, &tm_V, &bar[kBkKV], x * kBoxCols, u.idx * kTile, u.hk, u.b,
                          pol_kv);
            }
            ++nu;
          }
          for (int i = u.lo; i < u.hi && ok; ++i) {
            const int s = n & 1;
            const int m0 = i % p.rows.nm * p.rows.Mt, h0 = u.hk * p.rows.G + i / p.rows.nm * p.rows.Gt;
            const int64_t row = ((static_cast<int64_t>(u.b) * p.Hkv + u.hk) * q_tiles + i) * kTile;
            if (n >= 2 && !mbar_wait(&bar[kBkQEmpty0 + s], ((n >> 1) - 1) & 1, ctx, 402)) { ok = false; break; }
            mbar_arrive_expect_tx(&bar[kBkQFull0 + s], q_bytes + 2 * kTile * 4);
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x)
              tma_load_4d(smem + Cfg::kOffQ + s * Cfg::kTileBytes + x * kBoxBytes, &tm_Q, &bar[kBkQFull0 + s],
                          x * kBoxCols, m0, h0, u.b, pol_q);
            bulk_load(smem + Cfg::kOffL + s * 2 * kTile * 4, p.lse2 + row, kTile * 4, &bar[kBkQFull0 + s]);
            bulk_load(smem + Cfg::kOffL + (s * 2 + 1) * kTile * 4, p.delta + row, kTile * 4, &bar[kBkQFull0 + s]);
            ++n;
            if (no >= 2 && !mbar_wait(&bar[kBkOEmpty0 + s], ((no >> 1) - 1) & 1, ctx, 403)) { ok = false; break; }
            mbar_arrive_expect_tx(&bar[kBkOFull0 + s], q_bytes);
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x)
              tma_load_4d(smem + Cfg::kOffdO + s * Cfg::kTileBytes + x * kBoxBytes, &tm_dO, &bar[kBkOFull0 + s],
                          x * kBoxCols, m0, h0, u.b, pol_q);
            ++no;
          }
        }
      }
      if (lane == 0 && *abort_flag) {
        if (nu > 0) mbar_wait_drain(&bar[kBkKV], (nu - 1) & 1, p.timeout_ns);
        for (int i = (n > 2 ? n - 2 : 0); i < n; ++i)
          mbar_wait_drain(&bar[kBkQFull0 + (i & 1)], (i >> 1) & 1, p.timeout_ns);
        for (int i = (no > 2 ? no - 2 : 0); i < no; ++i)
          mbar_wait_drain(&bar[kBkOFull0 + (i & 1)], (i >> 1) & 1, p.timeout_ns);
      }
      __syncwarp();
    } else if (warp == 13) {
      // ---- MMA (the whole warp walks the units, lane 0 issues)
      constexpr uint32_t id_S = make_idesc_f16<kB>(kTile, kTile, false, false);
      constexpr uint32_t id_A = make_idesc_f16<kB>(kTile, D, false, true);
      const uint32_t base = smem_u32(smem);
      auto product = [&](uint32_t d, uint32_t a, uint32_t b) {
        const uint64_t da = make_sw128_desc(a, 16, 1024), db = make_sw128_desc(b, 16, 1024);
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          const uint32_t off = (x >> 2) * kBoxBytes + (x & 3) * 32;
          umma_f16_ss(d, desc_advance(da, off), desc_advance(db, off), id_S, x > 0 ? 1u : 0u);
        }
      };
      auto accumulate = [&](uint32_t d, uint32_t a, uint32_t b, bool keep) {
        const uint64_t db = make_sw128_desc(b, kBoxBytes, 1024);
#pragma unroll
        for (int x = 0; x < kTile / 16; ++x)
          umma_f16_ts(d, a + (x >> 2) * 64 + (x & 3) * 8, desc_advance(db, x * 2048), id_A, x > 0 || keep ? 1u : 0u);
      };
      int nu = 0;
      auto do_s = [&](int n, bool opens) {
        if (opens) {
          if (!mbar_wait(&bar[kBkKV], nu & 1, ctx, 410)) return false;
          ++nu;
        }
        if (!mbar_wait(&bar[kBkQFull0 + (n & 1)], (n >> 1) & 1, ctx, 411)) return false;
        tc_fence_after();
        product(tmem + Cfg::kColS, base + Cfg::kOffK, base + Cfg::kOffQ + (n & 1) * Cfg::kTileBytes);
        umma_commit(&bar[kBkSFull]);
        return true;
      };
      auto do_dp = [&](int n, bool closes) {
        if (!mbar_wait(&bar[kBkOFull0 + (n & 1)], (n >> 1) & 1, ctx, 412)) return false;
        tc_fence_after();
        product(tmem + Cfg::kColX, base + Cfg::kOffV, base + Cfg::kOffdO + (n & 1) * Cfg::kTileBytes);
        umma_commit(&bar[kBkXFull]);
        if (closes) umma_commit(&bar[kBkKVEmpty]);
        return true;
      };
      bool has = take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 409, ok);
      int n = 0, i = u.lo, lo = u.lo, hi = u.hi;
      if (has && lane == 0) ok = do_s(0, true) && do_dp(0, lo + 1 == hi);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      while (has && ok) {
        const bool keep = i > lo, closes = i + 1 == hi;
        bool more = true;
        int i1 = i + 1;
        if (closes) {
          more = take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 409, ok);
          i1 = u.lo;
        }
        if (lane == 0 && ok) {
          do {
            // the sums of the unit before have been read
            if (!keep && nu > 1 && !(ok = mbar_wait(&bar[kBkAccEmpty], (nu - 2) & 1, ctx, 413))) break;
            if (!(ok = mbar_wait(&bar[kBkPFull], n & 1, ctx, 414))) break;
            tc_fence_after();
            accumulate(tmem + Cfg::kColdV, tmem + Cfg::kColS, base + Cfg::kOffdO + (n & 1) * Cfg::kTileBytes, keep);
            umma_commit(&bar[kBkOEmpty0 + (n & 1)]);
            if (more && !(ok = do_s(n + 1, closes))) break;
            if (!(ok = mbar_wait(&bar[kBkDSFull], n & 1, ctx, 415))) break;
            tc_fence_after();
            accumulate(tmem + Cfg::kColdK, tmem + Cfg::kColX, base + Cfg::kOffQ + (n & 1) * Cfg::kTileBytes, keep);
            umma_commit(&bar[kBkQEmpty0 + (n & 1)]);
            if (closes) umma_commit(&bar[kBkAcc]);
            if (more && !(ok = do_dp(n + 1, i1 + 1 == u.hi))) break;
          } while (false);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        lo = u.lo;
        hi = u.hi;
        i = i1;
        has = more;
        ++n;
      }
      if (!ok && lane == 0) {
        umma_commit(&bar[kBkDrain]);
        mbar_wait_drain(&bar[kBkDrain], 0, p.timeout_ns);
      }
      __syncwarp();
    } else if (warp == 14) {
      if (lane == 0) feed_units<T, false>(p, ring, unit_full, unit_empty, ctx, 405);
      __syncwarp();
    } else {
      // ---- key tiles without a valid key: dK = dV = 0
      const int64_t thread = static_cast<int64_t>(blockIdx.x) * 32 + lane, threads = 32ll * gridDim.x;
      if (p.lens)
        for (int b = 0; b < p.B; ++b) {
          const int from = (valid_rows(p.lens, b, p.N) + kTile - 1) / kTile * kTile;
          if (from < p.N) {
            zero_rows<T, D>(p.dK, b, p.Hkv, from, p.N, thread, threads);
            zero_rows<T, D>(p.dV, b, p.Hkv, from, p.N, thread, threads);
          }
        }
    }
  } else if (warp < 8) {
    // ---- P^T and dS^T
    regs_raise<kBwdComputeRegs>();
    const int c = warp >> 2, r = threadIdx.x & 127;  // r: key within the tile (TMEM lane)
    const uint32_t lanes = static_cast<uint32_t>(r & 96) << 16;
    const uint32_t tS = tmem + Cfg::kColS + 64 * c + lanes, tX = tmem + Cfg::kColX + 64 * c + lanes;
    const float sl2 = p.scale * kLog2e;
    const float ds_mul = pow2(ds_exponent<T, D>(p, lane) - kPBias);
    int n = 0;
    while (take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 419, ok)) {
      // a key that does not count gets P = dS = 0, whatever K and V hold
      const bool valid = u.idx * kTile + r < u.n;
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
          a.x = ex2_approx(a.x);
          a.y = ex2_approx(a.y);
          b.x = ex2_approx(b.x);
          b.y = ex2_approx(b.y);
          s[4 * x] = __float_as_uint(a.x);
          s[4 * x + 1] = __float_as_uint(a.y);
          s[4 * x + 2] = __float_as_uint(b.x);
          s[4 * x + 3] = __float_as_uint(b.y);
          e[2 * x] = Elem<T>::pack(a.x, a.y);
          e[2 * x + 1] = Elem<T>::pack(b.x, b.y);
        }
        if (!valid) {
#pragma unroll
          for (int x = 0; x < 32; ++x) e[x] = 0u;
        }
        __syncwarp();
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
        if (!valid) {
#pragma unroll
          for (int x = 0; x < 32; ++x) e[x] = 0u;
        }
        __syncwarp();
        tmem_store_32(tX, e);
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBkDSFull]);
      }
    }
  } else {
    // ---- dV and dK: thread = key
    regs_lower<kBwdOtherRegs>();
    const int r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(r & 96) << 16;
    const float dk_mul = p.scale * pow2(-ds_exponent<T, D>(p, lane)), dv_mul = pow2(-kPBias);
    int nu = 0;
    while (take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 429, ok)) {
      if (!mbar_wait(&bar[kBkAcc], nu & 1, ctx, 430)) { ok = false; continue; }
      ++nu;
      __syncwarp();
      tc_fence_after();
      const int key = u.idx * kTile + r;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const View<T>& v = which == 0 ? p.dV : p.dK;
        store_sums<T, D>(tmem + (which == 0 ? Cfg::kColdV : Cfg::kColdK) + lanes,
                         key < p.N ? reinterpret_cast<uint8_t*>(v.at(u.b, u.hk, key)) : nullptr,
                         which == 0 ? dv_mul : dk_mul,
                         u.slot < 0 ? nullptr : p.part + ((static_cast<int64_t>(u.slot) * 2 + which) * kTile + r) * D, lane);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[kBkAccEmpty]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) publish_failure(*abort_flag, p.status);
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ===================================================================== join
// Items that fell to several CTAs: adds their partial sums in CTA order. Block
// (x, c - 1, z) looks at the boundary before CTA c of the dQ (z = 0) or the
// dK/dV kernel; the first boundary inside an item owns it. kJoinBlocks blocks
// share the item's two [128][D] sums, one thread per 4 columns.
constexpr int kJoinBlocks = 8;
struct JoinItem {
  BwdUnit u;
  int slots, from;  // partial sums, of CTAs from on
  int begins;       // CTA `from` begins in the item: its first slot, else its second
};

template <typename T, bool kQMajor>
__device__ JoinItem join_item(const BwdParams<T>& p, int grid, int c) {
  JoinItem it;
  it.slots = 0;
  BwdSchedule<T, kQMajor> sched(p, grid, c);
  if (!sched.by_steps || sched.pos >= sched.total || c >= sched.parts) return it;
  const int at = sched.pos;
  sched.end = sched.total;  // the whole item around the boundary
  sched.next(it.u);
  const int start = at - it.u.lo, stop = start + it.u.len;
  if (it.u.lo == 0 || sched.mark(c - 1) > start) return it;
  it.from = c - 1;
  it.begins = sched.mark(c - 1) == start ? 1 : 0;
  int e = c;
  while (e < sched.parts && sched.mark(e) < stop) ++e;
  it.slots = e - it.from;
  return it;
}

template <typename T, int D>
__global__ void __launch_bounds__(256)
    attn_bwd_join_kernel(const __grid_constant__ BwdParams<T> q, const __grid_constant__ BwdParams<T> kv, int grid_q,
                         int grid_k) {
  __shared__ JoinItem shared;
  const bool q_major = blockIdx.z == 0;
  const int c = blockIdx.y + 1;
  if (c >= (q_major ? grid_q : grid_k)) return;
  if (threadIdx.x == 0)
    shared = q_major ? join_item<T, true>(q, grid_q, c) : join_item<T, false>(kv, grid_k, c);
  __syncthreads();
  const JoinItem it = shared;
  if (it.slots == 0) return;
  const BwdParams<T>& p = q_major ? q : kv;
  const int ds_exp = ds_exponent<T, D>(p, threadIdx.x & 31);
  const float4* part = reinterpret_cast<const float4*>(p.part);
  for (int e = blockIdx.x * 256 + threadIdx.x; e < 2 * kTile * (D / 4); e += kJoinBlocks * 256) {
    const int which = e / (kTile * (D / 4)), row = e / (D / 4) % kTile, col = e % (D / 4);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < it.slots; ++k) {
      const int slot = 2 * (it.from + k) + (k == 0 && !it.begins ? 1 : 0);
      const float4 v = __ldcg(part + static_cast<int64_t>(slot) * (2 * kTile * (D / 4)) + e);
      a.x += v.x;
      a.y += v.y;
      a.z += v.z;
      a.w += v.w;
    }
    T* out = nullptr;
    float mul = p.scale * pow2(-ds_exp);
    if (q_major) {
      int m, g, s;
      const int tile = 2 * it.u.idx + which;
      if (tile < p.rows.tiles && p.rows.row(tile, row, m, g, s)) out = p.dQ.at(it.u.b, it.u.hk * p.rows.G + g, m);
    } else {
      const int key = it.u.idx * kTile + row;
      if (which == 0) mul = Elem<T>::kBF16 ? 1.f : pow2(-10);
      if (key < p.N) out = (which == 0 ? p.dV : p.dK).at(it.u.b, it.u.hk, key);
    }
    if (out)
      *reinterpret_cast<uint2*>(out + 4 * col) =
          make_uint2(Elem<T>::pack(mul * a.x, mul * a.y), Elem<T>::pack(mul * a.z, mul * a.w));
  }
}

}  // namespace fmha_sm100
