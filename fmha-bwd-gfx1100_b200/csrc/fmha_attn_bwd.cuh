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

// This thread's row of D sums in TMEM, to a partial-sum slot or, scaled, to
// its 16-bit output row (null: none).
template <typename T, int D>
__device__ __forceinline__ void store_sums(uint32_t taddr, T* out, float mul, float* part, int lane) {
  uint8_t* row = part ? reinterpret_cast<uint8_t*>(part) : reinterpret_cast<uint8_t*>(out);
  const float by = part ? 1.f : mul;
#pragma unroll 1
  for (int x = 0; x < D / 32; ++x) {
    uint32_t v[32];
    tmem_load_32(taddr + 32 * x, v);
    store_row_32(part != nullptr, row, x, v, by, lane, T());
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
// the TMA producer (warp 12), two MMA issuers (13, 15) and the scheduler (14),
// whose other lanes zero what has no keys. Registers: 2 * 128 * 184 + 2 * 128 *
// 72, the 512 * 128 of the launch.
constexpr int kBwdThreads = 512, kBwdComputeRegs = 184, kBwdOtherRegs = 72;
static_assert(2 * kBwdComputeRegs + 2 * kBwdOtherRegs == 4 * 128, "register split");
constexpr int kUnitReaders = 15;  // warps 0-13 and 15

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
  kBqDrain0 = 32,   // + tile
  kBqUnitFull0 = 34,
  kBqUnitEmpty0 = 38,
  kBqTail0 = 42,    // + slot: a last K tile has landed, its rows behind the keys not yet cleared
  kNumBqBars = 46,
};

// Zeroes the dS (16-bit pairs in TMEM) of the keys of the last 16 that count
// in part, at and past `left`; the products do not reach further.
__device__ __forceinline__ void clear_ds(uint32_t taddr, int left) {
  if ((left & 15) == 0) return;
  uint32_t v[8];
  const int c = left & ~15;
  tmem_load_8(taddr + c / 2, v);
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    if (c + 2 * x >= left) v[x] = 0u;
    else if (c + 2 * x + 1 >= left) v[x] &= 0xffffu;
  }
  tmem_store_8(taddr + c / 2, v);
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
      int count = 1;
      if ((i >= kBqKEmpty0 && i < kBqVFull0) || (i >= kBqVEmpty0 && i < kBqSFull0)) count = 2;
      if ((i >= kBqSRead0 && i < kBqXFull0) || (i >= kBqDSFull0 && i < kBqAcc0) || (i >= kBqAccEmpty0 && i < kBqDrain0))
        count = 4;
      if (i >= kBqUnitEmpty0 && i < kBqTail0) count = kUnitReaders;
      mbar_init(&bar[i], count);
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
      // ---- TMA producer
      if (elect_one()) {
        tma_prefetch_desc(&tm_Q);
        tma_prefetch_desc(&tm_K);
        tma_prefetch_desc(&tm_V);
        tma_prefetch_desc(&tm_dO);
        const uint64_t pol_q = l2_policy_evict_first(), pol_kv = l2_policy_evict_last();
        const uint32_t q_bytes = static_cast<uint32_t>(p.rows.Mt * p.rows.Gt) * 128u * (D / kBoxCols);
        int nq[2] = {0, 0}, nk = 0, nv = 0, tails = 0;
        auto load_k = [&](int j) {
          const int s = nk % SK;
          if (nk >= SK && !mbar_wait(&bar[kBqKEmpty0 + s], ((nk / SK) - 1) & 1, ctx, 302)) return false;
          const bool tail = j + 1 == u.hi && has_tail(u.n, u.hi);
          if (tail) tails |= 1 << s;
          uint64_t* fb = &bar[(tail ? kBqTail0 : kBqKFull0) + s];
          mbar_arrive_expect_tx(fb, Cfg::kTileBytes);
#pragma unroll
          for (int x = 0; x < D / kBoxCols; ++x)
            tma_load_4d(smem + Cfg::kOffK + s * Cfg::kTileBytes + x * kBoxBytes, &tm_K, fb, x * kBoxCols, j * kTile, u.hk,
                        u.b, pol_kv);
          ++nk;
          return true;
        };
        while (take_unit<false>(ring, unit_full, unit_empty, k, u, ctx, 300, ok)) {
#pragma unroll 1
          for (int t = 0; t < 2 && ok; ++t) {
            const int tile = 2 * u.idx + t;
            if (tile >= q_tiles) break;
            if (nq[t] > 0 && !(ok = mbar_wait(&bar[kBqQEmpty0 + t], (nq[t] - 1) & 1, ctx, 301))) break;
            const int m0 = tile % p.rows.nm * p.rows.Mt, h0 = u.hk * p.rows.G + tile / p.rows.nm * p.rows.Gt;
            mbar_arrive_expect_tx(&bar[kBqQFull0 + t], 2 * q_bytes);
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x) {
              tma_load_4d(smem + Cfg::kOffQ + t * Cfg::kTileBytes + x * kBoxBytes, &tm_Q, &bar[kBqQFull0 + t],
                          x * kBoxCols, m0, h0, u.b, pol_q);
              tma_load_4d(smem + Cfg::kOffdO + t * Cfg::kTileBytes + x * kBoxBytes, &tm_dO, &bar[kBqQFull0 + t],
                          x * kBoxCols, m0, h0, u.b, pol_q);
            }
            ++nq[t];
            if (t == 0) ok = load_k(u.lo);
          }
          for (int j = u.lo; j < u.hi && ok; ++j) {
            const int s = nv % SV;
            if (nv >= SV && !(ok = mbar_wait(&bar[kBqVEmpty0 + s], ((nv / SV) - 1) & 1, ctx, 303))) break;
            mbar_arrive_expect_tx(&bar[kBqVFull0 + s], Cfg::kTileBytes);
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x)
              tma_load_4d(smem + Cfg::kOffV + s * Cfg::kTileBytes + x * kBoxBytes, &tm_V, &bar[kBqVFull0 + s],
                          x * kBoxCols, j * kTile, u.hk, u.b, pol_kv);
            ++nv;
            if (j + 1 < u.hi) ok = load_k(j + 1);
          }
        }
        if (*abort_flag) {  // every copy in flight ends before the block does
          for (int t = 0; t < 2; ++t)
            if (nq[t] > 0) mbar_wait_drain(&bar[kBqQFull0 + t], (nq[t] - 1) & 1, p.timeout_ns);
          for (int i = (nk > SK ? nk - SK : 0); i < nk; ++i) {
            mbar_wait_drain(&bar[kBqKFull0 + i % SK], (i / SK) & 1, 1000000);
            if (tails >> (i % SK) & 1)
              for (int par = 0; par < 2; ++par) mbar_wait_drain(&bar[kBqTail0 + i % SK], par, 1000000);
          }
          for (int i = (nv > SV ? nv - SV : 0); i < nv; ++i)
            mbar_wait_drain(&bar[kBqVFull0 + i % SV], (i / SV) & 1, p.timeout_ns);
        }
      }
      __syncwarp();
    } else if (warp == 14) {
      if (lane == 0) {
        feed_units<T, true>(p, ring, unit_full, unit_empty, ctx, 305);
      } else if (p.lens) {
        // the other lanes: entries without keys have dQ = 0
        for (int b = 0; b < p.B; ++b)
          if (valid_rows(p.lens, b, p.N) == 0)
            zero_rows<T, D>(p.dQ, b, p.Hkv * p.rows.G, 0, p.rows.M, static_cast<int64_t>(blockIdx.x) * 31 + lane - 1,
                            31ll * gridDim.x);
      }
      __syncwarp();
    } else {
      // ---- MMA issuer of tile t: per step dP, dQ, and S of the next step. A
      // thread for each tile keeps one tile's wait from holding up the other's
      // products.
      const int t = warp == 13 ? 0 : 1;
      if (elect_one()) {
        constexpr uint32_t id_S = make_idesc_f16<kB>(kTile, kTile, false, false);
        constexpr uint32_t id_A = make_idesc_f16<kB>(kTile, D, false, true);
        const uint32_t sK = smem_u32(smem + Cfg::kOffK), sV = smem_u32(smem + Cfg::kOffV);
        const uint64_t dq = make_sw128_desc(smem_u32(smem + Cfg::kOffQ + t * Cfg::kTileBytes), 16, 1024);
        const uint64_t ddo = make_sw128_desc(smem_u32(smem + Cfg::kOffdO + t * Cfg::kTileBytes), 16, 1024);
        const uint32_t tR = tmem + 128 * t, tA = tmem + 256 + D * t;
        int g = 0, n = 0, nq = 0;  // steps of the CTA, steps and units of the tile
        auto product = [&](uint64_t da, uint32_t b) {  // A, B K-major over D
          const uint64_t db = make_sw128_desc(b, 16, 1024);
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            const uint32_t off = (x >> 2) * kBoxBytes + (x & 3) * 32;
            umma_f16_ss(tR, desc_advance(da, off), desc_advance(db, off), id_S, x > 0 ? 1u : 0u);
          }
        };
        while (take_unit<false>(ring, unit_full, unit_empty, k, u, ctx, 309 + 10 * t, ok)) {
          const bool alone = 2 * u.idx + 1 >= q_tiles;
          if (t == 1 && alone) {
            g += u.hi - u.lo;
            continue;
          }
          if (!(ok = mbar_wait(&bar[kBqQFull0 + t], nq & 1, ctx, 311 + 10 * t))) break;
          for (int j = u.lo - 1; j < u.hi; ++j) {
            if (j >= u.lo) {
              // dP_j over S_j once the warps have that in registers
              if (!(ok = mbar_wait(&bar[kBqVFull0 + g % SV], (g / SV) & 1, ctx, 312 + 10 * t))) break;
              if (!(ok = mbar_wait(&bar[kBqSRead0 + t], n & 1, ctx, 313 + 10 * t))) break;
              tc_fence_after();
              product(ddo, sV + (g % SV) * Cfg::kTileBytes);
              umma_commit(&bar[kBqXFull0 + t]);
              umma_commit(&bar[kBqVEmpty0 + g % SV]);
              if (alone) umma_commit(&bar[kBqVEmpty0 + g % SV]);
              if (j + 1 == u.hi) umma_commit(&bar[kBqQEmpty0 + t]);
              // dQ += dS_j K_j
              if (j == u.lo && nq > 0 && !(ok = mbar_wait(&bar[kBqAccEmpty0 + t], (nq - 1) & 1, ctx, 314 + 10 * t))) break;
              if (!(ok = mbar_wait(&bar[kBqDSFull0 + t], n & 1, ctx, 315 + 10 * t))) break;
              tc_fence_after();
              const uint64_t dk = make_sw128_desc(sK + (g % SK) * Cfg::kTileBytes, kBoxBytes, 1024);
              const uint32_t keep = j > u.lo ? 1u : 0u;
              const int left = u.n - j * kTile;
              if (left >= kTile) {
#pragma unroll
                for (int x = 0; x < kTile / 16; ++x)
                  umma_f16_ts(tA, tR + x * 8, desc_advance(dk, x * 2048), id_A, x > 0 ? 1u : keep);
              } else {
                for (int x = 0; x < (left + 15) / 16; ++x)
                  umma_f16_ts(tA, tR + x * 8, desc_advance(dk, x * 2048), id_A, x > 0 ? 1u : keep);
              }
              umma_commit(&bar[kBqKEmpty0 + g % SK]);
              if (alone) umma_commit(&bar[kBqKEmpty0 + g % SK]);
              if (j + 1 == u.hi) umma_commit(&bar[kBqAcc0 + t]);
              ++n;
              ++g;
            }
            if (j + 1 < u.hi) {  // S_(j+1)
              if (!(ok = mbar_wait(&bar[kBqKFull0 + g % SK], (g / SK) & 1, ctx, 310 + 10 * t))) break;
              tc_fence_after();
              product(dq, sK + (g % SK) * Cfg::kTileBytes);
              umma_commit(&bar[kBqSFull0 + t]);
            }
          }
          if (!ok) break;
          ++nq;
        }
        if (!ok) {
          umma_commit(&bar[kBqDrain0 + t]);
          mbar_wait_drain(&bar[kBqDrain0 + t], 0, p.timeout_ns);
        }
      }
      __syncwarp();
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
        auto weights = [&](uint32_t* v) {  // P of 64 columns, every fourth pair by polynomial
#pragma unroll
          for (int x = 0; x < 64; x += 2) {
            float2 a = fma_f32x2(make_float2(__uint_as_float(v[x]), __uint_as_float(v[x + 1])), make_float2(sl2, sl2),
                                 make_float2(nl, nl));
            if ((x & 7) == 6) {
              a = ex2_poly(a);
            } else {
              a.x = ex2_approx(a.x);
              a.y = ex2_approx(a.y);
            }
            v[x] = __float_as_uint(a.x);
            v[x + 1] = __float_as_uint(a.y);
          }
        };
        tmem_load_64_start(tR, s);
        tmem_load_64_wait(s);
        tmem_load_64_start(tR + 64, s + 64);
        weights(s);
        tmem_load_64_wait(s + 64);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBqSRead0 + t]);
        weights(s + 64);
        if (!mbar_wait(&bar[kBqXFull0 + t], ns & 1, ctx, 321)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          uint32_t dp[16], e[8];
          tmem_load_16(tR + 16 * q, dp);
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float2 a = fma_f32x2(make_float2(__uint_as_float(dp[2 * x]), __uint_as_float(dp[2 * x + 1])),
                                       make_float2(ds_mul, ds_mul), make_float2(nd, nd));
            const float2 d = mul_f32x2(a, make_float2(__uint_as_float(s[16 * q + 2 * x]), __uint_as_float(s[16 * q + 2 * x + 1])));
            e[x] = Elem<T>::pack(d.x, d.y);
          }
          tmem_store_8(tR + 8 * q, e);
        }
        if (u.n - j * kTile < kTile) {
          tmem_store_wait();
          clear_ds(tR, u.n - j * kTile);
        }
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBqDSFull0 + t]);
      }
    }
  } else {
    // ---- dQ: thread = row of each tile in turn; warp 8 also clears the last
    // K tile behind the last key, for the issuers that wait for it
    regs_lower<kBwdOtherRegs>();
    const int r = threadIdx.x & 127;
    const float out_mul = p.scale * pow2(-ds_exponent<T, D>(p, lane));
    int na0 = 0, na1 = 0, g = 0;
    uint32_t tail_turns = 0;
    while (take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 329, ok)) {
      g += u.hi - u.lo;
      if (warp == 8 && has_tail(u.n, u.hi)) {
        const int slot = (g - 1) % SK;
        if (!mbar_wait(&bar[kBqTail0 + slot], tail_turns >> slot & 1, ctx, 331)) ok = false;
        tail_turns ^= 1u << slot;
        __syncwarp();
        if (ok) clear_tail<D>(smem + Cfg::kOffK + slot * Cfg::kTileBytes, u.n - (u.hi - 1) * kTile, lane);
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(&bar[kBqKFull0 + slot]);
      }
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        const int tile = 2 * u.idx + t;
        if (tile >= q_tiles) continue;
        if (ok && !mbar_wait(&bar[kBqAcc0 + t], (t == 0 ? na0 : na1) & 1, ctx, 330)) ok = false;
        if (!ok) break;
        if (t == 0) ++na0;
        else ++na1;
        __syncwarp();
        tc_fence_after();
        int m, g, s;
        const bool real = p.rows.row(tile, r, m, g, s);
        T* out = real ? p.dQ.at(u.b, u.hk * p.rows.G + g, m) : nullptr;
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
// The warps form dS^T during dV and S^T of the next tile, and its P^T during
// dK and the next dP^T.
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
  kBkDrain0 = 16,   // + issuer
  kBkUnitFull0 = 18,
  kBkUnitEmpty0 = 22,
  kNumBkBars = 26,
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
      {
      int count = 1;
      if (i == kBkKVEmpty || i == kBkOEmpty0 || i == kBkOEmpty0 + 1 || i == kBkAcc) count = 2;
      if (i == kBkPFull || i == kBkDSFull) count = 8;
      if (i == kBkAccEmpty) count = 4;
      if (i >= kBkUnitEmpty0) count = kUnitReaders;
      mbar_init(&bar[i], count);
    }
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
      if (elect_one()) {
        tma_prefetch_desc(&tm_Q);
        tma_prefetch_desc(&tm_K);
        tma_prefetch_desc(&tm_V);
        tma_prefetch_desc(&tm_dO);
        const uint64_t pol_q = l2_policy_evict_last(), pol_kv = l2_policy_evict_first();
        const uint32_t q_bytes = static_cast<uint32_t>(box_rows) * 128u * (D / kBoxCols);
        int nu = 0, n = 0, no = 0;
        while (take_unit<false>(ring, unit_full, unit_empty, k, u, ctx, 400, ok)) {
          if (nu > 0 && !(ok = mbar_wait(&bar[kBkKVEmpty], (nu - 1) & 1, ctx, 401))) break;
          mbar_arrive_expect_tx(&bar[kBkKV], 2 * Cfg::kTileBytes);
#pragma unroll
          for (int x = 0; x < D / kBoxCols; ++x) {
            tma_load_4d(smem + Cfg::kOffK + x * kBoxBytes, &tm_K, &bar[kBkKV], x * kBoxCols, u.idx * kTile, u.hk, u.b,
                        pol_kv);
            tma_load_4d(smem + Cfg::kOffV + x * kBoxBytes, &tm_V, &bar[kBkKV], x * kBoxCols, u.idx * kTile, u.hk, u.b,
                        pol_kv);
          }
          ++nu;
          for (int i = u.lo; i < u.hi; ++i) {
            const int s = n & 1;
            const int m0 = i % p.rows.nm * p.rows.Mt, h0 = u.hk * p.rows.G + i / p.rows.nm * p.rows.Gt;
            const int64_t row = ((static_cast<int64_t>(u.b) * p.Hkv + u.hk) * q_tiles + i) * kTile;
            if (n >= 2 && !(ok = mbar_wait(&bar[kBkQEmpty0 + s], ((n >> 1) - 1) & 1, ctx, 402))) break;
            mbar_arrive_expect_tx(&bar[kBkQFull0 + s], q_bytes + 2 * kTile * 4);
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x)
              tma_load_4d(smem + Cfg::kOffQ + s * Cfg::kTileBytes + x * kBoxBytes, &tm_Q, &bar[kBkQFull0 + s],
                          x * kBoxCols, m0, h0, u.b, pol_q);
            bulk_load(smem + Cfg::kOffL + s * 2 * kTile * 4, p.lse2 + row, kTile * 4, &bar[kBkQFull0 + s]);
            bulk_load(smem + Cfg::kOffL + (s * 2 + 1) * kTile * 4, p.delta + row, kTile * 4, &bar[kBkQFull0 + s]);
            ++n;
            if (no >= 2 && !(ok = mbar_wait(&bar[kBkOEmpty0 + s], ((no >> 1) - 1) & 1, ctx, 403))) break;
            mbar_arrive_expect_tx(&bar[kBkOFull0 + s], q_bytes);
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x)
              tma_load_4d(smem + Cfg::kOffdO + s * Cfg::kTileBytes + x * kBoxBytes, &tm_dO, &bar[kBkOFull0 + s],
                          x * kBoxCols, m0, h0, u.b, pol_q);
            ++no;
          }
          if (!ok) break;
        }
        if (*abort_flag) {  // every copy in flight ends before the block does
          if (nu > 0) mbar_wait_drain(&bar[kBkKV], (nu - 1) & 1, p.timeout_ns);
          for (int i = (n > 2 ? n - 2 : 0); i < n; ++i)
            mbar_wait_drain(&bar[kBkQFull0 + (i & 1)], (i >> 1) & 1, p.timeout_ns);
          for (int i = (no > 2 ? no - 2 : 0); i < no; ++i)
            mbar_wait_drain(&bar[kBkOFull0 + (i & 1)], (i >> 1) & 1, p.timeout_ns);
        }
      }
      __syncwarp();
    } else if (warp == 14) {
      if (lane == 0) {
        feed_units<T, false>(p, ring, unit_full, unit_empty, ctx, 405);
      } else if (p.lens) {
        // the other lanes: key tiles without a valid key have dK = dV = 0
        const int64_t thread = static_cast<int64_t>(blockIdx.x) * 31 + lane - 1, threads = 31ll * gridDim.x;
        for (int b = 0; b < p.B; ++b) {
          const int from = (valid_rows(p.lens, b, p.N) + kTile - 1) / kTile * kTile;
          if (from < p.N) {
            zero_rows<T, D>(p.dK, b, p.Hkv, from, p.N, thread, threads);
            zero_rows<T, D>(p.dV, b, p.Hkv, from, p.N, thread, threads);
          }
        }
      }
      __syncwarp();
    } else {
      // ---- MMA issuers: warp 13 dV and S^T of the next row tile (TMEM S, P),
      // warp 15 dK and dP^T of the next (TMEM X), so that neither chain's
      // waits hold up the other's products.
      const int w = warp == 13 ? 0 : 1;
      if (elect_one()) {
        constexpr uint32_t id_S = make_idesc_f16<kB>(kTile, kTile, false, false);
        constexpr uint32_t id_A = make_idesc_f16<kB>(kTile, D, false, true);
        const uint32_t base = smem_u32(smem);
        const uint64_t da = make_sw128_desc(base + (w == 0 ? Cfg::kOffK : Cfg::kOffV), 16, 1024);  // K or V
        const uint32_t first = base + (w == 0 ? Cfg::kOffQ : Cfg::kOffdO);   // Q or dO slots: S^T, dP^T
        const uint32_t second = base + (w == 0 ? Cfg::kOffdO : Cfg::kOffQ);  // dO or Q slots: dV, dK
        const uint32_t tR = tmem + (w == 0 ? Cfg::kColS : Cfg::kColX), tA = tmem + (w == 0 ? Cfg::kColdV : Cfg::kColdK);
        uint64_t* landed = &bar[w == 0 ? kBkQFull0 : kBkOFull0];
        uint64_t* formed = &bar[w == 0 ? kBkPFull : kBkDSFull];
        int n = 0, nu = 0;
        while (take_unit<false>(ring, unit_full, unit_empty, k, u, ctx, 409 + 10 * w, ok)) {
          if (!(ok = mbar_wait(&bar[kBkKV], nu & 1, ctx, 410 + 10 * w))) break;
          for (int i = u.lo - 1; i < u.hi; ++i) {
            if (i >= u.lo) {
              if (i == u.lo && nu > 0 && !(ok = mbar_wait(&bar[kBkAccEmpty], (nu - 1) & 1, ctx, 413 + 10 * w))) break;
              if (!(ok = mbar_wait(formed, n & 1, ctx, 414 + 10 * w))) break;
              tc_fence_after();
              const uint64_t db = make_sw128_desc(second + (n & 1) * Cfg::kTileBytes, kBoxBytes, 1024);
#pragma unroll
              for (int x = 0; x < kTile / 16; ++x)
                umma_f16_ts(tA, tR + (x >> 2) * 64 + (x & 3) * 8, desc_advance(db, x * 2048), id_A,
                            x > 0 || i > u.lo ? 1u : 0u);
              umma_commit(&bar[(w == 0 ? kBkOEmpty0 : kBkQEmpty0) + (n & 1)]);
              if (i + 1 == u.hi) umma_commit(&bar[kBkAcc]);
              ++n;
            }
            if (i + 1 < u.hi) {
              if (!(ok = mbar_wait(landed + (n & 1), (n >> 1) & 1, ctx, 411 + 10 * w))) break;
              tc_fence_after();
              const uint64_t db = make_sw128_desc(first + (n & 1) * Cfg::kTileBytes, 16, 1024);
#pragma unroll
              for (int x = 0; x < D / 16; ++x) {
                const uint32_t off = (x >> 2) * kBoxBytes + (x & 3) * 32;
                umma_f16_ss(tR, desc_advance(da, off), desc_advance(db, off), id_S, x > 0 ? 1u : 0u);
              }
              umma_commit(&bar[w == 0 ? kBkSFull : kBkXFull]);
              // dO has two readers that do not wait for one another; Q's second, dK, waits for its first
              if (w == 1) umma_commit(&bar[kBkOEmpty0 + (n & 1)]);
              if (i + 2 == u.hi) umma_commit(&bar[kBkKVEmpty]);
            }
          }
          if (!ok) break;
          ++nu;
        }
        if (!ok) {
          umma_commit(&bar[kBkDrain0 + w]);
          mbar_wait_drain(&bar[kBkDrain0 + w], 0, p.timeout_ns);
        }
      }
      __syncwarp();
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
          if (x & 1) {
            b = ex2_poly(b);
          } else {
            b.x = ex2_approx(b.x);
            b.y = ex2_approx(b.y);
          }
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
#pragma unroll 1
      for (int which = 0; which < 2; ++which) {
        const View<T>& v = which == 0 ? p.dV : p.dK;
        store_sums<T, D>(tmem + (which == 0 ? Cfg::kColdV : Cfg::kColdK) + lanes,
                         key < p.N ? v.at(u.b, u.hk, key) : nullptr,
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
