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
// that hold no row have -LSE = -inf, hence P = 0.
//
// Work is divided by steps (one key tile for one pair of row tiles; one row
// tile for one key tile), counted on the device from the lengths. If whole
// items leave the SMs uneven, each CTA takes an equal run of steps instead;
// an item that falls to several CTAs leaves fp32 sums for the join, which adds
// them in order.
//
// P and dS are rounded to 16 bits for the tensor cores, after dS was formed
// from the fp32 P. In fp16, P is held times 2^10 and dS times 2^e, with an e for
// each kv head of an entry from its own largest finite |dO| and |V|, so that 2 d
// |dO| |V| 2^e <= 2^15: dS cannot overflow, and what the other heads and entries
// hold takes nothing from its precision. Within a head, dS below 2^-29 of that
// bound falls to fp16's subnormals.
#pragma once

#include "fmha_attn_fwd.cuh"

namespace fmha_sm100 {

template <typename T>
struct BwdParams {
  RowPack rows;       // S = 1, Gt divides G
  int B, Hkv, N, pairs;
  const int* lens;
  View<T> dQ, dK, dV;
  const float* nlse2;   // [B * Hkv * tiles * 128] -LSE log2e (+ 10 in fp16), packed rows
  const float* ndelta;  // the same rows' -D
  const float* top_do;  // [B * Hkv][row tiles], fp16 only: a tile's largest finite |dO|
  const float* top_v;   // [B * Hkv][key tiles], fp16 only: and |V| of its valid keys
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
  int exp;         // the power of two by which dS is held (ds_exponent)
};

// Steps that a division by steps has to save, as its partial sums cost about
// as much, and the least number of steps of a CTA under it: of a query-major
// step, which takes twice as long, half as many (with 4 of either 768 key-major
// steps take 50 us, with 8 36; with 8 of either 16 items of 12 query-major ones
// 55 instead of 42).
constexpr int kBwdSpare = 8, kBwdLeastQ = 4, kBwdLeastK = 8;
__host__ __device__ inline bool bwd_by_steps(int64_t whole, int64_t total, int64_t grid) {
  return whole > (total + grid - 1) / grid + kBwdSpare;
}
__host__ __device__ inline int bwd_parts(int64_t total, int grid, bool q_major) {
  const int least = q_major ? kBwdLeastQ : kBwdLeastK;
  const int64_t most = (total + least - 1) / least;
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
    // steps of the busiest CTA with whole items: all of them as long as the
    // longest, or the entries one after another, whichever bounds it better
    int most = 0, apart = 0;
    if (!p.lens) {
      most = len_of(key_tiles(0));
      items = items_of(key_tiles(0)) * p.B;
      total = items * most;
      apart = (items + grid - 1) / grid * most;
    } else {
      for (int e = 0; e < p.B; ++e) {
        const int nt = key_tiles(e), n = items_of(nt), len = len_of(nt);
        most = max(most, len);
        items += n;
        total += n * len;
        apart += (n + grid - 1) / grid * len;
      }
    }
    by_steps = bwd_by_steps(min((items + grid - 1) / grid * most, apart), total, grid);
    parts = bwd_parts(total, grid, kQMajor);
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

// The power of two by which a whole warp's fp16 holds dS of a unit's kv head
// (see the top): -25 to 54; 0 for bf16, and where all gradients are zero.
constexpr int kExpBias = 64;
template <typename T, int D>
__device__ __forceinline__ int ds_exponent(const BwdParams<T>& p, const BwdUnit& u, int lane) {
  if (Elem<T>::kBF16) return 0;
  const int64_t bh = static_cast<int64_t>(u.b) * p.Hkv + u.hk;
  const int key_tiles = (p.N + kTile - 1) / kTile;
  // no float here has a sign, so their bits compare as they do
  uint32_t x = 0, y = 0;
  for (int i = lane; i < p.rows.tiles; i += 32) x = max(x, __float_as_uint(__ldcg(p.top_do + bh * p.rows.tiles + i)));
  for (int i = lane; i * kTile < u.n; i += 32) y = max(y, __float_as_uint(__ldcg(p.top_v + bh * key_tiles + i)));
  x = __reduce_max_sync(0xffffffffu, x);
  y = __reduce_max_sync(0xffffffffu, y);
  if (x == 0 || y == 0) return 0;
  // below 2^ex and 2^ey
  const int ex = static_cast<int>(x >> 23) - 126, ey = static_cast<int>(y >> 23) - 126;
  return 15 - (D == 128 ? 8 : 7) - ex - ey;  // 2 d 2^ex 2^ey 2^e = 2^15
}

template <typename T, int D, bool kQMajor>
__device__ void feed_units(const BwdParams<T>& p, UnitRing* ring, uint64_t* full, uint64_t* empty, const WaitCtx& ctx,
                           int where) {
  BwdSchedule<T, kQMajor> sched(p, gridDim.x, blockIdx.x);
  const int lane = threadIdx.x & 31;
  BwdUnit u{};
  for (int k = 0;; ++k) {
    const bool more = sched.next(u);
    const int exp = more ? ds_exponent<T, D>(p, u, lane) : 0;
    bool ok = true;
    if (lane == 0)
      ok = put_unit(ring, full, empty, k, make_int4(u.b, u.hk, u.idx, u.slot),
                    make_int4(u.lo, u.hi, u.n, more ? kExpBias + exp : 0), ctx, where);
    if (!__all_sync(0xffffffffu, ok) || !more) return;
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
  u.exp = b.w - kExpBias;
  return true;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// ==================================================================== delta
// Per packed row: -LSE log2e (0 for a row without keys, -inf where the tile
// holds no row: P = 0) plus fp16's power of two of P, and -D. A block takes row
// tiles one by one, D / 8 threads a row, several rows' loads in flight. In fp16
// also a tile's largest finite |dO|, and a key tile's |V|. What the other kernels
// have no items for is zeroed here: dQ of entries without keys, dK and dV behind
// the last key (a tile's sums there would be NaN where Q or dO is). Bound by memory: 101
// MB (2 x 24 heads, 4096 rows of 128) take 25 to 31 us from DRAM; more blocks with
// fewer loads each were slower.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    attn_delta_kernel(View<T> dO, View<T> O, View<T> V, const float* __restrict__ LSE, BwdParams<T> p,
                      float* __restrict__ nlse2, float* __restrict__ ndelta, float* __restrict__ top_do,
                      float* __restrict__ top_v) {
  constexpr int kPer = D / 8, kStep = 256 / kPer, kBatch = 4;  // threads a row, rows a pass, passes at once
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int chunk = threadIdx.x % kPer, r0 = threadIdx.x / kPer;
  const int tiles = p.B * p.Hkv * p.rows.tiles;
  // largest magnitudes, two fp16 a word; infinities and NaN are left out
  uint32_t top = 0;
  auto widest = [&](const uint32_t (&w)[4]) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint32_t a = w[x] & 0x7fff7fffu;
      top = __vmaxu2(top, a & __vcmpltu2(a, 0x7c007c00u));
    }
  };
  // the block's, to `out`; each call's words are the other ones than the last's,
  // so that one barrier keeps them apart
  __shared__ uint32_t tops[2][8];
  int turn = 0;
  auto leave = [&](float* out) {
    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
    if (threadIdx.x % 32 == 0) tops[turn][threadIdx.x / 32] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < 8; ++w) top = max(top, tops[turn][w]);
      *out = __half2float(__ushort_as_half(static_cast<unsigned short>(top)));
    }
    turn ^= 1;
    top = 0;
  };
  for (int i = blockIdx.x; i < tiles; i += gridDim.x) {
    // kv heads innermost: with the usual [token][head] layouts, the blocks read neighbouring memory
    const int hk = i % p.Hkv, tile = i / p.Hkv % p.rows.tiles, b = i / p.Hkv / p.rows.tiles;
    const int64_t base = ((static_cast<int64_t>(b) * p.Hkv + hk) * p.rows.tiles + tile) * kTile;
    if (valid_rows(p.lens, b, p.N) == 0) {  // apart from the loads below, which must not wait for it
#pragma unroll 1
      for (int r = r0; r < kTile; r += kStep) {
        int m, g, s;
        if (p.rows.row(tile, r, m, g, s))
          reinterpret_cast<uint4*>(p.dQ.at(b, hk * p.rows.G + g, m))[chunk] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll 1
    for (int r = r0; r < kTile; r += kBatch * kStep) {
      uint4 x[kBatch], y[kBatch];
      float l[kBatch];
      bool real[kBatch];
#pragma unroll
      for (int i4 = 0; i4 < kBatch; ++i4) {  // all of the batch's loads first
        int m, g, s;
        real[i4] = p.rows.row(tile, r + i4 * kStep, m, g, s);
        x[i4] = y[i4] = make_uint4(0, 0, 0, 0);
        l[i4] = 0.f;
        if (real[i4]) {
          x[i4] = __ldg(reinterpret_cast<const uint4*>(dO.at(b, hk * p.rows.G + g, m)) + chunk);
          y[i4] = __ldg(reinterpret_cast<const uint4*>(O.at(b, hk * p.rows.G + g, m)) + chunk);
          l[i4] = __ldg(LSE + (static_cast<int64_t>(b) * p.Hkv * p.rows.G + hk * p.rows.G + g) * p.rows.M + m);
        }
      }
#pragma unroll
      for (int i4 = 0; i4 < kBatch; ++i4) {
        const uint32_t xw[4] = {x[i4].x, x[i4].y, x[i4].z, x[i4].w}, yw[4] = {y[i4].x, y[i4].y, y[i4].z, y[i4].w};
        float acc = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float2 a = Elem<T>::unpack(xw[t]), c = Elem<T>::unpack(yw[t]);
          acc = fmaf(a.x, c.x, acc);
          acc = fmaf(a.y, c.y, acc);
        }
        if (!Elem<T>::kBF16) widest(xw);
#pragma unroll
        for (int o = kPer / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o, kPer);
        if (chunk == 0) {
          const float nl = (l[i4] == -INFINITY ? 0.f : -l[i4] * kLog2e) + (Elem<T>::kBF16 ? 0.f : 10.f);
          nlse2[base + r + i4 * kStep] = real[i4] ? nl : -INFINITY;
          ndelta[base + r + i4 * kStep] = -acc;
        }
      }
    }
    if (!Elem<T>::kBF16) leave(top_do + base / kTile);
  }
  if (!Elem<T>::kBF16 || p.lens) {
    const int nt = (p.N + kTile - 1) / kTile, key_tiles = p.B * p.Hkv * nt;
    for (int i = blockIdx.x; i < key_tiles; i += gridDim.x) {
      const int bh = i / nt, hk = bh % p.Hkv, b = bh / p.Hkv;
      const int n = valid_rows(p.lens, b, p.N);
      if (Elem<T>::kBF16 && (i % nt + 1) * kTile <= n) continue;
#pragma unroll 4
      for (int r = r0; r < kTile; r += kStep) {
        const int key = i % nt * kTile + r;
        if (key >= n) {
          if (key < p.N) {
            reinterpret_cast<uint4*>(p.dK.at(b, hk, key))[chunk] = make_uint4(0, 0, 0, 0);
            reinterpret_cast<uint4*>(p.dV.at(b, hk, key))[chunk] = make_uint4(0, 0, 0, 0);
          }
        } else if (!Elem<T>::kBF16) {
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(V.at(b, hk, key)) + chunk);
          const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
          widest(xw);
        }
      }
      if (!Elem<T>::kBF16) leave(top_v + (static_cast<int64_t>(b) * p.Hkv + hk) * nt + i % nt);
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
// 2 x 24 heads, 4096 rows, 128 and 512 keys of 128: 66 to 70 us, 0.7 PFLOP/s,
// the tensor pipe 33 to 35 % busy; bound by a tile's chain S, P, dP, dS, product, of which
// the two tiles overlap about half.
// Both kernels: warpgroups 0 to 3 form P and dS, 4 stores the sums, 5 holds the
// TMA producer (warp 20), two MMA issuers (21, 23) and the scheduler (22). The
// dQ kernel holds 64 columns a thread and splits its registers, 4 * 128 * 96 +
// 2 * 128 * 48, the 768 * 80 of the launch; the other needs no more than 80.
// (With two warpgroups for P and dS a step took 10 % longer in both: a warp's
// own latencies were the longest part of the loop.)
constexpr int kBwdThreads = 768, kDqComputeRegs = 96, kDqOtherRegs = 48;
static_assert(4 * kDqComputeRegs + 2 * kDqOtherRegs == 6 * 80, "register split");
constexpr int kStoreWarp = 16, kLoadWarp = 20, kMmaWarp0 = 21, kUnitWarp = 22, kMmaWarp1 = 23;
constexpr int kBwdReaders = 23;  // of a unit: every warp but the scheduler

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
enum DqBar2 : int {
  kBqQFull0 = 0,    // + tile
  kBqQEmpty0 = 2,   // + tile: the unit's last S of the tile is done
  kBqKFull0 = 4,    // + slot (up to 4)
  kBqKEmpty0 = 8,
  kBqVFull0 = 12,
  kBqVEmpty0 = 16,
  kBqSFull0 = 20,   // + tile
  kBqSRead0 = 22,   // + tile: S is in registers (8 warps)
  kBqXFull0 = 24,   // + tile: dP
  kBqDSFull0 = 26,  // + tile: dS written (8 warps)
  kBqAcc0 = 28,     // + tile: the unit's dQ is complete
  kBqAccEmpty0 = 30,// + tile: and read (4 warps)
  kBqDrain0 = 32,   // + tile
  kBqUnitFull0 = 34,
  kBqUnitEmpty0 = 38,
  kBqTail0 = 42,    // + slot: a last K tile has landed, its rows behind the keys not yet cleared
  kBqOFull0 = 46,   // + tile: dO
  kBqOEmpty0 = 48,  // + tile: the unit's last dP of the tile is done
  kNumBqBars = 50,
};
static_assert(kNumBqBars * 8 + 8 <= 512, "barrier area");

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

  if (threadIdx.x < kNumBqBars) {
    const int i = threadIdx.x;
    int count = 1;
    if ((i >= kBqKEmpty0 && i < kBqVFull0) || (i >= kBqVEmpty0 && i < kBqSFull0)) count = 2;
    if ((i >= kBqSRead0 && i < kBqXFull0) || (i >= kBqDSFull0 && i < kBqAcc0)) count = 8;
    if (i >= kBqAccEmpty0 && i < kBqDrain0) count = 4;
    if (i >= kBqUnitEmpty0 && i < kBqTail0) count = kBwdReaders;
    mbar_init(&bar[i], count);
    if (i == 0) *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  WaitCtx ctx{abort_flag, p.timeout_ns};
  // nlse2, ndelta and the magnitudes come from the launch before; the launch after needs only those
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int q_tiles = p.rows.tiles;
  uint64_t *unit_full = &bar[kBqUnitFull0], *unit_empty = &bar[kBqUnitEmpty0];
  BwdUnit u{};
  int k = 0;
  bool ok = true;

  if (warp >= kLoadWarp) {
    regs_lower<kDqOtherRegs>();
    if (warp == kLoadWarp) {
      // ---- TMA producer
      if (elect_one()) {
        tma_prefetch_desc(&tm_Q);
        tma_prefetch_desc(&tm_K);
        tma_prefetch_desc(&tm_V);
        tma_prefetch_desc(&tm_dO);
        const uint64_t pol_q = l2_policy_evict_first(), pol_kv = l2_policy_evict_last();
        const uint32_t q_bytes = static_cast<uint32_t>(p.rows.Mt * p.rows.Gt) * 128u * (D / kBoxCols);
        uint32_t nq = 0;  // a byte each for Q and dO of both tiles
        int nk = 0, nv = 0, tails = 0;
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
          // Q before K, dO behind it: each as soon as its own last product of
          // the unit before is done
#pragma unroll 1
          for (int x4 = 0; x4 < 4 && ok; ++x4) {
            const int t = x4 & 1, tile = 2 * u.idx + t;
            const bool first = x4 < 2;  // Q, else dO
            if (x4 == 1) ok = load_k(u.lo);
            if (tile >= q_tiles || !ok) continue;
            const int full = first ? kBqQFull0 : kBqOFull0, empty = first ? kBqQEmpty0 : kBqOEmpty0;
            const int n = nq >> (8 * x4) & 1, any = nq >> (8 * x4 + 1) & 1;  // turns of its barrier, whether it was used
            if (any && !(ok = mbar_wait(&bar[empty + t], n ^ 1, ctx, 301))) break;
            nq ^= 1u << (8 * x4);
            nq |= 2u << (8 * x4);
            const int m0 = tile % p.rows.nm * p.rows.Mt, h0 = u.hk * p.rows.G + tile / p.rows.nm * p.rows.Gt;
            mbar_arrive_expect_tx(&bar[full + t], q_bytes);
            const CUtensorMap* tm = first ? &tm_Q : &tm_dO;
            uint8_t* dst = smem + (first ? Cfg::kOffQ : Cfg::kOffdO) + t * Cfg::kTileBytes;
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x)
              tma_load_4d(dst + x * kBoxBytes, tm, &bar[full + t], x * kBoxCols, m0, h0, u.b, pol_q);
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
          for (int x = 0; x < 4; ++x)
            if (nq >> (8 * x + 1) & 1)
              mbar_wait_drain(&bar[(x < 2 ? kBqQFull0 : kBqOFull0) + (x & 1)], (nq >> (8 * x) & 1) ^ 1, p.timeout_ns);
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
    } else if (warp == kUnitWarp) {
      feed_units<T, D, true>(p, ring, unit_full, unit_empty, ctx, 305);
      __syncwarp();
    } else {
      // ---- MMA issuer of tile t: per step dP, dQ, and S of the next step. A
      // thread for each tile keeps one tile's wait from holding up the other's
      // products.
      const int t = warp == kMmaWarp0 ? 0 : 1;
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
              if (j == u.lo && !(ok = mbar_wait(&bar[kBqOFull0 + t], nq & 1, ctx, 316 + 10 * t))) break;
              if (!(ok = mbar_wait(&bar[kBqVFull0 + g % SV], (g / SV) & 1, ctx, 312 + 10 * t))) break;
              if (!(ok = mbar_wait(&bar[kBqSRead0 + t], n & 1, ctx, 313 + 10 * t))) break;
              tc_fence_after();
              product(ddo, sV + (g % SV) * Cfg::kTileBytes);
              umma_commit(&bar[kBqXFull0 + t]);
              umma_commit(&bar[kBqVEmpty0 + g % SV]);
              if (alone) umma_commit(&bar[kBqVEmpty0 + g % SV]);
              if (j + 1 == u.hi) umma_commit(&bar[kBqOEmpty0 + t]);
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
                  umma_f16_ts(tA, tR + (x >> 2) * 64 + (x & 3) * 8, desc_advance(dk, x * 2048), id_A, x > 0 ? 1u : keep);
              } else {
                for (int x = 0; x < (left + 15) / 16; ++x)
                  umma_f16_ts(tA, tR + (x >> 2) * 64 + (x & 3) * 8, desc_advance(dk, x * 2048), id_A, x > 0 ? 1u : keep);
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
              if (j + 2 == u.hi) umma_commit(&bar[kBqQEmpty0 + t]);
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
  } else if (warp < kStoreWarp) {
    // ---- P and dS: two warpgroups a tile, thread = row (TMEM lane), columns
    // 64 c to 64 c + 63; dS lies in columns [64 c, 64 c + 32)
    regs_raise<kDqComputeRegs>();
    const int t = warp >> 3, c = warp >> 2 & 1, r = threadIdx.x & 127;
    const uint32_t tR = tmem + 128 * t + 64 * c + (static_cast<uint32_t>(r & 96) << 16);
    const float sl2 = p.scale * kLog2e;
    int ns = 0;
    while (take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 319, ok)) {
      const int tile = 2 * u.idx + t;
      if (tile >= q_tiles) continue;
      const int64_t row = ((static_cast<int64_t>(u.b) * p.Hkv + u.hk) * q_tiles + tile) * kTile + r;
      const float nl = __ldcg(p.nlse2 + row);
      const float ds_mul = pow2(u.exp - kPBias);
      const float nd = ds_mul * __ldcg(p.ndelta + row);
      for (int j = u.lo; j < u.hi; ++j, ++ns) {
        if (!mbar_wait(&bar[kBqSFull0 + t], ns & 1, ctx, 320)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        uint32_t s[64];
        tmem_load_32(tR, s);
        tmem_load_32(tR + 32, s + 32);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBqSRead0 + t]);
#pragma unroll
        for (int x = 0; x < 64; x += 2) {
          float2 a = fma_f32x2(make_float2(__uint_as_float(s[x]), __uint_as_float(s[x + 1])), make_float2(sl2, sl2),
                               make_float2(nl, nl));
          a = make_float2(ex2_approx(a.x), ex2_approx(a.y));
          s[x] = __float_as_uint(a.x);
          s[x + 1] = __float_as_uint(a.y);
        }
        if (!mbar_wait(&bar[kBqXFull0 + t], ns & 1, ctx, 321)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
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
        const int left = u.n - j * kTile - 64 * c;
        if (left > 0 && left < 64) {
          tmem_store_wait();
          clear_ds(tR, left);
        }
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBqDSFull0 + t]);
      }
    }
  } else {
    // ---- dQ: thread = row of each tile in turn; one warp also clears the
    // last K tile behind the last key, for the issuers that wait for it
    regs_lower<kDqOtherRegs>();
    const int r = threadIdx.x & 127;
    int na0 = 0, na1 = 0, g = 0;
    uint32_t tail_turns = 0;
    while (take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 329, ok)) {
      g += u.hi - u.lo;
      if (warp == kStoreWarp && has_tail(u.n, u.hi)) {
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
        float* part = p.part + ((static_cast<int64_t>(u.slot) * 2 + t) * kTile + r) * D;
        uint8_t* out = u.slot >= 0 ? reinterpret_cast<uint8_t*>(part)
                       : real      ? reinterpret_cast<uint8_t*>(p.dQ.at(u.b, u.hk * p.rows.G + g, m))
                                   : nullptr;
        store_sums<T, D, 16>(tmem + 256 + D * t + (static_cast<uint32_t>(r & 96) << 16), u.slot >= 0, out,
                         u.slot >= 0 ? 1.f : p.scale * pow2(-u.exp));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBqAccEmpty0 + t]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) publish_failure(*abort_flag, p.status);
  if (warp == kMmaWarp0) {
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
// 2 x 24 heads, 4096 rows, 128 and 512 keys of 128: 74 to 81 us, 0.80 to 0.87 PFLOP/s,
// the tensor pipe 38 to 42 % busy, bound by the same chain.
//
// Shared memory (D = 128): K, V 64 KB, Q x3, dO x2 160 KB, nlse2 and ndelta.
// (With two Q slots, S^T waited some 700 cycles a step for its Q: the slot is
// free only when dK of two steps before is done.) TMEM: S^T [0, 128), dP^T
// [128, 256), dV, dK behind.
template <int D>
struct DkvCfg2 {
  static constexpr int kTileBytes = (D / kBoxCols) * kBoxBytes;
  static constexpr int kOffK = 0, kOffV = kTileBytes;
  static constexpr int kOffQ = 2 * kTileBytes, kOffdO = 5 * kTileBytes;  // three and two slots
  static constexpr int kOffL = 7 * kTileBytes;                          // [dO slot][nlse2, ndelta][128]
  static constexpr int kOffRing = kOffL + 2 * 2 * kTile * 4;
  static constexpr int kOffBar = kOffRing + sizeof(UnitRing);
  static constexpr int kSmemBytes = kOffBar + 256;
  static constexpr uint32_t kColS = 0, kColX = 128, kColdV = 256, kColdK = 256 + D;
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

enum DkvBar2 : int {
  kBkKVFull0 = 28,  // K, V
  kBkKVEmpty0 = 0,  // the unit's last S^T, its last dP^T are done
  kBkQFull0 = 2,   // + slot (3)
  kBkQEmpty0 = 5,  // dK is done with it
  kBkOFull0 = 8,   // + slot (2): dO, nlse2, ndelta
  kBkOEmpty0 = 10, // dV is done with dO, and dK of the step (so the warps with ndelta)
  kBkSFull = 12,
  kBkPFull = 13,   // 16 warps
  kBkXFull = 14,
  kBkDSFull = 15,  // 16 warps
  kBkAcc = 16,     // both issuers
  kBkAccEmpty = 17, // 4 warps
  kBkDrain0 = 18,  // + issuer
  kBkUnitFull0 = 20,
  kBkUnitEmpty0 = 24,
  kNumBkBars = 30,
};
static_assert(kNumBkBars * 8 + 8 <= 256, "barrier area");

// 2^x of two values on the FMA pipe instead of the SFU, whose 16 results a
// clock would bound the kernel: x = n + f with n the nearest integer (taken
// from the low mantissa bits of x + 1.5 2^23) and 2^f on [-1/2, 1/2] by the
// polynomial 1 + f q(f) of degree 5 with the least largest relative error there
// (found by Remez exchange): 9.1e-8, 1.1e-7 with the coefficients in fp32 and
// 1.6e-7 as evaluated, like ex2.approx. 2^n is exact, with 0 for n = -127 and
// infinity for 128, so x is held to [-127, 128], NaN staying what it is.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;\n\tmin.NaN.f32 %0, %0, 0f43000000;" : "+f"(x.x));
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;\n\tmin.NaN.f32 %0, %0, 0f43000000;" : "+f"(x.y));
  auto both = [](float c) { return make_float2(c, c); };
  const float2 t = add_f32x2(x, both(12582912.f));
  const float2 f = fma_f32x2(add_f32x2(t, both(-12582912.f)), both(-1.f), x);
  float2 p = fma_f32x2(both(1.3264727e-3f), f, both(9.6715130e-3f));
  p = fma_f32x2(p, f, both(5.5507336e-2f));
  p = fma_f32x2(p, f, both(0.24022242f));
  p = fma_f32x2(p, f, both(0.69314700f));
  p = fma_f32x2(p, f, both(1.f));
  return mul_f32x2(p, make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                                  __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)));
}

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

  if (threadIdx.x < kNumBkBars) {
    const int i = threadIdx.x;
    int count = 1;
    if (i == kBkOEmpty0 || i == kBkOEmpty0 + 1 || i == kBkAcc) count = 2;
    if (i == kBkPFull || i == kBkDSFull) count = 16;
    if (i == kBkAccEmpty) count = 4;
    if (i >= kBkUnitEmpty0 && i < kBkKVFull0) count = kBwdReaders;
    mbar_init(&bar[i], count);
    if (i == 0) *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // rows of the Q and dO slots that no box fills are summed over with P = dS = 0
  const int box_rows = p.rows.Mt * p.rows.Gt;
  if (box_rows < kTile) {
    for (int i = threadIdx.x; i < 5 * Cfg::kTileBytes / 16; i += kBwdThreads)
      *reinterpret_cast<uint4*>(smem + Cfg::kOffQ + 16 * i) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  WaitCtx ctx{abort_flag, p.timeout_ns};
  uint64_t *unit_full = &bar[kBkUnitFull0], *unit_empty = &bar[kBkUnitEmpty0];
  BwdUnit u{};
  int k = 0;
  bool ok = true;
  // The launch before (attn_dq_kernel) let this one start after its own wait
  // for attn_delta_kernel, whose rows are thus there; attn_dq_kernel itself is
  // waited for at the end, for the launches after.

  if (warp >= kLoadWarp) {
    if (warp == kLoadWarp) {
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
#pragma unroll 1
          for (int y = 0; y < 2; ++y) {  // K, V
            if (nu > 0 && !(ok = mbar_wait(&bar[kBkKVEmpty0 + y], (nu - 1) & 1, ctx, 401))) break;
            mbar_arrive_expect_tx(&bar[kBkKVFull0 + y], Cfg::kTileBytes);
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x)
              tma_load_4d(smem + y * Cfg::kTileBytes + x * kBoxBytes, y == 0 ? &tm_K : &tm_V, &bar[kBkKVFull0 + y],
                          x * kBoxCols, u.idx * kTile, u.hk, u.b, pol_kv);
          }
          if (!ok) break;
          ++nu;
          for (int i = u.lo; i < u.hi; ++i) {
            const int s = n % 3, so = n & 1;
            const int m0 = i % p.rows.nm * p.rows.Mt, h0 = u.hk * p.rows.G + i / p.rows.nm * p.rows.Gt;
            const int64_t row = ((static_cast<int64_t>(u.b) * p.Hkv + u.hk) * q_tiles + i) * kTile;
            if (n >= 3 && !(ok = mbar_wait(&bar[kBkQEmpty0 + s], (n / 3 - 1) & 1, ctx, 402))) break;
            mbar_arrive_expect_tx(&bar[kBkQFull0 + s], q_bytes);
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x)
              tma_load_4d(smem + Cfg::kOffQ + s * Cfg::kTileBytes + x * kBoxBytes, &tm_Q, &bar[kBkQFull0 + s],
                          x * kBoxCols, m0, h0, u.b, pol_q);
            ++n;
            if (no >= 2 && !(ok = mbar_wait(&bar[kBkOEmpty0 + so], ((no >> 1) - 1) & 1, ctx, 403))) break;
            mbar_arrive_expect_tx(&bar[kBkOFull0 + so], q_bytes + 2 * kTile * 4);
#pragma unroll
            for (int x = 0; x < D / kBoxCols; ++x)
              tma_load_4d(smem + Cfg::kOffdO + so * Cfg::kTileBytes + x * kBoxBytes, &tm_dO, &bar[kBkOFull0 + so],
                          x * kBoxCols, m0, h0, u.b, pol_q);
            bulk_load(smem + Cfg::kOffL + so * 2 * kTile * 4, p.nlse2 + row, kTile * 4, &bar[kBkOFull0 + so]);
            bulk_load(smem + Cfg::kOffL + (so * 2 + 1) * kTile * 4, p.ndelta + row, kTile * 4, &bar[kBkOFull0 + so]);
            ++no;
          }
          if (!ok) break;
        }
        if (*abort_flag) {  // every copy in flight ends before the block does
          for (int y = 0; y < 2; ++y)
            if (nu > 0) mbar_wait_drain(&bar[kBkKVFull0 + y], (nu - 1) & 1, p.timeout_ns);
          for (int i = (n > 3 ? n - 3 : 0); i < n; ++i)
            mbar_wait_drain(&bar[kBkQFull0 + i % 3], (i / 3) & 1, p.timeout_ns);
          for (int i = (no > 2 ? no - 2 : 0); i < no; ++i)
            mbar_wait_drain(&bar[kBkOFull0 + (i & 1)], (i >> 1) & 1, p.timeout_ns);
        }
      }
      __syncwarp();
    } else if (warp == kUnitWarp) {
      feed_units<T, D, false>(p, ring, unit_full, unit_empty, ctx, 405);
      __syncwarp();
    } else {
      // ---- MMA issuers: the first dV and S^T of the next row tile (TMEM S, P),
      // the second dK and dP^T of the next (TMEM X), so that neither chain's
      // waits hold up the other's products.
      const int w = warp == kMmaWarp0 ? 0 : 1;
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
        const int slots1 = w == 0 ? 3 : 2, slots2 = w == 0 ? 2 : 3;
        int n = 0, nu = 0, s1 = 0, turn1 = 0, s2 = 0;  // steps and units; slots of `first` and `second`
        while (take_unit<false>(ring, unit_full, unit_empty, k, u, ctx, 409 + 10 * w, ok)) {
          if (!(ok = mbar_wait(&bar[kBkKVFull0 + w], nu & 1, ctx, 410 + 10 * w))) break;
          for (int i = u.lo - 1; i < u.hi; ++i) {
            if (i >= u.lo) {
              if (i == u.lo && nu > 0 && !(ok = mbar_wait(&bar[kBkAccEmpty], (nu - 1) & 1, ctx, 413 + 10 * w))) break;
              if (!(ok = mbar_wait(formed, n & 1, ctx, 414 + 10 * w))) break;
              tc_fence_after();
              const uint64_t db = make_sw128_desc(second + s2 * Cfg::kTileBytes, kBoxBytes, 1024);
#pragma unroll
              for (int x = 0; x < kTile / 16; ++x)
                umma_f16_ts(tA, tR + (x >> 1) * 32 + (x & 1) * 8, desc_advance(db, x * 2048), id_A,
                            x > 0 || i > u.lo ? 1u : 0u);
              umma_commit(&bar[kBkOEmpty0 + (n & 1)]);
              if (w == 1) umma_commit(&bar[kBkQEmpty0 + s2]);
              if (i + 1 == u.hi) umma_commit(&bar[kBkAcc]);
              if (++s2 == slots2) s2 = 0;
              ++n;
            }
            if (i + 1 < u.hi) {
              if (!(ok = mbar_wait(landed + s1, turn1, ctx, 411 + 10 * w))) break;
              tc_fence_after();
              const uint64_t db = make_sw128_desc(first + s1 * Cfg::kTileBytes, 16, 1024);
#pragma unroll
              for (int x = 0; x < D / 16; ++x) {
                const uint32_t off = (x >> 2) * kBoxBytes + (x & 3) * 32;
                umma_f16_ss(tR, desc_advance(da, off), desc_advance(db, off), id_S, x > 0 ? 1u : 0u);
              }
              umma_commit(&bar[w == 0 ? kBkSFull : kBkXFull]);
              if (i + 2 == u.hi) umma_commit(&bar[kBkKVEmpty0 + w]);
              if (++s1 == slots1) {
                s1 = 0;
                turn1 ^= 1;
              }
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
  } else if (warp < kStoreWarp) {
    // ---- P^T and dS^T: thread = key (TMEM lane), rows 32 c to 32 c + 31 of the
    // row tile; the 16-bit values lie in columns [32 c, 32 c + 16)
    const int c = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(r & 96) << 16;
    const uint32_t tS = tmem + Cfg::kColS + 32 * c + lanes, tX = tmem + Cfg::kColX + 32 * c + lanes;
    const float2 sl2 = make_float2(p.scale * kLog2e, p.scale * kLog2e);
    int n = 0;
    while (take_unit<true>(ring, unit_full, unit_empty, k, u, ctx, 419, ok)) {
      // a key that does not count gets P = dS = 0, whatever K and V hold
      const bool valid = u.idx * kTile + r < u.n;
      const float ds_mul = pow2(u.exp - kPBias);
      for (int i = u.lo; i < u.hi; ++i, ++n) {
        const float4* nl = reinterpret_cast<const float4*>(smem + Cfg::kOffL + (n & 1) * 2 * kTile * 4) + 8 * c;
        const float4* nd = nl + kTile / 4;
        if (!mbar_wait(&bar[kBkOFull0 + (n & 1)], (n >> 1) & 1, ctx, 420)) { ok = false; break; }
        if (!mbar_wait(&bar[kBkSFull], n & 1, ctx, 421)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        uint32_t s[32], e[16];
        tmem_load_32(tS, s);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float4 l = nl[x];
          float2 a = fma_f32x2(make_float2(__uint_as_float(s[4 * x]), __uint_as_float(s[4 * x + 1])), sl2,
                               make_float2(l.x, l.y));
          float2 b = fma_f32x2(make_float2(__uint_as_float(s[4 * x + 2]), __uint_as_float(s[4 * x + 3])), sl2,
                               make_float2(l.z, l.w));
          if (x % 4 < 1) a = ex2_poly(a);
          else a = make_float2(ex2_approx(a.x), ex2_approx(a.y));
          if (x % 4 < 1) b = ex2_poly(b);
          else b = make_float2(ex2_approx(b.x), ex2_approx(b.y));
          s[4 * x] = __float_as_uint(a.x);
          s[4 * x + 1] = __float_as_uint(a.y);
          s[4 * x + 2] = __float_as_uint(b.x);
          s[4 * x + 3] = __float_as_uint(b.y);
          e[2 * x] = Elem<T>::pack(a.x, a.y);
          e[2 * x + 1] = Elem<T>::pack(b.x, b.y);
        }
        if (!valid) {
#pragma unroll
          for (int x = 0; x < 16; ++x) e[x] = 0u;
        }
        __syncwarp();
        tmem_store_16(tS, e);
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBkPFull]);
        if (!mbar_wait(&bar[kBkXFull], n & 1, ctx, 422)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        uint32_t dp[32];
        tmem_load_32(tX, dp);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float4 d = nd[x];
          float2 a = add_f32x2(make_float2(__uint_as_float(dp[4 * x]), __uint_as_float(dp[4 * x + 1])), make_float2(d.x, d.y));
          float2 b =
              add_f32x2(make_float2(__uint_as_float(dp[4 * x + 2]), __uint_as_float(dp[4 * x + 3])), make_float2(d.z, d.w));
          if (!kB) {
            a = mul_f32x2(a, make_float2(ds_mul, ds_mul));
            b = mul_f32x2(b, make_float2(ds_mul, ds_mul));
          }
          a = mul_f32x2(a, make_float2(__uint_as_float(s[4 * x]), __uint_as_float(s[4 * x + 1])));
          b = mul_f32x2(b, make_float2(__uint_as_float(s[4 * x + 2]), __uint_as_float(s[4 * x + 3])));
          e[2 * x] = Elem<T>::pack(a.x, a.y);
          e[2 * x + 1] = Elem<T>::pack(b.x, b.y);
        }
        if (!valid) {
#pragma unroll
          for (int x = 0; x < 16; ++x) e[x] = 0u;
        }
        __syncwarp();
        tmem_store_16(tX, e);
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kBkDSFull]);
      }
    }
  } else {
    // ---- dV and dK: thread = key
    const int r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(r & 96) << 16;
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
        float* part = p.part + ((static_cast<int64_t>(u.slot) * 2 + which) * kTile + r) * D;
        uint8_t* out = u.slot >= 0 ? reinterpret_cast<uint8_t*>(part)
                       : key < u.n ? reinterpret_cast<uint8_t*>(v.at(u.b, u.hk, key))
                                   : nullptr;
        store_sums<T, D, 32>(tmem + (which == 0 ? Cfg::kColdV : Cfg::kColdK) + lanes, u.slot >= 0, out,
                         u.slot >= 0 ? 1.f : (which == 0 ? pow2(-kPBias) : p.scale * pow2(-u.exp)));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[kBkAccEmpty]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) publish_failure(*abort_flag, p.status);
  if (warp == kMmaWarp0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ===================================================================== join
// Items that fell to several CTAs: adds their partial sums in CTA order. Block
// (x, c - 1, z) looks at the boundary before CTA c of the dQ (z = 0) or the
// dK/dV kernel; the first boundary inside an item owns it. kJoinBlocks blocks
// share the item's two [128][D] sums, one thread per 4 columns. With nothing to
// join 5 us, so it is left out where no lengths can ask for it.
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
  const int ds_exp = ds_exponent<T, D>(p, it.u, threadIdx.x & 31);
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
      if (key < it.u.n) out = (which == 0 ? p.dV : p.dK).at(it.u.b, it.u.hk, key);
    }
    if (out)
      *reinterpret_cast<uint2*>(out + 4 * col) =
          make_uint2(Elem<T>::pack(mul * a.x, mul * a.y), Elem<T>::pack(mul * a.z, mul * a.w));
  }
}

}  // namespace fmha_sm100
