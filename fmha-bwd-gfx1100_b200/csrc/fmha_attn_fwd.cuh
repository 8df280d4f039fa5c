// Forward of attention on the tensor cores: O and LSE of packed query rows
// against the keys of one kv head, whole or split along the keys.
//
//   S = Q K^T,  p = 2^(S scale log2e - m),  O = sum p V / sum p,
//   LSE = (m + log2 sum p) ln 2
//
// with a running m for each row, in one pass over the keys.
//
// Rows. A tile is up to 128 query rows that read the same keys: Mt
// consecutive tokens of Gt query heads of the kv head's group of St batch
// entries that share the keys (St > 1 for a shared prefix only), tokens
// fastest. One tensor-map box of Q brings such a tile in, so a single token
// of many heads or samples fills a tile just as 128 tokens of one head do.
//
// Two tiles per CTA. Each tile has its own softmax warpgroup (thread = row),
// its own S (128 TMEM columns) and O accumulator (D columns); while one
// warpgroup computes p of its tile, the tensor core works for the other. p is
// written as 16-bit over the first 64 columns of S and read from there as the
// A operand of O += p V. The tensor core runs PV_t(j) and the next S_t(j+1) in
// the order of issue, so the completion of S_t(j+1) says that PV_t(j) has
// completed as well: between that and its own signal the warpgroup owns O_t.
//
// m moves only when a row's maximum exceeds it by more than 2^8 (its O is then
// scaled in TMEM by the softmax warpgroup, which owns it): p stays below 2^8
// (2^14 with fp16's bias below), and most steps rescale nothing.
//
// p is rounded to 16 bits (the tensor core's input type) after it went into
// the fp32 row sum. In fp16 m is lowered by kBias = 6, so that p down to 2^-20
// of the row's maximum keeps full precision (bf16 has fp32's range).
#pragma once

#include "fmha_attn.cuh"
#include "fmha_bwd_lse.cuh"  // ex2_approx, kLog2e

namespace fmha_sm100 {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoMax = -3.0e38f;  // the reference of a row before its first weight

// Units of work that one warp of a CTA works out and the others take from a
// ring in shared memory: the divisions are done once, and the other roles hold
// a unit's few numbers only. A unit is two int4; its last number is 0 behind
// the last unit.
constexpr int kUnitRing = 4;
struct UnitRing {
  int4 a[kUnitRing];
  int4 b[kUnitRing];
};
__device__ __forceinline__ bool put_unit(UnitRing* ring, uint64_t* full, uint64_t* empty, int k, int4 a, int4 b,
                                         const WaitCtx& ctx, int where) {
  const int i = k % kUnitRing;
  if (k >= kUnitRing && !mbar_wait(&empty[i], ((k / kUnitRing) - 1) & 1, ctx, where)) return false;
  ring->a[i] = a;
  ring->b[i] = b;
  mbar_arrive(&full[i]);
  return true;
}
// For a whole warp (kWarp) or one thread; false at the end, or with `ok`
// cleared (before or by the wait here).
template <bool kWarp>
__device__ __forceinline__ bool get_unit(const UnitRing* ring, uint64_t* full, uint64_t* empty, int& k, int4& a, int4& b,
                                         const WaitCtx& ctx, int where, bool& ok) {
  const int i = k % kUnitRing;
  if (ok && !mbar_wait(&full[i], (k / kUnitRing) & 1, ctx, where)) ok = false;
  if (kWarp) ok = __all_sync(0xffffffffu, ok);
  if (!ok) return false;
  a = ring->a[i];
  b = ring->b[i];
  if (kWarp) __syncwarp();
  if (!kWarp || (threadIdx.x & 31) == 0) mbar_arrive(&empty[i]);
  ++k;
  return b.w != 0;
}

// Quotient and remainder; most divisors here are 1 in most calls.
__device__ __forceinline__ void div_mod(int x, int d, int& q, int& r) {
  q = x;
  r = 0;
  if (d != 1) {
    q = static_cast<int>(static_cast<uint32_t>(x) / static_cast<uint32_t>(d));
    r = x - q * d;
  }
}

// How query rows fall into tiles (see above).
struct RowPack {
  int M, G, S;     // tokens, query heads of a kv head, batch entries that share keys
  int Mt, Gt, St;  // the box
  int nm, ng, ns;  // boxes along each
  int tiles;       // nm * ng * ns
  // tile t's box along each
  __device__ __forceinline__ void box(int t, int& im, int& ig, int& is) const {
    int u;
    div_mod(t, nm, u, im);
    div_mod(u, ng, is, ig);
  }
  // the oldest token of tile t
  __device__ __forceinline__ int oldest(int t) const {
    int im, ig, is;
    box(t, im, ig, is);
    return im * Mt;
  }
  // token, head within the group and entry of row r of tile t; false if there is no such row
  __device__ __forceinline__ bool row(int t, int r, int& m, int& g, int& s) const {
    int im, ig, is, rm = r, rg = 0, rs = 0;
    box(t, im, ig, is);
    if (Mt < 128) {
      int v;
      div_mod(r, Mt, v, rm);
      div_mod(v, Gt, rs, rg);
    }
    m = im * Mt + rm;
    g = ig * Gt + rg;
    s = is * St + rs;
    return m < M && rg < Gt && g < G && rs < St && s < S;
  }
};

// `divides`: boxes of whole groups, none of them reaching into the next kv head.
inline RowPack pack_rows(int M, int G, int S, bool divides = false) {
  RowPack p;
  p.M = M;
  p.G = G;
  p.S = S;
  p.Mt = M < 128 ? M : 128;
  p.Gt = std::min(G, 128 / p.Mt);
  while (divides && G % p.Gt != 0) --p.Gt;
  p.St = std::min(S, 128 / (p.Mt * p.Gt));
  p.nm = (M + p.Mt - 1) / p.Mt;
  p.ng = (G + p.Gt - 1) / p.Gt;
  p.ns = (S + p.St - 1) / p.St;
  p.tiles = p.nm * p.ng * p.ns;
  return p;
}

template <typename T>
struct FwdParams {
  RowPack rows;
  int B, Hkv, N;      // key batches, kv heads, key rows
  const int* lens;    // [B] or null
  int splits;         // parts of the keys (1: O and LSE are final)
  int pairs;          // tile pairs of one (batch, kv head)
  int items;          // B * Hkv * splits * pairs
  View<T> V;          // kOwn: the tensor of tm_V
  View<T> O;
  float* LSE;         // [batch][q head][token]
  float* part_o;      // splits > 1 or partial: [split][row][D], normalised
  float* part_lse;    // [split][row]
  bool partial;
  bool in_turn;       // partial, an item to a CTA: the softmax warps store it, a tile each warpgroup
  float scale;
  KernelStatus* status;
  uint64_t timeout_ns;
};

template <int D>
struct FwdCfg {
  static constexpr int kTileBytes = (D / kBoxCols) * kBoxBytes;  // 128 rows
  static constexpr int kSlots = D == 128 ? 5 : 8;                // K and V tiles, in the order of their use
  static constexpr int kOffQ = 0;                                // two tiles
  static constexpr int kOffKV = 2 * kTileBytes;
  static constexpr int kOffStat = kOffKV + kSlots * kTileBytes;  // float2 [2][128]
  static constexpr int kOffRing = kOffStat + 2 * 128 * 8;
  static constexpr int kOffBar = kOffRing + sizeof(UnitRing);
  static constexpr int kSmemBytes = kOffBar + 512;
  static constexpr int kThreads = 512;
  static constexpr uint32_t kColS = 0;    // + 128 * tile
  static constexpr uint32_t kColO = 256;  // + D * tile
  static_assert(kSmemBytes <= 232448, "shared memory budget");
  // warpgroups 0 and 1 softmax, 2 epilogue, 3 loads, MMA and schedule: 2 * 128
  // * 184 + 2 * 128 * 72 registers, the 512 * 128 of the launch
  static constexpr int kSoftmaxRegs = 184, kOtherRegs = 72;
  static_assert(2 * kSoftmaxRegs + 2 * kOtherRegs == 4 * 128, "register split");
  static constexpr int kReaders = 14;  // of a unit: warps 0-13
};

enum FwdBar : int {
  kFwQFull0 = 0,    // + tile
  kFwQEmpty0 = 2,   // + tile: the item's last S of the tile is done
  kFwKVFull0 = 4,   // + slot (up to 8)
  kFwKVEmpty0 = 12, // + slot
  kFwTail0 = 20,    // + slot: a V tile has landed that is_checked, and not yet cleared
  kFwSFull0 = 28,   // + tile
  kFwPFull0 = 30,   // + tile: the first 96 columns of p written (4 warps)
  kFwPRest0 = 32,   // + tile: and the others
  kFwOFull0 = 34,   // + tile: the item's last PV of the tile is done
  kFwOEmpty0 = 36,  // + tile: the epilogue has read O (4 warps)
  kFwStFull0 = 38,  // + tile: row maxima and sums written (4 warps)
  kFwStEmpty0 = 40, // + tile: and read (4 warps)
  kFwUnitFull0 = 42,
  kFwUnitEmpty0 = 46,
  kFwDrain = 50,
  kFwChecked = 51,  // kOwn: an item's V tiles have gone through hide_odd
  kFwSeen = 52,     // and the other epilogue warps know what it found (3 warps)
  kNumFwdBars = 53,
};
static_assert(kNumFwdBars * 8 + 12 <= 512, "barrier area");

// One item: a pair of row tiles of a (batch, kv head), a range of key tiles.
struct FwdItem {
  int b, hk, split, tile0, n;  // n: valid keys of the batch entry
  int lo, hi;                  // key tiles
  bool two;                    // the second tile exists
  int first;                   // kOwn: the first key tile that not all rows see whole
};

__device__ __forceinline__ FwdItem fwd_item(const int4& a, const int4& b) {
  return FwdItem{a.x, a.y, a.z, a.w, b.z, b.x, b.y, (b.w & 3) == 2, b.w >> 2};
}

// The items of this CTA. kv heads lie innermost: with the usual [token][head]
// layouts of Q and O, the CTAs then read and write neighbouring memory. kOwn: key
// tiles behind an item's newest token are left out, whatever they hold.
template <typename T, bool kOwn>
__device__ __forceinline__ void fwd_unit(const FwdParams<T>& p, int t, int4& a, int4& b) {
  int hk, pair, split, e;
  div_mod(t, p.Hkv, t, hk);
  div_mod(t, p.pairs, t, pair);
  div_mod(t, p.splits, e, split);
  const bool two = 2 * pair + 1 < p.rows.tiles;
  const int n = valid_rows(p.lens, e, p.N);
  int nt = (n + kTile - 1) / kTile, first = 0;
  if constexpr (kOwn) {
    int oldest = p.rows.oldest(2 * pair), newest = oldest;  // of both tiles, by their first rows
    if (two) {
      const int t = p.rows.oldest(2 * pair + 1);
      oldest = min(oldest, t);
      newest = max(newest, t);
    }
    newest = min(newest + p.rows.Mt, p.rows.M) - 1;
    const int all = n - (p.rows.M - 1);  // token m sees m more
    first = p.rows.M > 1 ? max(0, all + oldest) / kTile : nt;
    nt = (max(0, all + newest) + kTile - 1) / kTile;
  }
  int lo, hi, rest;
  // up to 2^23 tiles times 2 * 148 parts: 32 bits without a sign
  div_mod(static_cast<int>(static_cast<uint32_t>(nt) * split), p.splits, lo, rest);
  div_mod(static_cast<int>(static_cast<uint32_t>(nt) * (split + 1)), p.splits, hi, rest);
  a = make_int4(e, hk, split, 2 * pair);
  b = make_int4(lo, hi, n, first << 2 | (two ? 2 : 1));
}
// a, b: the first of them.
template <typename T, bool kOwn>
__device__ void feed_fwd(const FwdParams<T>& p, int4 a, int4 b, UnitRing* ring, uint64_t* full, uint64_t* empty,
                         const WaitCtx& ctx) {
  int k = 0;
  for (int t = blockIdx.x; t < p.items; ++k) {
    if (!put_unit(ring, full, empty, k, a, b, ctx, 205)) return;
    t += gridDim.x;
    if (t < p.items) fwd_unit<T, kOwn>(p, t, a, b);
  }
  put_unit(ring, full, empty, k, make_int4(0, 0, 0, 0), make_int4(0, 0, 0, 0), ctx, 205);
}

// Clears rows [left, left rounded up to 16) of a landed 128-row tile, by a
// warp: the products go over keys by 16, and would multiply what lies behind
// the last key by 0, whatever that is.
template <int D>
__device__ __forceinline__ void clear_tail(uint8_t* tile, int left, int lane) {
  const int rows = 16 - (left & 15);
  for (int i = lane; i < rows * (D / 8); i += 32) {
    const int row = left + i / (D / 8), c = i % (D / 8);
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kBoxBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
        make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
}
__device__ __forceinline__ bool has_tail(int n, int hi) { return hi * kTile > n && (n & 15) != 0; }

// kOwn: of the keys that some rows of an item see and others do not, an infinity
// or NaN in V would reach the latter as 0 times it. The landed V tiles that hold
// such keys are cleared of them (hide_odd) before their products, and the rows
// that do see them get them where they are stored (add_odd).
//
// Whether the epilogue looks at V tile j of an item before its products.
template <bool kOwn>
__device__ __forceinline__ bool is_checked(const FwdItem& it, int j) {
  return (j + 1 == it.hi && has_tail(it.n, it.hi)) || (kOwn && j >= it.first);
}
// Zeroes the elements of a word or four whose exponent is all ones.
template <typename T>
__device__ __forceinline__ bool drop_odd(uint32_t& w) {
  constexpr uint32_t kOnes = Elem<T>::kBF16 ? 0x7f807f80u : 0x7c007c00u;
  const uint32_t odd = __vcmpeq2(w & kOnes, kOnes);
  w &= ~odd;
  return odd != 0;
}
template <typename T>
__device__ __forceinline__ bool drop_odd(uint4& v) {
  bool odd = drop_odd<T>(v.x);
  odd |= drop_odd<T>(v.y);
  odd |= drop_odd<T>(v.z);
  odd |= drop_odd<T>(v.w);
  return odd;
}
// Rows [from, to) of a landed 128-row tile, by a warp; whether this lane found any.
template <typename T, int D>
__device__ __forceinline__ bool hide_odd(uint8_t* tile, int from, int to, int lane) {
  bool found = false;
#pragma unroll 1
  for (int i = lane; i < (to - from) * (D / 8); i += 32) {
    const int row = from + i / (D / 8), c = i % (D / 8);
    uint4* at = reinterpret_cast<uint4*>(tile + (c >> 3) * kBoxBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4));
    uint4 v = *at;
    if (!drop_odd<T>(v)) continue;
    *at = v;
    found = true;
  }
  if (found) fence_proxy_async_smem();
  return found;
}
// Adds the infinities and NaN of `count` rows of V (every weight is above 0) to a
// row of D finished sums; those that hide_odd left in place add nothing new.
template <typename T, int D>
__device__ __forceinline__ void add_odd(const T* v, int64_t stride, int count, float* out) {
  constexpr uint32_t kOnes = Elem<T>::kBF16 ? 0x7f80u : 0x7c00u;
#pragma unroll 1
  for (int c = 0; c < D; ++c) {
    float sum = 0.f;
#pragma unroll 1
    for (int k = 0; k < count; ++k) {
      const uint32_t x = reinterpret_cast<const uint16_t*>(v + k * stride)[c];
      if ((x & kOnes) == kOnes) sum += Elem<T>::unpack(x).x;
    }
    if (sum != 0.f) out[c] += sum;
  }
}

// 8 fp32 accumulators times `mul` as eight 16-bit values.
template <typename T>
__device__ __forceinline__ uint4 pack8(const uint32_t* a, float mul) {
  return make_uint4(Elem<T>::pack(mul * __uint_as_float(a[0]), mul * __uint_as_float(a[1])),
                    Elem<T>::pack(mul * __uint_as_float(a[2]), mul * __uint_as_float(a[3])),
                    Elem<T>::pack(mul * __uint_as_float(a[4]), mul * __uint_as_float(a[5])),
                    Elem<T>::pack(mul * __uint_as_float(a[6]), mul * __uint_as_float(a[7])));
}

// 32 bytes of one thread's row: one store where the row allows it.
__device__ __forceinline__ void store_32_bytes(uint8_t* at, const uint4& a, const uint4& b) {
  if ((reinterpret_cast<uintptr_t>(at) & 31u) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(a.x), "r"(a.y), "r"(a.z),
                 "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(at)[0] = a;
    reinterpret_cast<uint4*>(at)[1] = b;
  }
}

// This thread's row of D sums in TMEM, times `mul`, to its output row, fp32 or
// 16-bit (null: no row), C columns at a time.
template <typename T, int D, int C>
__device__ __forceinline__ void store_sums(uint32_t taddr, bool fp32, uint8_t* row, float mul) {
#pragma unroll 1
  for (int x = 0; x < D; x += C) {
    uint32_t v[C];
    __syncwarp();
    if constexpr (C == 32) tmem_load_32(taddr + x, v);
    else tmem_load_16(taddr + x, v);
    if (row == nullptr) continue;
    if (fp32) {
#pragma unroll
      for (int y = 0; y < C; ++y) v[y] = __float_as_uint(mul * __uint_as_float(v[y]));
#pragma unroll
      for (int y = 0; y < C; y += 8)
        store_32_bytes(row + 4 * (x + y), make_uint4(v[y], v[y + 1], v[y + 2], v[y + 3]),
                       make_uint4(v[y + 4], v[y + 5], v[y + 6], v[y + 7]));
    } else {
#pragma unroll
      for (int y = 0; y < C; y += 16)
        store_32_bytes(row + 2 * (x + y), pack8<T>(v + y, mul), pack8<T>(v + y + 8, mul));
    }
  }
}

// O and LSE of row `tok` of head g and entry s of an item's tile, from the
// sums in TMEM at taddr, their total l and its reference m; or a part of them.
// `odd`: hide_odd has found something, in this item or another.
template <typename T, int D, bool kOwn>
__device__ __forceinline__ void store_tile(const FwdParams<T>& p, const FwdItem& it, uint32_t taddr, int tok, int g, int s,
                                           bool real, float m, float l, int odd) {
  const bool keys = it.lo < it.hi;
  const int64_t all_rows = static_cast<int64_t>(p.B) * p.rows.S * p.Hkv * p.rows.G * p.rows.M;
  const int b = it.b * p.rows.S + s, h = it.hk * p.rows.G + g;
  // a sum of 0 has no keys behind it, or scores of -inf alone
  const float inv = keys && l != 0.f ? 1.f / l : 0.f;
  const float lse = keys ? (m + log2f(l)) * kLn2 : -INFINITY;
  const int64_t row = (static_cast<int64_t>(b) * p.Hkv * p.rows.G + h) * p.rows.M + tok;
  if (real) *(p.partial ? p.part_lse + it.split * all_rows + row : p.LSE + row) = lse;
  // bytes of this row's output, fp32 or 16-bit; null where there is no row
  uint8_t* out = reinterpret_cast<uint8_t*>(p.partial ? reinterpret_cast<void*>(p.part_o + (it.split * all_rows + row) * D)
                                                      : reinterpret_cast<void*>(p.O.at(b, h, tok)));
  if (!real) out = nullptr;
  if (keys) {
    store_sums<T, D, 32>(taddr, p.partial, out, inv);
    if (kOwn && odd && out) {  // behind a prefix sums are always parts
      const int all = it.n - (p.rows.M - 1), from = max(max(0, all), it.lo * kTile), to = min(all + tok, it.hi * kTile);
      add_odd<T, D>(p.V.at(it.b, it.hk, from), p.V.sr, to - from, reinterpret_cast<float*>(out));
    }
  } else if (out) {  // zeros
    const int chunks = D / (p.partial ? 4 : 8);
    for (int x = 0; x < chunks; ++x) reinterpret_cast<uint4*>(out)[x] = make_uint4(0, 0, 0, 0);
  }
}

// The instruction caches hold little next to these kernels' unrolled loops, and
// straight-line code that runs once an item is fetched at some 50 cycles a
// line: what is not the inner loop is kept short and rolled.

// Overwrites columns [left, 128) of this thread's row of S with -inf; none of
// the warp's rows has a left below `least`.
__device__ __forceinline__ void mask_columns(uint32_t taddr, int left, int least) {
#pragma unroll 1
  for (int c = max(least, 0) & ~15; c < 128; c += 16) {
    uint32_t v[16];
    tmem_load_16(taddr + c, v);
#pragma unroll
    for (int x = 0; x < 16; ++x)
      if (c + x >= left) v[x] = 0xff800000u;
    tmem_store_16(taddr + c, v);
  }
  tmem_store_wait();
}

// 32 weights of a row: p = 2^(s sl2 - m), summed into l and packed.
template <typename T>
__device__ __forceinline__ void weights_32(const uint32_t* s, float2 sc, float2 nm, float2& l0, float2& l1,
                                           uint32_t (&e)[16]) {
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    float2 a = fma_f32x2(make_float2(__uint_as_float(s[2 * x]), __uint_as_float(s[2 * x + 1])), sc, nm);
    a.x = ex2_approx(a.x);
    a.y = ex2_approx(a.y);
    if (x & 1) l1 = add_f32x2(l1, a);
    else l0 = add_f32x2(l0, a);
    e[x] = Elem<T>::pack(a.x, a.y);
  }
}

// 16384 rows, 1024 keys, 40 heads of 128, bf16: 343 to 366 us by the GPU's clock
// (0.94 to 1.0 PFLOP/s). A step of both tiles takes 3.7 K clocks, of which the
// exponentials take the SFU 2.0 K and the products the tensor core 2.0 K: each
// tile's softmax waits for the products between its p and its next S. Few steps
// are bound by latency: 3 to 4 us pass before the first S.
//
// kOwn: the keys of an entry's own tokens, behind a prefix: token m reads all but
// the M - 1 - m newest of them. It starts before the launch before it has ended,
// and waits for that at its end.
template <typename T, int D, bool kOwn>
__global__ void __launch_bounds__(FwdCfg<D>::kThreads, 1)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_Q, const __grid_constant__ CUtensorMap tm_K,
                    const __grid_constant__ CUtensorMap tm_V, const __grid_constant__ FwdParams<T> p) {
  using Cfg = FwdCfg<D>;
  constexpr int kSlots = Cfg::kSlots;
  constexpr bool kB = Elem<T>::kBF16;
  constexpr float kBias = kB ? 0.f : 6.f;
  // aligned by declaration: the tiles leave no room to align by hand
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // never, short of a toolchain that drops the alignment
    if (threadIdx.x == 0) publish_failure(1 + 200, p.status);
    return;
  }
  float2* stat = reinterpret_cast<float2*>(smem + Cfg::kOffStat);
  UnitRing* ring = reinterpret_cast<UnitRing*>(smem + Cfg::kOffRing);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + kNumFwdBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* odd_flag = abort_flag + 1;  // kOwn: hide_odd has found something in some item
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  int4 ua, ub;
  if (threadIdx.x < kNumFwdBars) {
    const int i = threadIdx.x;
    int count = 1;
    if ((i >= kFwPFull0 && i < kFwOFull0) || (i >= kFwOEmpty0 && i < kFwUnitFull0)) count = 4;
    if (i >= kFwUnitEmpty0 && i < kFwDrain) count = Cfg::kReaders;
    if (i == kFwSeen) count = 3;
    mbar_init(&bar[i], count);
    if (i == 0) {
      *abort_flag = 0;
      *odd_flag = 0;
    }
    fence_mbar_init();
  }
  if (warp == 12 && elect_one()) {
    tma_prefetch_desc(&tm_Q);
    tma_prefetch_desc(&tm_K);
    tma_prefetch_desc(&tm_V);
  }
  __syncwarp();
  if (warp == 13) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 14) fwd_unit<T, kOwn>(p, blockIdx.x, ua, ub);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  WaitCtx ctx{abort_flag, p.timeout_ns};
  uint64_t *unit_full = &bar[kFwUnitFull0], *unit_empty = &bar[kFwUnitEmpty0];
  int k = 0;
  bool ok = true;
  // a launch that joins the parts may start, and waits for them itself
  if (p.partial) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp >= 12) {
    regs_lower<Cfg::kOtherRegs>();
    if (warp == 12) {
      if (elect_one()) {
        // ---- TMA producer. Ring order: K_lo, then V_j, K_(j+1) in turn, the
        // order in which the MMA issuers use them.
        const uint64_t pol_q = l2_policy_evict_first(), pol_kv = l2_policy_evict_last();
        const uint32_t q_bytes = static_cast<uint32_t>(p.rows.Mt * p.rows.Gt * p.rows.St) * 128u * (D / kBoxCols);
        int nq0 = 0, nq1 = 0, g = 0, slot = 0, turn = 0, tails = 0;
        auto load_q = [&](const FwdItem& it, int t, int& n) {
          if (n > 0 && !mbar_wait(&bar[kFwQEmpty0 + t], (n - 1) & 1, ctx, 201)) return false;
          int im, ig, is;
          p.rows.box(it.tile0 + t, im, ig, is);
          mbar_arrive_expect_tx(&bar[kFwQFull0 + t], q_bytes);
#pragma unroll
          for (int x = 0; x < D / kBoxCols; ++x)
            tma_load_4d(smem + Cfg::kOffQ + t * Cfg::kTileBytes + x * kBoxBytes, &tm_Q, &bar[kFwQFull0 + t], x * kBoxCols,
                        im * p.rows.Mt, it.hk * p.rows.G + ig * p.rows.Gt, it.b * p.rows.S + is * p.rows.St, pol_q);
          ++n;
          return true;
        };
        auto load_kv = [&](const CUtensorMap* tm, const FwdItem& it, int j, int full) {
          if (g >= kSlots && !mbar_wait(&bar[kFwKVEmpty0 + slot], (turn - 1) & 1, ctx, 202)) return false;
          uint64_t* fb = &bar[full + slot];
          if (full == kFwTail0) tails |= 1 << slot;
          uint8_t* dst = smem + Cfg::kOffKV + slot * Cfg::kTileBytes;
          mbar_arrive_expect_tx(fb, Cfg::kTileBytes);
#pragma unroll
          for (int x = 0; x < D / kBoxCols; ++x)
            tma_load_4d(dst + x * kBoxBytes, tm, fb, x * kBoxCols, j * kTile, it.hk, it.b, pol_kv);
          ++g;
          if (++slot == kSlots) {
            slot = 0;
            ++turn;
          }
          return true;
        };
        while (get_unit<false>(ring, unit_full, unit_empty, k, ua, ub, ctx, 203, ok)) {
          const FwdItem it = fwd_item(ua, ub);
          if (it.lo == it.hi) continue;
          ok = load_q(it, 0, nq0) && load_kv(&tm_K, it, it.lo, kFwKVFull0) && (!it.two || load_q(it, 1, nq1));
          for (int j = it.lo; j < it.hi && ok; ++j)
            ok = load_kv(&tm_V, it, j, is_checked<kOwn>(it, j) ? kFwTail0 : kFwKVFull0) &&
                 (j + 1 == it.hi || load_kv(&tm_K, it, j + 1, kFwKVFull0));
        }
        if (*abort_flag) {
          // every copy in flight ends before the block does
          if (nq0 > 0) mbar_wait_drain(&bar[kFwQFull0], (nq0 - 1) & 1, p.timeout_ns);
          if (nq1 > 0) mbar_wait_drain(&bar[kFwQFull0 + 1], (nq1 - 1) & 1, p.timeout_ns);
          for (int i = (g > kSlots ? g - kSlots : 0); i < g; ++i) {
            mbar_wait_drain(&bar[kFwKVFull0 + i % kSlots], (i / kSlots) & 1, 1000000);
            if (tails >> (i % kSlots) & 1)
              for (int par = 0; par < 2; ++par) mbar_wait_drain(&bar[kFwTail0 + i % kSlots], par, 1000000);
          }
        }
      }
      __syncwarp();
    } else if (warp == 14) {
      if (lane == 0) feed_fwd<T, kOwn>(p, ua, ub, ring, unit_full, unit_empty, ctx);
      __syncwarp();
    } else if (warp == 13) {
      // ---- MMA. Per step, for each tile in turn: O += p V_j, then S of the
      // next step (of the next item, after the last one), which keeps the two
      // tiles half a step apart: with an issuer for each tile they drifted
      // into step and fought for the SFU and the tensor core by turns (357
      // against 327 us at 16384 rows, 1024 keys, 40 heads of 128).
      if (elect_one()) {
        constexpr uint32_t id_S = make_idesc_f16<kB>(kTile, kTile, false, false);
        constexpr uint32_t id_O = make_idesc_f16<kB>(kTile, D, false, true);
        const uint32_t sKV = smem_u32(smem + Cfg::kOffKV), sQ = smem_u32(smem + Cfg::kOffQ);
        int slot = 0, turn = 0;
        uint32_t turns = 0;  // bits: Q 0, 1; p 2, 3; O 4, 5; whether O was used 6, 7
        auto advance = [&] {
          if (++slot == kSlots) {
            slot = 0;
            turn ^= 1;
          }
        };
        auto next_item = [&](FwdItem& it) {
          while (get_unit<false>(ring, unit_full, unit_empty, k, ua, ub, ctx, 210, ok)) {
            it = fwd_item(ua, ub);
            if (it.lo < it.hi) return true;
          }
          return false;
        };
        FwdItem cur{}, nxt;
        bool more = next_item(cur);
        nxt = cur;
        int j = cur.lo - 1;  // the step before the first has no p V
        while (more && ok) {
          const bool start = j < cur.lo, last = j + 1 == cur.hi;
          // Whether S of a next step goes ahead. Behind the last step that is
          // of the next item, if this is not one without keys: to look for
          // further ones first would wait for units that are only put once
          // this item's O is done.
          bool ahead = true;
          if (last) {
            more = get_unit<false>(ring, unit_full, unit_empty, k, ua, ub, ctx, 210, ok);
            nxt = fwd_item(ua, ub);
            ahead = more && nxt.lo < nxt.hi;
          }
          if (!ok) break;
          const int jn = last ? nxt.lo : j + 1, vslot = slot;
          if (!start) {
            if (!(ok = mbar_wait(&bar[kFwKVFull0 + slot], turn, ctx, 212))) break;
            advance();
          }
          if (ahead && !(ok = mbar_wait(&bar[kFwKVFull0 + slot], turn, ctx, 216))) break;
#pragma unroll 1
          for (int t = 0; t < 2; ++t) {
            const uint32_t tS = tmem + Cfg::kColS + 128 * t, tO = tmem + Cfg::kColO + D * t;
            if (!start && (t == 0 || cur.two)) {
              if (j == cur.lo) {
                if ((turns >> (6 + t) & 1) && !(ok = mbar_wait(&bar[kFwOEmpty0 + t], (turns >> (4 + t) & 1) ^ 1, ctx, 213))) break;
                turns = (turns ^ (1u << (4 + t))) | 1u << (6 + t);
              }
              const uint32_t par = turns >> (2 + t) & 1, keep = j > cur.lo ? 1u : 0u;
              if (!(ok = mbar_wait(&bar[kFwPFull0 + t], par, ctx, 214))) break;
              tc_fence_after();
              const uint64_t dv = make_sw128_desc(sKV + vslot * Cfg::kTileBytes, kBoxBytes, 1024);
              const int left = cur.n - j * kTile;
              if (left >= kTile) {
#pragma unroll
                for (int x = 0; x < 6; ++x)
                  umma_f16_ts(tO, tS + x * 8, desc_advance(dv, x * 2048), id_O, x > 0 ? 1u : keep);
                if (!(ok = mbar_wait(&bar[kFwPRest0 + t], par, ctx, 215))) break;
                tc_fence_after();
#pragma unroll
                for (int x = 6; x < 8; ++x) umma_f16_ts(tO, tS + x * 8, desc_advance(dv, x * 2048), id_O, 1u);
              } else {
                if (!(ok = mbar_wait(&bar[kFwPRest0 + t], par, ctx, 215))) break;
                tc_fence_after();
#pragma unroll 1
                for (int x = 0; x < (left + 15) / 16; ++x)
                  umma_f16_ts(tO, tS + x * 8, desc_advance(dv, x * 2048), id_O, x > 0 ? 1u : keep);
              }
              turns ^= 4u << t;
              if (last) umma_commit(&bar[kFwOFull0 + t]);
            }
            if (t == 1 && !start) umma_commit(&bar[kFwKVEmpty0 + vslot]);
            if (ahead && (t == 0 || nxt.two)) {
              if (jn == nxt.lo) {
                if (!(ok = mbar_wait(&bar[kFwQFull0 + t], turns >> t & 1, ctx, 211))) break;
                turns ^= 1u << t;
              }
              tc_fence_after();
              const uint64_t dq = make_sw128_desc(sQ + t * Cfg::kTileBytes, 16, 1024);
              const uint64_t dk = make_sw128_desc(sKV + slot * Cfg::kTileBytes, 16, 1024);
#pragma unroll
              for (int x = 0; x < D / 16; ++x) {
                const uint32_t off = (x >> 2) * kBoxBytes + (x & 3) * 32;
                umma_f16_ss(tS, desc_advance(dq, off), desc_advance(dk, off), id_S, x > 0 ? 1u : 0u);
              }
              umma_commit(&bar[kFwSFull0 + t]);
              if (jn + 1 == nxt.hi) umma_commit(&bar[kFwQEmpty0 + t]);
            }
            if (t == 1 && ahead) umma_commit(&bar[kFwKVEmpty0 + slot]);
          }
          if (!ok) break;
          if (ahead) advance();
          else if (more) more = next_item(nxt);
          cur = nxt;
          j = ahead ? jn : nxt.lo - 1;
        }
        if (!ok) {
          umma_commit(&bar[kFwDrain]);
          mbar_wait_drain(&bar[kFwDrain], 0, p.timeout_ns);
        }
      }
      __syncwarp();
    }
  } else if (warp < 8) {
    // ---- softmax: warpgroup t owns tile t, thread = row (TMEM lane)
    regs_raise<Cfg::kSoftmaxRegs>();
    const int t = warp >> 2;
    const int r = threadIdx.x & 127;
    const uint32_t tS = tmem + Cfg::kColS + 128 * t + (static_cast<uint32_t>(r & 96) << 16);
    const uint32_t tO = tmem + Cfg::kColO + D * t + (static_cast<uint32_t>(r & 96) << 16);
    const float sl2 = p.scale * kLog2e;
    int ns = 0, nst = 0, no = 0;
    while (get_unit<true>(ring, unit_full, unit_empty, k, ua, ub, ctx, 230, ok)) {
      const FwdItem it = fwd_item(ua, ub);
      if (t == 1 && !it.two) continue;
      float m = 0.f;                                  // the row's reference, in powers of two
      float2 l0 = make_float2(0.f, 0.f), l1 = l0;     // its sum, in four shares
      for (int j = it.lo; j < it.hi; ++j, ++ns) {
        if (!mbar_wait(&bar[kFwSFull0 + t], ns & 1, ctx, 231)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        if constexpr (!kOwn) {
          if (it.n - j * kTile < kTile) mask_columns(tS, it.n - j * kTile, it.n - j * kTile);
        } else if (const int least = it.n - (p.rows.M - 1) - j * kTile; least < kTile) {
          int tok, g, s;
          p.rows.row(it.tile0 + t, r, tok, g, s);
          mask_columns(tS, least + min(tok, p.rows.M - 1), least);
        }
        uint32_t s[128];
        tmem_load_64(tS, s);
        tmem_load_64(tS + 64, s + 64);
        float mx[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) mx[x] = __uint_as_float(s[x]);
#pragma unroll
        for (int x = 4; x < 128; ++x) mx[x & 3] = fmaxf(mx[x & 3], __uint_as_float(s[x]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2 - kBias;
        if (j == it.lo) {
          m = fmaxf(top, kNoMax);  // finite, and below any score to come, where this tile has no weight
        } else if (__any_sync(0xffffffffu, top > m + 8.f)) {
          const bool move = top > m + 8.f;
          const float f = move ? ex2_approx(m - top) : 1.f;
          if (move) m = top;
          l0 = mul_f32x2(l0, make_float2(f, f));
          l1 = mul_f32x2(l1, make_float2(f, f));
#pragma unroll 1
          for (int x = 0; x < D / 16; ++x) {
            uint32_t o[16];
            tmem_load_16(tO + 16 * x, o);
#pragma unroll
            for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(f * __uint_as_float(o[y]));
            tmem_store_16(tO + 16 * x, o);
          }
          tmem_store_wait();
        }
        const float2 nm = make_float2(-m, -m), sc = make_float2(sl2, sl2);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t e[16];
          weights_32<T>(s + 32 * h, sc, nm, l0, l1, e);
          tmem_store_16(tS + 16 * h, e);
          if (h >= 2) {
            tmem_store_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar[(h == 2 ? kFwPFull0 : kFwPRest0) + t]);
          }
        }
      }
      if (!ok) continue;
      if (p.in_turn) {
        if (it.lo < it.hi) {
          if (!mbar_wait(&bar[kFwOFull0 + t], no & 1, ctx, 233)) { ok = false; continue; }
          if (kOwn && !mbar_wait(&bar[kFwChecked], no & 1, ctx, 234)) { ok = false; continue; }
          ++no;
        }
        __syncwarp();
        tc_fence_after();
        int tok, g, s;
        const bool real = p.rows.row(it.tile0 + t, r, tok, g, s);
        store_tile<T, D, kOwn>(p, it, tO, tok, g, s, real, m, (l0.x + l0.y) + (l1.x + l1.y), *odd_flag);
        tc_fence_before();
        __syncwarp();
        if (it.lo < it.hi && lane == 0) mbar_arrive(&bar[kFwOEmpty0 + t]);
        continue;
      }
      if (nst > 0 && !mbar_wait(&bar[kFwStEmpty0 + t], (nst - 1) & 1, ctx, 232)) { ok = false; continue; }
      stat[128 * t + r] = make_float2(m, (l0.x + l0.y) + (l1.x + l1.y));
      ++nst;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[kFwStFull0 + t]);
    }
  } else {
    // ---- epilogue: thread = row of each tile in turn. One warp also clears the
    // V tiles that are checked, for the issuer that waits for them.
    regs_lower<Cfg::kOtherRegs>();
    const int r = threadIdx.x & 127;
    int nst0 = 0, nst1 = 0, no0 = 0, no1 = 0, g = 0, ni = 0, odd = 0;
    uint32_t tail_turns = 0;  // a bit for each slot
    while (get_unit<true>(ring, unit_full, unit_empty, k, ua, ub, ctx, 240, ok)) {
      const FwdItem it = fwd_item(ua, ub);
      const bool keys = it.lo < it.hi;
      if (keys) {
        if (warp == 8) {
#pragma unroll 1
          for (int j = kOwn ? min(max(it.lo, it.first), it.hi - 1) : it.hi - 1; j < it.hi; ++j) {
            if (!is_checked<kOwn>(it, j)) continue;
            const int slot = (g + 2 * (j - it.lo) + 1) % kSlots;
            if (ok && !mbar_wait(&bar[kFwTail0 + slot], tail_turns >> slot & 1, ctx, 241)) ok = false;
            tail_turns ^= 1u << slot;
            __syncwarp();
            uint8_t* tile = smem + Cfg::kOffKV + slot * Cfg::kTileBytes;
            if (kOwn && ok && j >= it.first &&
                hide_odd<T, D>(tile, max(0, it.n - (p.rows.M - 1) - j * kTile), min(kTile, it.n - j * kTile), lane))
              *odd_flag = 1;
            if (ok && j + 1 == it.hi && has_tail(it.n, it.hi)) clear_tail<D>(tile, it.n - j * kTile, lane);
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(&bar[kFwKVFull0 + slot]);
          }
          // no further than one item ahead of the others
          if (kOwn && ok && ni > 0 && !mbar_wait(&bar[kFwSeen], (ni - 1) & 1, ctx, 245)) ok = false;
          __syncwarp();
          if (kOwn && ok && lane == 0) mbar_arrive(&bar[kFwChecked]);
        }
        g += 2 * (it.hi - it.lo);
      }
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        if ((t == 1 && !it.two) || p.in_turn) continue;
        if (ok && !mbar_wait(&bar[kFwStFull0 + t], (t == 0 ? nst0 : nst1) & 1, ctx, 242)) ok = false;
        if (!ok) break;
        if (t == 0) ++nst0;
        else ++nst1;
        const float2 ml = stat[128 * t + r];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[kFwStEmpty0 + t]);
        if (keys) {
          if (!mbar_wait(&bar[kFwOFull0 + t], (t == 0 ? no0 : no1) & 1, ctx, 243)) { ok = false; break; }
          if (kOwn && t == 0) {
            if (!mbar_wait(&bar[kFwChecked], ni & 1, ctx, 244)) { ok = false; break; }
            odd = *odd_flag;
            __syncwarp();
            if (warp != 8 && lane == 0) mbar_arrive(&bar[kFwSeen]);
          }
          if (t == 0) ++no0;
          else ++no1;
        }
        __syncwarp();
        tc_fence_after();
        int m, g, s;
        const bool real = p.rows.row(it.tile0 + t, r, m, g, s);
        store_tile<T, D, kOwn>(p, it, tmem + Cfg::kColO + D * t + (static_cast<uint32_t>(r & 96) << 16), m, g, s, real,
                               ml.x, ml.y, odd);
        tc_fence_before();
        __syncwarp();
        if (keys && lane == 0) mbar_arrive(&bar[kFwOEmpty0 + t]);
      }
      if (keys) ++ni;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) publish_failure(*abort_flag, p.status);
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (kOwn) asm volatile("griddepcontrol.wait;" ::: "memory");
}

constexpr int kJoinAhead = 4;
// Joins the parts of split keys: with weights w_i = exp(LSE_i - max LSE),
// O = sum w_i O_i / sum w_i and LSE = max LSE + log sum w_i, parts in order.
// D / 4 lanes to a row: they hold the parts' weights, and take 4 columns each.
// Bound by the latency of two loads in turn, so the first parts' O is asked for
// before their weights are known; 24 warps an SM matter more than more loads a
// thread (4 ahead: 18 us, 8 ahead and 16 warps: 20 for 333 x 777 in 3 parts).
// 19 parts of 2048 rows of 128: 4 us.
template <typename T, int D>
__global__ void __launch_bounds__(256, 6)
    attn_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_lse, int parts, int64_t rows,
                     View<T> O, float* __restrict__ LSE, int Hq, int M) {
  constexpr int L = D / 4;
  static_assert(L % kJoinAhead == 0, "a row's lanes hold whole batches of weights");
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / L;
  const int lane = threadIdx.x % L;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool real = at < rows;
  const int64_t row = real ? at : rows - 1;  // whole warps shuffle
  const float4* base = reinterpret_cast<const float4*>(part_o + row * D) + lane;
  const int64_t stride = rows * L;
  float4 v[kJoinAhead];  // the next parts' O, asked for before the weights are known
  auto load = [&](int from) {
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k)
      if (from + k < parts) v[k] = __ldcg(base + (from + k) * stride);
  };
  load(0);
  float top = -INFINITY;
  for (int k = lane; k < parts; k += L) top = fmaxf(top, __ldcg(part_lse + k * rows + row));
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top == -INFINITY) top = 0.f;  // no part has a key: all weights are 0
  float sum = 0.f, mine = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int from = 0; from < parts; from += kJoinAhead) {
    if (from % L == 0)
      mine = from + lane < parts ? ex2_approx((__ldcg(part_lse + (from + lane) * rows + row) - top) * kLog2e) : 0.f;
    if (from > 0) load(from);
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k) {
      if (from + k >= parts) break;
      const float w = __shfl_sync(0xffffffffu, mine, (from + k) % L, L);
      sum += w;
      acc.x = fmaf(w, v[k].x, acc.x);
      acc.y = fmaf(w, v[k].y, acc.y);
      acc.z = fmaf(w, v[k].z, acc.z);
      acc.w = fmaf(w, v[k].w, acc.w);
    }
  }
  if (!real) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;  // NaN stays
  const int m = static_cast<int>(row % M), h = static_cast<int>(row / M % Hq), b = static_cast<int>(row / M / Hq);
  *reinterpret_cast<uint2*>(O.at(b, h, m) + 4 * lane) =
      make_uint2(Elem<T>::pack(inv * acc.x, inv * acc.y), Elem<T>::pack(inv * acc.z, inv * acc.w));
  if (lane == 0) LSE[row] = sum == 0.f ? -INFINITY : top + logf(sum);
}

}  // namespace fmha_sm100
