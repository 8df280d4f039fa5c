// The backward of attention written straight from its formulas: one warp per
// output row, every product in fp32 on the CUDA cores. Right for every case;
// bounded by the re-reading of the other rows for every row.
#pragma once

#include "fmha_attn.cuh"

namespace fmha_sm100 {

template <typename T>
struct SimpleParams {
  View<T> Q, O, K, V, dO, dQ, dK, dV, Kp, Vp;
  float* LSE;
  const int *kv_lens, *prefix_lens;
  int B, Hq, Hkv, M, N, D, prefixes, Np;
  float scale;
};

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <typename T>
__device__ __forceinline__ float as_float(T x) {
  return static_cast<float>(x);
}

// dQ, one warp per query row.
template <typename T, int D>
__global__ void simple_dq_kernel(SimpleParams<T> p) {
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  const int lane = threadIdx.x & 31;
  if (row >= static_cast<int64_t>(p.B) * p.Hq * p.M) return;
  const int m = static_cast<int>(row % p.M), h = static_cast<int>(row / p.M % p.Hq), b = static_cast<int>(row / p.M / p.Hq);
  const int hk = h / (p.Hq / p.Hkv), n = valid_rows(p.kv_lens, b, p.N);
  constexpr int E = D / 32;
  float q[E], g[E], acc[E], delta = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = as_float(p.Q.at(b, h, m)[lane + 32 * e]) * p.scale;
    g[e] = as_float(p.dO.at(b, h, m)[lane + 32 * e]);
    delta = fmaf(g[e], as_float(p.O.at(b, h, m)[lane + 32 * e]), delta);
    acc[e] = 0.f;
  }
  delta = warp_sum(delta);
  const float lse = p.LSE[row];
  for (int j = 0; j < n; ++j) {
    const T *k = p.K.at(b, hk, j), *v = p.V.at(b, hk, j);
    float s = 0.f, dp = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s = fmaf(q[e], as_float(k[lane + 32 * e]), s);
      dp = fmaf(g[e], as_float(v[lane + 32 * e]), dp);
    }
    const float ds = expf(warp_sum(s) - lse) * (warp_sum(dp) - delta) * p.scale;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(ds, as_float(k[lane + 32 * e]), acc[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) p.dQ.at(b, h, m)[lane + 32 * e] = T(acc[e]);
}

// dK and dV, one warp per key row, over the query rows of its kv head's group.
template <typename T, int D>
__global__ void simple_dkv_kernel(SimpleParams<T> p) {
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  const int lane = threadIdx.x & 31;
  if (row >= static_cast<int64_t>(p.B) * p.Hkv * p.N) return;
  const int j = static_cast<int>(row % p.N), hk = static_cast<int>(row / p.N % p.Hkv), b = static_cast<int>(row / p.N / p.Hkv);
  const int G = p.Hq / p.Hkv;
  constexpr int E = D / 32;
  float dk[E], dv[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dk[e] = dv[e] = 0.f;
  if (j < valid_rows(p.kv_lens, b, p.N)) {
    float k[E], v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      k[e] = as_float(p.K.at(b, hk, j)[lane + 32 * e]) * p.scale;
      v[e] = as_float(p.V.at(b, hk, j)[lane + 32 * e]);
    }
    for (int h = hk * G; h < (hk + 1) * G; ++h) {
      for (int m = 0; m < p.M; ++m) {
        const T *q = p.Q.at(b, h, m), *g = p.dO.at(b, h, m), *o = p.O.at(b, h, m);
        float s = 0.f, dp = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float ge = as_float(g[lane + 32 * e]);
          s = fmaf(k[e], as_float(q[lane + 32 * e]), s);
          dp += ge * (v[e] - as_float(o[lane + 32 * e]));
        }
        const float w = expf(warp_sum(s) - p.LSE[(static_cast<int64_t>(b) * p.Hq + h) * p.M + m]);
        const float ds = w * warp_sum(dp) * p.scale;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          dk[e] = fmaf(ds, as_float(q[lane + 32 * e]), dk[e]);
          dv[e] = fmaf(w, as_float(g[lane + 32 * e]), dv[e]);
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    p.dK.at(b, hk, j)[lane + 32 * e] = T(dk[e]);
    p.dV.at(b, hk, j)[lane + 32 * e] = T(dv[e]);
  }
}

template <typename T>
int run_simple(const fmha_attn_t& a, cudaStream_t stream) {
  const SimpleParams<T> p{view_of<T>(a.Q), view_of<T>(a.O), view_of<T>(a.K), view_of<T>(a.V), view_of<T>(a.dO),
                          view_of<T>(a.dQ), view_of<T>(a.dK), view_of<T>(a.dV), view_of<T>(a.Kp), view_of<T>(a.Vp),
                          a.LSE, a.kv_lens, a.prefix_lens, a.batch, a.q_heads, a.kv_heads, a.M, a.N, a.K_dim,
                          a.prefixes, a.N_prefix, a.softmax_scale};
  auto blocks = [](int64_t rows) { return static_cast<unsigned>((rows + 7) / 8); };
  const unsigned gq = blocks(static_cast<int64_t>(a.batch) * a.q_heads * a.M);
  const unsigned gk = blocks(static_cast<int64_t>(a.batch) * a.kv_heads * a.N);
  auto go = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    simple_dq_kernel<T, D><<<gq, 256, 0, stream>>>(p);
    simple_dkv_kernel<T, D><<<gk, 256, 0, stream>>>(p);
  };
  if (a.K_dim == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 64>{});
  return kOk;
}

}  // namespace fmha_sm100
