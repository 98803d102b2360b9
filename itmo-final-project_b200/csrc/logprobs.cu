// Log probabilities of given tokens from rows of logits, with each row's entropy and its most probable tokens.
//
//   m = max z,  s = sum e^(z - m),  A = sum e^(z - m) (z - m)
//   log p_t = z_t - m - log s,      H = log s - A / s
//
// The reference reads them from torch.log_softmax over the whole vocabulary (eval_ppl,
// benchmarks/eval_llama.py:77-117, cross entropy of every token).  Here the logits are read once: every thread keeps
// a running (m, s, A) of its elements.
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace i4b {

namespace {

constexpr int kThreads = 512;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

template <int DT>
struct Logit;
template <>
struct Logit<I4B_F32> {
  using T = float;
  static constexpr int kVec = 4;
  __device__ __forceinline__ static float one(float v) { return v; }
  __device__ __forceinline__ static void many(const uint4& w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
  }
};
template <int DT>
struct Logit16 {
  using T = uint16_t;
  static constexpr int kVec = 8;
  __device__ __forceinline__ static float one(uint16_t v) { return Elem<DT>::to_f32(v); }
  __device__ __forceinline__ static void many(const uint4& w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = Elem<DT>::to_f32(uint16_t(u[i]));
      f[2 * i + 1] = Elem<DT>::to_f32(uint16_t(u[i] >> 16));
    }
  }
};
template <>
struct Logit<I4B_F16> : Logit16<I4B_F16> {};
template <>
struct Logit<I4B_BF16> : Logit16<I4B_BF16> {};

// Running statistics of a part of a row; m is the largest logit (NaN not counted), s and a are relative to it.
struct Stat {
  float m, s, a;
};

// (z - m) e^(z - m) summed where e > 0 only: 0 * -inf has no value.
__device__ __forceinline__ void add_one(Stat& st, float z) {
  if (z > st.m) {
    const float d = st.m == -INFINITY ? 0.0f : st.m - z, f = st.m == -INFINITY ? 0.0f : ex2(d * kLog2e);
    st.a = f > 0.0f ? (st.a + d * st.s) * f : 0.0f;  // d * s may overflow where f is 0
    st.s *= f;
    st.m = z;
  }
  const float d = z - st.m, e = ex2(d * kLog2e);
  st.s += z == -INFINITY ? 0.0f : e;
  if (e > 0.0f) st.a = fmaf(e, d, st.a);
}

__device__ __forceinline__ Stat merge(const Stat& x, const Stat& y) {
  Stat r;
  r.m = fmaxf(x.m, y.m);
  const float dx = x.m == -INFINITY ? 0.0f : x.m - r.m, dy = y.m == -INFINITY ? 0.0f : y.m - r.m;
  const float fx = ex2(dx * kLog2e), fy = ex2(dy * kLog2e);
  r.s = x.s * fx + y.s * fy;
  r.a = (fx > 0.0f ? (x.a + dx * x.s) * fx : 0.0f) + (fy > 0.0f ? (y.a + dy * y.s) * fy : 0.0f);
  return r;
}

// Whether (v, i) comes before (w, j) among the most probable tokens: larger value, then lower index; NaN last.
__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

template <int DT>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const typename Logit<DT>::T* __restrict__ x, int n,
                                                                  int64_t stride, const int64_t* __restrict__ targets,
                                                                  int top, float* __restrict__ logprobs,
                                                                  float* __restrict__ entropy,
                                                                  float* __restrict__ top_lp,
                                                                  int64_t* __restrict__ top_ids) {
  using E = Logit<DT>;
  constexpr int VEC = E::kVec;
  __shared__ Stat red[kThreads / 32];
  __shared__ float rv[kThreads / 32];
  __shared__ int ri[kThreads / 32];
  const int64_t row = blockIdx.x;
  const typename E::T* xr = x + row * stride;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // elements before the first 16-byte boundary and behind the last whole chunk go one by one
  const int head = min(n, int((16 - (reinterpret_cast<uintptr_t>(xr) & 15)) % 16 / sizeof(typename E::T)));
  const int chunks = (n - head) / VEC, tail = head + chunks * VEC;
  const uint4* xv = reinterpret_cast<const uint4*>(xr + head);
  Stat st = {-INFINITY, 0.0f, 0.0f};
  if (tid < head) add_one(st, E::one(xr[tid]));
  if (tid < n - tail) add_one(st, E::one(xr[tail + tid]));
  for (int ch = tid; ch < chunks; ch += kThreads) {
    float f[VEC];
    E::many(__ldg(xv + ch), f);
#pragma unroll
    for (int i = 0; i < VEC; ++i) add_one(st, f[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st = merge(st, {__shfl_xor_sync(0xFFFFFFFFu, st.m, o), __shfl_xor_sync(0xFFFFFFFFu, st.s, o),
                    __shfl_xor_sync(0xFFFFFFFFu, st.a, o)});
  if (lane == 0) red[warp] = st;
  __syncthreads();
  st = red[0];
  for (int w = 1; w < kThreads / 32; ++w) st = merge(st, red[w]);
  // a row that is -inf throughout has no distribution: log probabilities -inf, entropy 0
  const bool none = st.m == -INFINITY && st.s == 0.0f;
  const float ls = logf(st.s);
  auto logp = [&](float z) { return none ? -INFINITY : (z - st.m) - ls; };
  if (tid == 0) {
    const int64_t t = targets[row];
    logprobs[row] = t < 0 ? 0.0f : (t < n ? logp(E::one(xr[t])) : __int_as_float(0x7FC00000));
    entropy[row] = none ? 0.0f : ls - st.a / st.s;
  }
  float lv = INFINITY;
  int li = -1;
  for (int k = 0; k < top; ++k) {
    // the first element behind (lv, li)
    float bv = -INFINITY;
    int bi = INT32_MAX;
    bool any = false;
    for (int i = tid; i < n; i += kThreads) {
      float v = E::one(xr[i]);
      if (before(lv, li, v, i) && (!any || before(v, i, bv, bi))) bv = v, bi = i, any = true;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float v = __shfl_xor_sync(0xFFFFFFFFu, bv, o);
      const int i = __shfl_xor_sync(0xFFFFFFFFu, bi, o);
      if (before(v, i, bv, bi)) bv = v, bi = i;
    }
    __syncthreads();
    if (lane == 0) rv[warp] = bv, ri[warp] = bi;
    __syncthreads();
    bv = rv[0], bi = ri[0];
    for (int w = 1; w < kThreads / 32; ++w)
      if (before(rv[w], ri[w], bv, bi)) bv = rv[w], bi = ri[w];
    if (tid == 0) {
      top_lp[row * top + k] = logp(bv);
      top_ids[row * top + k] = bi < n ? bi : 0;
    }
    lv = bv, li = bi;
  }
}

}  // namespace

cudaError_t launch_token_logprobs(const void* x, int dtype, int64_t rows, int64_t n, int64_t stride,
                                  const int64_t* targets, int top, float* logprobs, float* entropy, float* top_lp,
                                  int64_t* top_ids, cudaStream_t s) {
  const dim3 grid{unsigned(rows)};
  if (dtype == I4B_F32)
    token_logprobs_kernel<I4B_F32><<<grid, kThreads, 0, s>>>(static_cast<const float*>(x), int(n), stride, targets, top,
                                                             logprobs, entropy, top_lp, top_ids);
  else if (dtype == I4B_F16)
    token_logprobs_kernel<I4B_F16><<<grid, kThreads, 0, s>>>(static_cast<const uint16_t*>(x), int(n), stride, targets,
                                                             top, logprobs, entropy, top_lp, top_ids);
  else
    token_logprobs_kernel<I4B_BF16><<<grid, kThreads, 0, s>>>(static_cast<const uint16_t*>(x), int(n), stride, targets,
                                                              top, logprobs, entropy, top_lp, top_ids);
  return cudaGetLastError();
}

}  // namespace i4b
