// Log probabilities of given tokens from rows of logits, with each row's entropy and its most probable tokens.
//
//   m = max z,  s = sum e^(z - m),  A = sum e^(z - m) (z - m)
//   log p_t = z_t - m - log s,      H = log s - A / s
//
// The reference reads them from torch.log_softmax over the whole vocabulary (eval_ppl,
// benchmarks/eval_llama.py:77-117, cross entropy of every token).  Here the logits are read once.  Every thread keeps
// a running (m, s, A) of its elements, in fp32; a row is one CTA's, or, when there are few rows, a cluster's.
//
// The most probable tokens: the threads' maxima, 32 groups of them, give a value that at least `top` logits reach (the
// top-th largest of the group maxima), and only the elements of the threads whose maximum reaches it are looked at
// again (from L2): some tens of candidates, which are put in order by counting.
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace i4b {

namespace {

constexpr int kCand = 512;  // candidates above, and at, the threshold that a CTA holds
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two fp32 operations in one instruction (sm_100).
__device__ __forceinline__ uint64_t pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Logits of a type: 16 bytes hold kVec of them; most() is the largest of a 16-byte chunk (a NaN does not count).
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
  __device__ __forceinline__ static float most(const uint4& w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
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
      if constexpr (DT == I4B_BF16) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
      } else {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
      }
    }
  }
  __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (DT == I4B_BF16)
      asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ static float most(const uint4& w) {
    const uint32_t m = max2(max2(w.x, w.y), max2(w.z, w.w));
    return fmaxf(one(uint16_t(m)), one(uint16_t(m >> 16)));
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

__device__ __forceinline__ void raise(Stat& st, float m) {  // to the larger m
  const float d = st.m == -INFINITY ? 0.0f : st.m - m, f = st.m == -INFINITY ? 0.0f : ex2(d * kLog2e);
  st.a = f > 0.0f ? (st.a + d * st.s) * f : 0.0f;  // d * s may overflow where f is 0
  st.s = st.s * f;                                 // (a NaN sum stays one)
  st.m = m;
}

// (z - m) e^(z - m) summed where e > 0 only: 0 * -inf has no value.
__device__ __forceinline__ void add_one(Stat& st, float z) {
  if (z > st.m) raise(st, z);
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

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// N chunks at once: their maximum first, then, in units of log 2, t = z log2(e) - m log2(e) in one packed operation of
// two elements, as are the two sums: 8.0 instructions per logit in the whole kernel.  m log2(e) is rounded, off by delta, and with it
// every t: the sums are put right for that afterwards, while |delta| <= 1 (|m| <= 2^24; beyond, 2^delta could leave
// fp32's range).  Every logit is first raised to m - 200 (e^-200 is 0 in fp32, its terms stay 0): a mask's -inf or lowest
// value would make 0 * inf.  Without that, masked batches had to go one by one: 198 instead of 90 us for 2048 x 128256
// bf16 with any -inf in each batch, 19.3 instead of 15.1 for 61 x 100003 fp32, against 88 instead of 90 where nothing is
// masked.  A NaN or a +inf leaves no finite sum; such a batch, and one of a larger |m|, is taken again one by one.
template <typename E, int N>
__device__ __forceinline__ void add_batch(Stat& st, const uint4 (&w)[N]) {
  float top = E::most(w[0]);
#pragma unroll
  for (int u = 1; u < N; ++u) top = fmaxf(top, E::most(w[u]));
  if (top > st.m) raise(st, top);
  const float m = st.m == -INFINITY ? 0.0f : st.m, low = m - 200.0f;  // (nothing but masked ones so far: all sums 0)
  const float ml = m * kLog2e, delta = fmaf(m, kLog2e, -ml);
  const uint64_t nm = pack(-ml, -ml), l2 = pack(kLog2e, kLog2e);
  uint64_t s2 = 0, a2 = 0;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float f[E::kVec];
    E::many(w[u], f);
#pragma unroll
    for (int i = 0; i < E::kVec; i += 2) {
      const uint64_t t2 = fma2(pack(max_nan(f[i], low), max_nan(f[i + 1], low)), l2, nm);
      const float2 t = unpack(t2);
      const uint64_t e = pack(ex2(t.x), ex2(t.y));
      s2 = add2(s2, e);
      a2 = fma2(e, t2, a2);
    }
  }
  const float2 s = unpack(s2), a = unpack(a2);
  const float ss = s.x + s.y, as = a.x + a.y;
  if (as - as == 0.0f && fabsf(m) <= 16777216.0f) {  // (the difference: finite)
    const float back = ex2(-delta);
    st.s = fmaf(ss, back, st.s);
    st.a = fmaf((as - delta * ss) * kLn2, back, st.a);
  } else {
#pragma unroll 1
    for (int u = 0; u < N; ++u) {
      uint4 x = w[0];
#pragma unroll
      for (int k = 1; k < N; ++k)
        if (u == k) x = w[k];
      float f[E::kVec];
      E::many(x, f);
#pragma unroll
      for (int i = 0; i < E::kVec; ++i) add_one(st, f[i]);
    }
  }
}

// Whether (v, i) comes before (w, j) among the most probable tokens: larger value, then lower index; never for a NaN.
__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

template <int kThreads>
struct Shared {
  Stat red[kThreads / 32], part;
  float col[kThreads / 32][32];
  float thr, bv[kThreads / 32];
  int bi[kThreads / 32];
  int above, ties, hits;
  int hit[kThreads];
  float cv[2 * kCand];
  int ci[2 * kCand];
  float sv[I4B_MAX_TOP];  // this CTA's best, in order; index -1: none
  int si[I4B_MAX_TOP];
};

// kThreads: 512 for few rows, 256 (four CTAs per SM, whose beginnings and ends overlap) when there are rows for all
// SMs: 88 us for 2048 x 128256 bf16 where 512 took 96 (90 since masked logits stay on the short way).
template <int DT, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
    token_logprobs_kernel(const typename Logit<DT>::T* __restrict__ x, int n, int64_t stride,
                          const int64_t* __restrict__ targets, int top, int parts, float* __restrict__ logprobs,
                          float* __restrict__ entropy, float* __restrict__ top_lp, int64_t* __restrict__ top_ids) {
  using E = Logit<DT>;
  constexpr int VEC = E::kVec, U = 4;
  __shared__ Shared<kThreads> sh;
  const int64_t row = blockIdx.x / parts;
  const int part = parts > 1 ? int(cluster_ctarank()) : 0;
  const typename E::T* xr = x + row * stride;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // elements before the first 16-byte boundary and behind the last whole chunk go one by one, the first with the first
  // part, the last with the last; a part's chunks are consecutive
  const int head = min(n, int((16 - (reinterpret_cast<uintptr_t>(xr) & 15)) % 16 / sizeof(typename E::T)));
  const int chunks = (n - head) / VEC, tail = head + chunks * VEC;
  const int c0 = int(int64_t(chunks) * part / parts), c1 = int(int64_t(chunks) * (part + 1) / parts);
  const int heads = part == 0 ? head : 0, tails = part == parts - 1 ? n - tail : 0;
  const uint4* xv = reinterpret_cast<const uint4*>(xr + head);
  Stat st = {-INFINITY, 0.0f, 0.0f};
  {
    uint4 w[U];
    int ch = c0 + tid;
    const bool first = ch + (U - 1) * kThreads < c1;
    if (first) {
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = __ldg(xv + ch + u * kThreads);
      for (ch += U * kThreads; ch + (U - 1) * kThreads < c1; ch += U * kThreads) {  // the next batch on its way
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = __ldg(xv + ch + u * kThreads);
        add_batch<E, U>(st, w);
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = v[u];
      }
    }
    uint4 r[U - 1];
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (ch + u * kThreads < c1) r[u] = __ldg(xv + ch + u * kThreads);
    if (first) add_batch<E, U>(st, w);
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (ch + u * kThreads < c1) {
        const uint4 one[1] = {r[u]};
        add_batch<E, 1>(st, one);
      }
    if (tid < heads) add_one(st, E::one(xr[tid]));
    if (tid < tails) add_one(st, E::one(xr[tail + tid]));
  }
  const float mine = st.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st = merge(st, {__shfl_xor_sync(0xFFFFFFFFu, st.m, o), __shfl_xor_sync(0xFFFFFFFFu, st.s, o),
                    __shfl_xor_sync(0xFFFFFFFFu, st.a, o)});
  if (lane == 0) sh.red[warp] = st;
  sh.col[warp][lane] = mine;
  if (tid == 0) sh.above = sh.ties = sh.hits = 0;
  __syncthreads();
  if (warp == 0) {
    st = lane < kThreads / 32 ? sh.red[lane] : Stat{-INFINITY, 0.0f, 0.0f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      st = merge(st, {__shfl_xor_sync(0xFFFFFFFFu, st.m, o), __shfl_xor_sync(0xFFFFFFFFu, st.s, o),
                      __shfl_xor_sync(0xFFFFFFFFu, st.a, o)});
    if (lane == 0) sh.part = st;
  }
  if (top > 0) {
    if (warp == 1) {  // the top-th largest of 32 group maxima
      float v = sh.col[0][lane];
#pragma unroll
      for (int w = 1; w < kThreads / 32; ++w) v = fmaxf(v, sh.col[w][lane]);
      int rank = 0;
      for (int i = 0; i < 32; ++i) {
        const float u = __shfl_sync(0xFFFFFFFFu, v, i);
        rank += u > v || (u == v && i < lane);
      }
      if (rank == top - 1) sh.thr = v;
    }
    __syncthreads();
    const float thr = sh.thr;
    if (mine >= thr) sh.hit[atomicAdd(&sh.hits, 1)] = tid;
    __syncthreads();
    // the elements of those threads: above the threshold, and at it
    auto look = [&](float v, int i) {
      if (v > thr) {
        const int at = atomicAdd(&sh.above, 1);
        if (at < kCand) sh.cv[at] = v, sh.ci[at] = i;
      } else if (v == thr) {
        const int at = atomicAdd(&sh.ties, 1);
        if (at < kCand) sh.cv[kCand + at] = v, sh.ci[kCand + at] = i;
      }
    };
    const int each = (c1 - c0 + kThreads - 1) / kThreads + 1, work = sh.hits * each;  // its chunks, and its single ones
    for (int i = tid; i < work; i += kThreads) {
      const int owner = sh.hit[i / each], k = i % each, ch = c0 + owner + k * kThreads;
      if (k == each - 1) {
        if (owner < heads) look(E::one(xr[owner]), owner);
        if (owner < tails) look(E::one(xr[tail + owner]), tail + owner);
      } else if (ch < c1) {
        float f[VEC];
        E::many(__ldg(xv + ch), f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) look(f[e], head + ch * VEC + e);
      }
    }
    __syncthreads();
    const int above = sh.above, ties = sh.ties;
    if (tid < I4B_MAX_TOP) sh.sv[tid] = -INFINITY, sh.si[tid] = -1;
    __syncthreads();
    if (above <= kCand) {
      for (int i = tid; i < above; i += kThreads) {
        int rank = 0;
        for (int j = 0; j < above; ++j) rank += before(sh.cv[j], sh.ci[j], sh.cv[i], sh.ci[i]);
        if (rank < top) sh.sv[rank] = sh.cv[i], sh.si[rank] = sh.ci[i];
      }
      if (above < top) {  // the lowest places among those at the threshold
        if (ties <= kCand) {
          for (int i = tid; i < ties; i += kThreads) {
            int rank = above;
            for (int j = 0; j < ties; ++j) rank += sh.ci[kCand + j] < sh.ci[kCand + i];
            if (rank < top) sh.sv[rank] = thr, sh.si[rank] = sh.ci[kCand + i];
          }
        } else {  // many: from the front until there are enough
          const int lo = part == 0 ? 0 : head + c0 * VEC, hi = part == parts - 1 ? n : head + c1 * VEC;
          int got = above;
          for (int i0 = lo; i0 < hi && got < top; i0 += kThreads) {
            const int i = i0 + tid;
            const bool is = i < hi && E::one(xr[i]) == thr;
            const uint32_t b = __ballot_sync(0xFFFFFFFFu, is);
            if (lane == 0) sh.bi[warp] = __popc(b);
            __syncthreads();
            int at = got, all = 0;
            for (int w = 0; w < kThreads / 32; ++w) {
              if (w < warp) at += sh.bi[w];
              all += sh.bi[w];
            }
            at += __popc(b & ((1u << lane) - 1u));
            if (is && at < top) sh.sv[at] = thr, sh.si[at] = i;
            got += all;
            __syncthreads();
          }
        }
      }
    } else {  // more than the lists hold (the part's largest logits all with few threads): one after the other
      const int lo = part == 0 ? 0 : head + c0 * VEC, hi = part == parts - 1 ? n : head + c1 * VEC;
      float lv = INFINITY;
      int li = -1;
      for (int k = 0; k < top; ++k) {
        float bv = -INFINITY;
        int bi = INT32_MAX;
        for (int i = lo + tid; i < hi; i += kThreads) {
          const float v = E::one(xr[i]);
          if (before(lv, li, v, i) && before(v, i, bv, bi)) bv = v, bi = i;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const float v = __shfl_xor_sync(0xFFFFFFFFu, bv, o);
          const int i = __shfl_xor_sync(0xFFFFFFFFu, bi, o);
          if (before(v, i, bv, bi)) bv = v, bi = i;
        }
        if (lane == 0) sh.bv[warp] = bv, sh.bi[warp] = bi;
        __syncthreads();
        bv = sh.bv[0], bi = sh.bi[0];
        for (int w = 1; w < kThreads / 32; ++w)
          if (before(sh.bv[w], sh.bi[w], bv, bi)) bv = sh.bv[w], bi = sh.bi[w];
        if (tid == 0) sh.sv[k] = bv, sh.si[k] = bi;
        lv = bv, li = bi;
        __syncthreads();
      }
    }
  }
  __syncthreads();
  st = sh.part;
  if (parts > 1) {
    cluster_sync();
    if (part == 0) {
      if (warp == 0) {
        if (lane > 0 && lane < parts) {
          st.m = ld_shared_cluster_f32(mapa_shared(smem_u32(&sh.part.m), uint32_t(lane)));
          st.s = ld_shared_cluster_f32(mapa_shared(smem_u32(&sh.part.s), uint32_t(lane)));
          st.a = ld_shared_cluster_f32(mapa_shared(smem_u32(&sh.part.a), uint32_t(lane)));
        } else if (lane > 0) {
          st = {-INFINITY, 0.0f, 0.0f};
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1)
          st = merge(st, {__shfl_xor_sync(0xFFFFFFFFu, st.m, o), __shfl_xor_sync(0xFFFFFFFFu, st.s, o),
                          __shfl_xor_sync(0xFFFFFFFFu, st.a, o)});
        if (lane == 0) sh.red[0] = st;
      }
      for (int i = tid; i < parts * top; i += kThreads) {
        const uint32_t r = uint32_t(i / top);
        sh.cv[i] = ld_shared_cluster_f32(mapa_shared(smem_u32(&sh.sv[i % top]), r));
        sh.ci[i] = __float_as_int(ld_shared_cluster_f32(mapa_shared(smem_u32(&sh.si[i % top]), r)));
      }
      __syncthreads();
      st = sh.red[0];
      if (tid < I4B_MAX_TOP) sh.sv[tid] = -INFINITY, sh.si[tid] = -1;  // (read by this CTA alone: rank 0's list is in cv)
      __syncthreads();
      for (int i = tid; i < parts * top; i += kThreads) {
        if (sh.ci[i] < 0) continue;
        int rank = 0;
        for (int j = 0; j < parts * top; ++j) rank += sh.ci[j] >= 0 && before(sh.cv[j], sh.ci[j], sh.cv[i], sh.ci[i]);
        if (rank < top) sh.sv[rank] = sh.cv[i], sh.si[rank] = sh.ci[i];
      }
      __syncthreads();
    }
    cluster_sync();  // no CTA leaves while the first may still read its shared memory
    if (part != 0) return;
  }
  // a row that is -inf throughout has no distribution: log probabilities -inf, entropy 0
  const bool none = st.m == -INFINITY && st.s == 0.0f;
  const float ls = logf(st.s);
  auto logp = [&](float z) { return none ? -INFINITY : (z - st.m) - ls; };
  if (tid == 0) {
    const int64_t t = targets[row];
    logprobs[row] = t < 0 ? 0.0f : (t < n ? logp(E::one(xr[t])) : __int_as_float(0x7FC00000));
    entropy[row] = none ? 0.0f : ls - st.a / st.s;
  }
  if (tid < top) {
    const int i = sh.si[tid];
    top_lp[row * top + tid] = i >= 0 && i < n ? logp(sh.sv[tid]) : __int_as_float(0x7FC00000);  // (only NaN are left)
    top_ids[row * top + tid] = i >= 0 && i < n ? i : 0;
  }
}

template <int DT>
cudaError_t launch(const void* x, int64_t rows, int64_t n, int64_t stride, const int64_t* targets, int top,
                   float* logprobs, float* entropy, float* top_lp, int64_t* top_ids, int sms, cudaStream_t s) {
  using T = typename Logit<DT>::T;
  // as many CTAs per row as keep all CTAs resident (two per SM), each with at least 16 KB
  int parts = 8;
  while (parts > 1 && (rows * parts > 2 * sms || n * int64_t(sizeof(T)) < parts * 16384)) parts /= 2;
  const bool many = rows >= 2 * sms;  // (parts is 1)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * parts));
  cfg.blockDim = dim3(many ? 256 : 512);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(parts);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, many ? token_logprobs_kernel<DT, 256> : token_logprobs_kernel<DT, 512>,
                            static_cast<const T*>(x), int(n), stride, targets, top, parts, logprobs, entropy, top_lp,
                            top_ids);
}

}  // namespace

cudaError_t launch_token_logprobs(const void* x, int dtype, int64_t rows, int64_t n, int64_t stride,
                                  const int64_t* targets, int top, float* logprobs, float* entropy, float* top_lp,
                                  int64_t* top_ids, int sms, cudaStream_t s) {
  if (dtype == I4B_F32) return launch<I4B_F32>(x, rows, n, stride, targets, top, logprobs, entropy, top_lp, top_ids, sms, s);
  if (dtype == I4B_F16) return launch<I4B_F16>(x, rows, n, stride, targets, top, logprobs, entropy, top_lp, top_ids, sms, s);
  return launch<I4B_BF16>(x, rows, n, stride, targets, top, logprobs, entropy, top_lp, top_ids, sms, s);
}

}  // namespace i4b
