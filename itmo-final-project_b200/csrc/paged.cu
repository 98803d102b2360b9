// Serving over a paged key-value cache: sequences of different lengths, their keys and values in fixed-size pages
// that a block table names.
//
//   paged_append   q, k = rotary(t, cos, sin); k and v -> page table[seq][slot / ps], row slot % ps
//   paged_attn     out = softmax(q . K^T * scale) . V over a sequence's positions, GQA; optionally
//                  weights[seq, kv head, j] += sum over the kv head's query heads of the probability of position j
//   paged_evict    the positions of highest accumulated weight and the most recent ones, kept in order, copied
//                  into new pages
//
// The reference has no counterpart: its decode benchmark runs transformers' attention over a StaticCache
// (benchmarks/eval_llama.py:121-183).  The contiguous, one-position forms are in decode_ops.cu.
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace i4b {

namespace {

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

template <bool F16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {  // round to nearest even
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// n / page_size for n < 2^31, by multiplication (page sizes need not be powers of two).
__device__ __forceinline__ int page_of(const PagedCache& c, int n) {
  return int(__umulhi(uint32_t(n), c.ps_mul) >> c.ps_shift);
}

// The page that holds position `pos` of sequence b, or -1: an entry outside the pool holds nothing.
__device__ __forceinline__ int page_entry(const PagedCache& c, const int32_t* row, int idx) {
  const int p = __ldg(row + idx);
  return uint32_t(p) < uint32_t(c.num_pages) ? p : -1;
}

// ------------------------------------------------------------------ append

// One CTA per token; a thread owns 8 dims of the head's first half and the matching 8 of the second (two 16-byte
// loads), so that rotate_half needs no exchange.  Rotation in fp32, rounded once.  Bound by bytes: every value is
// read once and written once; the token's row of the two tables comes from L1 after the first head.
template <bool F16, bool T32, int HD>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedCache c, const uint16_t* __restrict__ qkv,
                                                           int64_t sqkv, const void* __restrict__ cosT,
                                                           const void* __restrict__ sinT, int max_pos,
                                                           const int32_t* __restrict__ positions,
                                                           const int32_t* __restrict__ slots,
                                                           const int32_t* __restrict__ seqs,
                                                           uint16_t* __restrict__ q_out, int nq) {
  constexpr int TPH = HD / 16;  // threads per head
  const int64_t tok = blockIdx.x;
  const int p = positions[tok], slot = slots[tok], seq = seqs ? seqs[tok] : int(tok);
  const bool rot_ok = uint32_t(p) < uint32_t(max_pos);
  int page = -1, row = 0;
  if (uint32_t(seq) < uint32_t(c.seqs) && uint32_t(slot) < uint32_t(c.capacity)) {
    const int pi = page_of(c, slot);
    page = page_entry(c, c.table + int64_t(seq) * c.table_stride, pi);
    row = slot - pi * c.page_size;
  }
  if (!rot_ok) page = -1;
  const int heads = nq + 2 * c.kv_heads;
  const uint16_t* src0 = qkv + tok * sqkv;
  for (int i = threadIdx.x; i < heads * TPH; i += blockDim.x) {
    const int h = i / TPH, ch = i % TPH;
    const uint16_t* src = src0 + int64_t(h) * HD + 8 * ch;
    uint4 x0 = __ldg(reinterpret_cast<const uint4*>(src));
    uint4 x1 = __ldg(reinterpret_cast<const uint4*>(src + HD / 2));
    uint16_t* dst;
    if (h >= nq + c.kv_heads) {
      if (page < 0) continue;
      dst = c.v + page * c.vs_page + int64_t(h - nq - c.kv_heads) * c.vs_head + int64_t(row) * c.vs_token + 8 * ch;
    } else {
      if (h >= nq) {
        if (page < 0) continue;
        dst = c.k + page * c.ks_page + int64_t(h - nq) * c.ks_head + int64_t(row) * c.ks_token + 8 * ch;
      } else {
        dst = q_out + (tok * nq + h) * HD + 8 * ch;
      }
      if (!rot_ok) {  // a position without an angle: the query is zero, nothing is cached
        x0 = x1 = make_uint4(0u, 0u, 0u, 0u);
      } else {
        float co0[8], co1[8], si0[8], si1[8];
        if constexpr (T32) {
          const float* cp = static_cast<const float*>(cosT) + int64_t(p) * HD + 8 * ch;
          const float* sp = static_cast<const float*>(sinT) + int64_t(p) * HD + 8 * ch;
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            *reinterpret_cast<float4*>(co0 + e) = __ldg(reinterpret_cast<const float4*>(cp + e));
            *reinterpret_cast<float4*>(co1 + e) = __ldg(reinterpret_cast<const float4*>(cp + HD / 2 + e));
            *reinterpret_cast<float4*>(si0 + e) = __ldg(reinterpret_cast<const float4*>(sp + e));
            *reinterpret_cast<float4*>(si1 + e) = __ldg(reinterpret_cast<const float4*>(sp + HD / 2 + e));
          }
        } else {
          const uint16_t* cp = static_cast<const uint16_t*>(cosT) + int64_t(p) * HD + 8 * ch;
          const uint16_t* sp = static_cast<const uint16_t*>(sinT) + int64_t(p) * HD + 8 * ch;
          const uint4 a = __ldg(reinterpret_cast<const uint4*>(cp)), b = __ldg(reinterpret_cast<const uint4*>(cp + HD / 2));
          const uint4 d = __ldg(reinterpret_cast<const uint4*>(sp)), f = __ldg(reinterpret_cast<const uint4*>(sp + HD / 2));
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            *reinterpret_cast<float2*>(co0 + 2 * w) = unpack2<F16>(reinterpret_cast<const uint32_t*>(&a)[w]);
            *reinterpret_cast<float2*>(co1 + 2 * w) = unpack2<F16>(reinterpret_cast<const uint32_t*>(&b)[w]);
            *reinterpret_cast<float2*>(si0 + 2 * w) = unpack2<F16>(reinterpret_cast<const uint32_t*>(&d)[w]);
            *reinterpret_cast<float2*>(si1 + 2 * w) = unpack2<F16>(reinterpret_cast<const uint32_t*>(&f)[w]);
          }
        }
        uint32_t* a = reinterpret_cast<uint32_t*>(&x0);
        uint32_t* b = reinterpret_cast<uint32_t*>(&x1);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 u = unpack2<F16>(a[w]), v = unpack2<F16>(b[w]);
          a[w] = pack2<F16>(u.x * co0[2 * w] - v.x * si0[2 * w], u.y * co0[2 * w + 1] - v.y * si0[2 * w + 1]);
          b[w] = pack2<F16>(v.x * co1[2 * w] + u.x * si1[2 * w], v.y * co1[2 * w + 1] + u.y * si1[2 * w + 1]);
        }
      }
    }
    *reinterpret_cast<uint4*>(dst) = x0;
    *reinterpret_cast<uint4*>(dst + HD / 2) = x1;
  }
}

// ------------------------------------------------------------------ attention

// The cached positions of every (sequence, kv head, tile of 16 query heads) item are cut into tiles of 32; the
// items' tiles, one item behind the other, are dealt in equal consecutive runs to the grid's warps, each of which
// works by itself.  A run that holds an item whole writes its output; the pieces of an item that several runs share
// go to the workspace as (max, sum, unnormalised output) and paged_attn_join adds them in the runs' order.  The deal
// depends on the lengths alone, so results repeat bit by bit.
constexpr int kAttnWarps = 4;
constexpr int kAttnCtasPerSm = 2;
constexpr int kTile = 32;
constexpr int kMinTiles = 2;  // per warp: below this the join costs more than the split saves

// Tiles of sequence b before / in it, from the lengths; shared by the attention kernel and its join.
struct Deal {
  int H;      // items per sequence: kv heads x tiles of query heads
  int total;  // tiles of all items
  int per;    // tiles of a run
};

__device__ __forceinline__ int clamped_len(const PagedCache& c, const int32_t* lens, int b) {
  const int n = __ldg(lens + b);
  return n < 0 ? 0 : (n > c.capacity ? c.capacity : n);  // never reads past the table
}

__device__ __forceinline__ int run_tiles(int total, int workers) {
  const int per = (total + workers - 1) / workers;
  return per < kMinTiles ? kMinTiles : per;
}

struct Cursor {
  int b, h, tile, nt, len;
};

template <bool F16, int HD, bool TWO, bool WEIGHTS>
__global__ void __launch_bounds__(kAttnWarps * 32, kAttnCtasPerSm)
    paged_attn_kernel(const PagedCache c, const uint16_t* __restrict__ q, int64_t sqb, int64_t sqh,
                      const int32_t* __restrict__ lens, uint16_t* __restrict__ out, int nq, int HT, float scale_log2,
                      float* __restrict__ partials, float* __restrict__ logits, int64_t logit_stride,
                      float* __restrict__ ml) {
  constexpr int HC = HD / 32;              // 16-byte chunks of a key row that a lane owns
  constexpr int VC = HD / 64;              // 16-byte chunks of a value row that a lane owns
  constexpr int kHalf = kTile * HD * 2;    // bytes of a tile's keys (or values)
  constexpr int NB = 24576 / kHalf;        // halves in flight per warp
  constexpr int R = TWO ? 2 : 1;           // rows of 8 query heads
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int scan_tmp[kAttnWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint4* ring = reinterpret_cast<uint4*>(smem) + warp * (NB * kHalf / 16);
  int* pre = reinterpret_cast<int*>(smem + kAttnWarps * NB * kHalf);  // [B + 1] first tile of each sequence
  int* len = pre + c.seqs + 1;                                       // [B]
  const int H = c.kv_heads * HT, B = c.seqs, G = nq / c.kv_heads;

  // exclusive scan of the sequences' tiles
  {
    int base = 0;
    for (int b0 = 0; b0 < B; b0 += kAttnWarps * 32) {
      const int b = b0 + tid;
      const int L = b < B ? clamped_len(c, lens, b) : 0;
      int v = (L + kTile - 1) / kTile * H;
      const int own = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += u;
      }
      if (lane == 31) scan_tmp[warp] = v;
      __syncthreads();
      int add = base, all = 0;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        if (w < warp) add += scan_tmp[w];
        all += scan_tmp[w];
      }
      if (b < B) {
        pre[b] = add + v - own;
        len[b] = L;
      }
      base += all;
      __syncthreads();
    }
    if (tid == 0) pre[B] = base;
    __syncthreads();
  }
  const int total = pre[B];
  const int workers = int(gridDim.x) * kAttnWarps, worker = int(blockIdx.x) * kAttnWarps + warp;
  const int per = run_tiles(total, workers);
  const int64_t begin64 = int64_t(worker) * per;
  if (begin64 >= total) return;
  const int begin = int(begin64), ntiles = min(per, total - begin);

  Cursor cc;  // what is computed
  {
    int lo = 0, hi = B;  // pre[lo] <= begin < pre[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= begin) lo = mid; else hi = mid;
    }
    cc.b = lo;
    cc.len = len[lo];
    cc.nt = (cc.len + kTile - 1) / kTile;
    const int off = begin - pre[lo];
    cc.h = off / cc.nt;
    cc.tile = off - cc.h * cc.nt;
  }
  auto advance = [&](Cursor& x) {
    if (++x.tile < x.nt) return;
    x.tile = 0;
    if (++x.h < H) return;
    x.h = 0;
    do ++x.b;
    while (x.b < B && len[x.b] == 0);
    if (x.b < B) {
      x.len = len[x.b];
      x.nt = (x.len + kTile - 1) / kTile;
    }
  };

  // ---- loads: lane (g, t) copies for itself the keys 4g..4g+3, chunks t + 4h, and the values of positions
  // 8t..8t+7, chunks g + 8c: exactly the words its MMA fragments need, so no lane waits for another.
  Cursor ic = cc;  // what is requested
  int iu = 0, islot = 0;
  int kp = -1, vp = -1, krow = 0, vrow = 0;
  uint32_t vok = 0;  // bit n % 32: whether tile n's value page is there
  auto fetch_pages = [&]() {
    const int32_t* trow = c.table + int64_t(ic.b) * c.table_stride;
    const int kpos = ic.tile * kTile + 4 * g, vpos = ic.tile * kTile + 8 * t;
    kp = vp = -1;
    if (kpos < ic.len) {
      const int pi = page_of(c, kpos);
      krow = kpos - pi * c.page_size;
      kp = page_entry(c, trow, pi);
    }
    if (vpos < ic.len) {
      const int pi = page_of(c, vpos);
      vrow = vpos - pi * c.page_size;
      vp = page_entry(c, trow, pi);
    }
  };
  auto issue = [&]() {
    if (iu < 2 * ntiles) {
      uint4* dst = ring + islot * (kHalf / 16) + lane;
      const int kvh = HT == 1 ? ic.h : ic.h / HT;
      if ((iu & 1) == 0) {
        const int left = ic.len - (ic.tile * kTile + 4 * g);
        const uint16_t* src = c.k + int64_t(kp) * c.ks_page + int64_t(kvh) * c.ks_head + int64_t(krow) * c.ks_token + 8 * t;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool ok = kp >= 0 && j < left;
#pragma unroll
          for (int h = 0; h < HC; ++h)
            cp_async_16(dst + (j * HC + h) * 32, ok ? src + j * c.ks_token + 32 * h : c.k, ok ? 16u : 0u);
        }
      } else {
        const int left = ic.len - (ic.tile * kTile + 8 * t);
        const uint16_t* src = c.v + int64_t(vp) * c.vs_page + int64_t(kvh) * c.vs_head + int64_t(vrow) * c.vs_token + 8 * g;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool ok = vp >= 0 && j < left;  // rows behind the end arrive as zeros, whatever they hold
#pragma unroll
          for (int v = 0; v < VC; ++v)
            cp_async_16(dst + (j * VC + v) * 32, ok ? src + j * c.vs_token + 64 * v : c.v, ok ? 16u : 0u);
        }
        const uint32_t bit = 1u << ((iu >> 1) & 31);
        vok = vp >= 0 ? (vok | bit) : (vok & ~bit);
        if (iu + 1 < 2 * ntiles) {
          advance(ic);
          fetch_pages();
        }
      }
    }
    cp_async_commit();
    ++iu;
    islot = islot + 1 == NB ? 0 : islot + 1;
  };
  fetch_pages();
#pragma unroll
  for (int i = 0; i < NB; ++i) issue();

  uint32_t qa[2 * HC][4];
  float o[8 * VC][4], m[R], l[R];
  int cslot = 0, seg_first = 0, seg_tile0 = cc.tile;
  bool fresh = true;
  for (int n = 0; n < ntiles; ++n) {
    const int kvh = HT == 1 ? cc.h : cc.h / HT;
    const int head0 = kvh * G + (HT == 1 ? 0 : cc.h % HT) * 16;
    const int rows = min(16, kvh * G + G - head0);  // query heads of this item
    if (fresh) {
      fresh = false;
      const uint16_t* qr = q + int64_t(cc.b) * sqb + int64_t(head0) * sqh + 8 * t;
#pragma unroll
      for (int h = 0; h < HC; ++h) {
        uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
        if (g < rows) a = __ldg(reinterpret_cast<const uint4*>(qr + int64_t(g) * sqh + 32 * h));
        if (TWO && g + 8 < rows) b = __ldg(reinterpret_cast<const uint4*>(qr + int64_t(g + 8) * sqh + 32 * h));
        qa[2 * h][0] = a.x, qa[2 * h][2] = a.y, qa[2 * h + 1][0] = a.z, qa[2 * h + 1][2] = a.w;
        qa[2 * h][1] = b.x, qa[2 * h][3] = b.y, qa[2 * h + 1][1] = b.z, qa[2 * h + 1][3] = b.w;
      }
#pragma unroll
      for (int i = 0; i < 8 * VC; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r) m[r] = -INFINITY, l[r] = 0.0f;
    }
    // ---- scores: column n of block j is position 4n + j of the tile (as the keys were loaded)
    cp_async_wait<NB - 1>();
    float s[4][4];
    {
      const uint4* src = ring + cslot * (kHalf / 16) + lane;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int h = 0; h < HC; ++h) {
          const uint4 kf = src[(j * HC + h) * 32];
          if (h == 0)
            mma_16816_first<F16>(s[j], qa[0], kf.x, kf.y);
          else
            mma_16816<F16>(s[j], qa[2 * h], kf.x, kf.y);
          mma_16816<F16>(s[j], qa[2 * h + 1], kf.z, kf.w);
        }
      }
    }
    cslot = cslot + 1 == NB ? 0 : cslot + 1;
    issue();
    // ---- softmax over this tile; the lane's columns are positions 8t + j and 8t + 4 + j
    const int left = (vok >> (n & 31)) & 1u ? cc.len - (cc.tile * kTile + 8 * t) : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s[j][2 * r] = j < left ? s[j][2 * r] * scale_log2 : -INFINITY;
        s[j][2 * r + 1] = 4 + j < left ? s[j][2 * r + 1] * scale_log2 : -INFINITY;
      }
    if constexpr (WEIGHTS) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (g + 8 * r < rows) {
          float4* dst = reinterpret_cast<float4*>(logits + (int64_t(cc.b) * nq + head0 + g + 8 * r) * logit_stride +
                                                  cc.tile * kTile + 8 * t);
          dst[0] = make_float4(s[0][2 * r], s[1][2 * r], s[2][2 * r], s[3][2 * r]);
          dst[1] = make_float4(s[0][2 * r + 1], s[1][2 * r + 1], s[2][2 * r + 1], s[3][2 * r + 1]);
        }
    }
    bool grew = false;
    float mn[R], base[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mx = fmaxf(s[0][2 * r], s[0][2 * r + 1]);
#pragma unroll
      for (int j = 1; j < 4; ++j) mx = fmaxf(mx, fmaxf(s[j][2 * r], s[j][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
      mn[r] = fmaxf(m[r], mx);
      grew |= mn[r] > m[r];
      base[r] = mn[r] == -INFINITY ? 0.0f : mn[r];  // nothing seen yet: every probability is exp2(-inf) = 0
    }
    if (__any_sync(0xFFFFFFFFu, grew)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float f = ex2(m[r] - base[r]);  // m = -inf gives 0
        l[r] *= f;
        m[r] = mn[r];
#pragma unroll
        for (int i = 0; i < 8 * VC; ++i) o[i][2 * r] *= f, o[i][2 * r + 1] *= f;
      }
    }
    // probabilities; rounded to the values' type for the second product (half a step each, as the output is),
    // summed unrounded
    uint32_t pa[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t w = 0u;
        if (r < R) {
          const float p0 = ex2(s[j][2 * r] - base[r]), p1 = ex2(s[j][2 * r + 1] - base[r]);
          l[r] += p0 + p1;
          w = pack2<F16>(p0, p1);
        }
        pa[j >> 1][2 * (j & 1) + r] = w;
      }
    // ---- output: the pair (8t + j, 8t + 4 + j) of value rows meets the pair of probabilities of block j
    cp_async_wait<NB - 1>();
    {
      const uint4* src = ring + cslot * (kHalf / 16) + lane;
#pragma unroll
      for (int v = 0; v < VC; ++v)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint4 a0 = src[((2 * k) * VC + v) * 32], b0 = src[((2 * k + 4) * VC + v) * 32];
          const uint4 a1 = src[((2 * k + 1) * VC + v) * 32], b1 = src[((2 * k + 5) * VC + v) * 32];
          const uint32_t x0[4] = {a0.x, a0.y, a0.z, a0.w}, y0[4] = {b0.x, b0.y, b0.z, b0.w};
          const uint32_t x1[4] = {a1.x, a1.y, a1.z, a1.w}, y1[4] = {b1.x, b1.y, b1.z, b1.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            mma_16816<F16>(o[8 * v + 2 * w], pa[k], __byte_perm(x0[w], y0[w], 0x5410), __byte_perm(x1[w], y1[w], 0x5410));
            mma_16816<F16>(o[8 * v + 2 * w + 1], pa[k], __byte_perm(x0[w], y0[w], 0x7632), __byte_perm(x1[w], y1[w], 0x7632));
          }
        }
    }
    cslot = cslot + 1 == NB ? 0 : cslot + 1;
    issue();
    // ---- end of the item, or of this run
    if (cc.tile == cc.nt - 1 || n == ntiles - 1) {
      const bool whole = seg_tile0 == 0 && cc.tile == cc.nt - 1;
      float* part = partials + int64_t(2 * worker + (seg_first == 0 ? 0 : 1)) * (16 * (HD + 2));
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float ls = l[r] + __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
        ls += __shfl_xor_sync(0xFFFFFFFFu, ls, 2);
        if (g + 8 * r < rows) {
          if (whole) {
            const float inv = ls > 0.0f || ls != ls ? 1.0f / ls : 0.0f;  // no position: zeros (a NaN stays one)
            uint16_t* dst = out + (int64_t(cc.b) * nq + head0 + g + 8 * r) * HD;
#pragma unroll
            for (int v = 0; v < VC; ++v)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  w[i] = pack2<F16>(o[8 * v + 2 * i][2 * r + e] * inv, o[8 * v + 2 * i + 1][2 * r + e] * inv);
                *reinterpret_cast<uint4*>(dst + 8 * (2 * t + e + 8 * v)) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            if (WEIGHTS && t == 0)
              *reinterpret_cast<float2*>(ml + 2 * (int64_t(cc.b) * nq + head0 + g + 8 * r)) = make_float2(m[r], inv);
          } else {
            float* dst = part + (g + 8 * r) * HD;
#pragma unroll
            for (int v = 0; v < VC; ++v)
#pragma unroll
              for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                  *reinterpret_cast<float4*>(dst + 8 * (2 * t + e + 8 * v) + 4 * i) =
                      make_float4(o[8 * v + 4 * i][2 * r + e], o[8 * v + 4 * i + 1][2 * r + e],
                                  o[8 * v + 4 * i + 2][2 * r + e], o[8 * v + 4 * i + 3][2 * r + e]);
            if (t == 0) {
              part[16 * HD + 2 * (g + 8 * r)] = m[r];
              part[16 * HD + 2 * (g + 8 * r) + 1] = ls;
            }
          }
        }
      }
      fresh = true;
      seg_first = n + 1;
      seg_tile0 = 0;
    }
    advance(cc);
  }
  cp_async_wait<0>();
}

// One CTA per (sequence, query head): adds the pieces of an item that several runs share, in the runs' order, and
// writes zeros for an empty sequence.
template <bool F16, int HD>
__global__ void __launch_bounds__(128) paged_attn_join_kernel(const PagedCache c, const int32_t* __restrict__ lens,
                                                              uint16_t* __restrict__ out, int nq, int HT, int workers,
                                                              const float* __restrict__ partials,
                                                              float* __restrict__ ml) {
  constexpr int LX = HD / 4, SL = 128 / LX;  // float4 columns, slices over the pieces
  __shared__ int red[2][4];
  __shared__ float4 acc[SL][LX];
  __shared__ float accl[SL];
  const int b = blockIdx.y, head = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = nq / c.kv_heads, kvh = head / G, ht = (head % G) / 16, row = (head % G) % 16;
  const int H = c.kv_heads * HT;
  pdl_wait();
  int before = 0, total = 0;
  for (int i = tid; i < c.seqs; i += 128) {
    const int n = (clamped_len(c, lens, i) + kTile - 1) / kTile * H;
    total += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
    before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
  }
  if (lane == 0) red[0][warp] = total, red[1][warp] = before;
  __syncthreads();
  total = red[0][0] + red[0][1] + red[0][2] + red[0][3];
  before = red[1][0] + red[1][1] + red[1][2] + red[1][3];
  const int nt = (clamped_len(c, lens, b) + kTile - 1) / kTile;
  uint16_t* dst = out + (int64_t(b) * nq + head) * HD;
  if (nt == 0) {
    if (tid < HD / 2) reinterpret_cast<uint32_t*>(dst)[tid] = 0u;
    if (ml && tid == 0) *reinterpret_cast<float2*>(ml + 2 * (int64_t(b) * nq + head)) = make_float2(0.0f, 0.0f);
    return;
  }
  const int per = run_tiles(total, workers);
  const int t0 = before + (kvh * HT + ht) * nt, w0 = t0 / per, w1 = (t0 + nt - 1) / per;
  if (w0 == w1) return;  // written by the run itself
  const int first = 2 * w0 + (int64_t(w0) * per == t0 ? 0 : 1), pieces = w1 - w0 + 1;
  constexpr int64_t kPiece = 16 * (HD + 2);
  auto piece = [&](int i) { return partials + int64_t(i == 0 ? first : 2 * (w0 + i)) * kPiece; };
  const int x = tid % LX, s = tid / LX;
  float mx = -INFINITY;
  for (int i = 0; i < pieces; ++i) mx = fmaxf(mx, __ldcg(piece(i) + 16 * HD + 2 * row));
  const float base = mx == -INFINITY ? 0.0f : mx;
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
  for (int i = s; i < pieces; i += SL) {
    const float* p = piece(i);
    const float2 e = __ldcg(reinterpret_cast<const float2*>(p + 16 * HD + 2 * row));
    const float4 v = __ldcg(reinterpret_cast<const float4*>(p + row * HD + 4 * x));
    const float f = ex2(e.x - base);
    a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
    l = fmaf(e.y, f, l);
  }
  acc[s][x] = a;
  if (x == 0) accl[s] = l;
  __syncthreads();
  if (s != 0) return;
  for (int i = 1; i < SL; ++i) {
    const float4 v = acc[i][x];
    a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    l += accl[i];
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  *reinterpret_cast<uint2*>(dst + 4 * x) = make_uint2(pack2<F16>(a.x * inv, a.y * inv), pack2<F16>(a.z * inv, a.w * inv));
  if (ml && x == 0) *reinterpret_cast<float2*>(ml + 2 * (int64_t(b) * nq + head)) = make_float2(mx, inv);
}

// weights[b, kvh, j] += sum over the kv head's query heads of exp2(s_j - m) / l, from the stored scaled scores.
__global__ void __launch_bounds__(256) paged_attn_weights_kernel(const PagedCache c, const int32_t* __restrict__ lens,
                                                                 int nq, const float* __restrict__ logits,
                                                                 int64_t logit_stride, const float* __restrict__ ml,
                                                                 float* __restrict__ weights, int64_t swb, int64_t swh) {
  const int b = blockIdx.z, kvh = blockIdx.y, G = nq / c.kv_heads;
  pdl_wait();
  const int L = clamped_len(c, lens, b), j = 4 * (blockIdx.x * 256 + threadIdx.x);
  if (j >= L) return;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int r = 0; r < G; ++r) {
    const int64_t row = int64_t(b) * nq + kvh * G + r;
    const float2 e = __ldcg(reinterpret_cast<const float2*>(ml + 2 * row));
    const float4 s = __ldcg(reinterpret_cast<const float4*>(logits + row * logit_stride + j));
    const float base = e.x == -INFINITY ? 0.0f : e.x;
    sum.x = fmaf(ex2(s.x - base), e.y, sum.x);
    sum.y = fmaf(ex2(s.y - base), e.y, sum.y);
    sum.z = fmaf(ex2(s.z - base), e.y, sum.z);
    sum.w = fmaf(ex2(s.w - base), e.y, sum.w);
  }
  float* w = weights + b * swb + kvh * swh + j;
  const int n = min(4, L - j);
  w[0] += sum.x;
  if (n > 1) w[1] += sum.y;
  if (n > 2) w[2] += sum.z;
  if (n > 3) w[3] += sum.w;
}

// ------------------------------------------------------------------ eviction

// Weights as unsigned integers in the order of their values: NaN lowest, then -inf, ..., -0 = +0, ..., +inf.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0u;
  if (w == 0.0f) return 0x80000000u;
  const uint32_t u = __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;

// One CTA per (kv head, sequence): the order value of the `need`-th largest weight among the older positions by
// radix selection (four passes over 8 bits), then the kept positions in order.
__global__ void __launch_bounds__(kSelThreads) paged_evict_select_kernel(
    const float* weights, int64_t swb, int64_t swh, const int32_t* __restrict__ lens, int capacity, int budget,
    int recent, int32_t* __restrict__ new_lens, int32_t* __restrict__ kept, float* weights_out, int64_t sob,
    int64_t soh, int width) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t found[2];
  __shared__ uint32_t scan_tmp[32];
  const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* w = weights + b * swb + kvh * swh;
  float* wo = weights_out + b * sob + kvh * soh;
  int32_t* ko = kept + (int64_t(b) * gridDim.x + kvh) * budget;
  int L = __ldg(lens + b);
  L = L < 0 ? 0 : (L > capacity ? capacity : L);
  const int n = min(L, budget);
  if (kvh == 0 && tid == 0) new_lens[b] = n;
  const int old = L > budget ? L - recent : L;  // positions that compete
  uint32_t thr = 0u;
  uint32_t ties = 0u;  // how many of the positions at the threshold stay
  if (L > budget) {
    uint32_t need = uint32_t(budget - recent), mask = 0u;
    for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0u;
      __syncthreads();
      for (int i = tid; i < old; i += kSelThreads) {
        const uint32_t u = order_of(w[i]);
        if ((u & mask) == thr) atomicAdd(&hist[(u >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t above = 0u;
        int d = 255;
        for (; d > 0 && above + hist[d] < need; --d) above += hist[d];
        found[0] = uint32_t(d);
        found[1] = above;
      }
      __syncthreads();
      thr |= found[0] << shift;
      need -= found[1];
      mask |= 255u << shift;
      __syncthreads();
    }
    ties = need;
    if (budget == recent) thr = 0xFFFFFFFFu;  // nothing of the older positions stays (no weight has this value)
  }
  // kept positions in order: a scan over (ties before, kept before), both in one word pair
  uint32_t tie_base = 0u, kept_base = 0u;
  for (int i0 = 0; i0 < L; i0 += kSelThreads) {
    const int i = i0 + tid;
    float v = 0.0f;
    bool above = false, tie = false;
    if (i < L) {
      v = w[i];
      const uint32_t u = order_of(v);
      above = L <= budget || i >= old || u > thr;
      tie = !above && u == thr && ties > 0u;
    }
    const uint32_t bt = __ballot_sync(0xFFFFFFFFu, tie), below = (1u << lane) - 1u;
    if (lane == 0) scan_tmp[warp] = __popc(bt);
    __syncthreads();
    uint32_t tb = tie_base, tall = 0u;
    for (int k = 0; k < 32; ++k) {
      if (k < warp) tb += scan_tmp[k];
      tall += scan_tmp[k];
    }
    __syncthreads();
    const bool keep = above || (tie && tb + __popc(bt & below) < ties);
    const uint32_t bk = __ballot_sync(0xFFFFFFFFu, keep);
    if (lane == 0) scan_tmp[warp] = __popc(bk);
    __syncthreads();
    uint32_t kb = kept_base, kall = 0u;
    for (int k = 0; k < 32; ++k) {
      if (k < warp) kb += scan_tmp[k];
      kall += scan_tmp[k];
    }
    if (keep) {
      const uint32_t at = kb + __popc(bk & below);
      ko[at] = i;
      wo[at] = v;  // at <= i: in place, this position's weight and all later ones are read by now
    }
    tie_base += tall;
    kept_base += kall;
    __syncthreads();
  }
  for (int i = n + tid; i < budget; i += kSelThreads) ko[i] = -1;
  for (int i = n + tid; i < width; i += kSelThreads) wo[i] = 0.0f;
}

// Copies the kept rows into the new pages: a thread moves 16 bytes of keys and of values.
template <int HD>
__global__ void __launch_bounds__(256) paged_evict_copy_kernel(const PagedCache c, const int32_t* __restrict__ kept,
                                                               const int32_t* __restrict__ new_table,
                                                               int64_t new_stride, int budget) {
  constexpr int CH = HD / 8;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int i = (blockIdx.x * 256 + threadIdx.x) / CH, ch = threadIdx.x % CH;
  pdl_wait();
  if (i >= budget) return;
  const int pos = __ldcg(kept + (int64_t(b) * c.kv_heads + kvh) * budget + i);
  if (pos < 0) return;
  const int pi = page_of(c, pos), po = page_of(c, i);
  const int from = page_entry(c, c.table + int64_t(b) * c.table_stride, pi);
  const int to = page_entry(c, new_table + int64_t(b) * new_stride, po);
  if (to < 0) return;
  const int64_t r = pos - pi * c.page_size, ro = i - po * c.page_size;
  uint4 kk = make_uint4(0u, 0u, 0u, 0u), vv = kk;
  if (from >= 0) {
    kk = *reinterpret_cast<const uint4*>(c.k + from * c.ks_page + kvh * c.ks_head + r * c.ks_token + 8 * ch);
    vv = *reinterpret_cast<const uint4*>(c.v + from * c.vs_page + kvh * c.vs_head + r * c.vs_token + 8 * ch);
  }
  *reinterpret_cast<uint4*>(c.k + to * c.ks_page + kvh * c.ks_head + ro * c.ks_token + 8 * ch) = kk;
  *reinterpret_cast<uint4*>(c.v + to * c.vs_page + kvh * c.vs_head + ro * c.vs_token + 8 * ch) = vv;
}

// Launch that may start while its predecessor drains; the kernel waits (griddepcontrol.wait) before reading.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

template <bool F16, int HD, bool TWO, bool WEIGHTS>
cudaError_t attn(const PagedCache& c, const PagedAttn& a, const PagedAttnWorkspace& w, int sms, cudaStream_t s) {
  const int HT = (a.nq / c.kv_heads + 15) / 16;
  auto kern = paged_attn_kernel<F16, HD, TWO, WEIGHTS>;
  const size_t smem = size_t(kAttnWarps) * 24576 + (2 * size_t(c.seqs) + 1) * 4;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  const int ctas = sms * kAttnCtasPerSm;
  kern<<<ctas, kAttnWarps * 32, smem, s>>>(c, a.q, a.sqb, a.sqh, a.lens, a.out, a.nq, HT, a.scale * 1.4426950408889634f,
                                           w.partials, w.logits, w.logit_stride, w.ml);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  e = launch_after(paged_attn_join_kernel<F16, HD>, dim3(unsigned(a.nq), unsigned(c.seqs)), dim3(128), 0, s, c, a.lens,
                   a.out, a.nq, HT, ctas * kAttnWarps, static_cast<const float*>(w.partials), w.ml);
  if (e != cudaSuccess || !WEIGHTS || c.capacity == 0) return e;
  return launch_after(paged_attn_weights_kernel, dim3(unsigned((c.capacity + 1023) / 1024), unsigned(c.kv_heads), unsigned(c.seqs)),
                      dim3(256), 0, s, c, a.lens, a.nq, static_cast<const float*>(w.logits), w.logit_stride,
                      static_cast<const float*>(w.ml), a.weights, a.swb, a.swh);
}

template <bool F16, int HD>
cudaError_t attn_hd(const PagedCache& c, const PagedAttn& a, const PagedAttnWorkspace& w, int sms, cudaStream_t s) {
  const bool two = a.nq / c.kv_heads > 8;
  if (a.weights) return two ? attn<F16, HD, true, true>(c, a, w, sms, s) : attn<F16, HD, false, true>(c, a, w, sms, s);
  return two ? attn<F16, HD, true, false>(c, a, w, sms, s) : attn<F16, HD, false, false>(c, a, w, sms, s);
}

}  // namespace

void paged_set_page_size(PagedCache* c, int page_size) {
  int l = 0;
  while ((int64_t(1) << l) < page_size) ++l;
  c->page_size = page_size;
  c->ps_mul = uint32_t(((uint64_t(1) << (31 + l)) + page_size - 1) / uint64_t(page_size));
  c->ps_shift = l - 1;
}

size_t paged_attn_workspace(int seqs, int nq, int head_dim, int capacity, bool weights, int sms, void* base,
                            PagedAttnWorkspace* w) {
  const size_t pieces = size_t(sms) * kAttnCtasPerSm * kAttnWarps * 2;
  const size_t b0 = up256(pieces * 16 * (head_dim + 2) * 4);
  const int64_t stride = (int64_t(capacity) + kTile - 1) / kTile * kTile;
  const size_t b1 = weights ? up256(size_t(seqs) * nq * size_t(stride) * 4) : 0;
  const size_t b2 = weights ? up256(size_t(seqs) * nq * 8) : 0;
  if (w) {
    char* p = static_cast<char*>(base);
    w->partials = reinterpret_cast<float*>(p);
    w->logits = weights ? reinterpret_cast<float*>(p + b0) : nullptr;
    w->logit_stride = stride;
    w->ml = weights ? reinterpret_cast<float*>(p + b0 + b1) : nullptr;
  }
  return b0 + b1 + b2;
}

int64_t paged_attn_tiles(const PagedCache& c, int nq) {
  const int64_t ht = (nq / c.kv_heads + 15) / 16;
  return int64_t(c.seqs) * ((int64_t(c.capacity) + kTile - 1) / kTile) * c.kv_heads * ht;
}

cudaError_t launch_paged_attn(const PagedCache& c, const PagedAttn& a, const PagedAttnWorkspace& w, int sms,
                              cudaStream_t s) {
  if (c.f16) return c.head_dim == 64 ? attn_hd<true, 64>(c, a, w, sms, s) : attn_hd<true, 128>(c, a, w, sms, s);
  return c.head_dim == 64 ? attn_hd<false, 64>(c, a, w, sms, s) : attn_hd<false, 128>(c, a, w, sms, s);
}

cudaError_t launch_paged_append(const PagedCache& c, const uint16_t* qkv, int64_t sqkv, int64_t tokens, const void* cosT,
                                const void* sinT, bool table32, int max_pos, const int32_t* positions,
                                const int32_t* slots, const int32_t* seqs, uint16_t* q_out, int nq, cudaStream_t s) {
  const int threads = std::min(256, (((nq + 2 * c.kv_heads) * c.head_dim / 16) + 31) / 32 * 32);
  void (*kern)(const PagedCache, const uint16_t*, int64_t, const void*, const void*, int, const int32_t*, const int32_t*,
               const int32_t*, uint16_t*, int);
  if (c.head_dim == 64)
    kern = c.f16 ? (table32 ? paged_append_kernel<true, true, 64> : paged_append_kernel<true, false, 64>)
                 : (table32 ? paged_append_kernel<false, true, 64> : paged_append_kernel<false, false, 64>);
  else
    kern = c.f16 ? (table32 ? paged_append_kernel<true, true, 128> : paged_append_kernel<true, false, 128>)
                 : (table32 ? paged_append_kernel<false, true, 128> : paged_append_kernel<false, false, 128>);
  kern<<<unsigned(tokens), threads, 0, s>>>(c, qkv, sqkv, cosT, sinT, max_pos, positions, slots, seqs, q_out, nq);
  return cudaGetLastError();
}

cudaError_t launch_paged_evict(const PagedCache& c, const PagedEvict& e, cudaStream_t s) {
  paged_evict_select_kernel<<<dim3(unsigned(c.kv_heads), unsigned(c.seqs)), kSelThreads, 0, s>>>(
      e.weights, e.swb, e.swh, e.lens, std::min(c.capacity, e.width), e.budget, e.recent, e.new_lens, e.kept,
      e.weights_out, e.sob, e.soh, e.width);
  cudaError_t st = cudaGetLastError();
  if (st != cudaSuccess) return st;
  const int rows = 256 / (c.head_dim / 8);
  const dim3 grid(unsigned((e.budget + rows - 1) / rows), unsigned(c.kv_heads), unsigned(c.seqs));
  if (c.head_dim == 64)
    return launch_after(paged_evict_copy_kernel<64>, grid, dim3(256), 0, s, c, static_cast<const int32_t*>(e.kept),
                        e.new_table, e.new_stride, e.budget);
  return launch_after(paged_evict_copy_kernel<128>, grid, dim3(256), 0, s, c, static_cast<const int32_t*>(e.kept),
                      e.new_table, e.new_stride, e.budget);
}

}  // namespace i4b
