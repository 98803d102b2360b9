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

// 16 bytes global -> shared of data that is read once: the first to leave L2, so that what this kernel writes stays.
__device__ __forceinline__ uint64_t policy_evict_first() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void cp_async_once(void* dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "l"(policy)
               : "memory");
}

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

// The transpose of an 8 x 8 matrix of 16-bit values held two to a lane (row lane / 4, columns 2 (lane % 4) and + 1).
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
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

// A thread owns 8 dims of a head's first half and the matching 8 of the second (two 16-byte loads), so that
// rotate_half needs no exchange, for kHeads heads of one token, whose angles it reads once.  Rotation in fp32, rounded
// once.  Bound by bytes: every value is read once and written once, and a thread has all of its own in flight.
// 16381 tokens of 32 + 2 x 8 heads of 64 (206 MB; a plain copy of as much takes 34.9 us), heads per thread x threads:
// 6 x 128 34.8 us, 7 x 128 34.8, 6 x 256 36.1, 5 x 256 38.0, 4 x 256 41.1, 2 x 128 41.1, 8 x 128 43.9, 1 x 192 41.5.
constexpr int kAppendThreads = 128;
constexpr int kHeads = 6;

template <bool F16, bool T32, int HD>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(
    const PagedCache c, const uint16_t* __restrict__ qkv, int64_t sqkv, int64_t tokens, const void* __restrict__ cosT,
    const void* __restrict__ sinT, int max_pos, const int32_t* __restrict__ positions, const int32_t* __restrict__ slots,
    const int32_t* __restrict__ seqs, uint16_t* __restrict__ q_out, int nq, int per_token) {
  constexpr int TPH = HD / 16;  // threads per head
  const int64_t at = int64_t(blockIdx.x) * kAppendThreads + threadIdx.x, tok = at / per_token;
  if (tok >= tokens) return;
  const int unit = int(at - tok * per_token), ch = unit % TPH, h0 = unit / TPH, step = per_token / TPH;
  const int heads = nq + 2 * c.kv_heads;
  const int p = __ldg(positions + tok), slot = __ldg(slots + tok), seq = seqs ? __ldg(seqs + tok) : int(tok);
  const uint16_t* src0 = qkv + tok * sqkv + 8 * ch;
  uint4 x0[kHeads], x1[kHeads];
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    const int h = h0 + k * step;
    if (h < heads) {
      x0[k] = __ldg(reinterpret_cast<const uint4*>(src0 + int64_t(h) * HD));
      x1[k] = __ldg(reinterpret_cast<const uint4*>(src0 + int64_t(h) * HD + HD / 2));
    }
  }
  const bool rot_ok = uint32_t(p) < uint32_t(max_pos);
  float co0[8], co1[8], si0[8], si1[8];
  if (rot_ok) {
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
  }
  int page = -1, row = 0;
  if (rot_ok && uint32_t(seq) < uint32_t(c.seqs) && uint32_t(slot) < uint32_t(c.capacity)) {
    const int pi = page_of(c, slot);
    page = page_entry(c, c.table + int64_t(seq) * c.table_stride, pi);
    row = slot - pi * c.page_size;
  }
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    const int h = h0 + k * step;
    if (h >= heads) break;
    uint16_t* dst;
    if (h < nq)
      dst = q_out + (tok * nq + h) * HD + 8 * ch;
    else if (page < 0)
      continue;
    else if (h < nq + c.kv_heads)
      dst = c.k + page * c.ks_page + int64_t(h - nq) * c.ks_head + int64_t(row) * c.ks_token + 8 * ch;
    else
      dst = c.v + page * c.vs_page + int64_t(h - nq - c.kv_heads) * c.vs_head + int64_t(row) * c.vs_token + 8 * ch;
    if (!rot_ok) {  // a position without an angle: the query is zero, nothing is cached
      x0[k] = x1[k] = make_uint4(0u, 0u, 0u, 0u);
    } else if (h < nq + c.kv_heads) {
      uint32_t* a = reinterpret_cast<uint32_t*>(&x0[k]);
      uint32_t* b = reinterpret_cast<uint32_t*>(&x1[k]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 u = unpack2<F16>(a[w]), v = unpack2<F16>(b[w]);
        a[w] = pack2<F16>(u.x * co0[2 * w] - v.x * si0[2 * w], u.y * co0[2 * w + 1] - v.y * si0[2 * w + 1]);
        b[w] = pack2<F16>(v.x * co1[2 * w] + u.x * si1[2 * w], v.y * co1[2 * w + 1] + u.y * si1[2 * w + 1]);
      }
    }
    *reinterpret_cast<uint4*>(dst) = x0[k];
    *reinterpret_cast<uint4*>(dst + HD / 2) = x1[k];
  }
}

// ------------------------------------------------------------------ attention

// The cached positions of every (sequence, kv head, 16 query heads) item are cut into tiles; the items' tiles, one item
// behind the other, are cut into runs of consecutive tiles for the grid's warps, each of which works by itself.  A run
// that holds an item whole writes its output; the pieces of an item that several runs share go to the workspace as
// (max, sum, unnormalised output) and paged_attn_join adds them in the runs' order.  Where the runs begin depends on
// the lengths alone, so results repeat bit by bit, whichever warp takes which run.
//
// Every warp has one run of its own; when there is much to do, that is 5/8 of its share, and the rest lies in short
// runs that warps take from a counter: with equal shares alone the SMs, which do not see equal bandwidth, finished
// between 77 and 127 us (687 MB, mean 103).
// Both products are taken with the positions (or the head's dims) as the rows of the matrix instruction and the query
// heads as its 8 columns -- S^T = K Q^T, O^T = V^T P^T -- so that a group of 4 or 8 query heads fills half or all of
// it, not a quarter or half of 16 rows.  Between them P^T goes through an 8 x 8 transposition of registers.
//
// Bound by the bytes of K and V: the products are a few percent of what even mma.sync can do, so what counts is bytes
// in flight and whole 128-byte lines for each quarter of a warp.  Each warp keeps four units of 4 KB (two tiles' keys
// and values) on their way, in shared memory of its own: a quarter copies one row (or half of a 256-byte
// one), and the 16-byte words are placed so that neither that nor the reading of the MMA fragments meets a bank twice.
// (With every lane copying just the words of its own fragments, which needs no exchange, the values came in 32-byte
// pieces: 160 us against 129 for 687 MB at that stage.)
// Warps per CTA and CTAs per SM as measured (687 MB, fp16, head_dim 64; main kernel): 5 x 2 108 us, 7 x 1 107, 6 x 2 111,
// 8 x 1 110, 6 x 1 112, 4 x 2 122, 4 x 3 123, 10 x 1 127; on 74 MB 5 x 2 is the fastest too (17.0 us; 7 x 1 20.2).
constexpr int kAttnWarps = 5;
constexpr int kAttnCtas = 2;
constexpr int kUnit = 4096;  // bytes of a tile's keys, or values
constexpr int kUnits = 4;    // in flight per warp: keys and values of two tiles
constexpr int kMinTiles = 1;

// The probabilities enter the second product as the sum of two values of the cache's type, the rounded one and what that
// leaves; rounded once, they would be off as much as the output's own rounding is.  bf16 has fp32's exponents, both go
// into one sum.  fp16 ends at 2^-24: probabilities of 0 to 1 would lose what lies 17 below a row's largest score, all of
// the output where that slot's value is 0.  They are multiplied by 2^15 (1 becomes 32768), the rest, at most 8 there, by
// 2^11 once more and taken into a product of its own, added with 2^-11 for each tile: every probability within 2^-22 of
// itself, or within 2^-51.  (A second sum over the tiles would spill: the kernel is at its 168 registers.)  The factors
// are powers of two and leave the output before anything else sees it, so they round nothing.
constexpr float kP16 = 32768.0f, kRest16 = 2048.0f;

__host__ __device__ constexpr int attn_warp_smem(int head_dim, bool two) { return kUnits * kUnit + (two ? 2 : 1) * head_dim * 16; }

__host__ __device__ constexpr int tile_of(int head_dim) { return kUnit / 2 / head_dim; }  // 32 or 16 positions

// A piece of an item in the workspace: the outputs of its query heads, then (max, sum) of each; 16-byte aligned.
__host__ __device__ constexpr int piece_floats(int rows, int head_dim) { return rows * head_dim + (2 * rows + 3) / 4 * 4; }

__device__ __forceinline__ int clamped_len(const PagedCache& c, const int32_t* lens, int b) {
  const int n = __ldg(lens + b);
  return n < 0 ? 0 : (n > c.capacity ? c.capacity : n);  // never reads past the table
}

// How `total` tiles are cut into runs.  The first `workers` runs are the warps' own: of `own` tiles, the first `longer`
// of them of one more.  Where runs are shared, those of `more` tiles follow, and for the end ones of `last`: 2 tiles
// (16 KB), or as many as make a run 8 times its piece in the workspace.  Runs are shared from 8 `last` per warp on.
__host__ __device__ constexpr int last_tiles(int rows, int head_dim) {
  const int n = rows * head_dim * 4 * 8 / (2 * kUnit);
  return n < 2 ? 2 : n;
}

// Where the tables hold at most this many tiles per sequence a run is one item and there is nothing to join: one launch
// less (2.7 us of the host's time, 3.4 us of the device's) against 8 tiles by one warp.
constexpr int kWholeTiles = 8;

struct Deal {
  int total, workers, last, own, longer, more, long_end, more_end, more_runs;  // tiles: end of the own runs' longer ones, of ...
  __device__ Deal(int total_, int workers_, bool shared, int last_) : total(total_), workers(workers_), last(last_) {
    const int per = total / workers;
    if (shared && per >= 8 * last) {
      own = per * 5 / 8;
      longer = 0;
      more = max(2 * last, per / 8);
      more_runs = (total - workers * own - last * workers + more - 1) / more;  // (the last may end with the tiles)
    } else {
      own = max(per, kMinTiles);
      longer = per >= kMinTiles ? total - workers * per : 0;
      more = more_runs = 0;
    }
    long_end = longer * (own + 1);
    more_end = workers * own + longer + more_runs * more;
  }
  __device__ int64_t first(int r) const {
    if (r < workers) return int64_t(r) * own + min(r, longer);
    r -= workers;
    return r < more_runs ? int64_t(workers) * own + longer + int64_t(r) * more : more_end + last * int64_t(r - more_runs);
  }
  __device__ int tiles(int r) const {
    const int n = r < workers ? own + (r < longer ? 1 : 0) : (more == 0 ? 0 : (r < workers + more_runs ? more : last));
    return int(min(int64_t(n), total - first(r)));
  }
  __device__ int run_of(int tile) const {
    if (tile < long_end) return tile / (own + 1);
    if (tile < int64_t(workers) * own + longer) return longer + (tile - long_end) / own;
    if (tile < more_end) return workers + (tile - workers * own - longer) / more;
    return workers + more_runs + (tile - more_end) / last;
  }
};

// Runs per worker that a Deal makes at most: its own, (3/8 per + 2) / max(2 last, per / 8) < 4 and just over 1 at the end.
constexpr int kMostRuns = 7;

template <bool F16, int HD, bool TWO, bool WEIGHTS, bool WHOLE>
__global__ void __launch_bounds__(kAttnWarps * 32, kAttnCtas)
    paged_attn_kernel(const PagedCache c, const uint16_t* __restrict__ q, int64_t sqb, int64_t sqh,
                      const int32_t* __restrict__ lens, uint16_t* __restrict__ out, int nq, int HT, float scale_log2,
                      float* __restrict__ partials, float* __restrict__ logits, int64_t logit_stride,
                      float* __restrict__ ml, int* __restrict__ counter, int* __restrict__ starts) {
  constexpr int KT = tile_of(HD);         // positions of a tile
  constexpr int KI = KT / 16, KR = KT / 8; // blocks of 16 positions; key rows that a lane owns
  constexpr int HC = HD / 32;              // 16-byte chunks of a key row that a lane uses: t + 4h
  constexpr int VC = HD / 64;              // 16-byte chunks of a value row that a lane uses: g + 8v
  constexpr int R = TWO ? 2 : 1;           // blocks of 8 query heads
  static_assert(KR <= 4, "a lane's 2 KR value rows lie in one page: pages are multiples of 8");
  // Row r of block i is position KR * (r % 8) + KI * (r / 8) + i of the tile: lane (g, t) uses the KR consecutive key
  // rows from KR * g (rows g and g + 8 of every block) and the 2 KR value rows from 2 KR * t (k = 2t, 2t + 1, 2t + 8,
  // 2t + 9 of every block).  Key word (row j, chunk t + 4h) of lane (g, t) lies at 32 (HC j + h) + ((4g + t) ^ 4 (h & 1)),
  // value word (row j, chunk g + 8v) at 32 (VC j + v) + 8t + (g ^ 2t).
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int scan_tmp[kAttnWarps], queue[kAttnWarps][4][4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  constexpr int kWarpSmem = attn_warp_smem(HD, TWO);
  uint4* ring = reinterpret_cast<uint4*>(smem + warp * kWarpSmem);           // keys, keys, values, values, queries
  int* pre = reinterpret_cast<int*>(smem + kAttnWarps * kWarpSmem);  // [B + 1] first tile of each sequence
  int* len = pre + c.seqs + 1;                                            // [B]
  const int H = c.kv_heads * HT, B = c.seqs, G = nq / c.kv_heads;

  if (WHOLE) {
    for (int b = tid; b < B; b += kAttnWarps * 32) len[b] = clamped_len(c, lens, b);
    __syncthreads();
  } else {  // exclusive scan of the sequences' tiles
    int base = 0;
    for (int b0 = 0; b0 < B; b0 += kAttnWarps * 32) {
      const int b = b0 + tid;
      const int L = b < B ? clamped_len(c, lens, b) : 0;
      int v = (L + KT - 1) / KT * H;
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
  if (blockIdx.x == 0 && !WHOLE)
    for (int b = tid; b <= B; b += kAttnWarps * 32) starts[b] = pre[b];  // for the join
  const int worker = int(blockIdx.x) * kAttnWarps + warp;
  const Deal deal(WHOLE ? 0 : pre[B], int(gridDim.x) * kAttnWarps, counter != nullptr, last_tiles(min(16, G), HD));

  struct Item {
    int b, h, len, nt;  // sequence; kv head and tile of query heads; the sequence's length and tiles
  };
  auto next_item = [&](Item& x) {
    if (++x.h < H) return;
    x.h = 0;
    do ++x.b;
    while (x.b < B && len[x.b] == 0);
    if (x.b < B) {
      x.len = len[x.b];
      x.nt = (x.len + KT - 1) / KT;
    }
  };

  // ---- requests.  A tile's keys and values are requested as soon as those two tiles before have been used; its page
  // number is read half a tile before that, and an item's queries come with its first keys.
  Item ri = {};          // the item being requested, its tile, and what is the same for all its tiles
  int rtile, rleft = 0;  // and the tiles left in the run
  const int32_t* rtable;
  const uint16_t *rk, *rv;
  int items = 0, used = 0, held = 0, asked = 0;  // items requested, computed; whose queries are in shared memory, asked for
  auto enter = [&]() {
    const int kvh = HT == 1 ? ri.h : ri.h / HT;
    rtable = c.table + int64_t(ri.b) * c.table_stride;
    rk = c.k + kvh * c.ks_head + 8 * (lane & 7);
    rv = c.v + kvh * c.vs_head + 8 * (lane & 7);
    ++items;
  };
  int ahead = 0;            // (lane 0) the short run that this warp takes next
  auto take = [&](int r) {  // begin to request run r (or, of whole items, the first from there that is not empty), if there is one
    if constexpr (WHOLE) {
      rleft = 0;
      for (; r < B * H; r += deal.workers) {
        ri.b = r / H;
        ri.h = r - ri.b * H;
        ri.len = len[ri.b];
        rleft = ri.nt = (ri.len + KT - 1) / KT;
        rtile = 0;
        ahead = r + deal.workers;
        if (rleft > 0) {
          enter();
          return;
        }
        const int kvh = HT == 1 ? ri.h : ri.h / HT, head0 = kvh * G + (HT == 1 ? 0 : ri.h % HT) * 16;
        const int64_t at = int64_t(ri.b) * nq + head0;
        const int rows = min(16, kvh * G + G - head0);
        for (int i = lane; i < rows * (HD / 8); i += 32) reinterpret_cast<uint4*>(out + at * HD)[i] = make_uint4(0u, 0u, 0u, 0u);
        if (WEIGHTS && lane < rows) *reinterpret_cast<float2*>(ml + 2 * (at + lane)) = make_float2(0.0f, 0.0f);
      }
      return;
    }
    rleft = deal.tiles(r);
    if (rleft <= 0) return;
    if (deal.more > 0 && lane == 0) ahead = deal.workers + atomicAdd(counter, 1);
    const int begin = int(deal.first(r));
    int lo = 0, hi = B;  // pre[lo] <= begin < pre[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= begin) lo = mid; else hi = mid;
    }
    ri.b = lo;
    ri.len = len[lo];
    ri.nt = (ri.len + KT - 1) / KT;
    const int off = begin - pre[lo];
    ri.h = off / ri.nt;
    rtile = off - ri.h * ri.nt;
    enter();
  };
  take(worker);
  if (rleft <= 0) return;
  Item ci = ri;  // the item being computed, its tile, the tiles left in its run, and the run
  int ctile = rtile, cleft = rleft, run = worker, taken = 0, entered = 0;
  // this lane copies chunk lane % 8 (+ 8y) of rows 2 KR (lane / 8) + j, j < 2 KR, keys and values alike: one page
  const int lq = lane >> 3, l8 = lane & 7;
  const int kdst = 32 * (l8 >> 2) + 8 * lq + ((l8 & 3) ^ (4 * (l8 >> 2))), vdst = 8 * lq + (l8 ^ (2 * lq));
  const uint64_t once = policy_evict_first();
  int requested = 0;  // tiles whose keys were requested
  int page = -1, row = 0;
  auto fetch_page = [&]() {
    page = -1;
    const int pos = rtile * KT + 2 * KR * lq;
    if (rleft > 0 && pos < ri.len) {
      const int pi = page_of(c, pos);
      row = pos - pi * c.page_size;
      page = __ldg(rtable + pi);
    }
  };
  const uint16_t* vsrc = nullptr;  // the first of the rows of the tile whose values are requested next
  int left = 0;                    // how many of them exist
  uint32_t flags = 0;  // two bits for each of the last tiles (x & 7): every position there; the page of key rows KR g there
  auto request_keys = [&](uint4* dst) {
    __syncwarp();  // the slot has been read by every lane
    if (rleft > 0) {
      const bool ok = uint32_t(page) < uint32_t(c.num_pages);
      const uint32_t oks = __ballot_sync(0xFFFFFFFFu, ok);
      const bool full = (rtile + 1) * KT <= ri.len && oks == 0xFFFFFFFFu;
      const int sh = (requested & 7) * 2;
      flags = (flags & ~(3u << sh)) | ((full ? 1u : 0u) | (oks >> (8 * (g >> 1)) & 1u) << 1) << sh;
      vsrc = rv + page * c.vs_page + int64_t(row) * c.vs_token;
      left = ok ? ri.len - (rtile * KT + 2 * KR * lq) : 0;
      const uint16_t* src = rk + page * c.ks_page + int64_t(row) * c.ks_token;
      if (full) {
#pragma unroll
        for (int j = 0; j < 2 * KR; ++j, src += c.ks_token)
#pragma unroll
          for (int y = 0; y < HC / 2; ++y)
            cp_async_once(dst + 32 * (HC * (j % KR) + 2 * y) + (kdst ^ (4 * (j / KR))), src + 64 * y, once);
      } else {
#pragma unroll 1
        for (int j = 0; j < 2 * KR; ++j, src += c.ks_token)
#pragma unroll
          for (int y = 0; y < HC / 2; ++y)
            cp_async_16(dst + 32 * (HC * (j % KR) + 2 * y) + (kdst ^ (4 * (j / KR))), j < left ? src + 64 * y : c.k,
                        j < left ? 16u : 0u);
      }
      if (asked != items) {  // the item's first tile here: its queries too, unless the place still waits for its reader
        asked = items;
        if (held <= used) {
          held = items;
          const int kvh = HT == 1 ? ri.h : ri.h / HT, head0 = kvh * G + (HT == 1 ? 0 : ri.h % HT) * 16;
          const int rows = min(16, kvh * G + G - head0);
          const uint16_t* qr = q + int64_t(ri.b) * sqb + int64_t(head0 + g) * sqh + 8 * t;
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < HC; ++h) {
              const bool there = g + 8 * r < rows;
              cp_async_16(ring + kUnits * (kUnit / 16) + (r * HC + h) * 32 + lane, there ? qr + 8 * r * sqh + 32 * h : q,
                          there ? 16u : 0u);
            }
        }
      }
      ++requested;
      ++rtile;
      if (--rleft == 0) {
        if (deal.more > 0 || WHOLE) {  // left for the computation, two tiles behind: at most three runs wait there
          const int r = __shfl_sync(0xFFFFFFFFu, ahead, 0);
          take(r);
          if (lane == 0) {
            int* to = queue[warp][taken & 3];
            to[0] = rleft > 0 ? r : -1;
            to[1] = ri.b, to[2] = ri.h, to[3] = rtile;
          }
          ++taken;
        }
      } else if (rtile == ri.nt) {
        rtile = 0;
        next_item(ri);
        enter();
      }
    }
    cp_async_commit();
  };
  auto request_values = [&](uint4* dst, int x) {  // of tile x
    __syncwarp();
    if (x < requested) {
      const uint16_t* src = vsrc;
      if (flags >> ((x & 7) * 2) & 1u) {
#pragma unroll
        for (int j = 0; j < 2 * KR; ++j, src += c.vs_token)
#pragma unroll
          for (int v = 0; v < VC; ++v) cp_async_once(dst + 32 * (VC * j + v) + vdst, src + 64 * v, once);
      } else {
#pragma unroll 1
        for (int j = 0; j < 2 * KR; ++j, src += c.vs_token)
#pragma unroll
          for (int v = 0; v < VC; ++v)  // rows that do not exist arrive as zeros, whatever they hold
            cp_async_16(dst + 32 * (VC * j + v) + vdst, j < left ? src + 64 * v : c.v, j < left ? 16u : 0u);
      }
    }
    cp_async_commit();
  };
  constexpr int kSlot = kUnit / 16;
  fetch_page();
  request_keys(ring);
  request_values(ring + 2 * kSlot, 0);
  fetch_page();
  request_keys(ring + kSlot);
  request_values(ring + 3 * kSlot, 1);
  fetch_page();

  const int prows = min(16, G), piece = piece_floats(prows, HD);
  // A negative scale turns the queries' signs instead, so that the largest product has the largest score.
  const uint32_t flip = scale_log2 < 0.0f ? 0x80008000u : 0u;
  const float scl = fabsf(scale_log2);
  uint32_t qb[R][2 * HC][2];
  float o[R][4 * VC][4], m[R][2], l[R][2];  // of heads 2t and 2t + 1 of each block of 8
  int seg_tile0 = ctile;
  bool fresh = true, first_seg = true;  // of its run
  for (int n = 0;; ++n) {
    // ---- scores
    cp_async_wait<kUnits - 1>();
    __syncwarp();
    if (fresh) {
      fresh = false;
      const int kvh = HT == 1 ? ci.h : ci.h / HT, head0 = kvh * G + (HT == 1 ? 0 : ci.h % HT) * 16;
      const int rows = min(16, kvh * G + G - head0);  // query heads of this item
      const uint16_t* qr = q + int64_t(ci.b) * sqb + int64_t(head0) * sqh + 8 * t;
      const bool here = held == ++used;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int h = 0; h < HC; ++h) {
          uint4 a = make_uint4(0u, 0u, 0u, 0u);
          if (here)
            a = ring[kUnits * kSlot + (r * HC + h) * 32 + lane];
          else if (g + 8 * r < rows)
            a = __ldg(reinterpret_cast<const uint4*>(qr + int64_t(g + 8 * r) * sqh + 32 * h));
          qb[r][2 * h][0] = a.x ^ flip, qb[r][2 * h][1] = a.y ^ flip;
          qb[r][2 * h + 1][0] = a.z ^ flip, qb[r][2 * h + 1][1] = a.w ^ flip;
        }
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < 4 * VC; ++i) o[r][i][0] = o[r][i][1] = o[r][i][2] = o[r][i][3] = 0.0f;
        m[r][0] = m[r][1] = -INFINITY, l[r][0] = l[r][1] = 0.0f;
      }
    }
    float s[R][KI][4];  // rows g, g, g + 8, g + 8 of block i; heads 2t, 2t + 1, 2t, 2t + 1
    {
      const uint4* src = ring + (n & 1) * kSlot;
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int h = 0; h < HC; ++h) {
          const uint4 x = src[(i * HC + h) * 32 + (lane ^ (4 * (h & 1)))], y = src[((KI + i) * HC + h) * 32 + (lane ^ (4 * (h & 1)))];
          const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (h == 0)
              mma_16816_first<F16>(s[r][i], a0, qb[r][0][0], qb[r][0][1]);
            else
              mma_16816<F16>(s[r][i], a0, qb[r][2 * h][0], qb[r][2 * h][1]);
            mma_16816<F16>(s[r][i], a1, qb[r][2 * h + 1][0], qb[r][2 * h + 1][1]);
          }
        }
    }
    request_keys(ring + (n & 1) * kSlot);
    // ---- softmax; the lane's scores are those of its key rows KR * g + KI * e + i, entries [i][2 * e + head]
    const uint32_t f = flags >> ((n & 7) * 2);
    if (!(f & 1u)) {
      const int there = f >> 1 & 1u ? ci.len - (ctile * KT + KR * g) : 0;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < KI; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (KI * e + i >= there) s[r][i][2 * e] = s[r][i][2 * e + 1] = -INFINITY;
    }
    // The running maximum m: only when a score of the tile passes it (the lanes vote) is it found over the lanes, and
    // what is summed so far scaled.  No probability exceeds 1.
    bool grew = false;
    float mx[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        mx[r][u] = fmaxf(s[r][0][u], s[r][0][2 + u]);
#pragma unroll
        for (int i = 1; i < KI; ++i) mx[r][u] = fmaxf(mx[r][u], fmaxf(s[r][i][u], s[r][i][2 + u]));
        grew |= mx[r][u] * scl > m[r][u];
      }
    if (__any_sync(0xFFFFFFFFu, grew)) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float v = mx[r][u];
          v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 16));
          v = fmaxf(m[r][u], v == -INFINITY ? v : v * scl);
          const float k = v == -INFINITY ? 1.0f : ex2(m[r][u] - v);  // 0 for a head's first score
          m[r][u] = v;
          l[r][u] *= k;
#pragma unroll
          for (int i = 0; i < 4 * VC; ++i) o[r][i][u] *= k, o[r][i][2 + u] *= k;
        }
    }
    if constexpr (WEIGHTS) {
      const int kvh = HT == 1 ? ci.h : ci.h / HT, head0 = kvh * G + (HT == 1 ? 0 : ci.h % HT) * 16;
      const int rows = min(16, kvh * G + G - head0);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (2 * t + u + 8 * r < rows) {
            float* dst = logits + (int64_t(ci.b) * nq + head0 + 2 * t + u + 8 * r) * logit_stride + ctile * KT + KR * g;
            float w[KR];
#pragma unroll
            for (int i = 0; i < KR; ++i) {
              const float x = s[r][i % KI][2 * (i / KI) + u];
              w[i] = x == -INFINITY ? x : x * scl;
            }
            if constexpr (KR == 2) {
              *reinterpret_cast<float2*>(dst) = make_float2(w[0], w[1]);
            } else {
#pragma unroll
              for (int i = 0; i < KR; i += 4)
                *reinterpret_cast<float4*>(dst + i) = make_float4(w[i], w[i + 1], w[i + 2], w[i + 3]);
            }
          }
    }
    // probabilities, each as two values of the cache's type
    uint32_t pb[R][KI][2], pc[R][KI][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float n0 = m[r][0] == -INFINITY ? 0.0f : -m[r][0], n1 = m[r][1] == -INFINITY ? 0.0f : -m[r][1];
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x0 = s[r][i][2 * e], x1 = s[r][i][2 * e + 1];
          // rounded before the difference, as m and the stored scores are: the largest is exactly 2^0 however large it is
          float p0 = ex2(__fadd_rn(__fmul_rn(x0, scl), n0)), p1 = ex2(__fadd_rn(__fmul_rn(x1, scl), n1));
          if (!(f & 1u)) {  // (a scale of 0 would make a NaN of a place that is not there)
            p0 = x0 == -INFINITY ? 0.0f : p0;
            p1 = x1 == -INFINITY ? 0.0f : p1;
          }
          l[r][0] += p0, l[r][1] += p1;
          if constexpr (F16) p0 *= kP16, p1 *= kP16;
          const uint32_t w = pack2<F16>(p0, p1);
          const float2 back = unpack2<F16>(w);
          pb[r][i][e] = transpose8(w);
          const float u = F16 ? kRest16 : 1.0f;
          pc[r][i][e] = transpose8(pack2<F16>((p0 - back.x) * u, (p1 - back.y) * u));
        }
    }
    // ---- output: dims 8(g + 8v) + 2w and + 2w + 1 are rows g and g + 8 of block 4v + w
    cp_async_wait<kUnits - 1>();
    __syncwarp();
    {
      const uint4* src = ring + (2 + (n & 1)) * kSlot + 8 * t + (g ^ (2 * t));
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        float rest[R][4][4];
#pragma unroll
        for (int i = 0; i < KI; ++i) {
          const uint4 a = src[(i * VC + v) * 32], b = src[((KR + i) * VC + v) * 32];
          const uint4 d = src[((KI + i) * VC + v) * 32], e = src[((KR + KI + i) * VC + v) * 32];
          const uint32_t x0[4] = {a.x, a.y, a.z, a.w}, y0[4] = {b.x, b.y, b.z, b.w};
          const uint32_t x1[4] = {d.x, d.y, d.z, d.w}, y1[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t va[4] = {__byte_perm(x0[w], y0[w], 0x5410), __byte_perm(x0[w], y0[w], 0x7632),
                                    __byte_perm(x1[w], y1[w], 0x5410), __byte_perm(x1[w], y1[w], 0x7632)};
#pragma unroll
            for (int r = 0; r < R; ++r) {
              mma_16816<F16>(o[r][4 * v + w], va, pb[r][i][0], pb[r][i][1]);
              if constexpr (!F16)
                mma_16816<F16>(o[r][4 * v + w], va, pc[r][i][0], pc[r][i][1]);
              else if (i == 0)
                mma_16816_first<F16>(rest[r][w], va, pc[r][i][0], pc[r][i][1]);
              else
                mma_16816<F16>(rest[r][w], va, pc[r][i][0], pc[r][i][1]);
            }
          }
        }
        if constexpr (F16) {
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[r][4 * v + w][j] = fmaf(rest[r][w][j], 1.0f / kRest16, o[r][4 * v + w][j]);
        }
      }
    }
    request_values(ring + (2 + (n & 1)) * kSlot, n + 2);
    fetch_page();
    // ---- end of the item, or of this run
    --cleft;
    if (ctile == ci.nt - 1 || cleft == 0) {
      const int kvh = HT == 1 ? ci.h : ci.h / HT, head0 = kvh * G + (HT == 1 ? 0 : ci.h % HT) * 16;
      const int rows = min(16, kvh * G + G - head0);
      const bool whole = seg_tile0 == 0 && ctile == ci.nt - 1;
      if constexpr (F16) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 4 * VC; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[r][i][j] *= 1.0f / kP16;
      }
      float* part = partials + int64_t(2 * run + (first_seg ? 0 : 1)) * piece;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float ls = l[r][u] + __shfl_xor_sync(0xFFFFFFFFu, l[r][u], 4);
          ls += __shfl_xor_sync(0xFFFFFFFFu, ls, 8);
          ls += __shfl_xor_sync(0xFFFFFFFFu, ls, 16);
          const int row = 2 * t + u + 8 * r;
          if (row < rows) {
            if (whole) {
              const float inv = ls > 0.0f || ls != ls ? 1.0f / ls : 0.0f;  // no position: zeros (a NaN stays one)
              uint16_t* dst = out + (int64_t(ci.b) * nq + head0 + row) * HD;
#pragma unroll
              for (int v = 0; v < VC; ++v) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = pack2<F16>(o[r][4 * v + i][u] * inv, o[r][4 * v + i][2 + u] * inv);
                *reinterpret_cast<uint4*>(dst + 8 * (g + 8 * v)) = make_uint4(w[0], w[1], w[2], w[3]);
              }
              if (WEIGHTS && g == 0)
                *reinterpret_cast<float2*>(ml + 2 * (int64_t(ci.b) * nq + head0 + row)) = make_float2(m[r][u], inv);
            } else {
              float* dst = part + row * HD;
#pragma unroll
              for (int v = 0; v < VC; ++v)
#pragma unroll
                for (int i = 0; i < 4; i += 2)
                  *reinterpret_cast<float4*>(dst + 8 * (g + 8 * v) + 2 * i) =
                      make_float4(o[r][4 * v + i][u], o[r][4 * v + i][2 + u], o[r][4 * v + i + 1][u], o[r][4 * v + i + 1][2 + u]);
              if (g == 0) *reinterpret_cast<float2*>(part + HD * prows + 2 * row) = make_float2(m[r][u], ls);
            }
          }
        }
      fresh = true;
      first_seg = false;
      seg_tile0 = 0;
    }
    if (cleft == 0) {
      if (deal.more == 0 && !WHOLE) break;
      __syncwarp();
      const int* from = queue[warp][entered++ & 3];
      run = from[0];
      if (run < 0) break;
      ci.b = from[1], ci.h = from[2], ctile = seg_tile0 = from[3];
      ci.len = len[ci.b];
      ci.nt = (ci.len + KT - 1) / KT;
      cleft = WHOLE ? ci.nt : deal.tiles(run);
      first_seg = true;
    } else if (++ctile == ci.nt) {
      ctile = 0;
      next_item(ci);
    }
  }
  cp_async_wait<0>();
}

// Where the pieces of an item lie: none when one run held it whole.
struct Pieces {
  int count = 0, first = 0, r0 = 0;
  __device__ Pieces(const Deal& deal, int t0, int nt) {
    r0 = deal.run_of(t0);
    const int r1 = deal.run_of(t0 + nt - 1);
    if (r0 == r1) return;
    first = 2 * r0 + (deal.first(r0) == t0 ? 0 : 1);
    count = r1 - r0 + 1;
  }
  __device__ int64_t slot(int i) const { return i == 0 ? first : 2 * (r0 + i); }
};

struct JoinArgs {
  int seqs, kv_heads, nq, HT, workers, shared;
  uint16_t* out;
  const int* starts;
  const float* partials;
};

// A group of TPH threads, thread `tid` of them, for the `at`-th (sequence, query head): adds the pieces of an item that
// several runs share, in the runs' order, and writes zeros for an empty sequence.  Most items of a large batch lie in
// one run and have nothing to add; an item of few long sequences has hundreds of pieces, eight of which each thread has
// in flight.
template <bool F16, int HD, int TPH>
__device__ __forceinline__ void join_head(const JoinArgs& g, int64_t at, int tid) {
  constexpr int LX = HD / 4;                   // float4 columns
  constexpr int SL = TPH > LX ? TPH / LX : 1;  // slices over the pieces
  static_assert(TPH >= LX, "a warp covers a head's outputs");
  __shared__ float4 acc[TPH > 32 ? SL : 1][LX];
  __shared__ float2 accl[TPH > 32 ? SL : 1];
  const int b = int(at / g.nq), head = int(at - int64_t(b) * g.nq);
  const int G = g.nq / g.kv_heads, kvh = head / G, ht = (head % G) / 16, row = (head % G) % 16, prows = min(16, G);
  const int start = __ldcg(g.starts + b), nt = (__ldcg(g.starts + b + 1) - start) / (g.kv_heads * g.HT);
  uint16_t* dst = g.out + at * HD;
  if (nt == 0) {
    for (int i = tid; i < HD / 2; i += TPH) reinterpret_cast<uint32_t*>(dst)[i] = 0u;
    return;
  }
  const Deal deal(__ldcg(g.starts + g.seqs), g.workers, g.shared != 0, last_tiles(prows, HD));
  const Pieces where(deal, start + (kvh * g.HT + ht) * nt, nt);
  const int pieces = where.count;
  if (pieces == 0) return;  // written by the run itself
  auto piece = [&](int i) { return g.partials + where.slot(i) * piece_floats(prows, HD); };
  const int x = tid % LX, s = tid / LX;
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f, mx = -INFINITY;  // this thread's pieces, relative to their largest max
  constexpr int kBatch = 8;
  for (int i0 = s; i0 < pieces; i0 += kBatch * SL) {
    float2 e[kBatch];
    float4 v[kBatch];
    float top = mx;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * SL;
      e[k] = make_float2(-INFINITY, 0.0f);
      v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (i < pieces) {
        const float* p = piece(i);
        e[k] = __ldcg(reinterpret_cast<const float2*>(p + prows * HD + 2 * row));
        v[k] = __ldcg(reinterpret_cast<const float4*>(p + row * HD + 4 * x));
      }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) top = fmaxf(top, e[k].x);
    const float base = top == -INFINITY ? 0.0f : top, k0 = ex2(mx - base);
    a.x *= k0, a.y *= k0, a.z *= k0, a.w *= k0, l *= k0;
    mx = top;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float f = ex2(e[k].x - base);
      a.x = fmaf(v[k].x, f, a.x), a.y = fmaf(v[k].y, f, a.y), a.z = fmaf(v[k].z, f, a.z), a.w = fmaf(v[k].w, f, a.w);
      l = fmaf(e[k].y, f, l);
    }
  }
  if constexpr (TPH > 32) {
    acc[s][x] = a;
    if (x == 0) accl[s] = make_float2(mx, l);
    __syncthreads();
    if (s != 0) return;
    for (int i = 1; i < SL; ++i) mx = fmaxf(mx, accl[i].x);
    const float base = mx == -INFINITY ? 0.0f : mx;
    a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), l = 0.0f;
    for (int i = 0; i < SL; ++i) {
      const float4 v = acc[i][x];
      const float f = ex2(accl[i].x - base);
      a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
      l = fmaf(accl[i].y, f, l);
    }
  } else if constexpr (SL == 2) {
    const float top = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16)), f = ex2(mx - (top == -INFINITY ? 0.0f : top));
    a.x *= f, a.y *= f, a.z *= f, a.w *= f, l *= f, mx = top;
    a.x += __shfl_xor_sync(0xFFFFFFFFu, a.x, 16), a.y += __shfl_xor_sync(0xFFFFFFFFu, a.y, 16);
    a.z += __shfl_xor_sync(0xFFFFFFFFu, a.z, 16), a.w += __shfl_xor_sync(0xFFFFFFFFu, a.w, 16);
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
    if (s != 0) return;
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  *reinterpret_cast<uint2*>(dst + 4 * x) = make_uint2(pack2<F16>(a.x * inv, a.y * inv), pack2<F16>(a.z * inv, a.w * inv));
}

// TPH (a whole attention call in a captured loop): 32, eight heads in a CTA, from 2048 heads on, or from 512 where the
// tables hold at most 128 tiles (32 sequences up to 2047: 21.3 us, with 128 24.1; 24 up to 8191 at head_dim 128, 1536
// heads of some 40 pieces: 102.4, with 128 99.4); else 128 from 512 heads on or with such tables, else 512.
template <bool F16, int HD, int TPH>
__global__ void __launch_bounds__(TPH == 32 ? 256 : TPH) paged_attn_join_kernel(const JoinArgs g) {
  const int64_t at = TPH == 32 ? int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (at >= int64_t(g.seqs) * g.nq) return;
  pdl_wait();
  join_head<F16, HD, TPH>(g, at, threadIdx.x % TPH);
}

// weights[b, kvh, j] += sum over the kv head's query heads of exp2(s_j - m) / l, from the stored scaled scores, for the
// positions 4 (thread + 256 x), x = part, part + parts, ...; ml[r] = (m, 1 / l) of the kv head's r-th query head.
__device__ __forceinline__ void add_weights(const float2* ml, int G, const float* scores, int64_t score_stride, int L,
                                            float* w, int part, int parts) {
  for (int j = 4 * (part * 256 + int(threadIdx.x)); j < L; j += 1024 * parts) {
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int r = 0; r < G; ++r) {
      const float2 e = ml[r];
      const float4 s = __ldcg(reinterpret_cast<const float4*>(scores + r * score_stride + j));
      const float base = e.x == -INFINITY ? 0.0f : e.x;
      sum.x = fmaf(ex2(s.x - base), e.y, sum.x);
      sum.y = fmaf(ex2(s.y - base), e.y, sum.y);
      sum.z = fmaf(ex2(s.z - base), e.y, sum.z);
      sum.w = fmaf(ex2(s.w - base), e.y, sum.w);
    }
    const int n = min(4, L - j);
    w[j] += sum.x;
    if (n > 1) w[j + 1] += sum.y;
    if (n > 2) w[j + 2] += sum.z;
    if (n > 3) w[j + 3] += sum.w;
  }
}

constexpr int kMaxGroup = 1024;  // query heads per kv head

struct WeightArgs {
  const float* logits;
  int64_t logit_stride;
  const float2* ml;
  float* weights;
  int64_t swb, swh;
  int parts;  // CTAs per (sequence, kv head)
};

// After whole items alone: (m, 1 / l) of every head is there.
__global__ void __launch_bounds__(256) paged_attn_weights_kernel(const PagedCache c, const int32_t* __restrict__ lens,
                                                                 int nq, const WeightArgs a) {
  const int item = int(blockIdx.x), b = item / c.kv_heads, kvh = item % c.kv_heads, G = nq / c.kv_heads;
  __shared__ float2 ml[kMaxGroup];
  pdl_wait();
  for (int r = threadIdx.x; r < G; r += 256) ml[r] = __ldcg(a.ml + int64_t(b) * nq + kvh * G + r);
  __syncthreads();
  add_weights(ml, G, a.logits + (int64_t(b) * nq + kvh * G) * a.logit_stride, a.logit_stride, clamped_len(c, lens, b),
              a.weights + b * a.swb + kvh * a.swh, 0, 1);
}

// The join and the weights in one launch: the first CTAs join (TPH = 32 from 512 heads on, else 256), the others add
// the weights of a (sequence, kv head) each, for which they add up the pieces' sums (not the outputs) themselves.
template <bool F16, int HD, int TPH>
__global__ void __launch_bounds__(256) paged_attn_finish_kernel(const PagedCache c, const int32_t* __restrict__ lens,
                                                                const JoinArgs g, int join_ctas, const WeightArgs a) {
  __shared__ float2 ml[kMaxGroup];
  pdl_wait();
  if (int(blockIdx.x) < join_ctas) {
    const int64_t at = TPH == 32 ? int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (at < int64_t(g.seqs) * g.nq) join_head<F16, HD, TPH>(g, at, threadIdx.x % TPH);
    return;
  }
  const int id = int(blockIdx.x) - join_ctas, item = id / a.parts, b = item / g.kv_heads, kvh = item % g.kv_heads;
  const int G = g.nq / g.kv_heads, prows = min(16, G), lane = threadIdx.x & 31;
  const int L = clamped_len(c, lens, b);
  if (4 * 256 * (id % a.parts) >= L) return;
  const int start = __ldcg(g.starts + b), nt = (__ldcg(g.starts + b + 1) - start) / (g.kv_heads * g.HT);
  const Deal deal(__ldcg(g.starts + g.seqs), g.workers, g.shared != 0, last_tiles(prows, HD));
  for (int r = threadIdx.x >> 5; r < G; r += 8) {  // a warp per head
    const Pieces where(deal, start + (kvh * g.HT + r / 16) * nt, nt);
    if (where.count == 0) {
      if (lane == 0) ml[r] = __ldcg(a.ml + int64_t(b) * g.nq + kvh * G + r);
      continue;
    }
    float m = -INFINITY, l = 0.0f;
#pragma unroll 4
    for (int i = lane; i < where.count; i += 32) {
      const float2 e = __ldcg(reinterpret_cast<const float2*>(g.partials + where.slot(i) * piece_floats(prows, HD) + prows * HD +
                                                              2 * (r % 16)));
      const float top = fmaxf(m, e.x), base = top == -INFINITY ? 0.0f : top;
      l = l * ex2(m - base) + e.y * ex2(e.x - base);
      m = top;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, o), l2 = __shfl_xor_sync(0xFFFFFFFFu, l, o);
      const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.0f : top;
      l = l * ex2(m - base) + l2 * ex2(m2 - base);
      m = top;
    }
    if (lane == 0) ml[r] = make_float2(m, l > 0.0f || l != l ? 1.0f / l : 0.0f);
  }
  __syncthreads();
  add_weights(ml, G, a.logits + (int64_t(b) * g.nq + kvh * G) * a.logit_stride, a.logit_stride, L,
              a.weights + b * a.swb + kvh * a.swh, id % a.parts, a.parts);
}

// ------------------------------------------------------------------ eviction

// Weights as unsigned integers in the order of their values: NaN lowest, then -inf, ..., -0 = +0, ..., +inf.
__device__ __forceinline__ uint32_t order_of(uint32_t u) {
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
  return u & 0x80000000u ? (u == 0x80000000u ? u : ~u) : u | 0x80000000u;
}
// Of four at once; +0 to +inf, what accumulated weights are, take the short way.
__device__ __forceinline__ uint4 order_of(const uint4& w) {
  if (max(max(w.x, w.y), max(w.z, w.w)) <= 0x7F800000u)
    return make_uint4(w.x | 0x80000000u, w.y | 0x80000000u, w.z | 0x80000000u, w.w | 0x80000000u);
  return make_uint4(order_of(w.x), order_of(w.y), order_of(w.z), order_of(w.w));
}

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr int kSelMost = 49152;  // slots of a row that one CTA of a cluster can hold

// hist[i] += 1 in shared memory where `yes`: predicated, a branch around each would cost more than the addition.
__device__ __forceinline__ void count_if(uint32_t* hist, uint32_t i, bool yes) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p red.shared.add.u32 [%0], 1;\n\t}" ::"r"(smem_u32(hist + i)),
               "r"(uint32_t(yes))
               : "memory");
}
__device__ __forceinline__ uint2 ld_cluster_u64(const uint32_t* p, uint32_t rank) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_cluster_u32(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

// One cluster of `parts` CTAs per (kv head, sequence).  The row's weights lie in the CTAs' shared memory (read once,
// so that the output may be the input); three histograms, of 11, 11 and 10 bits of the order value, each added up over
// the cluster, give the `need`-th largest among the older positions; then every warp counts, and after one scan over
// the warps of the cluster writes, what stays of its consecutive positions.
__global__ void __launch_bounds__(kSelThreads, 2) paged_evict_select_kernel(
    const float* weights, int64_t swb, int64_t swh, const int32_t* __restrict__ lens, int capacity, int budget,
    int recent, int32_t* __restrict__ new_lens, int32_t* __restrict__ kept, float* weights_out, int64_t sob,
    int64_t soh, int width, int kv_heads, int parts) {
  extern __shared__ __align__(16) uint32_t row[];
  __shared__ __align__(8) uint32_t hist[kBins];
  __shared__ uint32_t sum[kSelWarps];
  __shared__ uint32_t found[2], wcount[2][kSelWarps], total[2];
  const int rank = parts > 1 ? int(cluster_ctarank()) : 0, item = int(blockIdx.x) / parts;
  const int kvh = item % kv_heads, b = item / kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* w = weights + b * swb + kvh * swh;
  float* wo = weights_out + b * sob + kvh * soh;
  int32_t* ko = kept + int64_t(item) * budget;
  int L = __ldg(lens + b);
  L = L < 0 ? 0 : (L > capacity ? capacity : L);
  const int n = min(L, budget);
  if (item % kv_heads == 0 && rank == 0 && tid == 0) new_lens[b] = n;
  const bool select = L > budget && budget > recent;
  const int old = L > budget ? L - recent : L;  // positions that compete; all others stay
  const int seg = ((L + parts - 1) / parts + 3) / 4 * 4, p0 = min(L, rank * seg), p1 = min(L, p0 + seg), np = p1 - p0;
  const int rival = min(np, max(0, old - p0));  // of this CTA's positions, those that compete
  auto everyone = [&]() {
    if (parts > 1)
      cluster_sync();
    else
      __syncthreads();
  };

  for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0u;
  __syncthreads();
  auto count4 = [&](int i, const uint4& k, uint32_t mask, uint32_t want, int shift, uint32_t low) {
    const uint32_t e[4] = {k.x, k.y, k.z, k.w};
    if (i + 4 <= rival) {
#pragma unroll
      for (int u = 0; u < 4; ++u) count_if(hist, (e[u] >> shift) & low, (e[u] & mask) == want);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) count_if(hist, (e[u] >> shift) & low, (e[u] & mask) == want && i + u < rival);
    }
  };
  const bool vec = (reinterpret_cast<uintptr_t>(w + p0) & 15) == 0;
#pragma unroll 4
  for (int i = 4 * tid; i < np; i += 4 * kSelThreads) {
    uint4 v;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(w + p0 + i);
    if (vec && i + 4 <= np) {
      v = *reinterpret_cast<const uint4*>(src);
    } else {
      v.x = src[0];
      v.y = i + 1 < np ? src[1] : 0u;
      v.z = i + 2 < np ? src[2] : 0u;
      v.w = i + 3 < np ? src[3] : 0u;
    }
    *reinterpret_cast<uint4*>(row + i) = v;
    if (select) count4(i, order_of(v), 0u, 0u, 21, 2047u);
  }
  uint32_t thr = L > budget ? 0xFFFFFFFFu : 0u;  // (no weight has that order value: nothing but the recent ones stays)
  uint32_t ties = 0u;                            // how many of the positions at the threshold stay
  everyone();                                    // the whole row has been read
  if (select) {
    uint32_t need = uint32_t(budget - recent);
    thr = 0u;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
      if (pass > 0) {
        const uint32_t mask = pass == 1 ? 0xFFE00000u : 0xFFFFFC00u;
        for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0u;
        __syncthreads();
#pragma unroll 4
        for (int i = 4 * tid; i < rival; i += 4 * kSelThreads)
          count4(i, order_of(*reinterpret_cast<const uint4*>(row + i)), mask, thr, shift, uint32_t(bins - 1));
        everyone();
      }
      // thread t owns bins 2t and 2t + 1 from the top; its count of the whole cluster, then a scan from the top
      const int top = bins - 1 - 2 * tid;
      uint32_t c0 = 0u, c1 = 0u;
      if (top > 0) {
        for (int r = 0; r < parts; ++r) {
          const uint2 c = parts > 1 ? ld_cluster_u64(&hist[top - 1], uint32_t(r)) : *reinterpret_cast<const uint2*>(&hist[top - 1]);
          c0 += c.y, c1 += c.x;
        }
      }
      uint32_t v = c0 + c1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += u;
      }
      if (lane == 31) sum[warp] = v;
      __syncthreads();
      const uint32_t above = v - c0 - c1 + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? sum[lane] : 0u);
      if (above < need && above + c0 >= need) found[0] = uint32_t(top), found[1] = above;
      if (above + c0 < need && above + c0 + c1 >= need) found[0] = uint32_t(top - 1), found[1] = above + c0;
      __syncthreads();
      thr |= found[0] << shift;
      need -= found[1];
      everyone();  // the histograms have been read
    }
    ties = need;
  }
  // each warp: consecutive positions, 128 at a time, four per lane; what stays as bits 0-3 (above the threshold, or not
  // competing) and 4-7 (at it)
  const int per = ((np + kSelWarps - 1) / kSelWarps + 127) / 128 * 128, q0 = min(np, warp * per), q1 = min(np, q0 + per);
  auto classify = [&](int i, uint4& v) {
    uint32_t m = 0u;
    if (i < q1) {
      v = *reinterpret_cast<const uint4*>(row + i);
      const uint4 k = order_of(v);
      const uint32_t e[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int u = 0; u < 4; ++u) m |= (e[u] > thr ? 1u << u : 0u) | (e[u] == thr ? 16u << u : 0u);
      if (L <= budget) m = 15u;
      if (i + 4 > rival) {  // some of them do not compete, or are not there
        const uint32_t stay = i >= rival ? 15u : (15u << (rival - i)) & 15u;
        m = (m & ~(stay | stay << 4)) | stay;
      }
      if (i + 4 > np) m &= ((1u << (np - i)) - 1u) * 17u;
    }
    return m;
  };
  uint32_t na = 0u, nt = 0u, known = 0u;  // the first four answers are kept
#pragma unroll 4
  for (int i = q0 + 4 * lane, k = 0; i - 4 * lane < q1; i += 128, k += 8) {
    uint4 v;
    const uint32_t m = classify(i, v);
    if (k < 32) known |= m << k;
    na += __popc(m & 15u), nt += __popc(m >> 4);
  }
  na = __reduce_add_sync(0xFFFFFFFFu, na), nt = __reduce_add_sync(0xFFFFFFFFu, nt);
  if (lane == 0) wcount[0][warp] = na, wcount[1][warp] = nt;
  __syncthreads();
  if (warp < 2) {  // exclusive scan over the CTA's warps, its sum for the cluster
    const uint32_t own = wcount[warp][lane];
    uint32_t v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, v, o);
      if (lane >= o) v += u;
    }
    wcount[warp][lane] = v - own;
    if (lane == 31) total[warp] = v;
  }
  everyone();
  uint32_t above = wcount[0][warp], tie = wcount[1][warp];
  for (int r = 0; r < rank; ++r) above += ld_cluster_u32(&total[0], uint32_t(r)), tie += ld_cluster_u32(&total[1], uint32_t(r));
#pragma unroll 1
  for (int i = q0 + 4 * lane, k = 0; i - 4 * lane < q1; i += 128, k += 8) {
    uint4 v;
    const uint32_t m = k < 32 ? known >> k & 255u : classify(i, v);
    if (__ballot_sync(0xFFFFFFFFu, m != 0u) == 0u) continue;
    const uint32_t own = __popc(m & 15u) | __popc(m >> 4) << 16;
    uint32_t scan = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, scan, o);
      if (lane >= o) scan += u;
    }
    const uint32_t all = __shfl_sync(0xFFFFFFFFu, scan, 31);
    uint32_t a = above + ((scan - own) & 0xFFFFu), t = tie + ((scan - own) >> 16);  // before this lane's positions
    if (m) {
      v = *reinterpret_cast<const uint4*>(row + i);
      const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool is_a = m >> u & 1u, is_t = m >> (4 + u) & 1u;
        if (is_a || (is_t && t < ties)) {
          const uint32_t at = a + min(t, ties);
          ko[at] = p0 + i + u;
          wo[at] = __uint_as_float(e[u]);
        }
        a += is_a, t += is_t;
      }
    }
    above += all & 0xFFFFu, tie += all >> 16;
  }
  for (int i = n + rank * kSelThreads + tid; i < budget; i += parts * kSelThreads) ko[i] = -1;
  if ((reinterpret_cast<uintptr_t>(wo) & 15) == 0) {
    const int n4 = (n + 3) / 4 * 4, w4 = width / 4 * 4;
    for (int i = n4 + 4 * (rank * kSelThreads + tid); i < w4; i += 4 * parts * kSelThreads)
      *reinterpret_cast<float4*>(wo + i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (rank == 0 && tid < 4 && n + tid < min(n4, width)) wo[n + tid] = 0.0f;
    if (rank == 0 && tid < 4 && w4 >= n4 && w4 + tid < width) wo[w4 + tid] = 0.0f;
  } else {
    for (int i = n + rank * kSelThreads + tid; i < width; i += parts * kSelThreads) wo[i] = 0.0f;
  }
  if (parts > 1) cluster_sync();  // no CTA leaves while another may still read its shared memory
}

// Copies the kept rows into the new pages: a thread moves 16 bytes of the keys and of the values of kCopyRows rows.
constexpr int kCopyRows = 4;
template <int HD>
__global__ void __launch_bounds__(256) paged_evict_copy_kernel(const PagedCache c, const int32_t* __restrict__ kept,
                                                               const int32_t* __restrict__ new_table,
                                                               int64_t new_stride, int budget) {
  constexpr int CH = HD / 8, ROWS = 256 / CH;
  const int kvh = blockIdx.y, b = blockIdx.z, ch = threadIdx.x % CH;
  const int i0 = blockIdx.x * (ROWS * kCopyRows) + threadIdx.x / CH;
  const int32_t* table = c.table + int64_t(b) * c.table_stride;
  pdl_wait();
  int pos[kCopyRows];
#pragma unroll
  for (int k = 0; k < kCopyRows; ++k) {
    const int i = i0 + k * ROWS;
    pos[k] = i < budget ? __ldcg(kept + (int64_t(b) * c.kv_heads + kvh) * budget + i) : -1;
  }
  int from[kCopyRows], to[kCopyRows];
#pragma unroll
  for (int k = 0; k < kCopyRows; ++k) {
    from[k] = to[k] = -1;
    if (uint32_t(pos[k]) < uint32_t(c.capacity)) {  // (-1 behind the last kept one)
      from[k] = page_entry(c, table, page_of(c, pos[k]));
      to[k] = page_entry(c, new_table + int64_t(b) * new_stride, page_of(c, i0 + k * ROWS));
    }
  }
  uint4 kk[kCopyRows], vv[kCopyRows];
#pragma unroll
  for (int k = 0; k < kCopyRows; ++k) {
    kk[k] = vv[k] = make_uint4(0u, 0u, 0u, 0u);  // (a page that holds nothing)
    if (from[k] >= 0) {
      const int r = pos[k] - page_of(c, pos[k]) * c.page_size;
      kk[k] = __ldcs(reinterpret_cast<const uint4*>(c.k + from[k] * c.ks_page + kvh * c.ks_head + int64_t(r) * c.ks_token + 8 * ch));
      vv[k] = __ldcs(reinterpret_cast<const uint4*>(c.v + from[k] * c.vs_page + kvh * c.vs_head + int64_t(r) * c.vs_token + 8 * ch));
    }
  }
#pragma unroll
  for (int k = 0; k < kCopyRows; ++k) {
    if (to[k] < 0) continue;
    const int i = i0 + k * ROWS, r = i - page_of(c, i) * c.page_size;
    *reinterpret_cast<uint4*>(c.k + to[k] * c.ks_page + kvh * c.ks_head + int64_t(r) * c.ks_token + 8 * ch) = kk[k];
    *reinterpret_cast<uint4*>(c.v + to[k] * c.vs_page + kvh * c.vs_head + int64_t(r) * c.vs_token + 8 * ch) = vv[k];
  }
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
  const bool whole = c.capacity <= kWholeTiles * tile_of(HD);
  auto kern = whole ? paged_attn_kernel<F16, HD, TWO, WEIGHTS, true> : paged_attn_kernel<F16, HD, TWO, WEIGHTS, false>;
  const size_t smem = size_t(kAttnWarps) * attn_warp_smem(HD, TWO) + (2 * size_t(c.seqs) + 1) * 4;
  cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  const int ctas = sms * kAttnCtas, workers = ctas * kAttnWarps;
  if (w.counter && (e = cudaMemsetAsync(w.counter, 0, sizeof(int), s)) != cudaSuccess) return e;
  kern<<<ctas, kAttnWarps * 32, smem, s>>>(c, a.q, a.sqb, a.sqh, a.lens, a.out, a.nq, HT, a.scale * 1.4426950408889634f,
                                           w.partials, w.logits, w.logit_stride, w.ml, w.counter, w.starts);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int64_t heads = int64_t(c.seqs) * a.nq;
  const JoinArgs g = {c.seqs, c.kv_heads, a.nq, HT, workers, w.counter ? 1 : 0, a.out, w.starts, w.partials};
  const int items = c.seqs * c.kv_heads;
  WeightArgs wa = {w.logits, w.logit_stride, reinterpret_cast<const float2*>(w.ml), a.weights, a.swb, a.swh, 1};
  if (WEIGHTS) {
    if (c.capacity == 0) return cudaSuccess;
    if (whole) return launch_after(paged_attn_weights_kernel, dim3(unsigned(items)), dim3(256), 0, s, c, a.lens, a.nq, wa);
    // four CTAs per SM over all items, whatever the tables could hold
    wa.parts = std::max(1, std::min((c.capacity + 1023) / 1024, 4 * sms / items));
    const int joins = int(heads >= 512 ? (heads + 7) / 8 : heads);
    return launch_after(heads >= 512 ? paged_attn_finish_kernel<F16, HD, 32> : paged_attn_finish_kernel<F16, HD, 256>,
                        dim3(unsigned(joins + items * wa.parts)), dim3(256), 0, s, c, a.lens, g, joins, wa);
  }
  if (whole) return cudaSuccess;
  const bool few = c.capacity <= 128 * tile_of(HD);  // pieces per head: at most 128
  if (heads >= (few ? 512 : 2048))
    return launch_after(paged_attn_join_kernel<F16, HD, 32>, dim3(unsigned((heads + 7) / 8)), dim3(256), 0, s, g);
  if (few || heads >= 512)
    return launch_after(paged_attn_join_kernel<F16, HD, 128>, dim3(unsigned(heads)), dim3(128), 0, s, g);
  return launch_after(paged_attn_join_kernel<F16, HD, 512>, dim3(unsigned(heads)), dim3(512), 0, s, g);
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

size_t paged_attn_workspace(int seqs, int nq, int kv_heads, int head_dim, int capacity, bool weights, int sms,
                            void* base, PagedAttnWorkspace* w) {
  const int G = nq / kv_heads, tile = tile_of(head_dim), HT = (G + 15) / 16;
  const int64_t workers = int64_t(sms) * kAttnCtas * kAttnWarps;
  const int64_t stride = (int64_t(capacity) + tile - 1) / tile * tile;
  const bool whole = capacity <= kWholeTiles * tile;
  // the lengths are on the device: runs are shared where the tables' whole capacity would call for it
  const int last = last_tiles(std::min(G, 16), head_dim);
  const bool shared = !whole && int64_t(seqs) * (stride / tile) * kv_heads * HT >= workers * 8 * last;
  const int64_t pieces = whole ? 0 : 2 * workers * (shared ? kMostRuns : 1);
  const size_t b0 = up256(size_t(pieces) * piece_floats(std::min(G, 16), head_dim) * 4), b1 = whole ? 0 : 256 + up256(4 * (size_t(seqs) + 1));
  const size_t b2 = weights ? up256(size_t(seqs) * nq * size_t(stride) * 4) : 0;
  const size_t b3 = weights ? up256(size_t(seqs) * nq * 8) : 0;
  if (w) {
    char* p = static_cast<char*>(base);
    w->partials = reinterpret_cast<float*>(p);
    w->counter = shared ? reinterpret_cast<int*>(p + b0) : nullptr;
    w->starts = reinterpret_cast<int*>(p + b0 + 256);
    w->logits = weights ? reinterpret_cast<float*>(p + b0 + b1) : nullptr;
    w->logit_stride = stride;
    w->ml = weights ? reinterpret_cast<float*>(p + b0 + b1 + b2) : nullptr;
  }
  return b0 + b1 + b2 + b3;
}

int64_t paged_attn_tiles(const PagedCache& c, int nq) {
  const int64_t ht = (nq / c.kv_heads + 15) / 16;
  return int64_t(c.seqs) * ((int64_t(c.capacity) + tile_of(c.head_dim) - 1) / tile_of(c.head_dim)) * c.kv_heads * ht;
}

cudaError_t launch_paged_attn(const PagedCache& c, const PagedAttn& a, const PagedAttnWorkspace& w, int sms,
                              cudaStream_t s) {
  if (c.f16) return c.head_dim == 64 ? attn_hd<true, 64>(c, a, w, sms, s) : attn_hd<true, 128>(c, a, w, sms, s);
  return c.head_dim == 64 ? attn_hd<false, 64>(c, a, w, sms, s) : attn_hd<false, 128>(c, a, w, sms, s);
}

cudaError_t launch_paged_append(const PagedCache& c, const uint16_t* qkv, int64_t sqkv, int64_t tokens, const void* cosT,
                                const void* sinT, bool table32, int max_pos, const int32_t* positions,
                                const int32_t* slots, const int32_t* seqs, uint16_t* q_out, int nq, cudaStream_t s) {
  const int heads = nq + 2 * c.kv_heads, per_token = (heads + kHeads - 1) / kHeads * (c.head_dim / 16);
  void (*kern)(const PagedCache, const uint16_t*, int64_t, int64_t, const void*, const void*, int, const int32_t*,
               const int32_t*, const int32_t*, uint16_t*, int, int);
  if (c.head_dim == 64)
    kern = c.f16 ? (table32 ? paged_append_kernel<true, true, 64> : paged_append_kernel<true, false, 64>)
                 : (table32 ? paged_append_kernel<false, true, 64> : paged_append_kernel<false, false, 64>);
  else
    kern = c.f16 ? (table32 ? paged_append_kernel<true, true, 128> : paged_append_kernel<true, false, 128>)
                 : (table32 ? paged_append_kernel<false, true, 128> : paged_append_kernel<false, false, 128>);
  const int64_t ctas = (tokens * per_token + kAppendThreads - 1) / kAppendThreads;
  if (ctas > INT32_MAX) return cudaErrorInvalidValue;
  kern<<<unsigned(ctas), kAppendThreads, 0, s>>>(c, qkv, sqkv, tokens, cosT, sinT, max_pos, positions, slots, seqs, q_out,
                                                 nq, per_token);
  return cudaGetLastError();
}

int paged_evict_most() { return 8 * kSelMost; }

cudaError_t launch_paged_evict(const PagedCache& c, const PagedEvict& e, int sms, cudaStream_t s) {
  // CTAs per row: as many as hold it at 64 KB each (two per SM), more while the SMs are not all busy and each still has
  // two positions per thread; rows beyond 8 x 64 KB take up to 192 KB each
  const int rows = c.seqs * c.kv_heads;
  int parts = 1;
  while (parts < 8 && c.capacity > parts * 16384) parts *= 2;
  while (parts < 8 && rows * parts * 2 <= sms && c.capacity > parts * 4096) parts *= 2;
  const size_t smem = size_t((c.capacity + parts - 1) / parts + 4) * 4;
  cudaError_t st = ensure_dynamic_smem(reinterpret_cast<const void*>(paged_evict_select_kernel), smem);
  if (st != cudaSuccess) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * parts));
  cfg.blockDim = dim3(kSelThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(parts);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  st = cudaLaunchKernelEx(&cfg, paged_evict_select_kernel, e.weights, e.swb, e.swh, e.lens, c.capacity, e.budget, e.recent,
                          e.new_lens, e.kept, e.weights_out, e.sob, e.soh, e.width, c.kv_heads, parts);
  if (st != cudaSuccess) return st;
  const int per = 256 / (c.head_dim / 8) * kCopyRows;
  const dim3 grid(unsigned((e.budget + per - 1) / per), unsigned(c.kv_heads), unsigned(c.seqs));
  if (c.head_dim == 64)
    return launch_after(paged_evict_copy_kernel<64>, grid, dim3(256), 0, s, c, static_cast<const int32_t*>(e.kept),
                        e.new_table, e.new_stride, e.budget);
  return launch_after(paged_evict_copy_kernel<128>, grid, dim3(256), 0, s, c, static_cast<const int32_t*>(e.kept),
                      e.new_table, e.new_stride, e.budget);
}

}  // namespace i4b
