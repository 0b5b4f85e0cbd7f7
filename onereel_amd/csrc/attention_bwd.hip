// Gradient of the packed varlen attention (attention.hip) for gfx950: dq, dk, dv of softmax(q k^T * scale) v per segment,
// bf16 in and out, fp32 accumulation, nothing kept from the forward pass but its output and its log-sum-exp.
//
//   P = exp(scale q k^T - lse)      delta = rowsum(do * o) - dlse      dS = P * (do v^T - delta)
//   dv = P^T do                     dq = scale dS k                    dk = scale dS^T q
//
// Two passes, each recomputing P: one over query tiles for dq (3 products), one over key tiles for dk and dv (4). One pass
// of 5 products would have to add dq into memory from every key tile, with atomics whose order changes the bits; the
// two passes sum every gradient in registers in a fixed order, so a call gives the same bits every time. Where a segment's
// keys fit one tile (cross-attention to a sentence) or its queries do, one pass would need no such sums; those calls take
// the two passes all the same, and read q and do, or k and v, twice.
//
// - A wavefront owns 32 rows (keys, or queries; 64 queries in long calls with heads of 64) of its work-group's tile and keeps their
//   operands and their fp32 gradient in registers; the rows of the other side stream past in blocks of 32 through a ring of
//   LDS slots filled by LDS DMA, three blocks ahead.
// - Both products of scores put the streamed rows on the MFMA rows and the owned rows on its columns, so a lane holds
//   scores of one owned row, and the bf16 P and dS of a lane are the B operand of the next products as they lie.
//   Their A operand is the streamed block transposed, read from the same slot by transposing LDS reads. The slot's
//   swizzle serves both kinds of read without bank conflicts.
// - P and dS are rounded to bf16 once, as the operands of the bf16 matrix cores (the forward pass rounds its P the same way);
//   scores, P, dS, delta and all sums are fp32. Calls of few scores (shape_of) carry what that rounding leaves out in a second
//   product.
// - Key rows may belong to several segments (overlapping ranges): the key axis is cut at every range boundary, so that all
//   rows of a key tile have the same segments, and the tile streams the queries of all of them. Rows past an end load as
//   zeros: a zero query row adds nothing to dk and dv, and the scores of key rows past the end are set to P = 0.
// - Tiles with long streamed axes (few queries against long keys, few keys against long queries, one long segment among short
//   ones) are split; the parts write fp32 partial gradients, and a last launch adds them in order.
// Measured: 3 x 9680 queries against overlapping 11440 keys, 16 heads of 128: dq 3.21 ms, dk and dv 4.09 ms, 1240 TFLOP/s of
// the 7 products executed (a large bf16 product of the vendor library reaches 1360 to 1490 on the same card), the matrix pipes
// busy 70 % of the cycles. With heads of 64 they are busy 49 % (dq) and 58 % (dk and dv), and the vector units, which have as
// many exponentials and conversions for half the matrix work, 60 % and 53 % (with heads of 128, 48 % and 39 %).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace onereel {

namespace {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

constexpr int kThreads = 256;        // 4 wavefronts
constexpr int kCUs = 256;
constexpr int kBlk = 32;             // streamed rows per block
constexpr int kRing = 4;             // LDS slots of the ring
constexpr int kPlanThreads = 1024;
constexpr int kMaxSeg = 4096;
constexpr int kHeader = 8;           // int32 words ahead of the tables
constexpr float kLog2e = 1.44269504088896340736f;

struct BwdArgs {
  const uint16_t *q, *k, *v, *o, *d_o;
  const float *lse, *dlse;
  uint16_t *dq, *dk, *dv;
  const int32_t *cu_q, *cu_k, *k_off, *k_len;
  int64_t qs, ks, os, dos;           // row strides (elements) of q, of k and v, of o, of do
  int64_t lse_stride;                // elements between the heads of lse and dlse
  int32_t n_seg, n_q, n_k, H;
  float scale;
  int32_t max_q_items, max_k_items;  // of one head
  int32_t slots_q, slots_k;          // partial gradients of tiles that a head may have; 0: no tile is split
  int32_t tq, tk;                    // rows of a query tile and of a key tile
  // workspace
  int32_t* head;                     // query items (calls that are planned ahead), key items, split query tiles, split key tiles
  i32x4* q_items;                    // first query, rows, first key, keys
  i32x4* k_items;                    // two an item: first key, rows, first and last segment that may read them; first query and
                                     // queries of the segment where only one may, part and parts, the part's slot
  i32x4 *q_split, *k_split;          // split tiles: first row, rows, first slot, parts
  float* stat;                       // [H][2][n_q]: -lse / scale, then -delta
  float* part_q;                     // [slots_q][H][tq][D]
  float* part_k;                     // [2][slots_k][H][tk][D]: dk, dv
};

// Blocks of 32 queries that a wavefront owns. One leaves room for two wavefronts on a SIMD, one's exponentials under the
// other's matrix work: 3 x 9680 queries x 11440 keys, 16 heads of 128, dq 3.41 ms against 3.88 with two blocks (one
// wavefront); dk and dv 4.80 against 5.36 ms with 32 and 64 keys. With heads of 64, two blocks fit twice too and halve the
// LDS reads per query, one block fits four times: 24 x 9680 x 9680 850 us with two and 890 with one, 2 x 3001 x 3001, 16 heads,
// 146 and 128, 8 x 700 x 700 16.6 and 12.4. So two where their tiles fill the GPU (dk and dv with 64 keys do not fit twice:
// 239 against 198 us).
int query_blocks(int64_t n_q, int H, int D) { return D == 64 && n_q / 256 * H >= 2 * kCUs ? 2 : 1; }
constexpr int kKeyTile = 128;

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }
// a value that is the same in every lane, in a scalar register
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ i32x4 uni(i32x4 x) { return i32x4{uni(x[0]), uni(x[1]), uni(x[2]), uni(x[3])}; }

// a segment's queries and keys, kept inside the tensors whatever the offsets say
__device__ __forceinline__ void seg_q(const BwdArgs& a, int s, int& lo, int& n) {
  lo = clampi(a.cu_q[s], 0, a.n_q);
  n = max(clampi(a.cu_q[s + 1], 0, a.n_q) - lo, 0);
}
__device__ __forceinline__ void seg_k(const BwdArgs& a, int s, int& lo, int& n) {
  const int64_t beg = (a.k_off ? a.k_off : a.cu_k)[s], end = (a.k_len ? a.k_len : a.cu_k + 1)[s];   // no branches: loads
  const int64_t len = a.k_len ? end : end - beg;                                                   // are under way at once
  lo = (int)min(max(beg, (int64_t)0), (int64_t)a.n_k);
  n = (int)max(min(beg + len, (int64_t)a.n_k) - lo, (int64_t)0);
}

// ------------------------------------------------------------------------------------------------------------------
// planner. Query tiles: every segment's queries in pieces of tq rows, then the rows behind the last segment (no keys: their
// gradient is zero). Key tiles: the key axis cut at the segments' key range boundaries, every interval in pieces of tk rows,
// with the first and last segment that cover it.
//
// Calls of up to kFewSeg segments need no launch for it: a block of the dq pass finds its query tile in a wavefront's scan of
// cu_q, and the first block of that pass writes the key tiles that the dk / dv pass reads (a planner launch of one block
// took 7 to 17 us, the dk / dv pass of 12 ragged sequences 49). With more segments one block plans both ahead.
constexpr int kFewSeg = 256;
// Of up to kSorted segments the tiles with the longest streamed axes come first, and long ones are split (parts_of): 12 ragged
// sequences of 1 to 899 rows, 16 heads of 128, dq in 36 us, 42 in the order of the segments, dk and dv in 36 and 40;
// 3 x 9680 queries against overlapping ranges, dk and dv, 4.14 ms and 4.33. A lane ranks one segment, so calls of more are neither
// sorted nor split. Segments with keys of their own lose nothing by it (64 of 198 rows 184 us, 65 of 195 185, 256 of 49 180);
// many that read the same keys do, whose tile streams all their queries alone: 64 ranges of 781 queries on the same 128 keys
// take 407 us, 65 of 769 2475 (one range of 50 000 queries 346).
constexpr int kSorted = 64;

// Parts of a tile that streams `blocks` blocks, in a call whose heads' tiles stream `total` blocks each: the nearest number that
// gives every one of 256 CUs a share of the call's blocks as long as a part, no part shorter than 4 blocks or so (with 8, passes
// of 1 to 2 heads with few segments take 14 to 17 us, so 11 to 14); and where such parts are 48 blocks long, nearly twice as many, since two work-groups on a CU fill each other's gaps. A tile of 2 parts
// or more has at most blocks / share + 1/2 <= 4/3 blocks / share of them, so a head's split tiles have at most
// 4/3 total / share, and never more than the workspace's slots: kMaxParts / H + 1, up to 932 over all heads (233 of them), 184 MB
// of dq, dk and dv. 24 calls of 1 to 24 segments of 1
// to 12720 rows, 1 to 8 heads: 2.4 to 6 times as fast where one segment outweighs the others, 1.5 times on (geometric)
// average, as with one number of parts for all tiles; 128 keys against 3 x 9680 queries, 16 heads: 488 us for dk and dv in 1
// part, 103 in 5, 80 in 10.
constexpr int kMaxParts = 700;
__device__ __forceinline__ int share_of(int64_t total, int H, int slots) {
  int64_t share = max((total * H + kCUs - 1) / kCUs, (int64_t)4);
  if (share >= 48) share = share * 9 / 16;
  return (int)min(max(share, (4 * total + 3 * slots - 1) / (3 * slots)), (int64_t)1 << 30);
}
__device__ __forceinline__ int parts_of(int blocks, int share) { return max((int)(((int64_t)blocks + share / 2) / share), 1); }

// exclusive sum over the block's threads; all: the total
template <int THREADS>
__device__ int block_scan(int v, int* wsum, int& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  if (lane == 63) wsum[w] = x;
  __syncthreads();
  int base = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) {
    const int y = wsum[i];
    if (i < w) base += y;
    all += y;
  }
  __syncthreads();
  return base + x - v;
}

// the tiles of n pieces (piece i: `count(i)` tiles), dealt out to the threads: emit(piece, tile of the piece, tile). first: n + 1
// ints of LDS
template <int THREADS, class Count, class Emit>
__device__ int deal_tiles(int n, int most, int* first, int* wsum, Count&& count, Emit&& emit) {
  const int t = threadIdx.x;
  int at = 0;
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    int all;
    const int x = block_scan<THREADS>(i0 + t < n ? count(i0 + t) : 0, wsum, all);
    if (i0 + t < n) first[i0 + t] = at + x;
    at += all;
  }
  if (t == 0) first[n] = at;
  __syncthreads();
  at = min(at, most);
  for (int x = t; x < at; x += THREADS) {
    int lo = 0, hi = n - 1;   // the last piece that starts at or before x
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= x) lo = mid; else hi = mid - 1;
    }
    emit(lo, x - first[lo], x);
  }
  return at;
}

template <int SEG>
struct PlanLds {
  int bnd[2 * SEG], lo_seg[2 * SEG + 1], hi_seg[2 * SEG + 1], first[2 * SEG + 2], wsum[16];
  unsigned long long total;
  int order[2 * kSorted + 1], blocks[2 * kSorted + 1], n_q[kSorted], k_lo[kSorted], k_end[kSorted];
};

template <int THREADS, int SEG>
__device__ void plan_keys(const BwdArgs& a, PlanLds<SEG>& l) {
  const int t = threadIdx.x, n = a.n_seg, tk = a.tk;
  // boundaries of the key ranges, sorted (a power of two of them, the rest past the end)
  int m = 2;
  while (m < 2 * n) m <<= 1;
  int* raw = l.first;   // unsorted, until the tiles are dealt out
  for (int i = t; i < m; i += THREADS) {
    int b = a.n_k;
    if (i < 2 * n) {
      int lo, len;
      seg_k(a, i >> 1, lo, len);
      b = i & 1 ? lo + len : lo;
    }
    raw[i] = b;
    l.bnd[i] = b;
  }
  for (int i = t; i <= m; i += THREADS) {
    l.lo_seg[i] = 0x7fffffff;
    l.hi_seg[i] = -1;
  }
  __syncthreads();
  if (m <= 512) {   // by rank: no barriers
    for (int i = t; i < m; i += THREADS) {
      const int b = raw[i];
      int rank = 0;
      for (int j = 0; j < m; ++j) rank += raw[j] < b || (raw[j] == b && j < i);
      l.bnd[rank] = b;
    }
    __syncthreads();
  } else {
    for (int size = 2; size <= m; size <<= 1)
      for (int d = size >> 1; d > 0; d >>= 1) {
        for (int i = t; i < m / 2; i += THREADS) {
          const int x = 2 * d * (i / d) + i % d, y = x + d;
          const bool up = (x & size) == 0;
          const int p = l.bnd[x], r = l.bnd[y];
          if ((p > r) == up) {
            l.bnd[x] = r;
            l.bnd[y] = p;
          }
        }
        __syncthreads();
      }
  }
  // interval i is [bnd[i - 1], bnd[i]): from 0 at i = 0, to n_k at i = m
  for (int s = t; s < n; s += THREADS) {
    int lo, len;
    seg_k(a, s, lo, len);
    if (len == 0) continue;
    int x = 0, y = m;   // the first boundary at lo
    while (x < y) {
      const int mid = (x + y) >> 1;
      if (l.bnd[mid] < lo) x = mid + 1; else y = mid;
    }
    for (int i = x + 1; i < m && l.bnd[i] <= lo + len; ++i) {
      if (l.bnd[i] == l.bnd[i - 1]) continue;
      atomicMin(&l.lo_seg[i], s);
      atomicMax(&l.hi_seg[i], s);
    }
  }
  __syncthreads();
  auto start = [&](int i) { return i > 0 ? l.bnd[i - 1] : 0; };
  auto length = [&](int i) { return (i < m ? l.bnd[i] : a.n_k) - start(i); };
  const bool sorted = SEG == kFewSeg && n <= kSorted;
  int share = 1 << 30;
  if (sorted) {
    // blocks of queries that read an interval; its rank among them
    if (t < n) {
      int lo, len;
      seg_q(a, t, lo, l.n_q[t]);
      seg_k(a, t, lo, len);
      l.k_lo[t] = lo;
      l.k_end[t] = lo + len;
    }
    if (t == 0) l.total = 0;
    __syncthreads();
    int mine = 0;
    if (t <= m) {
      if (length(t) > 0)
        for (int s = l.lo_seg[t]; s <= l.hi_seg[t]; ++s)
          if (l.k_lo[s] <= start(t) && start(t) < l.k_end[s]) mine += (l.n_q[s] + kBlk - 1) / kBlk;
      l.blocks[t] = mine;
      if (mine) atomicAdd(&l.total, (unsigned long long)mine * ((length(t) + tk - 1) / tk));
    }
    __syncthreads();
    if (a.slots_k) share = share_of((int64_t)l.total, a.H, a.slots_k);
    int rank = 0;
    if (t <= m) {
      for (int i = 0; i <= m; ++i) rank += l.blocks[i] > mine || (l.blocks[i] == mine && i < t);
      l.order[rank] = t;
    }
    __syncthreads();
  }
  auto nth = [&](int i) { return sorted ? l.order[i] : i; };
  auto parts = [&](int i) { return sorted ? parts_of(l.blocks[i], share) : 1; };
  auto tiles = [&](int i) { return (length(i) + tk - 1) / tk; };
  const int items = deal_tiles<THREADS>(
      m + 1, a.max_k_items, l.first, l.wsum, [&](int r) { return tiles(nth(r)) * parts(nth(r)); },
      [&](int r, int j, int x) {
        const int i = nth(r), n_parts = parts(i), at = j / n_parts * tk;
        int lo = 0, len = 0;
        if (l.lo_seg[i] == l.hi_seg[i]) seg_q(a, l.lo_seg[i], lo, len);
        a.k_items[2 * x] = i32x4{start(i) + at, min(tk, length(i) - at), l.lo_seg[i], l.hi_seg[i]};
        a.k_items[2 * x + 1] = i32x4{lo, len, j % n_parts | n_parts << 16, x};   // split tiles come first: the item is the slot
      });
  int n_split = 0;
  if (a.slots_k && sorted) {   // interval t's tiles, when split
    const int i = t <= m ? nth(t) : 0, n_parts = t <= m ? parts(i) : 1, n_tiles = n_parts > 1 ? tiles(i) : 0;
    const int base = block_scan<THREADS>(n_tiles, l.wsum, n_split);
    for (int j = 0; j < n_tiles; ++j)
      a.k_split[base + j] = i32x4{start(i) + j * tk, min(tk, length(i) - j * tk), l.first[t] + j * n_parts, n_parts};
  }
  if (t == 0) {
    a.head[1] = items;
    a.head[3] = n_split;
  }
}

__global__ __launch_bounds__(kPlanThreads) void bwd_plan_kernel(BwdArgs a) {
  __shared__ PlanLds<kMaxSeg> l;
  const int n = a.n_seg, tq = a.tq;
  auto piece = [&](int s, int& lo, int& len) {
    if (s < n) {
      seg_q(a, s, lo, len);
    } else {
      lo = clampi(a.cu_q[n], 0, a.n_q);
      len = a.n_q - lo;
    }
  };
  const int tiles = deal_tiles<kPlanThreads>(
      n + 1, a.max_q_items, l.first, l.wsum,
      [&](int s) {
        int lo, len;
        piece(s, lo, len);
        return (len + tq - 1) / tq;
      },
      [&](int s, int j, int x) {
        int lo, len, k0 = 0, nk = 0;
        piece(s, lo, len);
        if (s < n) seg_k(a, s, k0, nk);
        a.q_items[x] = i32x4{lo + j * tq, min(tq, len - j * tq), k0, nk};
      });
  if (threadIdx.x == 0) a.head[0] = tiles;
  __syncthreads();
  plan_keys<kPlanThreads, kMaxSeg>(a, l);
}

// The query items of a call of at most kFewSeg segments: how many there are, and the one with index x, from every
// wavefront's own scan.
struct QueryItems {
  static constexpr int N = kFewSeg / 64;
  int lo[N], len[N], k0[N], nk[N], incl[N], parts, n_seg_items, tail, tail_lo;
  static __device__ __forceinline__ int scan(int x, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(x, d);
      if (lane >= d) x += y;
    }
    return x;
  }
  __device__ __forceinline__ int count(const BwdArgs& a, int tq, int lane) {
    // every load at once: what follows waits for one round of them
#pragma unroll
    for (int i = 0; i < N; ++i) {
      lo[i] = len[i] = k0[i] = nk[i] = 0;
      if (64 * i < a.n_seg) {
        const int s = min(64 * i + lane, a.n_seg - 1);
        seg_q(a, s, lo[i], len[i]);
        seg_k(a, s, k0[i], nk[i]);
        if (64 * i + lane >= a.n_seg) len[i] = 0;
      }
    }
    tail_lo = uni(clampi(a.cu_q[a.n_seg], 0, a.n_q));
    tail = a.n_q - tail_lo;
    parts = 1;
    if (a.n_seg <= kSorted) {   // longest first, equal ones in order
      int rank = 0;
      for (int s = 0; s < a.n_seg; ++s) {
        const int x = __builtin_amdgcn_readlane(nk[0], s);
        rank += x > nk[0] || (x == nk[0] && s < lane);
      }
      rank = lane < a.n_seg ? 4 * rank : 4 * lane;
      lo[0] = __builtin_amdgcn_ds_permute(rank, lo[0]);
      len[0] = __builtin_amdgcn_ds_permute(rank, len[0]);
      k0[0] = __builtin_amdgcn_ds_permute(rank, k0[0]);
      nk[0] = __builtin_amdgcn_ds_permute(rank, nk[0]);
      if (a.slots_q) {
        const int blocks = (nk[0] + kBlk - 1) / kBlk;
        int64_t total = (int64_t)((len[0] + tq - 1) / tq) * blocks;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) total += __shfl_xor((long long)total, d);
        parts = parts_of(blocks, share_of(total, a.H, a.slots_q));
      }
    }
    int at = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      incl[i] = at;
      if (64 * i < a.n_seg) {
        incl[i] = at + scan(items(i, tq), lane);
        at = __shfl(incl[i], 63);
      }
    }
    n_seg_items = uni(at);
    return min(n_seg_items + (tail + tq - 1) / tq, a.max_q_items);
  }
  __device__ __forceinline__ int items(int i, int tq) const { return (len[i] + tq - 1) / tq * (i ? 1 : parts); }
  // first query, rows, first key, keys; the part and the parts
  __device__ __forceinline__ i32x4 at(int tq, int x, int& part, int& n_parts) const {
    i32x4 tile = {tail_lo + (x - n_seg_items) * tq, 0, 0, 0};
    tile[1] = min(tq, tail - (tile[0] - tail_lo));
    part = 0;
    n_parts = 1;
    bool found = x >= n_seg_items;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // the first lane whose sum passes x: its segment has tiles
      const uint64_t hit = __ballot(incl[i] > x && len[i] > 0);
      if (!found && hit) {
        const int l = __builtin_ctzll(hit), n = __shfl(len[i], l), j = x - __shfl(incl[i] - items(i, tq), l);
        if (i == 0) n_parts = uni(__shfl(parts, l));
        part = uni(j % n_parts);
        const int row = j / n_parts * tq;
        tile = i32x4{__shfl(lo[i], l) + row, min(tq, n - row), __shfl(k0[i], l), __shfl(nk[i], l)};
        found = true;
      }
    }
    return uni(tile);
  }
  // the split tiles, by one wavefront
  __device__ __forceinline__ void write_split(const BwdArgs& a, int tq, int lane) const {
    const int n = parts > 1 ? (len[0] + tq - 1) / tq : 0, end = scan(n, lane);
    for (int j = 0; j < n; ++j)
      a.q_split[end - n + j] = i32x4{lo[0] + j * tq, min(tq, len[0] - j * tq), incl[0] + (j - n) * parts, parts};
    if (lane == 63) a.head[2] = end;
  }
};

// ------------------------------------------------------------------------------------------------------------------
// streamed blocks: 32 rows of D bf16 in an LDS slot, row r's 16-byte chunk c at position c ^ swz(r). A b128 read of one
// chunk of 16 consecutive rows, and a transposing b64 read (4 rows x 32 columns per half wavefront), both touch every
// bank once: the low row bits move whole 64-byte pieces, the next ones chunks inside them.
template <int D>
__device__ __forceinline__ int swz(int r) {
  if constexpr (D == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(const lds_void*)p; }

template <int D>
struct Str {
  static constexpr int CH = D / 8;                 // 16-byte chunks per row
  static constexpr int KS = D / 16;                // MFMA steps over the head dims
  static constexpr int DB = D / 32;                // blocks of 32 head dims
  static constexpr int SLOT = kBlk * D * 2;        // bytes of one block
  static constexpr int LPB = kBlk * CH / kThreads; // DMA loads per lane and block
};

// one block of `rows` valid rows at `base` into LDS: the descriptor ends at the last valid row, the rows past it read zeros.
// Inline asm, so that the compiler adds no waits for these LDS writes to unrelated reads: the loop waits itself. One
// wait state is needed between the write of M0 and the LDS DMA that reads it (the s_nop).
template <int D>
__device__ __forceinline__ void dma_rows(const uint16_t* base, int64_t rs, int rows, const uint32_t* voff, uint32_t m0) {
  const uint64_t b = (uint64_t)base;
  const int32_t nrec = rows > 0 ? (int32_t)((rows - 1) * rs * 2 + D * 2) : 0;
  const i32x4 r = {__builtin_amdgcn_readfirstlane((int32_t)(uint32_t)b),
                   __builtin_amdgcn_readfirstlane((int32_t)(uint32_t)(b >> 32)), __builtin_amdgcn_readfirstlane(nrec),
                   0x00020000};
#pragma unroll
  for (int i = 0; i < Str<D>::LPB; ++i)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff[i]), "s"(r),
                 "s"(__builtin_amdgcn_readfirstlane(m0 + i * kThreads * 16))
                 : "memory");
}

// 64 statistics (32 rows of two arrays `apart` elements apart) into LDS, zeros past `rows`
__device__ __forceinline__ void dma_stats(const float* base, int64_t apart, int rows, int lane, uint32_t m0) {
  const uint64_t b = (uint64_t)base;
  const i32x4 r = {__builtin_amdgcn_readfirstlane((int32_t)(uint32_t)b),
                   __builtin_amdgcn_readfirstlane((int32_t)(uint32_t)(b >> 32)), (int32_t)0x7fffffff, 0x00020000};
  const uint32_t off = (lane & 31) < rows ? (uint32_t)((lane & 31) * 4 + (lane >> 5) * apart * 4) : 0x80000000u;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(off), "s"(r),
               "s"(__builtin_amdgcn_readfirstlane(m0))
               : "memory");
}

template <int N>
__device__ __forceinline__ void wait_loads_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Read addresses of a lane inside a slot: one register each, all others an XOR (and an immediate) away, since the dims of
// a step and the 4 rows of a transposing read are chunk bits that the swizzle only XORs.
template <int D>
struct Lds {
  uint32_t row;                    // dims 8 (lane / 32) .. of row lane % 32; step ks: ^ 32 ks
  uint32_t tr;                     // transposing: dims 0 .., rows 4 (lane / 32) + (0 .. 3); block db: ^ 64 db, rows + 8: + 8 rows, ^ 32
  __device__ __forceinline__ void init(int lane) {
    const int l32 = lane & 31, h = lane >> 5, r = lane & 15, g = (lane >> 4) & 1, rr = 4 * h + (r >> 2);
    row = l32 * D * 2 + (h ^ swz<D>(l32)) * 16;
    tr = rr * D * 2 + ((2 * g + ((r >> 1) & 1)) ^ swz<D>(rr)) * 16 + (r & 1) * 8;
  }
};

// `row` and `tr` here are the slot's address plus Lds::row and Lds::tr; `off` an offset of another slot at the same place
template <int D>
__device__ __forceinline__ bf16x8 row_frag(uint32_t row, int ks, uint32_t off) {
  return *(const __attribute__((address_space(3))) bf16x8*)(uintptr_t)((row ^ (32 * ks)) + off);
}

// dims 32 db + lane % 32 of the 8 rows that a lane's scores of step hs belong to: 16 hs + 4 (lane / 32) + {0..3, 8..11}
template <int D>
__device__ __forceinline__ bf16x8 tr_frag(uint32_t tr, int db, int hs, uint32_t off) {
  u32x2 x[2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
    x[t] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                                         (lds_bf16x4*)(uintptr_t)((tr ^ (64 * db + 32 * t)) + (16 * hs + 8 * t) * D * 2 + off)));
  const u32x4 y = {x[0][0], x[0][1], x[1][0], x[1][1]};
  return __builtin_bit_cast(bf16x8, y);
}

__device__ __forceinline__ bf16x8 pack8(const f32x16& x, int half) {
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = pack2(x[8 * half + 2 * i], x[8 * half + 2 * i + 1]);
  return __builtin_bit_cast(bf16x8, y);
}

// what the rounding of pack8(x, half) left out, rounded itself
__device__ __forceinline__ bf16x8 pack8_rest(const f32x16& x, int half, bf16x8 rounded) {
  const u32x4 r = __builtin_bit_cast(u32x4, rounded);
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    y[i] = pack2(x[8 * half + 2 * i] - bf2f((uint16_t)(r[i] & 0xffffu)), x[8 * half + 2 * i + 1] - bf2f((uint16_t)(r[i] >> 16)));
  return __builtin_bit_cast(bf16x8, y);
}

// operand of 32 owned rows: 8 dims 16 ks + 8 (lane / 32) of row lane % 32, zeros past `rows` by way of a buffer descriptor that
// ends there (with a branch around the loads they wait for one another)
template <int D>
__device__ __forceinline__ void load_owned(bf16x8 (&f)[Str<D>::KS], const uint16_t* p, int64_t rs, int rows, int lane) {
  const int l32 = lane & 31, h = lane >> 5;
  const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, rows > 0 ? (int)((rows - 1) * rs * 2 + D * 2) : 0, 0x00020000);
  const int at = (int)(l32 * rs * 2) + 16 * h;
#pragma unroll
  for (int ks = 0; ks < Str<D>::KS; ++ks)
    f[ks] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(r, at + 32 * ks, 0, 0));
}

// Gradient of 32 owned rows (dims on the accumulators' rows, owned row lane % 32 on the column) times f, bf16 or fp32, in whole
// lines by way of this wavefront's quarter of the ring at `lds`: stored as they lie, a lane's 4 dims at a time,
// dk and dv of 12720 keys against 64 queries take 62 us (16 bytes a write request), 47 so.
template <int D, class T>
__device__ __forceinline__ void store_rows(T* p, int64_t rs, const f32x16 (&acc)[Str<D>::DB], float f, int rows, int lane,
                                           uint32_t lds) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int BYTES = D * sizeof(T), CH = BYTES / 16, PER = 16 / sizeof(T);
  typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
  typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
  // chunk c (16 bytes) of row r lies at c ^ (r or r / 2), and in rows of bf16 the halves of a chunk are swapped from row 16
  auto at = [&](int r, int c) { return lds + r * BYTES + ((c ^ (CH == 8 ? r >> 1 : r)) & (CH - 1)) * 16; };
  const int l32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int db = 0; db < Str<D>::DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float x[4] = {acc[db][4 * g] * f, acc[db][4 * g + 1] * f, acc[db][4 * g + 2] * f, acc[db][4 * g + 3] * f};
      if constexpr (F32)
        *(lds_u32x4*)(uintptr_t)at(l32, 8 * db + 2 * g + h) = __builtin_bit_cast(u32x4, f32x4{x[0], x[1], x[2], x[3]});
      else
        *(lds_u32x2*)(uintptr_t)(at(l32, 4 * db + g) + 8 * (h ^ (l32 >> 4))) = u32x2{pack2(x[0], x[1]), pack2(x[2], x[3])};
    }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < CH / 2; ++i) {
    const int r = i * (64 / CH) + lane / CH, c = lane % CH;
    u32x4 y = *(const lds_u32x4*)(uintptr_t)at(r, c);
    if (!F32 && i >= CH / 4) y = u32x4{y[2], y[3], y[0], y[1]};
    if (r < rows) *(u32x4*)(p + r * rs + c * PER) = y;
  }
  __builtin_amdgcn_wave_barrier();
}

// This block's head and item of n_items x H; false: none. The blocks of one XCD (block index modulo 8) take consecutive items
// of few heads, which share their streamed rows in that XCD's L2. Few items are dealt out by their length instead (they
// come longest first), all heads' longest ahead of their shorter ones; where they all run at once, two work-groups on a
// CU, a CU's second one, a kCUs of blocks later, is the shorter the longer its first one is.
__device__ __forceinline__ bool item_of(int n_items, int H, int block, int& head, int& item) {
  const int64_t n = (int64_t)n_items * H;
  if (n <= 4 * kCUs) {
    if (block >= n) return false;
    const int first = (kCUs + H - 1) / H;
    item = block / H;
    head = block % H;
    if (n <= 2 * kCUs && item >= first) item = n_items - 1 - (item - first);
    return true;
  }
  const int64_t per = (n + 7) / 8, j = block >> 3, i = (block & 7) * per + j;
  if (j >= per || i >= n) return false;
  head = (int)(i / n_items);
  item = (int)(i % n_items);
  return true;
}

// ------------------------------------------------------------------------------------------------------------------
// dq: a block owns 128 T queries of one head and streams the keys and values of their segment
template <int D, int T, bool FEW, bool FINE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(FINE ? 1 : 2, D == 64 && T == 1 ? 4 : 2))) void bwd_q_kernel(BwdArgs a) {
  using C = Str<D>;
  __shared__ __attribute__((aligned(1024))) unsigned char ring[2 * kRing * C::SLOT];
  const int tid = threadIdx.x, lane = tid & 63, w = uni(tid >> 6);
  QueryItems qi;
  int n_items;
  if constexpr (FEW) {
    static_assert(sizeof(PlanLds<kFewSeg>) <= sizeof(ring), "plan");
    if (blockIdx.x < 8) {   // ahead of the blocks with an item, eight of them so that those keep their XCDs
      if (blockIdx.x == 0) plan_keys<kThreads, kFewSeg>(a, *(PlanLds<kFewSeg>*)ring);
      if (blockIdx.x == 1 && w == 0 && a.slots_q) {
        qi.count(a, 128 * T, lane);
        qi.write_split(a, 128 * T, lane);
      }
      return;
    }
    n_items = qi.count(a, 128 * T, lane);
  } else {
    n_items = uni(a.head[0]);
  }
  int head, item, part = 0, parts = 1;
  if (!item_of(n_items, a.H, blockIdx.x - (FEW ? 8 : 0), head, item)) return;
  i32x4 tile;
  if constexpr (FEW) tile = qi.at(128 * T, item, part, parts);
  else tile = uni(a.q_items[item]);
  const int row0 = tile[0] + w * 32 * T, n_keys = tile[3];
  const int rows = clampi(tile[1] - w * 32 * T, 0, 32 * T);

  uint32_t voff[C::LPB];
#pragma unroll
  for (int i = 0; i < C::LPB; ++i) {
    const int x = i * kThreads + tid, r = x / C::CH, c = x % C::CH;
    voff[i] = (uint32_t)(r * a.ks * 2 + (c ^ swz<D>(r)) * 16);
  }
  const uint32_t lds = lds_addr(ring), m0 = lds + w * 1024;
  const int blocks = (n_keys + kBlk - 1) / kBlk;
  const int b0 = (int)((int64_t)blocks * part / parts), b1 = (int)((int64_t)blocks * (part + 1) / parts);
  const uint16_t* kp = a.k + (int64_t)tile[2] * a.ks + (int64_t)head * D;
  const uint16_t* vp = a.v + (int64_t)tile[2] * a.ks + (int64_t)head * D;
  auto fetch = [&](int b) {
    const int n = b < b1 ? min(n_keys - b * kBlk, kBlk) : 0;
    const int64_t off = (int64_t)(b < b1 ? b : b0) * kBlk * a.ks;
    const uint32_t at = m0 + (b & (kRing - 1)) * C::SLOT;
    dma_rows<D>(kp + off, a.ks, n, voff, at);
    dma_rows<D>(vp + off, a.ks, n, voff, at + kRing * C::SLOT);
  };
  // the first blocks are under way while the owned rows load
#pragma unroll
  for (int b = 0; b < kRing - 1; ++b) fetch(b0 + b);

  // the owned queries, their output gradients and their statistics
  bf16x8 qf[T][C::KS], df[T][C::KS];
  float lse[T], dlse[T], neg_lse[T], neg_delta[T];
  f32x16 acc[T][C::DB];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int64_t at = head * a.lse_stride + min(row0 + 32 * t + (lane & 31), a.n_q - 1);
    lse[t] = a.lse[at];
    dlse[t] = (a.dlse ? a.dlse : a.lse)[at];
  }
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int n = clampi(rows - 32 * t, 0, 32);
    const int64_t r = row0 + 32 * t;
    bf16x8 of[C::KS];
    load_owned<D>(qf[t], a.q + r * a.qs + (int64_t)head * D, a.qs, n, lane);
    load_owned<D>(df[t], a.d_o + r * a.dos + (int64_t)head * D, a.dos, n, lane);
    load_owned<D>(of, a.o + r * a.os + (int64_t)head * D, a.os, n, lane);
    float d = 0.0f;
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) {
      const u32x4 x = __builtin_bit_cast(u32x4, of[ks]), y = __builtin_bit_cast(u32x4, df[t][ks]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d = fmaf(bf2f((uint16_t)(x[i] & 0xffffu)), bf2f((uint16_t)(y[i] & 0xffffu)), d);
        d = fmaf(bf2f((uint16_t)(x[i] >> 16)), bf2f((uint16_t)(y[i] >> 16)), d);
      }
    }
    d += __shfl_xor(d, 32);
    const bool mine = (lane & 31) < n;
    const int64_t at = r + (lane & 31);
    const float l = mine ? lse[t] : 0.0f;
    if (a.dlse) d -= mine ? dlse[t] : 0.0f;
    neg_lse[t] = -l * kLog2e;
    neg_delta[t] = -d;
    if (mine && lane < 32 && part == 0) {
      a.stat[(int64_t)2 * head * a.n_q + at] = -l / a.scale;
      a.stat[(int64_t)(2 * head + 1) * a.n_q + at] = -d;
    }
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[t][db][e] = 0.0f;
  }

  Lds<D> ad;
  ad.init(lane);
  const float c = a.scale * kLog2e;
  const f32x16 zero = {};
  const int end = min(n_keys, b1 * kBlk);
  auto step = [&](int b, auto tail) {
    wait_loads_barrier<(kRing - 2) * 2 * C::LPB>();
    fetch(b + kRing - 1);
    const uint32_t slot = lds + (b & (kRing - 1)) * C::SLOT, row = slot + ad.row, tr = slot + ad.tr;
    f32x16 s[T], dp[T];
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) {
      const bf16x8 kf = row_frag<D>(row, ks, 0), vf = row_frag<D>(row, ks, kRing * C::SLOT);
#pragma unroll
      for (int t = 0; t < T; ++t) s[t] = mfma(kf, qf[t][ks], ks ? s[t] : zero);
#pragma unroll
      for (int t = 0; t < T; ++t) dp[t] = mfma(vf, df[t][ks], ks ? dp[t] : zero);
    }
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[t][e] = __builtin_amdgcn_exp2f(fmaf(s[t][e], c, neg_lse[t]));
    if constexpr (decltype(tail)::value) {   // the key rows past the end
      const int n = end - b * kBlk - 4 * (lane >> 5);
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[t][e] = 8 * (e >> 2) + (e & 3) < n ? s[t][e] : 0.0f;
    }
    bf16x8 ds[T][2], rest[T][2];
#pragma unroll
    for (int t = 0; t < T; ++t) {
#pragma unroll
      for (int e = 0; e < 16; ++e) dp[t][e] = s[t][e] * (dp[t][e] + neg_delta[t]);
#pragma unroll
      for (int hs = 0; hs < 2; ++hs) {
        ds[t][hs] = pack8(dp[t], hs);
        if constexpr (FINE) rest[t][hs] = pack8_rest(dp[t], hs, ds[t][hs]);
      }
    }
#pragma unroll
    for (int db = 0; db < C::DB; ++db)
#pragma unroll
      for (int hs = 0; hs < 2; ++hs) {
        const bf16x8 kt = tr_frag<D>(tr, db, hs, 0);
#pragma unroll
        for (int t = 0; t < T; ++t) {
          acc[t][db] = mfma(kt, ds[t][hs], acc[t][db]);
          if constexpr (FINE) acc[t][db] = mfma(kt, rest[t][hs], acc[t][db]);
        }
      }
  };
  int b = b0;
#pragma unroll 1
  for (; (b + 1) * kBlk <= end; ++b) step(b, std::false_type{});
  if (b * kBlk < end) step(b, std::true_type{});
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the blocks asked for past the end, before the ring is used again
  __syncthreads();
  const uint32_t own = lds + w * (2 * kRing * C::SLOT / 4);
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int n = clampi(rows - 32 * t, 0, 32);
    if (parts == 1) {
      store_rows<D>(a.dq + ((int64_t)(row0 + 32 * t) * a.H + head) * D, (int64_t)a.H * D, acc[t], a.scale, n, lane, own);
    } else {   // split tiles come first: the item is the slot
      const int64_t row = ((int64_t)item * a.H + head) * 128 * T + w * 32 * T + 32 * t;
      store_rows<D>(a.part_q + row * D, D, acc[t], a.scale, n, lane, own);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// dk, dv: a block owns 128 keys of one head and streams the queries of every segment that reads them

// walks the blocks of 32 queries of the segments that cover a key tile
struct Walk {
  int seg, last, row, left;          // the segment, the last one to look at, the next query row and the rows after it
  __device__ __forceinline__ bool next_segment(const BwdArgs& a, int k0) {
    for (; seg <= last; ++seg) {
      int lo, n;
      seg_k(a, seg, lo, n);
      if (uni(lo) > k0 || uni(lo + n) <= k0) continue;
      seg_q(a, seg, row, left);
      row = uni(row);
      left = uni(left);
      if (left > 0) {
        ++seg;
        return true;
      }
    }
    left = 0;
    return false;
  }
};

template <int D, bool FINE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(FINE ? 1 : 2, 4))) void bwd_kv_kernel(BwdArgs a) {
  using C = Str<D>;
  constexpr int kStat = 256;         // bytes of one wavefront's statistics of a block
  __shared__ __attribute__((aligned(1024))) unsigned char ring[2 * kRing * C::SLOT + kRing * 4 * kStat];
  int head, item;
  if (!item_of(uni(a.head[1]), a.H, blockIdx.x, head, item)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const i32x4 tile = uni(a.k_items[2 * (int64_t)item]), only = uni(a.k_items[2 * (int64_t)item + 1]);
  const int part = only[2] & 0xffff, parts = only[2] >> 16;
  const int row0 = tile[0] + w * 32;
  const int rows = clampi(tile[1] - w * 32, 0, 32);

  uint32_t voq[C::LPB], vod[C::LPB];
#pragma unroll
  for (int i = 0; i < C::LPB; ++i) {
    const int x = i * kThreads + tid, r = x / C::CH, c = x % C::CH;
    voq[i] = (uint32_t)(r * a.qs * 2 + (c ^ swz<D>(r)) * 16);
    vod[i] = (uint32_t)(r * a.dos * 2 + (c ^ swz<D>(r)) * 16);
  }
  const uint32_t lds = lds_addr(ring), m0 = lds + w * 1024, st0 = lds + 2 * kRing * C::SLOT + w * kStat;

  // this part's blocks of the segments' blocks in order
  Walk walk{tile[3] + 1, tile[3], only[0], only[1]};
  int total = (only[1] + kBlk - 1) / kBlk;
  if (tile[2] < tile[3]) {
    Walk all{tile[2], tile[3], 0, 0};
    for (total = 0; all.next_segment(a, tile[0]);) total += (all.left + kBlk - 1) / kBlk;
    walk = Walk{tile[2], tile[3], 0, 0};
    walk.next_segment(a, tile[0]);
  }
  const int b0 = (int)((int64_t)total * part / parts), b1 = (int)((int64_t)total * (part + 1) / parts);
  for (int skip = b0; walk.left > 0;) {
    const int n = (walk.left + kBlk - 1) / kBlk;
    if (skip < n) {
      walk.row += skip * kBlk;
      walk.left -= skip * kBlk;
      break;
    }
    skip -= n;
    walk.next_segment(a, tile[0]);
  }
  auto fetch = [&](int b) {
    if (b < b1 && walk.left <= 0) walk.next_segment(a, tile[0]);
    const int n = b < b1 ? min(walk.left, kBlk) : 0, slot = b & (kRing - 1);
    const int64_t r = b < b1 ? walk.row : 0;
    const uint32_t at = m0 + slot * C::SLOT;
    dma_rows<D>(a.q + r * a.qs + (int64_t)head * D, a.qs, n, voq, at);
    dma_rows<D>(a.d_o + r * a.dos + (int64_t)head * D, a.dos, n, vod, at + kRing * C::SLOT);
    dma_stats(a.stat + (int64_t)2 * head * a.n_q + r, a.n_q, n, lane, st0 + slot * 4 * kStat);
    walk.row += kBlk;
    walk.left -= kBlk;
  };
  // the first blocks are under way while the owned rows load
#pragma unroll
  for (int b = 0; b < kRing - 1; ++b) fetch(b0 + b);

  bf16x8 kf[C::KS], vf[C::KS];
  f32x16 dk[C::DB], dv[C::DB];
  const int64_t own = (int64_t)row0 * a.ks + (int64_t)head * D;
  load_owned<D>(kf, a.k + own, a.ks, rows, lane);
  load_owned<D>(vf, a.v + own, a.ks, rows, lane);
#pragma unroll
  for (int db = 0; db < C::DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) dk[db][e] = dv[db][e] = 0.0f;

  Lds<D> ad;
  ad.init(lane);
  const float c = a.scale * kLog2e;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    wait_loads_barrier<(kRing - 2) * (2 * C::LPB + 1)>();
    fetch(b + kRing - 1);
    const int slot = b & (kRing - 1);
    const uint32_t row = lds + slot * C::SLOT + ad.row, tr = lds + slot * C::SLOT + ad.tr, st = st0 + slot * 4 * kStat;
    // -lse / scale and -delta start the sums of the scores and of do v^T: rows 8 g + 4 (lane / 32) ..
    f32x16 s0, d0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 x = *(const __attribute__((address_space(3))) f32x4*)(uintptr_t)(st + 32 * g + 16 * (lane >> 5));
      const f32x4 y = *(const __attribute__((address_space(3))) f32x4*)(uintptr_t)(st + 128 + 32 * g + 16 * (lane >> 5));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s0[4 * g + i] = x[i];
        d0[4 * g + i] = y[i];
      }
    }
    // The matrix work of a wavefront first: the other one on its SIMD fills the gaps with its exponentials (5.05 -> 4.60 ms,
    // 3 x 9680 queries x 11440 keys, 16 heads; dq gains nothing from it). Operands are read two steps early, which is what
    // the registers have room for, in an order set here: the compiler reads each pair just before its use (4.74 -> 4.35 ms).
    f32x16 s, dp;
    __builtin_amdgcn_s_setprio(1);
    bf16x8 fq[2] = {row_frag<D>(row, 0, 0), row_frag<D>(row, 1, 0)};
    bf16x8 fd[2] = {row_frag<D>(row, 0, kRing * C::SLOT), row_frag<D>(row, 1, kRing * C::SLOT)};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) {
      s = mfma(fq[ks & 1], kf[ks], ks ? s : s0);
      dp = mfma(fd[ks & 1], vf[ks], ks ? dp : d0);
      if (ks + 2 < C::KS) {
        fq[ks & 1] = row_frag<D>(row, ks + 2, 0);
        fd[ks & 1] = row_frag<D>(row, ks + 2, kRing * C::SLOT);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    // by halves: the first half's registers hold the first transposed operands while the second half is worked on
    bf16x8 p[2], ds[2], p_rest[2], ds_rest[2], ft[2][2];
#pragma unroll
    for (int hs = 0; hs < 2; ++hs) {
#pragma unroll
      for (int e = 8 * hs; e < 8 * hs + 8; ++e) {
        s[e] = __builtin_amdgcn_exp2f(s[e] * c);
        dp[e] *= s[e];
      }
      p[hs] = pack8(s, hs);
      ds[hs] = pack8(dp, hs);
      if constexpr (FINE) {
        p_rest[hs] = pack8_rest(s, hs, p[hs]);
        ds_rest[hs] = pack8_rest(dp, hs, ds[hs]);
      }
      ft[hs][0] = tr_frag<D>(tr, hs % C::DB, hs / C::DB, kRing * C::SLOT);
      ft[hs][1] = tr_frag<D>(tr, hs % C::DB, hs / C::DB, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < 2 * C::DB; ++i) {
      const int db = i % C::DB, hs = i / C::DB, n = i + 2;
      dv[db] = mfma(ft[i & 1][0], p[hs], dv[db]);
      dk[db] = mfma(ft[i & 1][1], ds[hs], dk[db]);
      if constexpr (FINE) {
        dv[db] = mfma(ft[i & 1][0], p_rest[hs], dv[db]);
        dk[db] = mfma(ft[i & 1][1], ds_rest[hs], dk[db]);
      }
      if (n < 2 * C::DB) {
        ft[i & 1][0] = tr_frag<D>(tr, n % C::DB, n / C::DB, kRing * C::SLOT);
        ft[i & 1][1] = tr_frag<D>(tr, n % C::DB, n / C::DB, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the blocks asked for past the end, before the ring is used again
  __syncthreads();
  const uint32_t mine = lds + w * (2 * kRing * C::SLOT / 4);
  if (parts == 1) {
    const int64_t at = ((int64_t)row0 * a.H + head) * D, rs = (int64_t)a.H * D;
    store_rows<D>(a.dk + at, rs, dk, a.scale, rows, lane, mine);
    store_rows<D>(a.dv + at, rs, dv, 1.0f, rows, lane, mine);
  } else {
    float* at = a.part_k + (((int64_t)only[3] * a.H + head) * kKeyTile + w * 32) * D;
    store_rows<D>(at, D, dk, a.scale, rows, lane, mine);
    store_rows<D>(at + (int64_t)a.slots_k * a.H * kKeyTile * D, D, dv, 1.0f, rows, lane, mine);
  }
}

// the partial gradients of split tiles, added in the order of the parts: 8 elements a thread of dq, then of dk and dv
template <int D>
__global__ __launch_bounds__(kThreads) void bwd_add_kernel(BwdArgs a) {
  constexpr int ROWS = kThreads * 8 / D;
  const int qc = a.tq / ROWS, kc = a.tk / ROWS;
  const int64_t nq = a.slots_q ? (int64_t)a.head[2] * a.H * qc : 0, nk = a.slots_k ? (int64_t)a.head[3] * a.H * kc : 0;
  for (int64_t i = blockIdx.x; i < nq + 2 * nk; i += gridDim.x) {
    const bool is_q = i < nq;
    const int which = is_q ? 0 : (int)((i - nq) / nk), tile_rows = is_q ? a.tq : a.tk, chunks = is_q ? qc : kc;
    const int64_t x = is_q ? i : (i - nq) % nk;
    const int head = (int)(x / chunks % a.H), row = (int)(x % chunks) * ROWS + threadIdx.x / (D / 8), col = threadIdx.x % (D / 8) * 8;
    const i32x4 tile = (is_q ? a.q_split : a.k_split)[x / chunks / a.H];
    if (row >= tile[1]) continue;
    const int64_t apart = (int64_t)a.H * tile_rows * D;
    const float* p = (is_q ? a.part_q : a.part_k + which * a.slots_k * apart) + tile[2] * apart + ((int64_t)head * tile_rows + row) * D + col;
    f32x4 lo = {}, hi = {};
#pragma unroll 8
    for (int j = 0; j < tile[3]; ++j) {
      lo += *(const f32x4*)(p + j * apart);
      hi += *(const f32x4*)(p + j * apart + 4);
    }
    *(u32x4*)((is_q ? a.dq : which ? a.dv : a.dk) + ((int64_t)(tile[0] + row) * a.H + head) * D + col) =
        u32x4{pack2(lo[0], lo[1]), pack2(lo[2], lo[3]), pack2(hi[0], hi[1]), pack2(hi[2], hi[3])};
  }
}

// ------------------------------------------------------------------------------------------------------------------
// tiles and parts of a call, from its sizes alone (the offsets are on the device)
struct Shape {
  int tq, tk;                        // rows of a query tile and of a key tile
  int64_t max_q_items, max_k_items;
  int slots_q, slots_k;
  bool fine;                         // see shape_of
};

// Partial gradients of tiles that a head may have: parts_of's limits, of at most `tiles` tiles of at most `blocks` blocks. None in
// calls of more than 16 rounds of work-groups, whose longest tiles come first.
int slots_of(int32_t n_seg, int64_t tiles, int64_t blocks, int H) {
  if (n_seg > kSorted || (tiles - n_seg / 2) * H > 32 * kCUs || blocks < 12) return 0;
  return (int)std::min<int64_t>(kMaxParts / H + 1, tiles * blocks / 3 + 1);
}

// fine: whether P and dS go into their products as two bf16 numbers, the rounded value and what that rounding left out: in calls
// of few scores, which latency bounds, counted as heads x query rows x the longest segment's keys (the offsets are on the device). A result rounded once has its own rounding and that of its operand, 1.41 times the
// error of its own rounding alone with many scores and up to 1.55 times with few, where the roundings do not average out;
// with the second product it is 1.00 times. Kernel times with one product / two: 13.5 / 14.2 us at 2 heads x 64 x 64
// scores (D 64), 18.8 / 20.3 at 4 x 128 x 128; above the limit 31.5 / 35.6 at 8 x 256 x 256 (D 128), 75.8 / 87.0 at
// 8 x 1400 x 1400.
Shape shape_of(int32_t n_seg, int32_t n_q, int32_t n_k, int32_t max_q, int32_t max_k, int32_t H, int32_t D) {
  Shape s;
  s.fine = (int64_t)H * n_q * max_k <= (int64_t)1 << 18;
  s.tq = 128 * (s.fine ? 1 : query_blocks(n_q, H, D));
  s.tk = kKeyTile;
  const int64_t q_tiles = n_q / s.tq + n_seg + 1, k_tiles = n_k / s.tk + 2 * (int64_t)n_seg + 1;
  s.slots_q = slots_of(n_seg, q_tiles, ((int64_t)max_k + kBlk - 1) / kBlk, H);
  // overlapping ranges: a key tile may stream every segment's queries
  s.slots_k = slots_of(n_seg, n_k / s.tk + n_seg + 1, std::min((int64_t)n_q / kBlk, (int64_t)max_q / kBlk * n_seg) + n_seg, H);
  s.max_q_items = q_tiles + s.slots_q;
  s.max_k_items = k_tiles + s.slots_k;
  return s;
}

struct Layout {
  int64_t q_items, k_items, q_split, k_split, stat, part_q, part_k, bytes;
};
Layout layout_of(const Shape& s, int32_t n_q, int32_t H, int32_t D) {
  Layout l;
  int64_t at = kHeader * 4;
  auto take = [&](int64_t n) {
    const int64_t was = (at + 255) & ~(int64_t)255;
    at = was + n;
    return was;
  };
  l.q_items = take(s.max_q_items * 16);
  l.k_items = take(s.max_k_items * 32);
  l.q_split = take((int64_t)s.slots_q * 16);
  l.k_split = take((int64_t)s.slots_k * 16);
  l.stat = take((int64_t)2 * H * n_q * 4);
  l.part_q = take((int64_t)s.slots_q * H * s.tq * D * 4);
  l.part_k = take((int64_t)s.slots_k * 2 * H * s.tk * D * 4);
  l.bytes = (at + 255) & ~(int64_t)255;
  return l;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

template <int D, int T, bool FINE>
void launch(const BwdArgs& a, const Shape& s, hipStream_t st) {
  auto grid = [](int64_t items) { return dim3((unsigned)((items + 7) / 8 * 8)); };
  const dim3 gq = grid(s.max_q_items * a.H), gk = grid(s.max_k_items * a.H), t(kThreads);
  if (a.n_seg <= kFewSeg) {
    hipLaunchKernelGGL((bwd_q_kernel<D, T, true, FINE>), dim3(gq.x + 8), t, 0, st, a);
  } else {
    hipLaunchKernelGGL(bwd_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
    if (a.n_q > 0) hipLaunchKernelGGL((bwd_q_kernel<D, T, false, FINE>), gq, t, 0, st, a);
  }
  if (a.n_k > 0) hipLaunchKernelGGL((bwd_kv_kernel<D, FINE>), gk, t, 0, st, a);
  if (s.slots_q || s.slots_k) hipLaunchKernelGGL(bwd_add_kernel<D>, dim3(8 * kCUs), t, 0, st, a);
}

}  // namespace
}  // namespace onereel

using namespace onereel;

extern "C" int64_t or_varlen_bwd_workspace_size(int32_t n_seg, int32_t n_q, int32_t n_k, int32_t max_q, int32_t max_k,
                                                int32_t H, int32_t D) {
  if (n_seg < 1 || n_seg > kMaxSeg || n_q < 0 || n_k < 0 || max_q < 0 || max_k < 0 || H < 1 || H > 256 ||
      (D != 64 && D != 128))
    return fail_arg("or_varlen_bwd_workspace_size: 1 to %d segments, 1 to 256 heads of 64 or 128 and sizes of at least 0 are "
                    "needed", kMaxSeg);
  return layout_of(shape_of(n_seg, n_q, n_k, max_q, max_k, H, D), n_q, H, D).bytes;
}

extern "C" int or_varlen_bwd(const or_varlen_bwd_args* p, void* stream) {
  if (!p) return fail_arg("or_varlen_bwd: args is NULL");
  const or_varlen_bwd_args& x = *p;
  if (x.D != 64 && x.D != 128) return fail_arg("or_varlen_bwd: head_dim must be 64 or 128 (got %d)", x.D);
  if (x.H < 1 || x.H > 256) return fail_arg("or_varlen_bwd: 1 to 256 heads (got %d)", x.H);
  if (x.n_seg < 1 || x.n_seg > kMaxSeg) return fail_arg("or_varlen_bwd: 1 to %d segments (got %d)", kMaxSeg, x.n_seg);
  if (x.n_q < 0 || x.n_k < 0 || x.max_q < 0 || x.max_k < 0) return fail_arg("or_varlen_bwd: negative sizes");
  if (!(x.scale > 0.0f) || !isfinite(x.scale)) return fail_arg("or_varlen_bwd: scale must be positive and finite");
  if (x.n_q == 0 && x.n_k == 0) return 0;
  if (x.n_q > 0 && (!x.q || !x.o || !x.d_o || !x.lse || !x.dq))
    return fail_arg("or_varlen_bwd: q, o, do, lse and dq are required");
  if (x.n_k > 0 && (!x.k || !x.v || !x.dk || !x.dv)) return fail_arg("or_varlen_bwd: k, v, dk and dv are required");
  if (!x.cu_q || (!x.cu_k && !(x.k_off && x.k_len)))
    return fail_arg("or_varlen_bwd: cu_q and cu_k (or k_off and k_len) are required");
  const int64_t row = (int64_t)x.H * x.D, far = (int64_t)1 << 24;
  for (int64_t s : {x.q_row_stride, x.k_row_stride, x.o_row_stride, x.do_row_stride})
    if (s < row || s % 8 || s > far)
      return fail_arg("or_varlen_bwd: row strides must be multiples of 8 elements from H * D = %lld to 2^24",
                      (long long)row);
  if (!aligned16(x.q) || !aligned16(x.k) || !aligned16(x.v) || !aligned16(x.o) || !aligned16(x.d_o) || !aligned16(x.dq) ||
      !aligned16(x.dk) || !aligned16(x.dv))
    return fail_arg("or_varlen_bwd: pointers must be 16-byte aligned");
  if (x.lse_stride < x.n_q) return fail_arg("or_varlen_bwd: lse_stride must cover the query rows");
  const Shape s = shape_of(x.n_seg, x.n_q, x.n_k, x.max_q, x.max_k, x.H, x.D);
  const Layout l = layout_of(s, x.n_q, x.H, x.D);
  if (!x.workspace || x.workspace_bytes < l.bytes || !aligned16(x.workspace))
    return fail_arg("or_varlen_bwd: a 16-byte aligned workspace of %lld bytes is needed", (long long)l.bytes);
  // a head's second row of statistics lies 4 n_q bytes after the first, within the 32 bits of a buffer offset
  if ((int64_t)x.n_q * 4 + 256 >= (int64_t)0x7fffffff) return fail_arg("or_varlen_bwd: n_q must stay under 2^29");
  if (std::max(s.max_q_items, s.max_k_items) * x.H >= (int64_t)1 << 24)   // 2^32 threads
    return fail_arg("or_varlen_bwd: too many tiles");
  char* ws = (char*)x.workspace;
  BwdArgs a;
  a.q = (const uint16_t*)x.q;
  a.k = (const uint16_t*)x.k;
  a.v = (const uint16_t*)x.v;
  a.o = (const uint16_t*)x.o;
  a.d_o = (const uint16_t*)x.d_o;
  a.lse = x.lse;
  a.dlse = x.dlse;
  a.dq = (uint16_t*)x.dq;
  a.dk = (uint16_t*)x.dk;
  a.dv = (uint16_t*)x.dv;
  a.cu_q = x.cu_q;
  a.cu_k = x.cu_k;
  a.k_off = x.k_off;
  a.k_len = x.k_len;
  a.qs = x.q_row_stride;
  a.ks = x.k_row_stride;
  a.os = x.o_row_stride;
  a.dos = x.do_row_stride;
  a.lse_stride = x.lse_stride;
  a.n_seg = x.n_seg;
  a.n_q = x.n_q;
  a.n_k = x.n_k;
  a.H = x.H;
  a.scale = x.scale;
  a.slots_q = s.slots_q;
  a.slots_k = s.slots_k;
  a.tq = s.tq;
  a.tk = s.tk;
  a.max_q_items = (int32_t)s.max_q_items;
  a.max_k_items = (int32_t)s.max_k_items;
  a.head = (int32_t*)ws;
  a.q_items = (i32x4*)(ws + l.q_items);
  a.k_items = (i32x4*)(ws + l.k_items);
  a.q_split = (i32x4*)(ws + l.q_split);
  a.k_split = (i32x4*)(ws + l.k_split);
  a.stat = (float*)(ws + l.stat);
  a.part_q = (float*)(ws + l.part_q);
  a.part_k = (float*)(ws + l.part_k);
  hipStream_t st = (hipStream_t)stream;
  if (x.D == 128) s.fine ? launch<128, 1, true>(a, s, st) : launch<128, 1, false>(a, s, st);
  else if (s.fine) launch<64, 1, true>(a, s, st);
  else s.tq == 128 ? launch<64, 1, false>(a, s, st) : launch<64, 2, false>(a, s, st);
  return check_hip(hipGetLastError(), "attention backward launch");
}
