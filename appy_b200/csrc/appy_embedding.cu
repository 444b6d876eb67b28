// Embedding lookup and its gradient.
//
//   out[n, :]  = scale * W[token[n], :]                       (zeros where the token is outside [0, rows))
//   dW[v, :] (+)= scale * sum over { n : token[n] = v } of g[n, :]
//
// The gradient is a sum over iterations that store to one row: a loop over tokens is not parallel, and atomics on
// the row would add in an order that changes from run to run.  Here the positions are sorted by token (stable, so
// the sum of a row runs in the order of its positions), and the sorted positions are cut into shares of equal
// length, one per warp and 32 packs of columns, whatever their tokens: a frequent token takes many warps, rare ones
// share a warp.  A row that lies inside a share is written by it; a row cut by a share's border leaves float32 pieces
// in the workspace, and the warp that hands in the last piece folds them in share order.  Sums are float32
// throughout, rounded once.
//
// Up to 65536 positions one cluster of blocks sorts, and the blocks beside it clear the rows without tokens meanwhile: with a
// large vocabulary most of the gradient's bytes are those zeros, and the sort is hidden behind them.
#include <cooperative_groups.h>

#include "operators.cuh"

namespace {
using namespace appy_op;
namespace cg = cooperative_groups;

template <class I> APPY_DEV i64 token_at(const void* tokens, i64 n) { return (i64)__ldg(static_cast<const I*>(tokens) + n); }
APPY_DEV i64 token_of(const void* tokens, bool wide, i64 n) {
  return wide ? token_at<i64>(tokens, n) : token_at<int>(tokens, n);
}

// ------------------------------------------------------------------------------------------------ lookup
// Rows of at least 32 packs: a warp takes a stretch of one row, so that no pack needs an index of its own (65536 rows
// of 4096 bfloat16 117 us; the flat form, at 118 instructions per 32 packs, four fifths of all issue slots, 144).  Shorter
// rows: flat over the packs of the output, pack i of row i / per_row; neighbouring threads read one row, so token
// loads are broadcasts.
const int kLookupBlock = 256;

template <class T, int V, int U>
__global__ void __launch_bounds__(kLookupBlock) k_lookup(const T* __restrict__ w, i64 ldw, i64 rows, unsigned per_row,
                                                         const void* __restrict__ tokens, bool wide, i64 n, float scale,
                                                         T* __restrict__ out, i64 ldo) {
  const i64 total = n * per_row, base = (i64)blockIdx.x * (kLookupBlock * U) + threadIdx.x;
  i64 tok[U], row[U];
  unsigned col[U];
  Pack<T, V> k[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const i64 i = base + u * kLookupBlock;
    tok[u] = -1;
    if (i < total) {
      row[u] = total <= 0xffffffffll ? (i64)((unsigned)i / per_row) : i / per_row;
      col[u] = (unsigned)(i - row[u] * per_row);
      tok[u] = token_of(tokens, wide, row[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    k[u] = zero_pack<T, V>();
    if (tok[u] >= 0 && tok[u] < rows) k[u] = ld_keep<T, V>(w + tok[u] * ldw + (i64)col[u] * V);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (base + u * kLookupBlock >= total) continue;
    if (scale != 1.f && tok[u] >= 0 && tok[u] < rows) {
      float f[V];
      unpack<T, V>(k[u], f);
#pragma unroll
      for (int x = 0; x < V; ++x) f[x] *= scale;
      k[u] = pack<T, V>(f);
    }
    st_stream<T, V>(out + row[u] * ldo + (i64)col[u] * V, k[u]);
  }
}

// A warp takes `stretch` neighbouring packs of a row (elements, where packs cannot move it), U of them in flight a lane.
template <class T, int V, int U>
__global__ void __launch_bounds__(kLookupBlock) k_lookup_rows(const T* __restrict__ w, i64 ldw, i64 rows, i64 per_row, int parts, int stretch,
                                                              const void* __restrict__ tokens, bool wide, i64 n, float scale,
                                                              T* __restrict__ out, i64 ldo) {
  const int lane = threadIdx.x & 31;
  const i64 unit = (i64)blockIdx.x * (kLookupBlock / 32) + (threadIdx.x >> 5), row = unit / parts;
  if (row >= n) return;
  const i64 lo = (unit - row * parts) * stretch, tok = token_of(tokens, wide, row);
  const int count = (int)min((i64)stretch, per_row - lo);
  const bool known = tok >= 0 && tok < rows;
  const T* const from = w + (known ? tok * ldw : 0) + lo * V;
  T* const to = out + row * ldo + lo * V;
  for (int c = lane; c < count; c += 32 * U) {
    Pack<T, V> k[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      k[u] = zero_pack<T, V>();
      if (known && c + 32 * u < count) k[u] = ld_keep<T, V>(from + (c + 32 * u) * V);
    }
    if (scale != 1.f && known) {                   // the zeros of an unknown token stay +0 whatever the scale
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[V];
        unpack<T, V>(k[u], f);
        floats<V>(mul<V>(vec<V>(f), all<V>(scale)), f);
        k[u] = pack<T, V>(f);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c + 32 * u < count) st_stream<T, V>(to + (c + 32 * u) * V, k[u]);
  }
}

// ------------------------------------------------------------------------------------------------ sort by token
// Stable radix sort of (key, position), least significant digit first.  The key of a position is its token, or
// `rows` for one that is dropped, so dropped positions come last.  A block owns a contiguous range of positions;
// k_count counts its digits, k_place adds up what lies before them and writes the range out in order.
const int kSortBlock = 256, kSortItems = 16, kSortTile = kSortBlock * kSortItems, kSortMaxBlocks = 256, kDigits = 512;

struct SortPass {
  const void* tokens;        // first pass: keys come from here, positions are the index
  bool wide;
  i64 rows;
  const int* key_in;
  const int* pos_in;
  int* key_out;
  int* pos_out;
  int* counts;               // [block][digit]
  int n, per_block, shift, digits;
  int* zero;                 // counters that the sum wants at zero
  int zeros;
};

APPY_DEV int sort_key(const SortPass& p, int i) {
  if (!p.tokens) return __ldg(p.key_in + i);
  const i64 t = token_of(p.tokens, p.wide, i);
  return (int)(t >= 0 && t < p.rows ? t : p.rows);
}

__global__ void __launch_bounds__(kSortBlock) k_count(SortPass p) {
  __shared__ int hist[kDigits];
  for (int d = threadIdx.x; d < p.digits; d += kSortBlock) hist[d] = 0;
  for (int x = blockIdx.x * kSortBlock + threadIdx.x; x < p.zeros; x += gridDim.x * kSortBlock) p.zero[x] = 0;
  __syncthreads();
  const i64 lo = (i64)blockIdx.x * p.per_block, hi = lo + p.per_block < p.n ? lo + p.per_block : p.n;
  for (i64 i = lo + threadIdx.x; i < hi; i += kSortBlock) atomicAdd(&hist[(sort_key(p, (int)i) >> p.shift) & (p.digits - 1)], 1);
  __syncthreads();
  for (int d = threadIdx.x; d < p.digits; d += kSortBlock) p.counts[blockIdx.x * p.digits + d] = hist[d];
}

__global__ void __launch_bounds__(kSortBlock) k_place(SortPass p) {
  const int kWarps = kSortBlock / 32, kRounds = kSortItems;
  __shared__ int base[kDigits];                  // where the next key with this digit goes
  __shared__ int warp_count[kWarps][kDigits];
  __shared__ int warp_sum[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nblocks = gridDim.x;
  // base[d] = keys with a smaller digit anywhere + keys with this digit in earlier blocks
  const int per_thread = (p.digits + kSortBlock - 1) / kSortBlock;       // 1 or 2 neighbouring digits per thread
  int total[2] = {0, 0}, before[2] = {0, 0};
  for (int b = 0; b < nblocks; ++b)
    for (int x = 0; x < per_thread; ++x) {
      const int d = threadIdx.x * per_thread + x;
      if (d >= p.digits) continue;
      const int c = __ldg(p.counts + b * p.digits + d);
      if (b < (int)blockIdx.x) before[x] += c;
      total[x] += c;
    }
  int sum = total[0] + total[1], incl = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(APPY_FULL_MASK, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int excl = incl - sum;
  for (int w = 0; w < warp; ++w) excl += warp_sum[w];
  for (int x = 0; x < per_thread; ++x) {
    const int d = threadIdx.x * per_thread + x;
    if (d < p.digits) base[d] = excl + before[x];
    excl += total[x];
  }
  const i64 lo = (i64)blockIdx.x * p.per_block, hi = lo + p.per_block < p.n ? lo + p.per_block : p.n;
  for (i64 tile = lo; tile < hi; tile += kSortTile) {
    for (int d = threadIdx.x; d < kWarps * p.digits; d += kSortBlock) warp_count[d / p.digits][d % p.digits] = 0;
    __syncthreads();
    // a warp takes 32 * kRounds consecutive positions, 32 at a time: lane order is position order
    int key[kRounds], pos[kRounds], rank[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const i64 i = tile + warp * (32 * kRounds) + r * 32 + lane;
      key[r] = -1;
      if (i < hi) {
        key[r] = sort_key(p, (int)i);
        pos[r] = p.tokens ? (int)i : __ldg(p.pos_in + i);
      }
    }
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int d = key[r] < 0 ? -1 : (key[r] >> p.shift) & (p.digits - 1);
      const unsigned peers = __match_any_sync(APPY_FULL_MASK, d);
      const unsigned below = peers & ((1u << lane) - 1);
      rank[r] = d < 0 ? 0 : warp_count[warp][d] + __popc(below);
      __syncwarp();
      if (d >= 0 && below == 0) warp_count[warp][d] += __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    // counts of the warps -> first place of each warp's keys; base moves on past the tile
    for (int d = threadIdx.x; d < p.digits; d += kSortBlock) {
      int at = base[d];
      for (int w = 0; w < kWarps; ++w) {
        const int c = warp_count[w][d];
        warp_count[w][d] = at;
        at += c;
      }
      base[d] = at;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      if (key[r] >= 0) {
        const int to = warp_count[warp][(key[r] >> p.shift) & (p.digits - 1)] + rank[r];
        p.key_out[to] = key[r];
        p.pos_out[to] = pos[r];
      }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ sort and clear
// The same sort in one launch for up to 16 * 4096 positions: a cluster of blocks of 1024 threads, ITEMS keys a thread,
// which meet at cluster barriers instead of launch boundaries.  Pairs travel between passes through global memory
// (L2).  All other blocks of the grid clear rows: each finds out from the tokens which of its rows have none.
const int kOneBlock = 1024, kOneWarps = kOneBlock / 32, kClearRows = 65536;

struct OneSort {
  const void* tokens;
  bool wide;
  int n, rows, passes, digit_bits;
  int* key;                  // results
  int* pos;
  u64* between;              // [2][n] (key, position) pairs
  int* counts;               // [blocks of the cluster][kDigits]
  int* zero;                 // counters that the sum wants at zero
  int zeros;
  char* out;                 // NULL: nothing to clear
  i64 row_bytes, ld_bytes;
};

APPY_DEV void clear_bytes(char* p, i64 bytes, int lane) {        // p and bytes are even; one warp
  const i64 head = min((i64)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15), bytes), body = (bytes - head) / 16;
  for (i64 x = 2 * lane; x < head; x += 64) *reinterpret_cast<unsigned short*>(p + x) = 0;
  for (i64 x = lane; x < body; x += 32) __stcs(reinterpret_cast<uint4*>(p + head) + x, make_uint4(0, 0, 0, 0));
  for (i64 x = head + body * 16 + 2 * lane; x < bytes; x += 64) *reinterpret_cast<unsigned short*>(p + x) = 0;
}

template <int ITEMS, int C>
__global__ void __launch_bounds__(kOneBlock, 1) k_sort_clear(OneSort a) {
  __shared__ __align__(16) unsigned short warp_count[kOneWarps][kDigits];
  __shared__ int base[kDigits];
  __shared__ int warp_sum[kDigits / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (blockIdx.x >= C) {                           // clears rows [lo, hi), kClearRows at a time
    unsigned* const seen = reinterpret_cast<unsigned*>(&warp_count[0][0]);
    const i64 part = blockIdx.x - C, parts = gridDim.x - C;
    const i64 lo = a.rows * part / parts, hi = a.rows * (part + 1) / parts;
    for (i64 r0 = lo; r0 < hi; r0 += kClearRows) {
      const int count = (int)min((i64)kClearRows, hi - r0);
      for (int x = tid; x < (count + 31) / 32; x += kOneBlock) seen[x] = 0;
      __syncthreads();
      for (int i = tid; i < a.n; i += 4 * kOneBlock) {
        i64 t[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) t[u] = i + u * kOneBlock < a.n ? token_of(a.tokens, a.wide, i + u * kOneBlock) - r0 : -1;
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (t[u] >= 0 && t[u] < count) atomicOr(&seen[t[u] >> 5], 1u << (t[u] & 31));
      }
      __syncthreads();
      for (int r = warp; r < count; r += kOneWarps)
        if (!(seen[r >> 5] >> (r & 31) & 1)) clear_bytes(a.out + (r0 + r) * a.ld_bytes, a.row_bytes, lane);
      __syncthreads();
    }
    return;
  }
  const int block = blockIdx.x, digits = 1 << a.digit_bits, per = (a.n + C - 1) / C, lo = min(block * per, a.n), hi = min(lo + per, a.n);
  for (int x = block * kOneBlock + tid; x < a.zeros; x += C * kOneBlock) a.zero[x] = 0;
  auto meet = [] {
    if constexpr (C > 1) cg::this_cluster().sync();
    else __syncthreads();
  };
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.digit_bits;
    for (int x = tid; x < kOneWarps * kDigits / 8; x += kOneBlock) reinterpret_cast<uint4*>(&warp_count[0][0])[x] = make_uint4(0, 0, 0, 0);
    int key[ITEMS], pos[ITEMS], rank[ITEMS];
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const int i = lo + warp * (32 * ITEMS) + r * 32 + lane;
      key[r] = -1;
      if (i < hi) {
        if (pass == 0) {
          const i64 t = token_of(a.tokens, a.wide, i);
          key[r] = (int)(t >= 0 && t < a.rows ? t : a.rows);
          pos[r] = i;
        } else {
          const u64 k = __ldcg(a.between + (i64)((pass - 1) & 1) * a.n + i);
          key[r] = (int)(k >> 32);
          pos[r] = (int)k;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const int d = key[r] < 0 ? -1 : (key[r] >> shift) & (digits - 1);
      const unsigned peers = __match_any_sync(APPY_FULL_MASK, d);
      const unsigned below = peers & ((1u << lane) - 1);
      rank[r] = d < 0 ? 0 : warp_count[warp][d] + __popc(below);
      __syncwarp();
      if (d >= 0 && below == 0) warp_count[warp][d] += (unsigned short)__popc(peers);
      __syncwarp();
    }
    __syncthreads();
    int mine = 0;
    if (tid < digits) {
#pragma unroll 8
      for (int w = 0; w < kOneWarps; ++w) {
        const int c = warp_count[w][tid];
        warp_count[w][tid] = (unsigned short)mine;
        mine += c;
      }
      if (C > 1) __stcg(a.counts + block * kDigits + tid, mine);
    }
    if (C > 1) meet();
    if (tid < kDigits) {
      int total = 0, before = 0;
      if (tid < digits) {
#pragma unroll
        for (int b = 0; b < C; ++b) {
          const int c = C > 1 ? __ldcg(a.counts + b * kDigits + tid) : mine;
          before += b < block ? c : 0;
          total += c;
        }
      }
      int incl = total;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(APPY_FULL_MASK, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) warp_sum[warp] = incl;
      base[tid] = incl - total + before;
    }
    __syncthreads();
    if (tid < kDigits) {
      int add = 0;
      for (int w = 0; w < warp; ++w) add += warp_sum[w];
      base[tid] += add;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
      if (key[r] >= 0) {
        const int d = (key[r] >> shift) & (digits - 1), to = base[d] + warp_count[warp][d] + rank[r];
        if (pass == a.passes - 1) {
          a.key[to] = key[r];
          a.pos[to] = pos[r];
        } else {
          __stcg(a.between + (i64)(pass & 1) * a.n + to, (u64)key[r] << 32 | (unsigned)pos[r]);
        }
      }
    if (pass < a.passes - 1) meet();
  }
}

// Rows without tokens become zero, for sorted keys.  A block takes 32 rows: lane r of warp 0 looks row r up.
__global__ void __launch_bounds__(256) k_clear_rows(const int* __restrict__ key, int n, i64 rows, char* out, i64 row_bytes, i64 ld_bytes) {
  __shared__ unsigned empty;
  const i64 row0 = (i64)blockIdx.x * 32;
  if (threadIdx.x < 32) {
    const i64 row = row0 + threadIdx.x;
    int first = 0, last = n;
    while (first < last) {
      const int mid = first + (last - first) / 2;
      if (__ldg(key + mid) < row) first = mid + 1; else last = mid;
    }
    const bool none = row < rows && (first == n || __ldg(key + first) != row);
    const unsigned m = __ballot_sync(APPY_FULL_MASK, none);
    if (threadIdx.x == 0) empty = m;
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < 32; r += 8)
    if (empty >> r & 1) clear_bytes(out + (row0 + r) * ld_bytes, row_bytes, threadIdx.x & 31);
}

// ------------------------------------------------------------------------------------------------ sum by token
const int kSumBlock = 256, kSumWarps = kSumBlock / 32, kSumAhead = 4;

struct SumArgs {
  const int* key;            // sorted; keys >= rows are dropped positions
  const int* pos;
  int n, rows, share, shares, col_warps;
  i64 width, ldg, ldo;
  float scale;
  bool accumulate;
  float* pieces;             // [share][head, tail][width padded to packs]
  i64 piece_ld;
  int* arrived;              // [share][col_warps]: pieces handed in of the row that runs out of this share
};

// One thread writes an element of a row.  Adding to float32 by `red` has nothing to wait for, but it takes subnormal operands
// and results for zero.  From 2^-101 on that cannot be seen: a subnormal it is added to is less than half a step of the sum,
// and what it cancels with is a multiple of 2^-125, so the difference is zero or normal.  Packs with smaller values, zeros
// among them, are loaded, added up and stored (16384 x 2048 float32 into 32000 rows: all packs that way 83 us, 63 so).
template <class O, int V> APPY_DEV void write_row(O* out, i64 at, const float (&acc)[V], float scale, bool accumulate) {
  float f[V], least = __int_as_float(0x7f800000);
#pragma unroll
  for (int x = 0; x < V; ++x) f[x] = acc[x] * scale;
  if (accumulate) {
    if constexpr (sizeof(O) == 4) {
#pragma unroll
      for (int x = 0; x < V; ++x) least = fminf(least, fabsf(f[x]));
      if (least >= __int_as_float((127 - 101) << 23)) {
        if constexpr (V >= 4) {
#pragma unroll
          for (int x = 0; x < V; x += 4)
            asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(out + at + x), "f"(f[x]), "f"(f[x + 1]), "f"(f[x + 2]),
                         "f"(f[x + 3]) : "memory");
        } else {
#pragma unroll
          for (int x = 0; x < V; ++x) asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(out + at + x), "f"(f[x]) : "memory");
        }
        return;
      }
    }
    float old[V];
    unpack<O, V>(ld_plain<O, V>(out + at), old);
#pragma unroll
    for (int x = 0; x < V; ++x) f[x] += old[x];
  }
  st_plain<O, V>(out + at, pack<O, V>(f));
}

// written by other blocks of this launch: not from L1
template <int V> APPY_DEV Pack<float, V> ld_shared(const float* p) {
  if constexpr (V == 8) return {Raw32{__ldcg(reinterpret_cast<const uint4*>(p)), __ldcg(reinterpret_cast<const uint4*>(p) + 1)}};
  else return {__ldcg(reinterpret_cast<const typename Raw<4 * V>::type*>(p))};
}

// Hands in a piece of row `cur` (the head of this share, or its tail); the warp that hands in the last one folds the
// row.  Not inlined: the sum's loop would be many times as long.
template <class O, int V>
__device__ __noinline__ void hand_in(const SumArgs& a, O* out, int share, int col_warp, int cur, bool head, bool runs_on, Pack<float, V> sum) {
  const int lane = threadIdx.x & 31;
  const i64 col = ((i64)col_warp * 32 + lane) * V;
  const bool live = col < a.width;
  if (live) st_plain<float, V>(a.pieces + ((i64)share * 2 + !head) * a.piece_ld + col, sum);
  // the shares that the row begins and ends in: it runs on over a border if the key there is still the row's
  int owner = share, last = share;
  if (head)
    for (;;) {
      const int at = owner - lane;
      const int run = __ffs(~__ballot_sync(APPY_FULL_MASK, at > 0 && __ldg(a.key + (i64)at * a.share - 1) == cur));      // 0: all 32
      owner -= run ? run - 1 : 32;
      if (run) break;
    }
  if (runs_on)
    for (;;) {
      const i64 at = (i64)(last + 1 + lane) * a.share;
      const int run = __ffs(~__ballot_sync(APPY_FULL_MASK, at < a.n && __ldg(a.key + at) == cur));
      last += run ? run - 1 : 32;
      if (run) break;
    }
  __threadfence();
  __syncwarp();
  int n = 0;
  if (lane == 0) n = atomicAdd(a.arrived + (i64)owner * a.col_warps + col_warp, 1);
  n = __shfl_sync(APPY_FULL_MASK, n, 0);
  if (n != last - owner) return;
  __threadfence();
  if (!live) return;
  const float* from = a.pieces + (i64)owner * 2 * a.piece_ld + col;
  float total[V];
  unpack<float, V>(ld_shared<V>(from + a.piece_ld), total);
  int s = owner + 1;
  for (; s + 4 <= last + 1; s += 4) {              // a frequent token has hundreds of pieces: four at a time
    Pack<float, V> k[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) k[u] = ld_shared<V>(from + (i64)(s - owner + u) * 2 * a.piece_ld);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float f[V];
      unpack<float, V>(k[u], f);
#pragma unroll
      for (int x = 0; x < V; ++x) total[x] += f[x];
    }
  }
  for (; s <= last; ++s) {
    float f[V];
    unpack<float, V>(ld_shared<V>(from + (i64)(s - owner) * 2 * a.piece_ld), f);
#pragma unroll
    for (int x = 0; x < V; ++x) total[x] += f[x];
  }
  write_row<O, V>(out, (i64)cur * a.ldo + col, total, a.scale, a.accumulate);
}

// A warp takes one share and 32 packs of columns, kSumAhead rows in flight before it adds up the kSumAhead before
// them: 24 warps to an SM with 4 to 8 rows of 512 bytes each keep 48 to 96 KB in flight.  At 80 registers the 16-bit packs
// spill 108 bytes.  Two blocks to an SM with 128 registers, which spill nothing: 51 us for 53 (16384 x 4096 bfloat16 into 600
// rows) but 64 for 60 (5003 x 769 float32).
template <class T, class O, int V>
__global__ void __launch_bounds__(kSumBlock, 3) k_sum_rows(const __grid_constant__ SumArgs a, const T* __restrict__ g, O* __restrict__ out) {
  constexpr int U = kSumAhead;
  const int lane = threadIdx.x & 31;
  const i64 unit = (i64)blockIdx.x * kSumWarps + (threadIdx.x >> 5);
  const int share = (int)(unit / a.col_warps), col_warp = (int)(unit - (i64)share * a.col_warps);
  if (share >= a.shares) return;
  const i64 col = ((i64)col_warp * 32 + lane) * V;
  const bool live = col < a.width;
  const int lo = share * a.share, hi = min(lo + a.share, a.n);
  // keys and positions of 32 rows, one per lane, and of the next 32
  int key = a.rows, pos = 0, key_next = a.rows, pos_next = 0;
  if (lo + lane < hi) key = __ldg(a.key + lo + lane), pos = __ldg(a.pos + lo + lane);
  if (lo + 32 + lane < hi) key_next = __ldg(a.key + lo + 32 + lane), pos_next = __ldg(a.pos + lo + 32 + lane);
  const int before = lo > 0 ? __ldg(a.key + lo - 1) : -1;
  int cur = __shfl_sync(APPY_FULL_MASK, key, 0);
  if (cur >= a.rows) return;
  bool open_left = before == cur;                  // the current row began in an earlier share
  float acc[V];
#pragma unroll
  for (int x = 0; x < V; ++x) acc[x] = 0.f;
  const T* const from = g + (live ? col : 0);
  Pack<T, V> k[2][U];
  // rows past the share and dropped ones read the first row again, for nothing, and are not added
  auto issue = [&](Pack<T, V> (&to)[U], int pos32, int b) {
#pragma unroll
    for (int u = 0; u < U; ++u) to[u] = ld_stream<T, V>(from + (i64)__shfl_sync(APPY_FULL_MASK, pos32, b + u) * a.ldg);
  };
  issue(k[0], key < a.rows ? pos : 0, 0);
  for (int s0 = lo; s0 < hi; s0 += 32) {
    const bool here = key < a.rows;                // dropped keys come last, so these are the first lanes
    const int count = __popc(__ballot_sync(APPY_FULL_MASK, here));
    const int left = __shfl_up_sync(APPY_FULL_MASK, key, 1);
    const unsigned turns = __ballot_sync(APPY_FULL_MASK, here && key != (lane ? left : cur));      // rows that begin here
    const int at = here ? pos : 0, at_next = key_next < a.rows ? pos_next : 0;
#pragma unroll
    for (int b = 0; b < 32; b += U) {
      if (b + U < 32) issue(k[(b / U + 1) & 1], at, b + U);
      else issue(k[0], at_next, 0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (turns >> (b + u) & 1) {
          if (open_left) hand_in<O, V>(a, out, share, col_warp, cur, true, false, pack<float, V>(acc));
          else if (live) write_row<O, V>(out, (i64)cur * a.ldo + col, acc, a.scale, a.accumulate);
          open_left = false;
          cur = __shfl_sync(APPY_FULL_MASK, key, b + u);
          unpack<T, V>(k[(b / U) & 1][u], acc);
        } else if (b + u < count) {
          float f[V];
          unpack<T, V>(k[(b / U) & 1][u], f);
#pragma unroll
          for (int x = 0; x < V; ++x) acc[x] += f[x];
        }
      }
    }
    if (count < 32) break;
    key = key_next;
    pos = pos_next;
    key_next = a.rows;
    if (s0 + 64 + lane < hi) key_next = __ldg(a.key + s0 + 64 + lane), pos_next = __ldg(a.pos + s0 + 64 + lane);
  }
  const bool runs_on = hi < a.n && __ldg(a.key + hi) == cur;
  if (open_left || runs_on) hand_in<O, V>(a, out, share, col_warp, cur, open_left, runs_on, pack<float, V>(acc));
  else if (live) write_row<O, V>(out, (i64)cur * a.ldo + col, acc, a.scale, a.accumulate);
}

// ------------------------------------------------------------------------------------------------ few positions
// Up to kFewTokens positions need no sort: a warp takes one position and 32 packs of columns, and, if it is the first
// with its token, adds up the rows of all positions with that token, which it finds by looking through the tokens in
// shared memory.  The blocks behind those clear the rows without tokens.  One launch.  (Rows of 1024 bfloat16 added to
// float32 ones, microseconds here / by way of the sort: 16 positions 4 / 20, 512 positions 12 / 21, but 512 positions of
// one token, which one warp per 256 columns adds up, 59 / 22; so no more than 256.)
const int kFewTokens = 256;

struct FewArgs {
  const void* tokens;
  bool wide;
  int n, rows, col_warps, blocks;
  i64 width, ldg, ldo;
  float scale;
  bool accumulate;
  i64 row_bytes, ld_bytes;
};

template <class T, class O, int V>
__global__ void __launch_bounds__(256) k_few(FewArgs a, const T* __restrict__ g, O* __restrict__ out) {
  __shared__ int token[kFewTokens];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < kFewTokens; i += 256) {
    const i64 t = i < a.n ? token_of(a.tokens, a.wide, i) : -1;
    token[i] = t >= 0 && t < a.rows ? (int)t : -1;
  }
  __syncthreads();
  if ((int)blockIdx.x >= a.blocks) {
    const i64 part = (i64)blockIdx.x - a.blocks, parts = (i64)gridDim.x - a.blocks;
    const i64 lo = a.rows * part / parts, hi = a.rows * (part + 1) / parts;
    __shared__ unsigned seen[kClearRows / 8 / 32];
    const int chunk = kClearRows / 8;
    for (i64 r0 = lo; r0 < hi; r0 += chunk) {
      const int count = (int)min((i64)chunk, hi - r0);
      for (int x = tid; x < (count + 31) / 32; x += 256) seen[x] = 0;
      __syncthreads();
      for (int i = tid; i < a.n; i += 256) {
        const i64 t = token[i] - r0;
        if (token[i] >= 0 && t >= 0 && t < count) atomicOr(&seen[t >> 5], 1u << (t & 31));
      }
      __syncthreads();
      for (int r = warp; r < count; r += 8)
        if (!(seen[r >> 5] >> (r & 31) & 1)) clear_bytes(reinterpret_cast<char*>(out) + (r0 + r) * a.ld_bytes, a.row_bytes, lane);
      __syncthreads();
    }
    return;
  }
  const int unit = blockIdx.x * 8 + warp, i = unit / a.col_warps, col_warp = unit - i * a.col_warps;
  if (i >= a.n) return;
  const int mine = token[i];
  if (mine < 0) return;
  for (int x = 0; x < i; x += 32)                  // an earlier position has the token: its warp sees to it
    if (__any_sync(APPY_FULL_MASK, x + lane < i && token[x + lane] == mine)) return;
  const i64 col = ((i64)col_warp * 32 + lane) * V;
  const bool live = col < a.width;
  const T* const from = g + (live ? col : 0);
  float acc[V];
#pragma unroll
  for (int x = 0; x < V; ++x) acc[x] = 0.f;
  for (int x = i / 32 * 32; x < a.n; x += 32) {
    unsigned m = __ballot_sync(APPY_FULL_MASK, token[x + lane] == mine);
    while (m) {
      constexpr int U = 8;                         // rows in flight: one warp sees to a frequent token alone
      Pack<T, V> k[U];
      unsigned left = m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (left) k[u] = ld_stream<T, V>(from + (i64)(x + __ffs(left) - 1) * a.ldg);
        left &= left - 1;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!m) break;
        m &= m - 1;
        float f[V];
        unpack<T, V>(k[u], f);
#pragma unroll
        for (int y = 0; y < V; ++y) acc[y] += f[y];
      }
    }
  }
  if (live) write_row<O, V>(out, (i64)mine * a.ldo + col, acc, a.scale, a.accumulate);
}

// ------------------------------------------------------------------------------------------------ host side
int bits_of(i64 v) {
  int b = 0;
  while (v) { ++b; v >>= 1; }
  return b;
}
size_t round256(size_t v) { return (v + 255) / 256 * 256; }

struct GradPlan {
  int cluster, items;        // one sort launch, or (cluster 0) two per pass
  int blocks, per_block, passes, digit_bits, share, shares, col_warps, counters;
  size_t counts_at, key_at[2], pos_at[2], between_at, pieces_at, arrived_at, bytes;
  i64 piece_ld;
};

GradPlan grad_plan(i64 n, i64 rows, i64 width, int vec) {
  GradPlan p;
  // 2048 keys a block up to 16 blocks, then up to 4096: a wider cluster has fewer rounds per pass but slower barriers
  // (16384 keys: 8 and 16 blocks alike, 4 blocks 6 us more; 4096 keys: 1 to 8 blocks within 2 us)
  p.cluster = 1;
  while (p.cluster < 16 && n > (i64)p.cluster * 2 * kOneBlock) p.cluster *= 2;
  const i64 items = (n + (i64)p.cluster * kOneBlock - 1) / ((i64)p.cluster * kOneBlock);
  p.items = items <= 1 ? 1 : items <= 2 ? 2 : 4;
  if (items > 4) p.cluster = 0;
  const i64 tiles = std::max<i64>(1, (n + kSortTile - 1) / kSortTile);
  const i64 per = (tiles + kSortMaxBlocks - 1) / kSortMaxBlocks;
  p.per_block = (int)(per * kSortTile);
  p.blocks = (int)((tiles + per - 1) / per);
  const int bits = std::max(1, bits_of(rows));                 // keys run from 0 to rows
  p.passes = (bits + 8) / 9;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  const i64 packs = std::max<i64>(1, (width + vec - 1) / vec);
  p.col_warps = (int)((packs + 31) / 32);
  // shares of 32 to 1024 positions, so many that the warps make two rounds on all SMs (24 of them to an SM at a time)
  const i64 want = (i64)148 * 24 * 2;
  const i64 share = (n * p.col_warps / want + 31) / 32 * 32;
  p.share = (int)std::min<i64>(1024, std::max<i64>(32, share));
  p.shares = (int)((n + p.share - 1) / p.share);
  p.counters = (int)std::min<i64>((i64)p.shares * p.col_warps, 0x7fffffff);
  p.piece_ld = packs * vec;
  size_t at = 0;
  p.counts_at = at; at += round256((size_t)std::max(p.blocks, 16) * kDigits * sizeof(int));
  for (int x = 0; x < 2; ++x) {
    p.key_at[x] = at; at += round256((size_t)n * sizeof(int));
    p.pos_at[x] = at; at += round256((size_t)n * sizeof(int));
  }
  p.between_at = at; at += round256(p.cluster ? (size_t)n * 2 * sizeof(u64) : 0);
  p.arrived_at = at; at += round256((size_t)p.shares * p.col_warps * sizeof(int));
  p.pieces_at = at; at += round256((size_t)p.shares * 2 * p.piece_ld * sizeof(float));
  p.bytes = at;
  return p;
}

template <int ITEMS, int C> int launch_one(const OneSort& a, bool clear, cudaStream_t s) {
  const auto kernel = k_sort_clear<ITEMS, C>;
  cudaLaunchConfig_t cfg = {};
  // one block to an SM, and as many clusters as run at once: a GPC of 16 to 20 SMs holds one of 16 blocks, two of 8
  const int fit = std::max(2 * C, C >= 8 ? std::min(128, sm_count()) / C * C : sm_count() / C * C);
  cfg.gridDim = dim3((unsigned)(clear ? fit : C));
  cfg.blockDim = dim3(kOneBlock);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  if (C > 8) {
    static signed char fits[16] = {0};             // per instantiation and device: 0 not known yet
    int dev = 0;
    cudaGetDevice(&dev);
    signed char known = dev >= 0 && dev < 16 ? fits[dev] : 0;
    if (!known) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return appy_fail_cuda(e, "embedding gradient set-up");
      known = cluster_fits(kernel, cfg) ? 1 : -1;
      if (dev >= 0 && dev < 16) fits[dev] = known;
    }
    if (known < 0) return kNoCluster;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return appy_fail_cuda(e, "embedding gradient sort launch");
  }
  return finish("embedding gradient sort launch");
}
// The forms that grad_plan asks for: one key a thread only in a block alone, four only in 16 blocks.
int launch_one(int items, int cluster, const OneSort& a, bool clear, cudaStream_t s) {
  if (items == 1) return launch_one<1, 1>(a, clear, s);
  if (items == 4) return launch_one<4, 16>(a, clear, s);
  switch (cluster) {
    case 1: return launch_one<2, 1>(a, clear, s);
    case 2: return launch_one<2, 2>(a, clear, s);
    case 4: return launch_one<2, 4>(a, clear, s);
    case 8: return launch_one<2, 8>(a, clear, s);
    default: return launch_one<2, 16>(a, clear, s);
  }
}

template <class T, class O, int V> int launch_sums(const SumArgs& a, const T* g, O* out, cudaStream_t s) {
  const i64 units = (i64)a.shares * a.col_warps;
  k_sum_rows<T, O, V><<<(unsigned)((units + kSumWarps - 1) / kSumWarps), kSumBlock, 0, s>>>(a, g, out);
  return finish("embedding gradient sum launch");
}

// Positions, rows and keys are int on the device: the end of the last share or tile, and the 64 positions that a warp looks ahead,
// must not pass 2^31.
bool grad_sizes(i64 n, i64 rows, i64 width) { return n >= 0 && n <= 0x7fff0000 && rows >= 0 && rows < 0x7fffffff && width >= 0; }

int grad_vec(const void* g, int dtype, i64 ldg, const void* out, int out_dtype, i64 ldo, i64 width) {
  // one pack per thread and position: 8 16-bit columns or 4 float32 ones, if rows start where such packs may
  const int V = dtype == APPY_F32 ? 4 : 8, so = element_size(out_dtype);
  const bool ok = width % V == 0 && ldg % V == 0 && ldo % V == 0 && aligned(g, 16) && aligned(out, so * V > 16 ? 16 : so * V);
  return ok ? V : 1;
}

}  // namespace

extern "C" {

int appy_embedding(const void* dweight, int dtype, int64_t ldw, int64_t rows, int64_t width, const void* dtokens, int token_dtype,
                   int64_t n, float scale, void* dout, int64_t ldo, void* stream) {
  static const char fn[] = "appy_embedding";
  const int size = element_size(dtype);
  if (!size) return fail_named(fn, "dtype must be APPY_F32, APPY_F16 or APPY_BF16");
  if (token_dtype != APPY_I32 && token_dtype != APPY_I64) return fail_named(fn, "token_dtype must be APPY_I32 or APPY_I64");
  if (rows < 0 || width < 0 || n < 0) return fail_named(fn, "negative size");
  if (n == 0 || width == 0) return APPY_OK;
  if (!dtokens || !dout || (!dweight && rows)) return fail_named(fn, "NULL argument");
  if (ldw < width || ldo < width) return fail_named(fn, "ldw and ldo must be at least width");
  if (width > 0x7fffffff) return fail_named(fn, "width must be below 2^31");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = token_dtype == APPY_I64;
  const int V = 16 / size;
  const bool vec = width % V == 0 && ldw % V == 0 && ldo % V == 0 && aligned(dweight, 16) && aligned(dout, 16);
  const i64 per_row = vec ? width / V : width, stretch = vec ? 128 : 512, parts = (per_row + stretch - 1) / stretch;
  const bool flat = vec && per_row < 32;
  const i64 blocks = flat ? (n * per_row + kLookupBlock * 4 - 1) / (kLookupBlock * 4) : (n * parts + kLookupBlock / 32 - 1) / (kLookupBlock / 32);
  if (blocks > 0x7fffffff) return fail_named(fn, "too many elements for one launch");
  return APPY_OP_DTYPE(dtype, {
    constexpr int W = 16 / sizeof(T);
    const T* w = static_cast<const T*>(dweight);
    T* out = static_cast<T*>(dout);
    if (flat)
      k_lookup<T, W, 4><<<(unsigned)blocks, kLookupBlock, 0, s>>>(w, ldw, rows, (unsigned)per_row, dtokens, wide, n, scale, out, ldo);
    else if (vec)
      k_lookup_rows<T, W, 4><<<(unsigned)blocks, kLookupBlock, 0, s>>>(w, ldw, rows, per_row, (int)parts, (int)stretch, dtokens, wide, n, scale, out, ldo);
    else
      k_lookup_rows<T, 1, 8><<<(unsigned)blocks, kLookupBlock, 0, s>>>(w, ldw, rows, per_row, (int)parts, (int)stretch, dtokens, wide, n, scale, out, ldo);
    return finish("embedding launch");
  });
}

int appy_embedding_grad_bytes(int64_t n, int64_t rows, int64_t width, size_t* bytes) {
  static const char fn[] = "appy_embedding_grad_bytes";
  if (!bytes) return fail_named(fn, "NULL argument");
  if (!grad_sizes(n, rows, width)) return fail_named(fn, "sizes must not be negative, n at most 2^31 - 2^16, rows below 2^31 - 1");
  size_t most = 0;
  for (int vec : {1, 4, 8}) most = std::max(most, grad_plan(n, rows, width, vec).bytes);
  *bytes = std::max<size_t>(most, 256);
  return APPY_OK;
}

int appy_embedding_grad(const void* dgrad, int dtype, int64_t ldg, const void* dtokens, int token_dtype, int64_t n, int64_t rows,
                        int64_t width, float scale, int accumulate, void* dout, int out_dtype, int64_t ldo, void* dworkspace,
                        size_t workspace_bytes, void* stream) {
  static const char fn[] = "appy_embedding_grad";
  if (!element_size(dtype)) return fail_named(fn, "dtype must be APPY_F32, APPY_F16 or APPY_BF16");
  if (out_dtype != dtype && out_dtype != APPY_F32) return fail_named(fn, "out_dtype must be dtype or APPY_F32");
  if (token_dtype != APPY_I32 && token_dtype != APPY_I64) return fail_named(fn, "token_dtype must be APPY_I32 or APPY_I64");
  if (!grad_sizes(n, rows, width)) return fail_named(fn, "sizes must not be negative, n at most 2^31 - 2^16, rows below 2^31 - 1");
  if (rows == 0 || width == 0) return APPY_OK;
  if (!dout || (n && (!dgrad || !dtokens || !dworkspace))) return fail_named(fn, "NULL argument");
  if (ldg < width || ldo < width) return fail_named(fn, "ldg and ldo must be at least width");
  const int V = grad_vec(dgrad, dtype, ldg, dout, out_dtype, ldo, width);
  const GradPlan p = grad_plan(n, rows, width, V);
  if (n && (workspace_bytes < p.bytes || !aligned(dworkspace, 256))) return fail_named(fn, "workspace too small or not aligned to 256 bytes");
  if (n <= kFewTokens && n * p.col_warps > 0x7fffffff) return fail_named(fn, "too many elements for one launch");
  if (n && n <= kFewTokens) {
    const int blocks = (int)((n * p.col_warps + 7) / 8);
    const FewArgs a{dtokens, token_dtype == APPY_I64, (int)n, (int)rows, p.col_warps, blocks, width, ldg, ldo, scale, accumulate != 0,
                    width * element_size(out_dtype), ldo * element_size(out_dtype)};
    // clearing: four blocks to an SM beside the sums
    const unsigned grid = (unsigned)(blocks + (accumulate ? 0 : std::min<i64>(rows, 4 * (i64)sm_count())));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return APPY_OP_DTYPE(dtype, {
      const T* g = static_cast<const T*>(dgrad);
      constexpr int W = 16 / sizeof(T);
      if (out_dtype == APPY_F32) {
        float* out = static_cast<float*>(dout);
        if (V == 1) k_few<T, float, 1><<<grid, 256, 0, s>>>(a, g, out);
        else k_few<T, float, W><<<grid, 256, 0, s>>>(a, g, out);
      } else {
        T* out = static_cast<T*>(dout);
        if (V == 1) k_few<T, T, 1><<<grid, 256, 0, s>>>(a, g, out);
        else k_few<T, T, W><<<grid, 256, 0, s>>>(a, g, out);
      }
      return finish("embedding gradient launch");
    });
  }
  if ((i64)p.shares * p.col_warps > 0x7fffffff) return fail_named(fn, "too many elements for one launch");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  char* const ws = static_cast<char*>(dworkspace);
  const bool wide = token_dtype == APPY_I64, clear = !accumulate;
  const i64 row_bytes = width * element_size(out_dtype), ld_bytes = ldo * element_size(out_dtype);
  char* const out_bytes = static_cast<char*>(dout);
  int* key[2];
  int* pos[2];
  for (int x = 0; x < 2; ++x) {
    key[x] = reinterpret_cast<int*>(ws + p.key_at[x]);
    pos[x] = reinterpret_cast<int*>(ws + p.pos_at[x]);
  }
  int* const arrived = reinterpret_cast<int*>(ws + p.arrived_at);
  int last = 0, rc = kNoCluster;
  if (p.cluster && n) {
    const OneSort q{dtokens, wide, (int)n, (int)rows, p.passes, p.digit_bits, key[0], pos[0], reinterpret_cast<u64*>(ws + p.between_at),
                    reinterpret_cast<int*>(ws + p.counts_at), arrived, p.counters, out_bytes, row_bytes, ld_bytes};
    rc = launch_one(p.items, p.cluster, q, clear, s);
    if (rc && rc != kNoCluster) return rc;
  }
  if (rc == kNoCluster) {                          // many positions, or no cluster that wide
    if (n)
      for (int pass = 0; pass < p.passes; ++pass) {
        SortPass q{pass ? nullptr : dtokens, wide, rows, key[(pass + 1) & 1], pos[(pass + 1) & 1], key[pass & 1], pos[pass & 1],
                   reinterpret_cast<int*>(ws + p.counts_at), (int)n, p.per_block, pass * p.digit_bits, 1 << p.digit_bits,
                   arrived, pass ? 0 : p.counters};
        k_count<<<p.blocks, kSortBlock, 0, s>>>(q);
        if (int rc = finish("embedding gradient count launch")) return rc;
        k_place<<<p.blocks, kSortBlock, 0, s>>>(q);
        if (int rc = finish("embedding gradient place launch")) return rc;
      }
    last = (p.passes - 1) & 1;
    if (clear) {
      k_clear_rows<<<(unsigned)((rows + 31) / 32), 256, 0, s>>>(key[last], (int)n, rows, out_bytes, row_bytes, ld_bytes);
      if (int rc = finish("embedding gradient clear launch")) return rc;
    }
  }
  if (!n) return APPY_OK;
  const SumArgs a{key[last], pos[last], (int)n, (int)rows, p.share, p.shares, p.col_warps, width, ldg, ldo, scale, accumulate != 0,
                  reinterpret_cast<float*>(ws + p.pieces_at), p.piece_ld, arrived};
  return APPY_OP_DTYPE(dtype, {
    const T* g = static_cast<const T*>(dgrad);
    if (out_dtype == APPY_F32) {
      float* out = static_cast<float*>(dout);
      return V == 1 ? launch_sums<T, float, 1>(a, g, out, s) : launch_sums<T, float, 16 / sizeof(T)>(a, g, out, s);
    }
    T* out = static_cast<T*>(dout);
    return V == 1 ? launch_sums<T, T, 1>(a, g, out, s) : launch_sums<T, T, 16 / sizeof(T)>(a, g, out, s);
  });
}

}  // extern "C"
