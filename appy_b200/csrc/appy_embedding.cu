// Embedding lookup and its gradient.
//
//   out[n, :]  = scale * W[token[n], :]                       (zeros where the token is outside [0, rows))
//   dW[v, :] (+)= scale * sum over { n : token[n] = v } of g[n, :]
//
// The gradient is a sum over iterations that store to one row: a loop over tokens is not parallel, and atomics on
// the row would add in an order that changes from run to run.  Here the positions are sorted by token (stable, so
// the sum of a row runs in the order of its positions), and the sorted positions are cut into shares of equal
// length, one per group of threads, whatever their tokens: a frequent token takes many groups, rare ones share a
// group.  A row that lies inside a share is written by it; a row cut by a share's border leaves float32 pieces in
// the workspace, which a second kernel folds in share order.  Sums are float32 throughout, rounded once.
#include "operators.cuh"

namespace {
using namespace appy_op;

template <class I> APPY_DEV i64 token_at(const void* tokens, i64 n) { return (i64)__ldg(static_cast<const I*>(tokens) + n); }
APPY_DEV i64 token_of(const void* tokens, bool wide, i64 n) {
  return wide ? token_at<i64>(tokens, n) : token_at<int>(tokens, n);
}

// ------------------------------------------------------------------------------------------------ lookup
// Flat over the packs of the output: pack i belongs to row i / per_row.  A thread has U packs a block apart in
// flight (token, then row); neighbouring threads read one row, so token loads are broadcasts.
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
};

APPY_DEV int sort_key(const SortPass& p, int i) {
  if (!p.tokens) return __ldg(p.key_in + i);
  const i64 t = token_of(p.tokens, p.wide, i);
  return (int)(t >= 0 && t < p.rows ? t : p.rows);
}

__global__ void __launch_bounds__(kSortBlock) k_count(SortPass p) {
  __shared__ int hist[kDigits];
  for (int d = threadIdx.x; d < p.digits; d += kSortBlock) hist[d] = 0;
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

// ------------------------------------------------------------------------------------------------ sum by token
const int kSumBlock = 256;

struct SumArgs {
  const int* key;            // sorted; keys >= rows are dropped positions
  const int* pos;
  int n, rows, share, shares;
  i64 width, ldg, ldo;
  float scale;
  bool accumulate;
  float* pieces;             // [share][head, tail][width padded to packs]
  i64 piece_ld;
};

template <class O, int V> APPY_DEV void write_row(O* out, i64 at, const float (&acc)[V], float scale, bool accumulate) {
  float f[V];
#pragma unroll
  for (int x = 0; x < V; ++x) f[x] = acc[x] * scale;
  if (accumulate) {
    float old[V];
    unpack<O, V>(ld_plain<O, V>(out + at), old);
#pragma unroll
    for (int x = 0; x < V; ++x) f[x] += old[x];
  }
  st_plain<O, V>(out + at, pack<O, V>(f));
}

// A group of `group` threads (a power of two, 32..256) takes one share and V columns per thread.
template <class T, class O, int V, int U>
__global__ void __launch_bounds__(kSumBlock) k_sum_rows(SumArgs a, const T* __restrict__ g, O* __restrict__ out, int group) {
  const int share = blockIdx.x * (kSumBlock / group) + threadIdx.x / group;
  const i64 col = ((i64)blockIdx.y * group + threadIdx.x % group) * V;
  if (share >= a.shares || col >= a.width) return;
  const int lo = share * a.share, hi = min(lo + a.share, a.n);
  int cur = __ldg(a.key + lo);
  if (cur >= a.rows) return;
  bool open_left = lo > 0 && __ldg(a.key + lo - 1) == cur;      // the current row began in an earlier share
  float* const head = a.pieces + (i64)share * 2 * a.piece_ld + col;
  float acc[V];
#pragma unroll
  for (int x = 0; x < V; ++x) acc[x] = 0.f;
  for (int s = lo; s < hi; s += U) {
    int key[U];
    Pack<T, V> k[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      key[u] = s + u < hi ? __ldg(a.key + s + u) : a.rows;
      k[u] = zero_pack<T, V>();
      if (key[u] < a.rows) k[u] = ld_stream<T, V>(g + (i64)__ldg(a.pos + s + u) * a.ldg + col);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (key[u] != cur && cur < a.rows && !(s + u >= hi)) {     // the current row ends here
        if (open_left) st_plain<float, V>(head, pack<float, V>(acc));
        else write_row<O, V>(out, (i64)cur * a.ldo + col, acc, a.scale, a.accumulate);
        open_left = false;
        cur = key[u];
#pragma unroll
        for (int x = 0; x < V; ++x) acc[x] = 0.f;
      }
      if (key[u] < a.rows) {
        float f[V];
        unpack<T, V>(k[u], f);
#pragma unroll
        for (int x = 0; x < V; ++x) acc[x] += f[x];
      }
    }
  }
  if (cur >= a.rows) return;
  const bool open_right = hi < a.n && __ldg(a.key + hi) == cur;
  if (open_left) st_plain<float, V>(head, pack<float, V>(acc));
  else if (open_right) st_plain<float, V>(head + a.piece_ld, pack<float, V>(acc));
  else write_row<O, V>(out, (i64)cur * a.ldo + col, acc, a.scale, a.accumulate);
}

// One block per (share whose last row begins in it and runs on, 32 packs): warps take contiguous parts of the
// row's head pieces, their sums are added in order.
const int kFoldWarps = 8;

template <class O, int V>
__global__ void __launch_bounds__(32 * kFoldWarps) k_fold_rows(SumArgs a, O* __restrict__ out) {
  __shared__ float part[kFoldWarps][32 * V];
  const int share = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int lo = share * a.share, hi = min(lo + a.share, a.n);
  if (hi >= a.n) return;
  const int cur = __ldg(a.key + hi - 1);
  if (cur >= a.rows || __ldg(a.key + hi) != cur) return;
  if (__ldg(a.key + lo) == cur && lo > 0 && __ldg(a.key + lo - 1) == cur) return;      // began earlier
  int first = hi, last = a.n;                      // the row's end: first position with a larger key
  while (first < last) {
    const int mid = first + (last - first) / 2;
    if (__ldg(a.key + mid) <= cur) first = mid + 1; else last = mid;
  }
  const int end_share = (first - 1) / a.share, pieces = end_share - share;
  const i64 col = ((i64)blockIdx.y * 32 + lane) * V;
  const bool live = col < a.width;
  float acc[V];
#pragma unroll
  for (int x = 0; x < V; ++x) acc[x] = 0.f;
  const int per = (pieces + kFoldWarps - 1) / kFoldWarps;
  if (live) {
    if (warp == 0) unpack<float, V>(ld_plain<float, V>(a.pieces + ((i64)share * 2 + 1) * a.piece_ld + col), acc);
    const int b = share + 1 + warp * per, e = min(b + per, end_share + 1);
#pragma unroll 4
    for (int s = b; s < e; ++s) {
      float f[V];
      unpack<float, V>(ld_plain<float, V>(a.pieces + (i64)s * 2 * a.piece_ld + col), f);
#pragma unroll
      for (int x = 0; x < V; ++x) acc[x] += f[x];
    }
  }
#pragma unroll
  for (int x = 0; x < V; ++x) part[warp][lane * V + x] = acc[x];
  __syncthreads();
  if (warp == 0 && live) {
    for (int w = 1; w < kFoldWarps; ++w)
#pragma unroll
      for (int x = 0; x < V; ++x) acc[x] += part[w][lane * V + x];
    write_row<O, V>(out, (i64)cur * a.ldo + col, acc, a.scale, a.accumulate);
  }
}

// Rows without tokens become zero.  A block takes 32 rows: lane r of warp 0 looks row r up among the sorted keys.
template <class O, int V>
__global__ void __launch_bounds__(256) k_clear_rows(const int* __restrict__ key, int n, i64 rows, i64 width, O* __restrict__ out, i64 ldo) {
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
  for (unsigned m = empty; m; m &= m - 1) {
    O* const r = out + (row0 + __ffs(m) - 1) * ldo;
    for (i64 c = (i64)threadIdx.x * V; c < width; c += 256 * V) st_stream<O, V>(r + c, zero_pack<O, V>());
  }
}

// ------------------------------------------------------------------------------------------------ host side
int bits_of(i64 v) {
  int b = 0;
  while (v) { ++b; v >>= 1; }
  return b;
}
size_t round256(size_t v) { return (v + 255) / 256 * 256; }

struct GradPlan {
  int blocks, per_block, passes, digit_bits, share, shares, group, col_blocks, vec;
  size_t counts_at, key_at[2], pos_at[2], pieces_at, bytes;
  i64 piece_ld;
};

// V = elements of 16 bytes of the wider of the two types where rows allow it, else 1.
GradPlan grad_plan(i64 n, i64 rows, i64 width, int vec) {
  GradPlan p;
  const i64 tiles = std::max<i64>(1, (n + kSortTile - 1) / kSortTile);
  const i64 per = (tiles + kSortMaxBlocks - 1) / kSortMaxBlocks;
  p.per_block = (int)(per * kSortTile);
  p.blocks = (int)((tiles + per - 1) / per);
  const int bits = std::max(1, bits_of(rows));                 // keys run from 0 to rows
  p.passes = (bits + 8) / 9;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  p.vec = vec;
  const i64 packs = std::max<i64>(1, (width + vec - 1) / vec);
  p.group = 32;
  while (p.group < kSumBlock && p.group < packs) p.group *= 2;
  p.col_blocks = (int)((packs + p.group - 1) / p.group);
  // shares: enough groups to fill the GPU (8 blocks of 256 threads per SM), 32 to 1024 positions each
  const i64 want = std::max<i64>(1, (i64)148 * 8 * (kSumBlock / p.group) / p.col_blocks);
  p.share = (int)std::min<i64>(1024, std::max<i64>(32, (n + want - 1) / want));
  p.shares = (int)((n + p.share - 1) / p.share);
  p.piece_ld = packs * vec;
  size_t at = 0;
  p.counts_at = at; at += round256((size_t)p.blocks * kDigits * sizeof(int));
  for (int x = 0; x < 2; ++x) {
    p.key_at[x] = at; at += round256((size_t)n * sizeof(int));
    p.pos_at[x] = at; at += round256((size_t)n * sizeof(int));
  }
  p.pieces_at = at; at += round256((size_t)p.shares * 2 * p.piece_ld * sizeof(float));
  p.bytes = at;
  return p;
}

template <class T, class O, int V>
int launch_sums(const GradPlan& p, const SumArgs& a, const T* g, O* out, cudaStream_t s) {
  if (!a.accumulate && a.rows > 0) {
    k_clear_rows<O, V><<<(unsigned)((a.rows + 31) / 32), 256, 0, s>>>(a.key, a.n, a.rows, a.width, out, a.ldo);
    if (int rc = finish("embedding gradient clear launch")) return rc;
  }
  if (!a.n) return APPY_OK;
  const int per_block = kSumBlock / p.group;
  k_sum_rows<T, O, V, 8><<<dim3((unsigned)((p.shares + per_block - 1) / per_block), (unsigned)p.col_blocks), kSumBlock, 0, s>>>(
      a, g, out, p.group);
  if (int rc = finish("embedding gradient sum launch")) return rc;
  if (p.shares < 2) return APPY_OK;
  k_fold_rows<O, V><<<dim3((unsigned)(p.shares - 1), (unsigned)((p.piece_ld / V + 31) / 32)), 32 * kFoldWarps, 0, s>>>(a, out);
  return finish("embedding gradient fold launch");
}

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
  const i64 per_row = vec ? width / V : width, total = n * per_row, blocks = (total + kLookupBlock * 4 - 1) / (kLookupBlock * 4);
  if (blocks > 0x7fffffff) return fail_named(fn, "too many elements for one launch");
  return APPY_OP_DTYPE(dtype, {
    const T* w = static_cast<const T*>(dweight);
    T* out = static_cast<T*>(dout);
    if (vec)
      k_lookup<T, 16 / sizeof(T), 4><<<(unsigned)blocks, kLookupBlock, 0, s>>>(w, ldw, rows, (unsigned)per_row, dtokens, wide, n, scale, out, ldo);
    else
      k_lookup<T, 1, 4><<<(unsigned)blocks, kLookupBlock, 0, s>>>(w, ldw, rows, (unsigned)per_row, dtokens, wide, n, scale, out, ldo);
    return finish("embedding launch");
  });
}

int appy_embedding_grad_bytes(int64_t n, int64_t rows, int64_t width, size_t* bytes) {
  static const char fn[] = "appy_embedding_grad_bytes";
  if (!bytes) return fail_named(fn, "NULL argument");
  if (rows < 0 || width < 0 || n < 0 || n >= 0x7fffffff || rows >= 0x7fffffff) return fail_named(fn, "sizes must be in [0, 2^31 - 1)");
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
  if (rows < 0 || width < 0 || n < 0 || n >= 0x7fffffff || rows >= 0x7fffffff) return fail_named(fn, "sizes must be in [0, 2^31 - 1)");
  if (rows == 0 || width == 0) return APPY_OK;
  if (!dout || (n && (!dgrad || !dtokens || !dworkspace))) return fail_named(fn, "NULL argument");
  if (ldg < width || ldo < width) return fail_named(fn, "ldg and ldo must be at least width");
  const int V = grad_vec(dgrad, dtype, ldg, dout, out_dtype, ldo, width);
  const GradPlan p = grad_plan(n, rows, width, V);
  if (n && (workspace_bytes < p.bytes || !aligned(dworkspace, 256))) return fail_named(fn, "workspace too small or not aligned to 256 bytes");
  if (p.col_blocks > 65535 || (p.piece_ld / V + 31) / 32 > 65535) return fail_named(fn, "width is too large");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  char* const ws = static_cast<char*>(dworkspace);
  int* key[2];
  int* pos[2];
  for (int x = 0; x < 2; ++x) {
    key[x] = reinterpret_cast<int*>(ws + p.key_at[x]);
    pos[x] = reinterpret_cast<int*>(ws + p.pos_at[x]);
  }
  if (n)
    for (int pass = 0; pass < p.passes; ++pass) {
      SortPass q{pass ? nullptr : dtokens, token_dtype == APPY_I64, rows, key[(pass + 1) & 1], pos[(pass + 1) & 1], key[pass & 1],
                 pos[pass & 1], reinterpret_cast<int*>(ws + p.counts_at), (int)n, p.per_block, pass * p.digit_bits, 1 << p.digit_bits};
      k_count<<<p.blocks, kSortBlock, 0, s>>>(q);
      if (int rc = finish("embedding gradient count launch")) return rc;
      k_place<<<p.blocks, kSortBlock, 0, s>>>(q);
      if (int rc = finish("embedding gradient place launch")) return rc;
    }
  const int last = (p.passes - 1) & 1;
  const SumArgs a{key[last], pos[last], (int)n, (int)rows, p.share, p.shares, width, ldg, ldo, scale, accumulate != 0,
                  reinterpret_cast<float*>(ws + p.pieces_at), p.piece_ld};
  return APPY_OP_DTYPE(dtype, {
    const T* g = static_cast<const T*>(dgrad);
    if (out_dtype == APPY_F32) {
      float* out = static_cast<float*>(dout);
      return V == 1 ? launch_sums<T, float, 1>(p, a, g, out, s) : launch_sums<T, float, 16 / sizeof(T)>(p, a, g, out, s);
    }
    T* out = static_cast<T*>(dout);
    return V == 1 ? launch_sums<T, T, 1>(p, a, g, out, s) : launch_sums<T, T, 16 / sizeof(T)>(p, a, g, out, s);
  });
}

}  // extern "C"
