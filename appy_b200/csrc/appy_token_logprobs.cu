// Log probabilities of given tokens, entropy and top alternatives of each row of logits, and the gradient.
//
// With z = logits / temperature, m the row's maximum, k = log2(e) / temperature:
//   d[j] = (x[j] - m) * k,  S = sum 2^d[j],  Q = sum 2^d[j] d[j]
//   logprob[j] = ln2 (d[j] - log2 S),   entropy = ln2 (log2 S - Q / S)
//   d logits[j] = ( g (1[j = token] - p[j]) - gH p[j] (log p[j] + entropy) ) / temperature
// One pass over the row: every thread keeps its own m, S and Q and rescales them when its maximum grows.  S and Q
// are float32 sums of at most a few hundred terms per thread, joined as a tree.
//
// Masked logits may be -inf, the type's lowest value, or any large finite one.  The fused form of d takes the rounded product
// m k for the reference, which at x = m is off by up to half a step of that product, so it is used where this is at most a
// quarter; a row (or a thread's part of it) whose maximum lies farther out takes x - m first (see `Scaled`).  d is held above
// -1000, where its weight has long been zero.  A row of -inf only is empty: log probability -inf, entropy 0, no gradient.  A
// row with a NaN or +inf is NaN throughout.
//
// Top alternatives: a thread remembers its best pack.  The `top`-th largest of 64 groups' bests bounds the answer
// from below, so only packs not below it are looked at again, and the few elements found are ranked by
// (value, lowest index first), which makes the answer independent of the order in which they were found.
#include <cooperative_groups.h>

#include <type_traits>

#include "operators.cuh"

namespace {
using namespace appy_op;
namespace cg = cooperative_groups;

const int kTopMax = 32;

APPY_DEV float neg_inf() { return __int_as_float(0xff800000); }
APPY_DEV float quiet_nan() { return __int_as_float(0x7fffffff); }
APPY_DEV float exp2_fast(float x) {                      // 2^x to 2 units in the last place, 0 below -126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
APPY_DEV float max_nan(float a, float b) {               // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// k and a bound: a maximum within +-limit has a product with k below 2^22, whose half step is at most 2^-2
struct Scale { float k, limit, span, inv_temperature; };      // span: 2^(-span k) is below float32

// d = (x - m) * k.  For a maximum within the limit as one fused multiply-add against the rounded product m * k: that product is a
// reference like any other, as long as every use of this m has the same one (so it must not be contracted into a
// difference of two of them).  Beyond it the maximum itself is the reference: at x = m the fused form would give the rounding
// of the product, 439 for m = -1e10 and 6e21 for -1e30 at temperature 1, and its weight would be infinite or zero.
struct Scaled {
  float m, mk;
  bool far;                                              // maximum beyond the limit (or no maximum yet)
  APPY_DEV Scaled(float m_, const Scale& s) {
    m = m_;
    mk = __fmul_rn(m_, s.k);
    far = !(fabsf(m_) < s.limit);
  }
  APPY_DEV float fast(float x, const Scale& s) const { return fmaxf(fmaf(x, s.k, -mk), -1000.f); }
  APPY_DEV float slow(float x, const Scale& s) const { return fmaxf((x - m) * s.k, -1000.f); }
};

// Part of a row's softmax: maximum, sum of 2^d, sum of 2^d d.
struct Part {
  float m, s, q;
};
APPY_DEV Part rescaled(const Part& p, float m, const Scale& s) {
  if (p.s == 0.f) return {m, 0.f, 0.f};
  const Scaled now(m, s), was(p.m, s);
  // the old reference against the new: each is its maximum times k, rounded (within the limit) or not
  float d = was.mk - now.mk;
  if (__builtin_expect(now.far || was.far, 0)) d = !was.far ? -fmaf(m, s.k, -was.mk) : now.far ? (p.m - m) * s.k : fmaf(p.m, s.k, -now.mk);
  d = fmaxf(d, -1000.f);
  const float c = exp2_fast(d);
  return {m, p.s * c, c * (p.q + p.s * d)};
}
APPY_DEV Part joined(const Part& a, const Part& b, const Scale& s) {
  const float m = max_nan(a.m, b.m);
  const Part x = rescaled(a, m, s), y = rescaled(b, m, s);
  return {m, x.s + y.s, x.q + y.q};
}

// orders as the values do, NaN above +inf, -0 with +0
APPY_DEV unsigned ordered(float v) {
  const unsigned b = v != v ? 0x7fffffffu : __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
APPY_DEV float unordered(unsigned o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
APPY_DEV u64 key_of(float v, int index) { return ((u64)ordered(v) << 32) | (unsigned)~index; }

// How a row splits into single elements up to the first 16-byte boundary, packs, and single elements behind them.
struct Split {
  int head, packs, tail0;
  template <class T, int V> static APPY_DEV Split of(const T* row, int cols) {
    const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    Split s;
    s.head = mis ? min(V - mis, cols) : 0;
    s.packs = (cols - s.head) / V;
    s.tail0 = s.head + s.packs * V;
    return s;
  }
};

struct Best { unsigned value; int at; };                 // ordered value and first index of the best pack

// Maximum of a pack (NaN if one is), and the pack with everything below `bound` raised to it; 16-bit types two at a time.
template <class T, int V> APPY_DEV float pack_max(const Pack<T, V>& k) {
  if constexpr (sizeof(T) == 2 && V > 1) {
    typename Pack<T, V>::Bits u;
    u.raw = k.raw;
    unsigned m = u.w[0];
#pragma unroll
    for (int i = 1; i < V / 2; ++i) {
      if constexpr (std::is_same<T, bf16>::value) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(u.w[i]));
      else asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(u.w[i]));
    }
    float lo, hi;
    unpack2(m, lo, hi, T());
    return max_nan(lo, hi);
  } else {
    float x[V];
    unpack<T, V>(k, x);
    float m = x[0];
#pragma unroll
    for (int v = 1; v < V; ++v) m = max_nan(m, x[v]);
    return m;
  }
}
template <class T, int V> APPY_DEV void unpack_from(const Pack<T, V>& k, unsigned bound, float (&x)[V]) {
  if constexpr (sizeof(T) == 2 && V > 1) {
    typename Pack<T, V>::Bits u;
    u.raw = k.raw;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same<T, bf16>::value) asm("max.bf16x2 %0, %0, %1;" : "+r"(u.w[i]) : "r"(bound));
      else asm("max.f16x2 %0, %0, %1;" : "+r"(u.w[i]) : "r"(bound));
      unpack2(u.w[i], x[2 * i], x[2 * i + 1], T());
    }
  } else {
    unpack<T, V>(k, x);
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = fmaxf(x[v], sizeof(T) == 2 ? neg_inf() : __uint_as_float(bound));
  }
}
// The bound for a maximum: so far below that the weight is zero, as two elements of T (or one float32).  False: none
// that is finite in T, or the maximum is far out; d is then held up one by one.
template <class T> APPY_DEV bool bound_of(const Scaled& d, const Scale& s, unsigned& bound) {
  const float b = d.m - s.span;
  if constexpr (sizeof(T) == 4) {
    bound = __float_as_uint(b);
  } else if constexpr (std::is_same<T, bf16>::value) {
    const unsigned short h = __bfloat16_as_ushort(__float2bfloat16_rd(b));
    bound = h | (unsigned)h << 16;
  } else {
    if (!(b > -65504.f)) return false;
    const unsigned short h = __half_as_ushort(__float2half_rd(b));
    bound = h | (unsigned)h << 16;
  }
  return !d.far;                                         // else m - span may be m
}

// One thread's part of a row: softmax with its own maximum, S and Q as pairs of sums.
template <class T> struct Running {
  float m;
  bool fine;                 // a finite bound: whole packs at a time
  unsigned bound;
  Vec<2> s, q;
  APPY_DEV void start() {
    m = neg_inf();
    fine = false;
    bound = 0;
    s = q = all<2>(0.f);
  }
  APPY_DEV Part part() const {
    float a[2], b[2];
    floats<2>(s, a);
    floats<2>(q, b);
    return {m, a[0] + a[1], b[0] + b[1]};
  }
  APPY_DEV void raise(float to, const Scale& sc) {
    const Part p = rescaled(part(), max_nan(to, m), sc);         // a NaN stays
    m = p.m;
    const float a[2] = {p.s, 0.f}, b[2] = {p.q, 0.f};
    s = vec<2>(a);
    q = vec<2>(b);
    fine = bound_of<T>(Scaled(m, sc), sc, bound);
  }
  template <int V> APPY_DEV void add_pack(const Pack<T, V>& k, const Scaled& d, const Scale& sc) {
    if (fine && V > 1) {
      float x[V];
      unpack_from<T, V>(k, bound, x);
#pragma unroll
      for (int v = 0; v < V; v += 2) {
        const float pr[2] = {x[v], x[V > 1 ? v + 1 : v]};
        const Vec<2> t = fma<2>(vec<2>(pr), all<2>(sc.k), all<2>(-d.mk));
        float e[2];
        floats<2>(t, e);
        e[0] = exp2_fast(e[0]);
        e[1] = exp2_fast(e[1]);
        const Vec<2> w = vec<2>(e);
        s = add<2>(s, w);
        q = fma<2>(w, t, q);
      }
    } else if (fabsf(m) < __int_as_float(0x7f800000)) {
      float x[V], es = 0.f, eq = 0.f;
      unpack<T, V>(k, x);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float t = d.far ? d.slow(x[v], sc) : d.fast(x[v], sc), e = exp2_fast(t);
        es += e;
        eq = fmaf(e, t, eq);
      }
      const float a[2] = {es, 0.f}, b[2] = {eq, 0.f};
      s = add<2>(s, vec<2>(a));
      q = add<2>(q, vec<2>(b));
    }
  }
  // U packs whose first elements are at `at`, `at + step`, ..
  template <int V, int U, bool TOP> APPY_DEV void take(const Pack<T, V> (&k)[U], int at, int step, Best& best, const Scale& sc) {
    float top = neg_inf();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float pm = pack_max<T, V>(k[u]);
      if (TOP) {
        const unsigned o = ordered(pm);
        if (o > best.value) best = {o, at + u * step};
      }
      top = u ? max_nan(top, pm) : pm;
    }
    if (!(top <= m)) raise(top, sc);
    const Scaled d(m, sc);
#pragma unroll
    for (int u = 0; u < U; ++u) add_pack<V>(k[u], d, sc);
  }
};

struct LogprobArgs {
  const void* logits;
  i64 ld;
  int cols;
  const void* tokens;
  bool wide;
  Scale scale;
  int top;
  float* logprobs;
  float* entropy;
  float* stats;              // [rows][3]: maximum, log2 S, entropy
  float* top_logprobs;
  void* top_tokens;
};

const float kLn2 = 0.693147180559945309f;

// logprob of a logit from the row's statistics
APPY_DEV float logprob_of(float x, float m, float log2s, const Scale& s) {
  if (!(m < __int_as_float(0x7f800000))) return quiet_nan();
  if (x == neg_inf()) return neg_inf();
  const Scaled d(m, s);
  const float t = d.far ? (x - m) * s.k : fmaf(x, s.k, -d.mk);
  return t < -1e38f ? (x - m) * s.inv_temperature : (t - log2s) * kLn2;
}

struct LargerKey {
  template <class K> static APPY_DEV K id() { return 0; }
  template <class K> static APPY_DEV K op(K a, K b) { return a > b ? a : b; }
};
struct NoTop {};
template <int NT> struct TopState {
  static constexpr int kGroups = NT < 64 ? NT : 64, kCandidates = NT < 64 ? 512 : 1024;
  u64 key[NT];
  u64 found[kCandidates];
  u64 list[kTopMax];
  u64 bound;
  int count;
};

// The `top` largest keys of this block's part of the row, largest first, in t.list (0: there are fewer).
template <class T, int V, int NT> APPY_DEV void select_top(TopState<NT>& t, const Best& best, bool any, const T* row, const Split& sp, int lo, int hi,
                                                   bool edges, int cols, int top) {
  constexpr int kBlock = NT, kGroups = TopState<NT>::kGroups, kCandidates = TopState<NT>::kCandidates;
  const int tid = threadIdx.x;
  t.key[tid] = any ? ((u64)best.value << 32) | (unsigned)~best.at : 0;
  if (tid < kTopMax) t.list[tid] = 0;
  if (tid == 0) t.count = 0, t.bound = 0;
  __syncthreads();
  u64 mine = 0;
  if (tid < kGroups) {
    for (int x = tid; x < kBlock; x += kGroups) mine = max(mine, t.key[x]);
  }
  const u64 own = t.key[tid];
  __syncthreads();
  if (tid < kGroups) t.key[tid] = mine;
  __syncthreads();
  if (tid < kGroups && mine) {
    int above = 0;
    for (int x = 0; x < kGroups; ++x) above += t.key[x] > mine;
    if (above == top - 1) t.bound = mine;            // keys differ, so one group at most
  }
  __syncthreads();
  const u64 bound = t.bound;
  auto look = [&](float v, int pack_at, int at) {
    if ((((u64)ordered(v) << 32) | (unsigned)~pack_at) < bound) return;
    const int n = atomicAdd(&t.count, 1);
    if (n < kCandidates) t.found[n] = key_of(v, at);
  };
  const bool again = any && own >= bound;
  if (again && edges) {
    if (tid < sp.head) look(to_f32(row[tid]), tid, tid);
    if (sp.tail0 + tid < cols) look(to_f32(row[sp.tail0 + tid]), sp.tail0 + tid, sp.tail0 + tid);
  }
  // the packs of a thread that has candidates are looked through by its whole warp
  for (unsigned who = __ballot_sync(APPY_FULL_MASK, again); who; who &= who - 1) {
    const int other = (tid & ~31) + __ffs(who) - 1;
    for (int p = lo + other + (tid & 31) * kBlock; p < hi; p += 32 * kBlock) {
      const int at = sp.head + p * V;
      float x[V];
      unpack<T, V>(ld_keep<T, V>(row + at), x);
#pragma unroll
      for (int v = 0; v < V; ++v) look(x[v], at, at + v);
    }
  }
  __syncthreads();
  const int count = t.count;
  if (count <= kCandidates) {
    for (int x = tid; x < count; x += kBlock) {
      const u64 k = t.found[x];
      int above = 0;
      for (int y = 0; y < count; ++y) above += t.found[y] > k;
      if (above < top) t.list[above] = k;
    }
    __syncthreads();
    return;
  }
  // many equal or unluckily placed values: one maximum after another
  u64 last = ~(u64)0;
  for (int r = 0; r < top; ++r) {
    u64 k = 0;
    auto see = [&](float v, int at) {
      const u64 c = key_of(v, at);
      if (c < last && c > k) k = c;
    };
    if (edges && tid < sp.head) see(to_f32(row[tid]), tid);
    for (int p = lo + tid; p < hi; p += kBlock) {
      const int at = sp.head + p * V;
      float x[V];
      unpack<T, V>(ld_keep<T, V>(row + at), x);
#pragma unroll
      for (int v = 0; v < V; ++v) see(x[v], at + v);
    }
    if (edges && sp.tail0 + tid < cols) see(to_f32(row[sp.tail0 + tid]), sp.tail0 + tid);
    k = appy_block_reduce<LargerKey, u64>(k, t.key);
    if (tid == 0) t.list[r] = k;
    last = k;
    if (!k) break;
  }
  __syncthreads();
}

// One cluster of C blocks per row; block `rank` takes an equal share of the packs, block 0 the elements around them.
template <class T, int V, int NT, int C, bool TOP>
__global__ void __launch_bounds__(NT, 1024 / NT > 16 ? 16 : 1024 / NT) k_logprobs(LogprobArgs a) {
  constexpr int U = NT == 32 ? 2 : 4, kBlock = NT, kWarps = NT / 32;
  __shared__ Part warp_part[kWarps];
  __shared__ Part parts[C];
  __shared__ u64 lists[TOP ? C : 1][TOP ? kTopMax : 1];
  __shared__ typename std::conditional<TOP, TopState<NT>, NoTop>::type top_state;
  const int tid = threadIdx.x, rank = C > 1 ? blockIdx.x % C : 0;
  const i64 n = blockIdx.x / C;
  const T* const row = static_cast<const T*>(a.logits) + n * a.ld;
  const Split sp = Split::of<T, V>(row, a.cols);
  const int per = (sp.packs + C - 1) / C, lo = min(rank * per, sp.packs), hi = min(lo + per, sp.packs);
  const bool edges = rank == 0;
  i64 token = -1;
  float token_logit = 0.f;
  if (rank == 0 && tid == 0) {
    token = a.wide ? __ldg(static_cast<const i64*>(a.tokens) + n) : (i64)__ldg(static_cast<const int*>(a.tokens) + n);
    if (token >= 0 && token < a.cols) token_logit = to_f32(row[token]);
  }
  Running<T> run;
  run.start();
  Best best = {0, 0};
  bool any = false;
  auto single = [&](int at) {
    Pack<T, 1> k[1] = {ld_keep<T, 1>(row + at)};
    run.template take<1, 1, TOP>(k, at, 0, best, a.scale);
    any = true;
  };
  if (edges)
    for (int at = tid; at < sp.head; at += kBlock) single(at);
  const T* const body = row + sp.head;
  int p0 = lo + tid;
  for (; p0 + (U - 1) * kBlock < hi; p0 += kBlock * U) {
    Pack<T, V> k[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = ld_stream<T, V>(body + (i64)(p0 + u * kBlock) * V);
    run.template take<V, U, TOP>(k, sp.head + p0 * V, kBlock * V, best, a.scale);
    any = true;
  }
  for (; p0 < hi; p0 += kBlock) {
    Pack<T, V> k[1] = {ld_stream<T, V>(body + (i64)p0 * V)};
    run.template take<V, 1, TOP>(k, sp.head + p0 * V, 0, best, a.scale);
    any = true;
  }
  if (edges)
    for (int at = sp.tail0 + tid; at < a.cols; at += kBlock) single(at);
  Part p = run.part();
  for (int o = 16; o; o >>= 1) {
    const Part y = {__shfl_xor_sync(APPY_FULL_MASK, p.m, o), __shfl_xor_sync(APPY_FULL_MASK, p.s, o), __shfl_xor_sync(APPY_FULL_MASK, p.q, o)};
    p = joined(p, y, a.scale);
  }
  if ((tid & 31) == 0) warp_part[tid >> 5] = p;
  if constexpr (TOP) select_top<T, V, NT>(top_state, best, any, row, sp, lo, hi, edges, a.cols, a.top);
  __syncthreads();
  if (tid == 0) {
    p = warp_part[0];
    for (int w = 1; w < kWarps; ++w) p = joined(p, warp_part[w], a.scale);
  }
  if (C > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();                                      // block 0 runs
    if (tid == 0) *cluster.map_shared_rank(&parts[rank], 0) = p;
    if constexpr (TOP)
      if (tid < kTopMax) *cluster.map_shared_rank(&lists[rank][tid], 0) = top_state.list[tid];
    cluster.sync();
    if (rank) return;
    if (tid == 0) {
      p = parts[0];
      for (int r = 1; r < C; ++r) p = joined(p, parts[r], a.scale);
    }
    if constexpr (TOP) {
      for (int x = tid; x < C * a.top; x += kBlock) {
        const u64 k = lists[x / a.top][x % a.top];
        if (!k) continue;
        int above = 0;                                   // keys above this one in each block's list, which falls
#pragma unroll
        for (int r = 0; r < C; ++r) {
          int n = 0;
#pragma unroll
          for (int step = 32; step; step >>= 1)
            if (n + step <= a.top && lists[r][n + step - 1] > k) n += step;
          above += n;
        }
        if (above < a.top) top_state.list[above] = k;
      }
    }
  }
  if (tid == 0) {
    const bool empty = p.m == neg_inf(), bad = !(p.m < __int_as_float(0x7f800000));
    const float log2s = empty ? 0.f : log2f(p.s);
    const float h = bad ? quiet_nan() : empty ? 0.f : (log2s - p.q / p.s) * kLn2;
    const bool known = token >= 0 && token < a.cols;
    a.logprobs[n] = !known ? 0.f : empty ? neg_inf() : logprob_of(token_logit, p.m, log2s, a.scale);
    a.entropy[n] = h;
    a.stats[n * 3] = p.m;
    a.stats[n * 3 + 1] = log2s;
    a.stats[n * 3 + 2] = h;
    parts[0] = {p.m, log2s, 0.f};
  }
  if constexpr (TOP) {
    __syncthreads();
    if (tid < a.top) {
      const u64 k = top_state.list[tid];
      const Part r = parts[0];
      const float x = unordered((unsigned)(k >> 32));
      const int at = (int)~(unsigned)k;
      a.top_logprobs[n * a.top + tid] = r.m == neg_inf() ? neg_inf() : logprob_of(x, r.m, r.s, a.scale);
      if (a.wide) static_cast<i64*>(a.top_tokens)[n * a.top + tid] = at;
      else static_cast<int*>(a.top_tokens)[n * a.top + tid] = at;
    }
  }
}

// ------------------------------------------------------------------------------------------------ gradient
struct LogprobGradArgs {
  const void* logits;
  i64 ld;
  int cols;
  const void* tokens;
  bool wide;
  Scale scale;
  const float* stats;
  const float* g;
  i64 g_stride;
  const float* gh;
  i64 gh_stride;
  void* out;
  i64 ldo;
  int chunks;
};

const int kGradBlock = 256, kGradU = 4;

// A block takes kGradBlock * U packs of one row; where input and output rows are not aligned alike, V is 1.
template <class T, int V>
__global__ void __launch_bounds__(kGradBlock) k_logprobs_grad(LogprobGradArgs a) {
  constexpr int U = kGradU * (V == 1 ? 4 : 1);
  const int tid = threadIdx.x, chunk = blockIdx.x % a.chunks;
  const i64 n = blockIdx.x / a.chunks;
  const T* const row = static_cast<const T*>(a.logits) + n * a.ld;
  T* const out = static_cast<T*>(a.out) + n * a.ldo;
  const Split sp = V == 1 ? Split{0, a.cols, a.cols} : Split::of<T, V>(row, a.cols);
  const float m = __ldg(a.stats + n * 3), log2s = __ldg(a.stats + n * 3 + 1), h = __ldg(a.stats + n * 3 + 2);
  i64 token = a.wide ? __ldg(static_cast<const i64*>(a.tokens) + n) : (i64)__ldg(static_cast<const int*>(a.tokens) + n);
  if (token < 0 || token >= a.cols) token = -1;
  const float g = a.g && token >= 0 ? __ldg(a.g + n * a.g_stride) : 0.f, gh = a.gh ? __ldg(a.gh + n * a.gh_stride) : 0.f;
  const bool empty = m == neg_inf(), bad = !(m < __int_as_float(0x7f800000));
  // d logits = p * (c0 + c1 * log2 p) + [j = token] * c2
  const float c0 = -(g + gh * h) * a.scale.inv_temperature, c1 = -gh * kLn2 * a.scale.inv_temperature, c2 = empty ? 0.f : g * a.scale.inv_temperature;
  const Scaled d(m, a.scale);
  unsigned bound;
  const bool fine = bound_of<T>(d, a.scale, bound) && !empty && !bad && V > 1;
  auto one = [&](float x, int at) {
    const float t = (d.far ? d.slow(x, a.scale) : d.fast(x, a.scale)) - log2s;
    float r = exp2_fast(t) * fmaf(c1, t, c0);
    if (empty) r = 0.f;
    if (at == (int)token) r += c2;
    return bad ? quiet_nan() : r;
  };
  const int p0 = chunk * (kGradBlock * U) + tid;
  Pack<T, V> k[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (p0 + u * kGradBlock < sp.packs) k[u] = ld_stream<T, V>(row + sp.head + (i64)(p0 + u * kGradBlock) * V);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (p0 + u * kGradBlock < sp.packs) {
      const int at = sp.head + (p0 + u * kGradBlock) * V;
      float x[V];
      if (fine) {
        unpack_from<T, V>(k[u], bound, x);
        const Vec<V> t = add<V>(fma<V>(vec<V>(x), all<V>(a.scale.k), all<V>(-d.mk)), all<V>(-log2s));
        float e[V];
        floats<V>(t, e);
#pragma unroll
        for (int v = 0; v < V; ++v) e[v] = exp2_fast(e[v]);
        floats<V>(mul<V>(vec<V>(e), fma<V>(t, all<V>(c1), all<V>(c0))), x);
        if ((unsigned)((int)token - at) < (unsigned)V) {
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (at + v == (int)token) x[v] += c2;
        }
      } else {
        unpack<T, V>(k[u], x);
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = one(x[v], at + v);
      }
      st_stream<T, V>(out + at, pack<T, V>(x));
    }
  if (V > 1 && chunk == 0) {
    if (tid < sp.head) out[tid] = from_f32<T>(one(to_f32(row[tid]), tid));
    const int at = sp.tail0 + tid;
    if (at < a.cols) out[at] = from_f32<T>(one(to_f32(row[at]), at));
  }
}

// ------------------------------------------------------------------------------------------------ host side
template <class T, int V, int NT, int C, bool TOP> int launch_c(const LogprobArgs& a, i64 rows, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * C));
  cfg.blockDim = dim3(NT);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_logprobs<T, V, NT, C, TOP>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return appy_fail_cuda(e, "token logprobs launch");
  }
  return finish("token logprobs launch");
}

template <class T, bool TOP> int launch_logprobs(const LogprobArgs& a, i64 rows, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  // A block per row, of so many threads that each has some packs: short rows would otherwise wait at barriers for
  // threads without work.  Few long rows: a cluster of up to 8 blocks per row, as long as every thread still has two.
  // B200, bfloat16, 20 alternatives, microseconds for blocks of 32 / 128 / 256 threads:
  //   8192 x 1000: 47 / 68 / 111,  8192 x 8192: 80 / 99 / 127,  8 x 1000: 14 / 8 / 10,  1000 x 8192: 25 / 17 / 21,
  //   4000 x 16384: 73 / 68 / 84,  1000 x 32768: 96 / 31 / 35;  none, 4096 x 131072: 256 threads 198, 512 threads 226;
  //   8 x 131072: clusters of 8 blocks 12.4, of 16 blocks 20.5.
  const i64 packs = a.cols / V, sms = sm_count();
  if (rows >= 8 * sms && packs <= 1024) return launch_c<T, V, 32, 1, TOP>(a, rows, s);
  if (packs <= 256 || (rows >= sms && packs <= 4096)) return launch_c<T, V, 128, 1, TOP>(a, rows, s);
  int c = 1;
  while (c < 8 && rows * c < 2 * sms && packs >= 512 * 2 * c) c *= 2;
  switch (c) {
    case 1: return launch_c<T, V, 256, 1, TOP>(a, rows, s);
    case 2: return launch_c<T, V, 512, 2, TOP>(a, rows, s);
    case 4: return launch_c<T, V, 512, 4, TOP>(a, rows, s);
    default: return launch_c<T, V, 512, 8, TOP>(a, rows, s);
  }
}

Scale scale_of(float temperature) {
  const float k = 1.44269504088896341f / temperature;
  return {k, 4194304.f / k, 200.f / k, 1.f / temperature};
}

int check_logits(const char* fn, int dtype, int token_dtype, i64 rows, i64 cols, i64 ld, float temperature) {
  if (!element_size(dtype)) return fail_named(fn, "dtype must be APPY_F32, APPY_F16 or APPY_BF16");
  if (token_dtype != APPY_I32 && token_dtype != APPY_I64) return fail_named(fn, "token_dtype must be APPY_I32 or APPY_I64");
  if (rows < 0 || cols < 1 || cols > 0x7fff0000) return fail_named(fn, "rows must not be negative, cols must be in [1, 2^31 - 2^16]");
  if (rows > 1 && ld < cols) return fail_named(fn, "ld must be at least cols");
  if (!(temperature >= 1e-4f && temperature <= 1e4f)) return fail_named(fn, "temperature must be in [1e-4, 1e4]");
  return APPY_OK;
}

}  // namespace

extern "C" {

int appy_token_logprobs(const void* dlogits, int dtype, int64_t ld, int64_t rows, int64_t cols, const void* dtokens, int token_dtype,
                        float temperature, int top, float* dlogprobs, float* dentropy, float* dstats, float* dtop_logprobs,
                        void* dtop_tokens, void* stream) {
  static const char fn[] = "appy_token_logprobs";
  if (int rc = check_logits(fn, dtype, token_dtype, rows, cols, ld, temperature)) return rc;
  if (top < 0 || top > kTopMax || top > cols) return fail_named(fn, "top must be in [0, 32] and not above cols");
  if (rows == 0) return APPY_OK;
  if (rows > 0x7fffffff / 8) return fail_named(fn, "too many rows for one launch");
  if (!dlogits || !dtokens || !dlogprobs || !dentropy || !dstats || (top && (!dtop_logprobs || !dtop_tokens))) return fail_named(fn, "NULL argument");
  LogprobArgs a{dlogits, ld, (int)cols, dtokens, token_dtype == APPY_I64, scale_of(temperature), top,
                dlogprobs, dentropy, dstats, dtop_logprobs, dtop_tokens};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return APPY_OP_DTYPE(dtype, { return top ? launch_logprobs<T, true>(a, rows, s) : launch_logprobs<T, false>(a, rows, s); });
}

int appy_token_logprobs_grad(const void* dlogits, int dtype, int64_t ld, int64_t rows, int64_t cols, const void* dtokens, int token_dtype,
                             float temperature, const float* dstats, const float* dgrad_logprobs, int64_t grad_logprobs_stride,
                             const float* dgrad_entropy, int64_t grad_entropy_stride, void* dout, int64_t ldo, void* stream) {
  static const char fn[] = "appy_token_logprobs_grad";
  if (int rc = check_logits(fn, dtype, token_dtype, rows, cols, ld, temperature)) return rc;
  if (rows > 1 && ldo < cols) return fail_named(fn, "ldo must be at least cols");
  if (rows == 0) return APPY_OK;
  if (!dlogits || !dtokens || !dstats || !dout) return fail_named(fn, "NULL argument");
  const int size = element_size(dtype), V = 16 / size;
  const bool alike = ((reinterpret_cast<uintptr_t>(dlogits) ^ reinterpret_cast<uintptr_t>(dout)) & 15) == 0 &&
                     (rows == 1 || (ld - ldo) % V == 0);
  const i64 packs = alike ? cols / V : cols, per = (i64)kGradBlock * kGradU * (alike ? 1 : 4), chunks = std::max<i64>(1, (packs + per - 1) / per);
  if (rows * chunks > 0x7fffffff) return fail_named(fn, "too many elements for one launch");
  LogprobGradArgs a{dlogits, ld, (int)cols, dtokens, token_dtype == APPY_I64, scale_of(temperature), dstats,
                    dgrad_logprobs, grad_logprobs_stride, dgrad_entropy, grad_entropy_stride, dout, ldo, (int)chunks};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return APPY_OP_DTYPE(dtype, {
    if (alike) k_logprobs_grad<T, 16 / sizeof(T)><<<(unsigned)(rows * chunks), kGradBlock, 0, s>>>(a);
    else k_logprobs_grad<T, 1><<<(unsigned)(rows * chunks), kGradBlock, 0, s>>>(a);
    return finish("token logprobs gradient launch");
  });
}

}  // extern "C"
