// Gated linear recurrence along tokens, channel by channel, and its gradient:
//
//   f = sigmoid(gate),   h[t] = f[t] * h[t-1] + (1 - f[t]) * x[t],   h[-1] = initial
//
// The map from h[t-1] to h[t] is affine, and affine maps compose: (A, B) after (A', B') is (A A', A B' + B).  So the
// tokens of a tile are cut into short runs, one per thread, each thread composes its run, the runs' maps are joined
// (within a warp by shuffles, across warps through shared memory, across the blocks of a cluster through their
// shared memory), and every thread replays its run from the state that it then knows.  Gates and products stay in
// registers between the two passes: global memory is read once and written once.
//
// The gradient is the same recurrence backwards.  With lam[t] = dh[t] + mu[t+1] (dh: gradient of h[t] from outside),
//   mu[t] = f[t] * lam[t],  dx[t] = (1 - f[t]) * lam[t],  dgate[t] = lam[t] * (h[t-1] - x[t]) * f[t] * (1 - f[t]),
// mu past the last token is the gradient of the last state, mu[0] that of the initial one.
//
// A block takes 64 channels (32 where rows do not allow packs) of one sequence and walks along it; with few
// sequences and channels a cluster of blocks takes neighbouring stretches of tokens in each step, so that the whole
// machine loads at a time.  States are float32; each result is rounded once.
#include <cooperative_groups.h>

#include "operators.cuh"

namespace {
using namespace appy_op;
namespace cg = cooperative_groups;

const int kBlock = 128;

// ------------------------------------------------------------------------------------------------ V floats at a time
// Two float32 of one 64-bit register per instruction where V is even: these kernels issue a dozen operations per
// element, and products and sums of pairs cost half of that.
template <int V> struct Vec { u64 p[V / 2]; };
template <> struct Vec<1> { float p[1]; };

APPY_DEV u64 pair(float lo, float hi) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
APPY_DEV float mul1(float a, float b) { return a * b; }
APPY_DEV float add1(float a, float b) { return a + b; }
APPY_DEV float fma1(float a, float b, float c) { return fmaf(a, b, c); }
APPY_DEV u64 mul1(u64 a, u64 b) { u64 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
APPY_DEV u64 add1(u64 a, u64 b) { u64 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
APPY_DEV u64 fma1(u64 a, u64 b, u64 c) { u64 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }

template <int V> APPY_DEV Vec<V> vec(const float (&f)[V]) {
  Vec<V> r;
  if constexpr (V == 1) {
    r.p[0] = f[0];
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = pair(f[2 * i], f[2 * i + 1]);
  }
  return r;
}
template <int V> APPY_DEV Vec<V> all(float x) {
  float f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = x;
  return vec<V>(f);
}
template <int V> APPY_DEV void floats(const Vec<V>& a, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = a.p[0];
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) asm("mov.b64 {%0, %1}, %2;" : "=f"(f[2 * i]), "=f"(f[2 * i + 1]) : "l"(a.p[i]));
  }
}
#define APPY_EACH(expr)                                                    \
  Vec<V> r;                                                                \
  _Pragma("unroll") for (int i = 0; i < (V == 1 ? 1 : V / 2); ++i) r.p[i] = expr; \
  return r
template <int V> APPY_DEV Vec<V> mul(const Vec<V>& a, const Vec<V>& b) { APPY_EACH(mul1(a.p[i], b.p[i])); }
template <int V> APPY_DEV Vec<V> add(const Vec<V>& a, const Vec<V>& b) { APPY_EACH(add1(a.p[i], b.p[i])); }
template <int V> APPY_DEV Vec<V> fma(const Vec<V>& a, const Vec<V>& b, const Vec<V>& c) { APPY_EACH(fma1(a.p[i], b.p[i], c.p[i])); }
#undef APPY_EACH

// f = sigmoid(g) and i = 1 - f, each to a few units in the last place whichever is small: with e = exp(-g),
// f = 1 / (1 + e) and i = e f.  A gate below -87 counts as -87, so that e stays finite: f is 1.6e-38 there, not less.
template <int V> APPY_DEV void sigmoid_pair(float (&g)[V], Vec<V>& f, Vec<V>& i) {
#pragma unroll
  for (int v = 0; v < V; ++v) asm("max.NaN.f32 %0, %0, %1;" : "+f"(g[v]) : "f"(-87.f));
  float t[V];
  floats<V>(mul<V>(vec<V>(g), all<V>(-1.44269504088896341f)), t);
#pragma unroll
  for (int v = 0; v < V; ++v) asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t[v]));
  const Vec<V> e = vec<V>(t);
  float d[V];
  floats<V>(add<V>(e, all<V>(1.f)), d);
#pragma unroll
  for (int v = 0; v < V; ++v) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d[v]));
  f = vec<V>(d);
  i = mul<V>(e, f);
}

struct Rows {                // element (sequence s, token t, channel c) is at base + s * seq + t * row + c
  void* base;
  i64 seq, row;
};

struct ScanArgs {
  Rows x, gate, h;           // forward: h is written; gradient: h is read
  Rows dh, dx, dgate;        // gradient only; dh NULL: zeros
  const float* initial;      // [sequences][width], NULL: zeros
  const float* dlast;        // gradient only, NULL: zeros
  float* final_state;        // last state, or the gradient of the initial one
  const void* offsets;       // NULL: every sequence has `tokens` tokens
  bool wide, fill;
  i64 sequences, tokens, width;
  int tiles;
};

APPY_DEV i64 offset_at(const ScanArgs& a, i64 s) {
  const i64 v = a.wide ? __ldg(static_cast<const i64*>(a.offsets) + s) : (i64)__ldg(static_cast<const int*>(a.offsets) + s);
  return v < 0 ? 0 : v > a.tokens ? a.tokens : v;
}

template <class T> APPY_DEV T* row_ptr(const Rows& r, i64 seq, i64 first, i64 t, i64 c) {
  return static_cast<T*>(r.base) + seq * r.seq + (first + t) * r.row + c;
}

// Packed rows that no sequence covers are set to zero where the caller asks for it.
template <class T, int V> APPY_DEV void clear_rows(const Rows& r, i64 lo, i64 hi, i64 col, bool live, int sub, int subs) {
  if (!live) return;
  for (i64 t = lo + sub; t < hi; t += subs) st_stream<T, V>(row_ptr<T>(r, 0, 0, t, col), zero_pack<T, V>());
}

// What a thread reads of one step: LT tokens of V channels of each of NA arrays (gate, x; gradient: also dh and h of
// the token before).  Packs go through a ring of `S` stages in shared memory by cp.async, S - 1 steps ahead; a thread
// reads back only what it copied itself, so the ring needs no barrier.  Elements of 2 bytes, which cp.async cannot
// move, are loaded into registers one step ahead instead (S = 1).
template <class T, int V, int LT, int NA, int S> struct Feed {
  typedef typename Raw<sizeof(T) * V>::type R;
  static constexpr int kBytes = S > 1 ? S * NA * LT * kBlock * (int)sizeof(R) : 0;
  const char* from[NA];      // this thread's first row of the next step to fetch
  i64 row[NA], step[NA];     // bytes from one token to the next in walking order, and from one step to the next
  R held[S > 1 ? 1 : NA][S > 1 ? 1 : LT];
  R* ring;

  APPY_DEV void start(int a, const T* p, i64 row_bytes, i64 step_tokens) {
    from[a] = reinterpret_cast<const char*>(p);
    row[a] = row_bytes;
    step[a] = row_bytes * step_tokens;
  }
  // rows 0 .. n[a]-1 of the step are there for array a
  APPY_DEV void fetch(int stage, const int (&n)[NA]) {
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      const int lim = n[a];
#pragma unroll
      for (int j = 0; j < LT; ++j) {
        const R* src = reinterpret_cast<const R*>(from[a] + j * row[a]);
        if constexpr (S > 1) {
          const unsigned dst = (unsigned)__cvta_generic_to_shared(ring + ((stage * NA + a) * LT + j) * kBlock + threadIdx.x);
          if (j < lim) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(sizeof(R)) : "memory");
        } else {
          if (j < lim) held[a][j] = ld_raw_cs(src);
        }
      }
      from[a] += step[a];
    }
    if constexpr (S > 1) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  APPY_DEV void arrived() {
    if constexpr (S > 1) asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
  }
  APPY_DEV void get(int stage, int a, int j, float (&f)[V]) const {
    Pack<T, V> k;
    if constexpr (S > 1) k.raw = ring[((stage * NA + a) * LT + j) * kBlock + threadIdx.x];
    else k.raw = held[a][j];
    unpack<T, V>(k, f);
  }
};

// Maps that the blocks of a cluster hand to one another: every block writes its (A, B) of a channel into the same
// place of every block's shared memory, where the bytes count towards a barrier; no block waits for stores of another
// kind.  Two buffers alternate: a block sends step k + 2 only after it has everybody's k + 1, which they send after
// they have read k.
template <int C, int CH> struct Exchange {
  u64 map[2][C][CH];
  u64 full[2];
};
APPY_DEV unsigned shared_address(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
APPY_DEV unsigned in_block(unsigned address, int rank) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
  return r;
}
APPY_DEV bool wait_full(unsigned barrier, unsigned parity) {           // false: gave up
  for (unsigned tries = 0; tries < (1u << 22); ++tries) {          // some tenths of a second
    unsigned done;
    asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done) : "r"(barrier), "r"(parity) : "memory");
    if (done) return true;
  }
  return false;
}

// V channels per thread, CP threads along the channels, LT tokens per thread, C blocks per cluster, S stages.
template <class T, int V, int CP, int LT, int S, int C, int MIN_BLOCKS, bool BACK>
__global__ void __launch_bounds__(kBlock, MIN_BLOCKS) k_scan(ScanArgs a) {
  constexpr int CH = CP * V, SUBS = kBlock / CP, L = SUBS * LT, NA = BACK ? 4 : 2;
  static_assert(CH <= kBlock, "one thread per channel carries the state");
  extern __shared__ __align__(16) unsigned char ring_memory[];
  __shared__ __align__(16) float run_a[SUBS][CH], run_b[SUBS][CH], enter[SUBS][CH];
  __shared__ __align__(16) Exchange<C, (C > 1 ? CH : 1)> exchange;
  const int tid = threadIdx.x, sub = tid / CP, pc = (tid % CP) * V;
  const int rank = C > 1 ? blockIdx.x % C : 0;
  const i64 unit = blockIdx.x / C, seq = unit / a.tiles;
  const i64 chan0 = (unit % a.tiles) * CH, col = chan0 + pc;
  const bool live = col < a.width;
  i64 first = 0, len = a.tokens, seq_at = seq;
  if (a.offsets) {
    first = offset_at(a, seq);
    const i64 end = offset_at(a, seq + 1);
    len = end > first ? end - first : 0;
    seq_at = 0;
    if (a.fill && rank == 0) {
      if (seq == 0) {
        clear_rows<T, V>(BACK ? a.dx : a.h, 0, first, col, live, sub, SUBS);
        if (BACK) clear_rows<T, V>(a.dgate, 0, first, col, live, sub, SUBS);
      }
      if (seq == a.sequences - 1) {
        clear_rows<T, V>(BACK ? a.dx : a.h, end, a.tokens, col, live, sub, SUBS);
        if (BACK) clear_rows<T, V>(a.dgate, end, a.tokens, col, live, sub, SUBS);
      }
    }
  }
  const bool owner = tid < CH && chan0 + tid < a.width;      // one thread per channel carries the state along
  float carry = 0.f;
  if (owner && (BACK ? a.dlast : a.initial)) carry = (BACK ? a.dlast : a.initial)[seq * a.width + chan0 + tid];
  const i64 steps = (len + (i64)L * C - 1) / ((i64)L * C);
  // this thread's run in the first step, in walking order (backwards for the gradient)
  const i64 tau0 = (i64)rank * L + sub * LT, t0 = BACK ? len - 1 - tau0 : tau0;
  const int dir = BACK ? -1 : 1;
  Feed<T, V, LT, NA, S> feed;
  feed.ring = reinterpret_cast<typename Feed<T, V, LT, NA, S>::R*>(ring_memory);
  feed.start(0, row_ptr<const T>(a.gate, seq_at, first, t0, col), dir * a.gate.row * (i64)sizeof(T), (i64)L * C);
  feed.start(1, row_ptr<const T>(a.x, seq_at, first, t0, col), dir * a.x.row * (i64)sizeof(T), (i64)L * C);
  if constexpr (BACK) {
    feed.start(2, row_ptr<const T>(a.dh, seq_at, first, t0, col), dir * a.dh.row * (i64)sizeof(T), (i64)L * C);
    feed.start(3, row_ptr<const T>(a.h, seq_at, first, t0 - 1, col), dir * a.h.row * (i64)sizeof(T), (i64)L * C);
  }
  char* to = reinterpret_cast<char*>(row_ptr<T>(BACK ? a.dx : a.h, seq_at, first, t0, col));
  char* to_gate = BACK ? reinterpret_cast<char*>(row_ptr<T>(a.dgate, seq_at, first, t0, col)) : nullptr;
  const i64 to_row = dir * (BACK ? a.dx.row : a.h.row) * (i64)sizeof(T), gate_row = dir * a.dgate.row * (i64)sizeof(T);
  auto rows_left = [&](i64 k, i64 of) {                      // rows of this thread's run in step k that lie in [.., of)
    const i64 n = live ? of - (k * L * C + tau0) : 0;
    return n > LT ? LT : n < 0 ? 0 : (int)n;
  };
  auto fetch = [&](int to_stage, i64 k) {
    const int n = rows_left(k, len);
    if constexpr (BACK) feed.fetch(to_stage, {n, n, a.dh.base ? n : 0, rows_left(k, len - 1)});      // the first token has none before it
    else feed.fetch(to_stage, {n, n});
  };
  for (int k = 0; k < (S > 1 ? S - 1 : 1); ++k) fetch(k, k);
  if constexpr (C > 1) {                           // every block of the cluster runs, its barriers set up, before it is written to
    if (tid < 2) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&exchange.full[tid])) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    cg::this_cluster().sync();
  }
  int stage = 0;
  for (i64 k = 0; k < steps; ++k) {
    const int n = rows_left(k, len);
    if constexpr (S > 1) {
      fetch(stage == 0 ? S - 1 : stage - 1, k + S - 1);
      feed.arrived();
    }
    Vec<V> f[LT], u[LT];                           // forward: gate and (1 - gate) * x; gradient: gate and dh
    Vec<V> in[BACK ? LT : 1], w[BACK ? LT : 1];    // gradient: 1 - gate and (h[t-1] - x) * gate * (1 - gate)
#pragma unroll
    for (int j = 0; j < LT; ++j) {
      float g[V], x[V];
      feed.get(stage, 0, j, g);
      feed.get(stage, 1, j, x);
      Vec<V> i;
      sigmoid_pair<V>(g, f[j], i);
      if constexpr (!BACK) {
        u[j] = mul<V>(i, vec<V>(x));
      } else {
        float hp[V], d[V];
        feed.get(stage, 2, j, d);
        feed.get(stage, 3, j, hp);
        u[j] = a.dh.base ? vec<V>(d) : all<V>(0.f);
        if (k * L * C + tau0 + j == len - 1 && live) {
#pragma unroll
          for (int v = 0; v < V; ++v) hp[v] = a.initial ? a.initial[seq * a.width + col + v] : 0.f;
        }
        in[j] = i;
        w[j] = mul<V>(fma<V>(vec<V>(x), all<V>(-1.f), vec<V>(hp)), mul<V>(f[j], i));
      }
    }
    if (n < LT) {                                  // tokens past the end change nothing
#pragma unroll
      for (int j = 0; j < LT; ++j)
        if (j >= n) f[j] = all<V>(1.f), u[j] = all<V>(0.f);
    }
    if constexpr (S == 1) fetch(0, k + 1);
    // this thread's run as one map
    Vec<V> A = f[0], B = BACK ? mul<V>(f[0], u[0]) : u[0];
#pragma unroll
    for (int j = 1; j < LT; ++j) {
      A = mul<V>(A, f[j]);
      B = BACK ? mul<V>(f[j], add<V>(B, u[j])) : fma<V>(f[j], B, u[j]);
    }
    float o[V];
    floats<V>(A, o);
    st_plain<float, V>(&run_a[sub][pc], pack<float, V>(o));
    floats<V>(B, o);
    st_plain<float, V>(&run_b[sub][pc], pack<float, V>(o));
    __syncthreads();
    // the channels' threads join the runs' maps (in a cluster first the blocks') and leave each run its state
    if (tid < CH) {
      float s = carry;
      if constexpr (C > 1) {
        const int buf = (int)(k & 1);
        float ba = 1.f, bb = 0.f;
#pragma unroll
        for (int q = 0; q < SUBS; ++q) {
          bb = run_a[q][tid] * bb + run_b[q][tid];
          ba *= run_a[q][tid];
        }
        const unsigned full = shared_address(&exchange.full[buf]), place = shared_address(&exchange.map[buf][rank][tid]);
        if (tid == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full), "n"(C * CH * 8) : "memory");
        const u64 map = pair(ba, bb);
#pragma unroll
        for (int r = 0; r < C; ++r)
          asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(in_block(place, r)), "l"(map),
                       "r"(in_block(full, r)) : "memory");
        if (!wait_full(full, (unsigned)(k >> 1) & 1)) carry = __int_as_float(0x7fffffff);      // cannot happen; shows as NaN
#pragma unroll
        for (int r = 0; r < C; ++r) {
          if (r == rank) s = carry;
          float ra, rb;
          asm("mov.b64 {%0, %1}, %2;" : "=f"(ra), "=f"(rb) : "l"(exchange.map[buf][r][tid]));
          carry = ra * carry + rb;
        }
      }
#pragma unroll
      for (int q = 0; q < SUBS; ++q) {
        enter[q][tid] = s;
        s = run_a[q][tid] * s + run_b[q][tid];
      }
      if (C == 1) carry = s;
    }
    __syncthreads();
    unpack<float, V>(ld_plain<float, V>(&enter[sub][pc]), o);
    Vec<V> s = vec<V>(o);
#pragma unroll
    for (int j = 0; j < LT; ++j) {
      if constexpr (!BACK) {
        s = fma<V>(f[j], s, u[j]);
        floats<V>(s, o);
        if (j < n) st_stream<T, V>(reinterpret_cast<T*>(to + j * to_row), pack<T, V>(o));
      } else {
        const Vec<V> lam = add<V>(u[j], s);
        s = mul<V>(f[j], lam);
        float og[V];
        floats<V>(mul<V>(in[j], lam), o);
        floats<V>(mul<V>(w[j], lam), og);
        if (j < n) {
          st_stream<T, V>(reinterpret_cast<T*>(to + j * to_row), pack<T, V>(o));
          st_stream<T, V>(reinterpret_cast<T*>(to_gate + j * gate_row), pack<T, V>(og));
        }
      }
    }
    to += to_row * L * C;
    if (BACK) to_gate += gate_row * L * C;
    stage = stage + 1 == S ? 0 : stage + 1;
  }
  if (a.final_state && owner && rank == 0) a.final_state[seq * a.width + chan0 + tid] = carry;
}

// ------------------------------------------------------------------------------------------------ host side
template <class T, int V, int CP, int LT, int S, int C, int MIN_BLOCKS, bool BACK> int launch_c(ScanArgs a, cudaStream_t s) {
  const char* const fn = BACK ? "appy_gated_scan_grad" : "appy_gated_scan";
  const auto kernel = k_scan<T, V, CP, LT, S, C, MIN_BLOCKS, BACK>;
  a.tiles = (int)((a.width + CP * V - 1) / (CP * V));
  const i64 blocks = a.sequences * a.tiles * C;
  if (blocks > 0x7fffffff) return fail_named(fn, "too many sequences for one launch");
  const int dyn = Feed<T, V, LT, BACK ? 4 : 2, S>::kBytes;
  static bool ready[16] = {false};                 // per instantiation and device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 16 || !ready[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, dyn);
    if (e == cudaSuccess && C > 8) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return appy_fail_cuda(e, "gated scan set-up");
    if (dev >= 0 && dev < 16) ready[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kBlock);
  cfg.dynamicSmemBytes = dyn;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return appy_fail_cuda(e, "gated scan launch");
  }
  return finish("gated scan launch");
}

// CP1, S1: threads along the channels and stages of a block on its own, CPC, SC: in a cluster (narrower tiles make
// more clusters, fewer stages leave room for as many blocks beside the exchange)
template <class T, int V, int CP1, int CPC, int LT, int S1, int SC, int MIN_BLOCKS, bool BACK> int launch_scan(const ScanArgs& a, cudaStream_t s) {
  // blocks of their own if they come to two per SM; else clusters along the tokens, up to 16 blocks, as long as the
  // cluster's step is not longer than the tokens
  const i64 slots = 2 * (i64)sm_count();
  if (a.sequences * ((a.width + CP1 * V - 1) / (CP1 * V)) >= slots) return launch_c<T, V, CP1, LT, S1, 1, MIN_BLOCKS, BACK>(a, s);
  const i64 units = a.sequences * ((a.width + CPC * V - 1) / (CPC * V)), L = kBlock / CPC * LT;
  int c = 1;
  while (c < 16 && units * c < 2 * slots && L * c < a.tokens) c *= 2;
  switch (c) {
    case 1: return launch_c<T, V, CPC, LT, SC, 1, MIN_BLOCKS, BACK>(a, s);
    case 2: return launch_c<T, V, CPC, LT, SC, 2, MIN_BLOCKS, BACK>(a, s);
    case 4: return launch_c<T, V, CPC, LT, SC, 4, MIN_BLOCKS, BACK>(a, s);
    case 8: return launch_c<T, V, CPC, LT, SC, 8, MIN_BLOCKS, BACK>(a, s);
    default: return launch_c<T, V, CPC, LT, SC, 16, MIN_BLOCKS, BACK>(a, s);
  }
}

bool packs(const Rows& r, int V, int size) { return !r.base || (r.seq % V == 0 && r.row % V == 0 && aligned(r.base, (size_t)V * size)); }

int check_shape(const char* fn, int dtype, const void* offsets, int offsets_dtype, i64 sequences, i64 tokens, i64 width) {
  if (!element_size(dtype)) return fail_named(fn, "dtype must be APPY_F32, APPY_F16 or APPY_BF16");
  if (offsets && offsets_dtype != APPY_I32 && offsets_dtype != APPY_I64) return fail_named(fn, "offsets_dtype must be APPY_I32 or APPY_I64");
  if (sequences < 0 || tokens < 0 || width < 0) return fail_named(fn, "negative size");
  if (width > 0x3fffffff) return fail_named(fn, "width is too large");
  return APPY_OK;
}

}  // namespace

extern "C" {

int appy_gated_scan(const void* dx, int64_t x_seq, int64_t x_row, const void* dgate, int64_t gate_seq, int64_t gate_row, int dtype,
                    const void* doffsets, int offsets_dtype, int64_t sequences, int64_t tokens, int64_t width,
                    const float* dinitial, void* dh, int64_t h_seq, int64_t h_row, float* dlast, int fill, void* stream) {
  static const char fn[] = "appy_gated_scan";
  if (int rc = check_shape(fn, dtype, doffsets, offsets_dtype, sequences, tokens, width)) return rc;
  if (sequences == 0 || width == 0) return APPY_OK;
  if (tokens && (!dx || !dgate || !dh)) return fail_named(fn, "NULL argument");
  ScanArgs a = {};
  a.x = {const_cast<void*>(dx), x_seq, x_row};
  a.gate = {const_cast<void*>(dgate), gate_seq, gate_row};
  a.h = {dh, h_seq, h_row};
  a.initial = dinitial;
  a.final_state = dlast;
  a.offsets = doffsets;
  a.wide = offsets_dtype == APPY_I64;
  a.fill = fill != 0;
  a.sequences = sequences;
  a.tokens = tokens;
  a.width = width;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int size = element_size(dtype);
  const bool vec = width % 4 == 0 && packs(a.x, 4, size) && packs(a.gate, 4, size) && packs(a.h, 4, size);
  return APPY_OP_DTYPE(dtype, {
    constexpr bool wide = sizeof(T) == 4;
    return vec ? launch_scan<T, 4, wide ? 8 : 16, 8, wide ? 4 : 8, 3, 2, 4, false>(a, s) : launch_scan<T, 1, 32, 32, 16, wide ? 3 : 1, wide ? 3 : 1, 4, false>(a, s);
  });
}

int appy_gated_scan_grad(const void* ddh, int64_t dh_seq, int64_t dh_row, const void* dx, int64_t x_seq, int64_t x_row,
                         const void* dgate, int64_t gate_seq, int64_t gate_row, const void* dh, int64_t h_seq, int64_t h_row,
                         int dtype, const void* doffsets, int offsets_dtype, int64_t sequences, int64_t tokens, int64_t width,
                         const float* dinitial, const float* dgrad_last, void* dgrad_x, int64_t gx_seq, int64_t gx_row,
                         void* dgrad_gate, int64_t gg_seq, int64_t gg_row, float* dgrad_initial, int fill, void* stream) {
  static const char fn[] = "appy_gated_scan_grad";
  if (int rc = check_shape(fn, dtype, doffsets, offsets_dtype, sequences, tokens, width)) return rc;
  if (sequences == 0 || width == 0) return APPY_OK;
  if (tokens && (!dx || !dgate || !dh || !dgrad_x || !dgrad_gate)) return fail_named(fn, "NULL argument");
  ScanArgs a = {};
  a.dh = {const_cast<void*>(ddh), dh_seq, dh_row};
  a.x = {const_cast<void*>(dx), x_seq, x_row};
  a.gate = {const_cast<void*>(dgate), gate_seq, gate_row};
  a.h = {const_cast<void*>(dh), h_seq, h_row};
  a.dx = {dgrad_x, gx_seq, gx_row};
  a.dgate = {dgrad_gate, gg_seq, gg_row};
  a.initial = dinitial;
  a.dlast = dgrad_last;
  a.final_state = dgrad_initial;
  a.offsets = doffsets;
  a.wide = offsets_dtype == APPY_I64;
  a.fill = fill != 0;
  a.sequences = sequences;
  a.tokens = tokens;
  a.width = width;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int size = element_size(dtype);
  const bool vec = width % 4 == 0 && packs(a.x, 4, size) && packs(a.gate, 4, size) && packs(a.h, 4, size) && packs(a.dh, 4, size) &&
                   packs(a.dx, 4, size) && packs(a.dgate, 4, size);
  return APPY_OP_DTYPE(dtype, {
    constexpr bool wide = sizeof(T) == 4;
    return vec ? launch_scan<T, 4, wide ? 8 : 16, 8, 4, wide ? 2 : 3, 2, wide ? 3 : 4, true>(a, s) : launch_scan<T, 1, 32, 32, 8, wide ? 3 : 1, wide ? 3 : 1, 4, true>(a, s);
  });
}

}  // extern "C"
