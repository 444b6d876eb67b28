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
// mu past the last token is the gradient of the last state, mu[0] that of the initial one.  h[t-1] is read as the forward pass
// left it, rounded to the type of x: half a step of it in 16 bits is the largest error of dgate, about that of rounding dgate
// itself (bfloat16: off by 0.0018 of its size, 0.0016 with float32 states).  The states in float32 would cost a
// third more bytes in the forward pass and a sixth more in this one.
//
// A block takes 64 or 32 channels of one sequence and walks along it; with few sequences and channels a cluster of
// blocks takes neighbouring stretches of tokens in each step, so that the whole machine loads at a time.  States are float32; each result is rounded once.
#include <cooperative_groups.h>
#include <cuda.h>

#include <type_traits>

#include "operators.cuh"

namespace {
using namespace appy_op;
namespace cg = cooperative_groups;

// f = sigmoid(g) and i = 1 - f: with e = exp(-g), f = 1 / (1 + e) and i = e f, so that neither is a difference.  The exponent
// -g log2(e) is rounded once, so the smaller of the two is off by up to (1.3 |g| + 8) 2^-24 of itself, the larger by a few
// 2^-24.  A gate below -87 counts as -87, so that e stays finite: f is 1.6e-38 there, not less.  From 87.4 on e is below the
// normal range and counts as zero: f is 1 and i is 0.
template <class T, int V> APPY_DEV void bounded_gate(Pack<T, V> k, float (&g)[V]) {
  if constexpr (sizeof(T) == 2 && V > 1) {         // two at a time, as they came
    typename Pack<T, V>::Bits u;
    u.raw = k.raw;
    const unsigned bound = pack2(-87.f, -87.f, T());
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same<T, bf16>::value) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(u.w[i]) : "r"(bound));
      else asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(u.w[i]) : "r"(bound));
    }
    k.raw = u.raw;
    unpack<T, V>(k, g);
  } else {
    unpack<T, V>(k, g);
#pragma unroll
    for (int v = 0; v < V; ++v) asm("max.NaN.f32 %0, %0, %1;" : "+f"(g[v]) : "f"(-87.f));
  }
}
template <int V> APPY_DEV void sigmoid_pair(const float (&g)[V], Vec<V>& f, Vec<V>& i) {
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

APPY_DEV float quiet_nan() { return __int_as_float(0x7fffffff); }

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
template <class T, int V> APPY_DEV void clear_rows(const Rows& r, i64 lo, i64 hi, i64 col, i64 width, int sub, int subs) {
  for (i64 t = lo + sub; t < hi; t += subs)
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (col + v < width) *row_ptr<T>(r, 0, 0, t, col + v) = from_f32<T>(0.f);
}

APPY_DEV unsigned shared_address(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
// Each try suspends the warp for up to about 4 us; false: it gave up after about a second.
APPY_DEV bool wait_full(unsigned barrier, unsigned parity) {
  for (unsigned tries = 0; tries < (1u << 18); ++tries) {
    unsigned done;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done) : "r"(barrier), "r"(parity), "r"(1000u) : "memory");
    if (done) return true;
  }
  return false;
}
APPY_DEV void expect_bytes(unsigned barrier, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"(bytes) : "memory");
}

// The arrays that a step reads: gate, x; for the gradient also dh and h of the token before.
template <int NA> struct Maps { CUtensorMap m[NA]; };
struct NoMaps {};

// What the blocks of a cluster tell one another about a step.  Each channel has an owner among the blocks: every block
// sends it the channel's map (A, B) over its stretch of the step, the owner, which also carries the channel's state from
// step to step, sends every block the state that its stretch begins with.  Both travel as st.async, whose bytes count
// towards a barrier of the receiver, so no block waits for stores of another kind, and a step costs 2 CH messages per
// block however large the cluster is (all maps to all blocks were C CH, and the step 3.4 us for C = 16).
// Two buffers alternate: a channel's map of step k + 2 is sent after its state of step k + 1 has come, which its owner
// sends after it has read the maps of step k, and its state of step k + 2 after all blocks' maps of step k + 2, which
// they send after they have read their state of step k.
template <int C, int CH> struct Exchange {
  u64 map[2][C][CH / C];
  float state[2][CH];
  u64 maps_full[2], states_full[2];
};
APPY_DEV unsigned in_block(unsigned address, int rank) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
  return r;
}

// V channels per thread, CP threads along the channels, LT tokens per thread, NT threads, C blocks per cluster.
//
// Where rows start on 16-byte boundaries, TMA brings the tiles of a step (L tokens of CH channels of each array) into a
// ring of S stages, some steps ahead (S > 1, V = 4); what lies outside the arrays arrives as zeros.  Elsewhere every
// thread loads its elements into registers one step ahead (S = 1, V = 1).
//
// While the maps of step k + 1 travel (to the other warps; in a cluster to the owners and back), step k is replayed and
// the maps of step k + 2 are made: a step waits for nobody in the middle, and one barrier per step is enough.
template <class T, int V, int CP, int LT, int S, int NT, int C, bool BACK> struct Shape {
  static constexpr int CH = CP * V, SUBS = NT / CP, L = SUBS * LT, NA = BACK ? 4 : 2;
  struct Shared {
    T ring[S > 1 ? S : 1][2][S > 1 ? L * CH : 8];                // gate and x; gradient: gate and dh
    T late[S > 1 && BACK ? S : 1][2][S > 1 && BACK ? L * CH : 8];      // gradient: x and h of the token before
    float run_a[2][SUBS][CH], run_b[2][SUBS][CH], enter[2][SUBS][CH];
    Exchange<C, CH> exchange;
    u64 loaded[S], late_loaded[S];
  };
};

template <class T, int V, int CP, int LT, int S, int NT, int C, int MIN_BLOCKS, bool BACK>
__global__ void __launch_bounds__(NT, MIN_BLOCKS)
k_scan(const ScanArgs a, const __grid_constant__ typename std::conditional<(S > 1), Maps<BACK ? 4 : 2>, NoMaps>::type maps) {
  typedef Shape<T, V, CP, LT, S, NT, C, BACK> Sh;
  constexpr int CH = Sh::CH, SUBS = Sh::SUBS, L = Sh::L, NA = Sh::NA;
  // The maps of a step are joined by all threads: a warp takes WC channels, G lanes of it share a channel's runs.
  constexpr int WC = CH / (NT / 32), G = 32 / WC, PER = SUBS / G;
  static_assert(G * WC == 32 && PER * G == SUBS, "every run of every channel belongs to one lane");
  // The gradient needs x and h only when it replays a step; from a ring they are read as late as that.
  constexpr bool KEEP = !BACK || S == 1;
  extern __shared__ __align__(128) unsigned char shared_memory[];
  typename Sh::Shared& sh = *reinterpret_cast<typename Sh::Shared*>(shared_memory);
  const int tid = threadIdx.x, lane = tid & 31, sub = tid / CP, pc = (tid % CP) * V;
  const int join_ch = tid / 32 * WC + lane % WC, join_run = lane / WC * PER;
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
        clear_rows<T, V>(BACK ? a.dx : a.h, 0, first, col, a.width, sub, SUBS);
        if (BACK) clear_rows<T, V>(a.dgate, 0, first, col, a.width, sub, SUBS);
      }
      if (seq == a.sequences - 1) {
        clear_rows<T, V>(BACK ? a.dx : a.h, end, a.tokens, col, a.width, sub, SUBS);
        if (BACK) clear_rows<T, V>(a.dgate, end, a.tokens, col, a.width, sub, SUBS);
      }
    }
  }
  // The state before the step whose maps are joined next: in a block of its own in all G lanes of a channel, in a
  // cluster in C threads of the channel's owner.
  constexpr int OWN = CH / C;
  const int carry_ch = C == 1 ? join_ch : rank * OWN + tid % OWN;
  float carry = 0.f;
  const float* const start = BACK ? a.dlast : a.initial;
  if (start && chan0 + carry_ch < a.width) carry = start[seq * a.width + chan0 + carry_ch];
  const i64 steps = (len + (i64)L * C - 1) / ((i64)L * C);
  // this thread's run in the first step, in walking order (backwards for the gradient)
  const i64 tau0 = (i64)rank * L + sub * LT, t0 = BACK ? len - 1 - tau0 : tau0;
  constexpr int dir = BACK ? -1 : 1;
  char* to = reinterpret_cast<char*>(row_ptr<T>(BACK ? a.dx : a.h, seq_at, first, t0, col));
  char* to_gate = BACK ? reinterpret_cast<char*>(row_ptr<T>(a.dgate, seq_at, first, t0, col)) : nullptr;
  const i64 to_row = dir * (BACK ? a.dx.row : a.h.row) * (i64)sizeof(T), gate_row = dir * a.dgate.row * (i64)sizeof(T);
  auto rows_left = [&](i64 k, i64 of) {            // rows of this thread's run in step k that lie in [.., of)
    const i64 n = live ? of - (k * L * C + tau0) : 0;
    return n > LT ? LT : n < 0 ? 0 : (int)n;
  };
  // A wait that gives up, which cannot happen, shows as NaN in all that its block writes.  In a cluster the block stops with the
  // step, so the others, which wait for its next message, give up too, and none of them leaves before the rest.
  bool in_time = true;
  auto wait = [&](const u64* barrier, unsigned parity) { in_time = in_time && wait_full(shared_address(barrier), parity); };
  auto meet = [&] {                                // in a cluster all threads learn whether one gave up, before they send
    if constexpr (C > 1) in_time = __syncthreads_and(in_time);
    else __syncthreads();
  };

  // ---- reading: array 0 gate, 1 x, 2 dh, 3 h of the token before
  Pack<T, V> held[S > 1 ? 1 : NA][S > 1 ? 1 : LT];
  int make_stage = 0, replay_stage = 0;
  unsigned make_parity = 0, replay_parity = 0;
  auto next = [](int& stage, unsigned& parity) {
    stage = stage + 1 == S ? 0 : stage + 1;
    if (stage == 0) parity ^= 1;
  };
  auto load = [&](u64* loaded, i64 k, auto& ring, int x, int y) {        // two arrays of step k by TMA
    if (tid != 0 || k >= steps) return;
    const int stage = (int)(k % S);
    const unsigned barrier = shared_address(&loaded[stage]);
    const bool first_too = x != 2 || a.dh.base, second_too = y != 2 || a.dh.base;
    expect_bytes(barrier, (first_too + second_too) * (unsigned)(L * CH * sizeof(T)));
    if constexpr (S > 1) {
      const i64 base = (k * C + rank) * L, t = first + (BACK ? len - base - L : base);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int array = q ? y : x;
        if (q ? second_too : first_too)
          asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                           shared_address(&ring[stage][q][0])),
                       "l"(&maps.m[array]), "r"((int)chan0), "r"((int)(array == 3 ? t - 1 : t)), "r"((int)seq_at), "r"(barrier)
                       : "memory");
      }
    }
  };
  const T* from[NA];                               // S = 1: this thread's first row of the step to fetch next
  i64 from_row[NA];
  if constexpr (S == 1) {
#pragma unroll
    for (int x = 0; x < NA; ++x) {
      const Rows& r = x == 0 ? a.gate : x == 1 ? a.x : x == 2 ? a.dh : a.h;
      from[x] = row_ptr<const T>(r, seq_at, first, x == 3 ? t0 - 1 : t0, col);
      from_row[x] = dir * r.row;
    }
  }
  auto fetch = [&](i64 k) {                        // what step k is made from (registers: all of it)
    if constexpr (S > 1) {
      load(sh.loaded, k, sh.ring, 0, BACK ? 2 : 1);
    } else {
      const int n = rows_left(k, len), n_before = BACK ? rows_left(k, len - 1) : 0;      // the first token has none before it
#pragma unroll
      for (int x = 0; x < NA; ++x) {
        const int lim = x == 3 ? n_before : x == 2 && !a.dh.base ? 0 : n;
#pragma unroll
        for (int j = 0; j < LT; ++j)
          if (j < lim) held[x][j] = ld_stream<T, V>(from[x] + j * from_row[x]);
        from[x] += from_row[x] * L * C;
      }
    }
  };
  auto fetch_late = [&](i64 k) {
    if constexpr (S > 1 && BACK) load(sh.late_loaded, k, sh.late, 1, 3);
  };
  const int at_row = BACK ? L - 1 - sub * LT : sub * LT;
  auto word = [&](const auto& ring, int stage, int q, int x, int j) -> Pack<T, V> {
    if constexpr (S > 1) return ld_plain<T, V>(&ring[stage][q][(at_row + dir * j) * CH + pc]);
    else return held[x][j];
  };

  struct Step {
    Vec<V> f[LT];                                  // gate
    Vec<V> i[BACK ? LT : 1];                       // gradient: 1 - gate
    Vec<V> u[BACK ? 1 : LT];                       // forward: (1 - gate) * x
    Pack<T, V> dh[BACK ? LT : 1];                  // gradient, as it came
    Vec<V> w[BACK && KEEP ? LT : 1];               // gradient: h[t-1] - x
  };
  auto dh_of = [&](Pack<T, V> word) {
    float d[V];
    unpack<T, V>(word, d);
    return a.dh.base ? vec<V>(d) : all<V>(0.f);
  };
  auto difference = [&](int stage, int first_token, int j) {      // h[t-1] - x
    float x[V], hp[V];
    unpack<T, V>(word(sh.late, stage, 0, 1, j), x);
    unpack<T, V>(word(sh.late, stage, 1, NA - 1, j), hp);
    if (j == first_token) {
#pragma unroll
      for (int v = 0; v < V; ++v) hp[v] = a.initial && col + v < a.width ? a.initial[seq * a.width + col + v] : 0.f;
    }
    return fma<V>(vec<V>(x), all<V>(-1.f), vec<V>(hp));
  };
  // gates and maps of step k
  auto make = [&](i64 k, Step& st) {
    const int buf = (int)(k & 1), n = rows_left(k, len), n_before = BACK ? rows_left(k, len - 1) : n;      // one less where the sequence begins
    if constexpr (S > 1) wait(&sh.loaded[make_stage], make_parity);
    Vec<V> u[LT];
#pragma unroll
    for (int j = 0; j < LT; ++j) {
      float g[V];
      bounded_gate<T, V>(word(sh.ring, make_stage, 0, 0, j), g);
      Vec<V> i;
      sigmoid_pair<V>(g, st.f[j], i);
      if constexpr (BACK) {
        st.i[j] = i;
        st.dh[j] = word(sh.ring, make_stage, 1, NA - 2, j);
        u[j] = dh_of(st.dh[j]);
        if constexpr (KEEP) st.w[j] = difference(make_stage, n - n_before == 1 ? n_before : -1, j);
      } else {
        float x[V];
        unpack<T, V>(word(sh.ring, make_stage, 1, 1, j), x);
        u[j] = mul<V>(i, vec<V>(x));
      }
    }
    if (n < LT) {                                  // tokens past the end change nothing
#pragma unroll
      for (int j = 0; j < LT; ++j)
        if (j >= n) st.f[j] = all<V>(1.f), u[j] = all<V>(0.f);
    }
    Vec<V> A = st.f[0], B = BACK ? mul<V>(st.f[0], u[0]) : u[0];
#pragma unroll
    for (int j = 0; j < LT; ++j) {
      if constexpr (!BACK) st.u[j] = u[j];
      if (j == 0) continue;
      A = mul<V>(A, st.f[j]);
      B = BACK ? mul<V>(st.f[j], add<V>(B, u[j])) : fma<V>(st.f[j], B, u[j]);
    }
    next(make_stage, make_parity);
    float o[V];
    floats<V>(A, o);
    st_plain<float, V>(&sh.run_a[buf][sub][pc], pack<float, V>(o));
    floats<V>(B, o);
    st_plain<float, V>(&sh.run_b[buf][sub][pc], pack<float, V>(o));
  };
  // joins the maps of step k: this lane's PER runs, the G lanes of the channel (in a cluster the blocks, for which
  // `send` and `join` come apart), and leaves each run the state it starts from
  float ma[PER], mb[PER], before_a, before_b;
  auto send = [&](i64 k) {
    const int buf = (int)(k & 1);
    float A = 1.f, B = 0.f;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      ma[q] = sh.run_a[buf][join_run + q][join_ch];
      mb[q] = sh.run_b[buf][join_run + q][join_ch];
      B = ma[q] * B + mb[q];
      A *= ma[q];
    }
#pragma unroll
    for (int o = WC; o < 32; o *= 2) {
      const float pa = __shfl_up_sync(APPY_FULL_MASK, A, o), pb = __shfl_up_sync(APPY_FULL_MASK, B, o);
      if (lane >= o) {
        B = A * pb + B;
        A *= pa;
      }
    }
    before_a = 1.f;
    before_b = 0.f;
    if constexpr (G > 1) {
      const float pa = __shfl_up_sync(APPY_FULL_MASK, A, WC), pb = __shfl_up_sync(APPY_FULL_MASK, B, WC);
      if (lane >= WC) before_a = pa, before_b = pb;
    }
    if constexpr (C > 1) {
      const unsigned full = shared_address(&sh.exchange.maps_full[buf]);
      if (tid == 0) {
        expect_bytes(full, CH * 8);
        expect_bytes(shared_address(&sh.exchange.states_full[buf]), CH * 4);
      }
      if (lane >= 32 - WC)                         // the last of a channel's lanes has the block's map
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(
                         in_block(shared_address(&sh.exchange.map[buf][rank][join_ch % OWN]), join_ch / OWN)),
                     "l"(pair(A, B)), "r"(in_block(full, join_ch / OWN))
                     : "memory");
    }
  };
  auto answer = [&](i64 k) {                       // the owner's part: thread (channel, block)
    if (tid >= CH) return;
    const int buf = (int)(k & 1), ch = tid % OWN, to_rank = tid / OWN;
    wait(&sh.exchange.maps_full[buf], (unsigned)(k >> 1) & 1);
    if (!in_time) return;
    float s = carry;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      if (r == to_rank) s = carry;
      float ra, rb;
      asm("mov.b64 {%0, %1}, %2;" : "=f"(ra), "=f"(rb) : "l"(sh.exchange.map[buf][r][ch]));
      carry = ra * carry + rb;
    }
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(
                     in_block(shared_address(&sh.exchange.state[buf][rank * OWN + ch]), to_rank)),
                 "r"(__float_as_uint(s)), "r"(in_block(shared_address(&sh.exchange.states_full[buf]), to_rank))
                 : "memory");
  };
  auto join = [&](i64 k) {
    const int buf = (int)(k & 1);
    float s = carry;
    if constexpr (C > 1) {
      wait(&sh.exchange.states_full[buf], (unsigned)(k >> 1) & 1);
      s = sh.exchange.state[buf][join_ch];
    }
    s = before_a * s + before_b;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      sh.enter[buf][join_run + q][join_ch] = s;
      s = ma[q] * s + mb[q];
    }
    if constexpr (C == 1) carry = __shfl_sync(APPY_FULL_MASK, s, 32 - WC + lane % WC);
  };
  auto replay = [&](i64 k, const Step& st) {
    const int buf = (int)(k & 1), n = rows_left(k, len), n_before = BACK ? rows_left(k, len - 1) : n;
    if constexpr (S > 1 && BACK) wait(&sh.late_loaded[replay_stage], replay_parity);
    float o[V];
    unpack<float, V>(ld_plain<float, V>(&sh.enter[buf][sub][pc]), o);
    Vec<V> state = vec<V>(o);
#pragma unroll
    for (int j = 0; j < LT; ++j) {
      if constexpr (!BACK) {
        state = fma<V>(st.f[j], state, st.u[j]);
        floats<V>(state, o);
        if (j < n) st_stream<T, V>(reinterpret_cast<T*>(to + j * to_row), pack<T, V>(o));
      } else {
        Vec<V> w;
        if constexpr (KEEP) w = st.w[j];
        else w = difference(replay_stage, n - n_before == 1 ? n_before : -1, j);
        const Vec<V> lam = add<V>(dh_of(st.dh[j]), state);
        state = mul<V>(st.f[j], lam);
        float og[V];
        const Vec<V> d = mul<V>(st.i[j], lam);
        floats<V>(d, o);
        floats<V>(mul<V>(w, mul<V>(st.f[j], d)), og);
        if (j < n) {
          st_stream<T, V>(reinterpret_cast<T*>(to + j * to_row), pack<T, V>(o));
          st_stream<T, V>(reinterpret_cast<T*>(to_gate + j * gate_row), pack<T, V>(og));
        }
      }
    }
    if constexpr (BACK) next(replay_stage, replay_parity);
    to += to_row * L * C;
    if (BACK) to_gate += gate_row * L * C;
  };
  if (S > 1 || C > 1) {                            // barriers, before anybody counts on them
    if (tid < S) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&sh.loaded[tid])) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&sh.late_loaded[tid])) : "memory");
    }
    if (tid < 2) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&sh.exchange.maps_full[tid])) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&sh.exchange.states_full[tid])) : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if constexpr (C > 1) cg::this_cluster().sync();          // every block of the cluster runs before it is written to
    else __syncthreads();
  }
  for (int k = 0; k < S; ++k) {
    fetch(k);
    fetch_late(k);
  }
  if (steps > 0) {
    Step even, odd;
    // A stage is free once all threads have done with its step: made it, or, for what comes late, replayed it.
    auto refill = [&](i64 made) {
      if constexpr (S > 1) fetch(made + S);
    };
    auto advance = [&](i64 k, Step& st) {          // st: step k, then step k + 2
      const bool more = k + 1 < steps;
      if (more) send(k + 1);
      if (C == 1 && more) join(k + 1);
      replay(k, st);
      if (C > 1 && more) answer(k + 1);
      if (k + 2 < steps) {
        make(k + 2, st);
        if constexpr (S == 1) fetch(k + 3);
      }
      if (C > 1 && more) join(k + 1);
      meet();
      refill(k + 2);
      fetch_late(k + S);
    };
    make(0, even);
    if constexpr (S == 1) fetch(1);
    meet();
    refill(0);
    send(0);
    if constexpr (C > 1) answer(0);
    if (steps > 1) {
      make(1, odd);
      if constexpr (S == 1) fetch(2);
    }
    join(0);
    meet();
    refill(1);
    for (i64 k = 0; k < steps && (C == 1 || in_time); k += 2) {
      advance(k, even);
      if (k + 1 < steps && (C == 1 || in_time)) advance(k + 1, odd);
    }
  }
  if (S > 1 || C > 1) {
    if (__builtin_expect(__syncthreads_or(!in_time), 0)) {
      carry = quiet_nan();
      to = reinterpret_cast<char*>(row_ptr<T>(BACK ? a.dx : a.h, seq_at, first, t0, col));
      if (BACK) to_gate = reinterpret_cast<char*>(row_ptr<T>(a.dgate, seq_at, first, t0, col));
      for (i64 k = 0; k < steps; ++k) {
        const int n = rows_left(k, len);
        for (int j = 0; j < n; ++j)
          for (int v = 0; v < V; ++v) {
            reinterpret_cast<T*>(to + j * to_row)[v] = from_f32<T>(quiet_nan());
            if (BACK) reinterpret_cast<T*>(to_gate + j * gate_row)[v] = from_f32<T>(quiet_nan());
          }
        to += to_row * L * C;
        to_gate += BACK ? gate_row * L * C : 0;
      }
      if constexpr (C > 1) cg::this_cluster().sync();
      for (int x = 0; x < 10; ++x) __nanosleep(100000);          // for what is on its way to this block
    }
  }
  if (a.final_state && (C == 1 ? lane < WC : tid < OWN) && chan0 + carry_ch < a.width) a.final_state[seq * a.width + chan0 + carry_ch] = carry;
}

// One token of every sequence, the step of a serving loop: no scan, a thread per channel.
template <class T> __global__ void __launch_bounds__(256) k_scan_token(ScanArgs a) {
  const i64 i = (i64)blockIdx.x * 256 + threadIdx.x, seq = i / a.width, col = i - seq * a.width;
  if (seq >= a.sequences) return;
  float g[1] = {to_f32(*row_ptr<const T>(a.gate, seq, 0, 0, col))};
  const float x = to_f32(*row_ptr<const T>(a.x, seq, 0, 0, col));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(g[0]) : "f"(-87.f));
  Vec<1> f, in;
  sigmoid_pair<1>(g, f, in);
  const float h = fmaf(f.p[0], a.initial ? a.initial[i] : 0.f, in.p[0] * x);
  *row_ptr<T>(a.h, seq, 0, 0, col) = from_f32<T>(h);
  if (a.final_state) a.final_state[i] = h;
}

// ------------------------------------------------------------------------------------------------ host side
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// The array as (channel, token, sequence), read in boxes of `channels` by `tokens`.
template <class T> bool encode(CUtensorMap* m, const Rows& r, const ScanArgs& a, int channels, int tokens) {
  const i64 sequences = a.offsets ? 1 : a.sequences;
  const cuuint64_t dims[3] = {(cuuint64_t)a.width, (cuuint64_t)a.tokens, (cuuint64_t)sequences};
  const cuuint64_t strides[2] = {(cuuint64_t)r.row * sizeof(T), (cuuint64_t)(sequences > 1 ? r.seq : r.row) * sizeof(T)};
  const cuuint32_t box[3] = {(cuuint32_t)channels, (cuuint32_t)tokens, 1}, unit[3] = {1, 1, 1};
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : std::is_same<T, f16>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode_tiled()(m, type, 3, r.base, dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

const int kNoTma = -1000;                          // not a status: TMA cannot describe the arrays, read them without it

template <class T, int V, int CP, int LT, int S, int NT, int C, int MIN_BLOCKS, bool BACK> int launch_c(ScanArgs a, cudaStream_t s) {
  typedef Shape<T, V, CP, LT, S, NT, C, BACK> Sh;
  const char* const fn = BACK ? "appy_gated_scan_grad" : "appy_gated_scan";
  const auto kernel = k_scan<T, V, CP, LT, S, NT, C, MIN_BLOCKS, BACK>;
  a.tiles = (int)((a.width + Sh::CH - 1) / Sh::CH);
  const i64 blocks = a.sequences * a.tiles * C;
  if (blocks > 0x7fffffff) return fail_named(fn, "too many sequences for one launch");
  typename std::conditional<(S > 1), Maps<BACK ? 4 : 2>, NoMaps>::type maps;
  if constexpr (S > 1) {
    const Rows* rows[4] = {&a.gate, &a.x, a.dh.base ? &a.dh : &a.gate, &a.h};
    for (int x = 0; x < Sh::NA; ++x)
      if (!encode<T>(&maps.m[x], *rows[x], a, Sh::CH, Sh::L)) return kNoTma;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = sizeof(typename Sh::Shared);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  static signed char fits[16] = {0};               // per instantiation and device: 0 not known yet
  int dev = 0;
  cudaGetDevice(&dev);
  signed char known = dev >= 0 && dev < 16 ? fits[dev] : 0;
  if (!known) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(typename Sh::Shared));
    if (e == cudaSuccess && C > 8) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return appy_fail_cuda(e, "gated scan set-up");
    known = C <= 8 || cluster_fits(kernel, cfg) ? 1 : -1;
    if (dev >= 0 && dev < 16) fits[dev] = known;
  }
  if (known < 0) return kNoCluster;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, maps);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return appy_fail_cuda(e, "gated scan launch");
  }
  return finish("gated scan launch");
}

// Variants, each with the time of the one it was chosen over (B200, bfloat16 unless said, forward / gradient):
//   many (sequence, 64 channels) pairs, four per SM: 64-channel blocks of 4 tokens per thread, four to an SM
//     (64 x 512 x 2048: 71 us; 32-channel blocks of 8 tokens per thread 96 us), and short sequences (16 x 100 x 2048:
//     8 / 12 us; the others 12 / 14 us);
//   fewer: 32-channel blocks, twice as many; forward 8 tokens per thread and two blocks to an SM (8 x 2048 x 2048:
//     47 us; the first variant 53 us), gradient 4 tokens per thread and four blocks (73 us; the first variant 94 us);
//   fewer than two 32-channel blocks per SM: clusters along the tokens, as many blocks as keep to two per SM, which
//     is where all clusters run at once (65536 x 1024: 8 blocks 109 us, 16 blocks 160 us, one block 493 us);
//     packed sequences, whose lengths are uneven, up to twelve per SM (37 sequences of 0 to 8000 tokens of 648 float32
//     channels: two blocks 87 / 154 us, one 85 / 176 us).
template <class T, bool BACK> int launch_packed(const ScanArgs& a, cudaStream_t s) {
  constexpr bool wide = sizeof(T) == 4;
  constexpr int S = wide || BACK ? 2 : 4, LT = BACK ? 4 : 8;
  const i64 sms = sm_count(), units = a.sequences * ((a.width + 31) / 32), wide_units = a.sequences * ((a.width + 63) / 64);
  if (wide_units >= 4 * sms || a.tokens <= 128) return launch_c<T, 4, 16, 4, S, 128, 1, BACK && wide ? 3 : 4, BACK>(a, s);
  const i64 most = a.offsets ? 12 * sms : 2 * sms;
  int c = 1;
  while (c < 16 && units * 2 * c <= most && (i64)16 * LT * c < a.tokens) c *= 2;
  if (c == 16) {
    const int rc = launch_c<T, 4, 8, LT, S, 128, 16, 2, BACK>(a, s);
    if (rc != kNoCluster) return rc;
  }
  switch (c) {
    case 1: return launch_c<T, 4, 8, LT, S, 128, 1, BACK ? (wide ? 3 : 4) : 2, BACK>(a, s);
    case 2: return launch_c<T, 4, 8, LT, S, 128, 2, 2, BACK>(a, s);
    case 4: return launch_c<T, 4, 8, LT, S, 128, 4, 2, BACK>(a, s);
    default: return launch_c<T, 4, 8, LT, S, 128, 8, 2, BACK>(a, s);
  }
}
// Rows that TMA cannot read: the same with direct loads (two channels a thread, for packed arithmetic, 72 / 177 us for
// 8 x 2048 x 1001 bfloat16: the loads are what takes the time).  As many blocks to a cluster as keep to four per SM, for packed
// sequences, whose lengths are uneven, to twelve.  Times for 1, 2, 4 blocks, the chosen one marked; bfloat16:
//   8 x 2048 x 1001: 56, 46*, 48 / 137, 101*, 104 us;  16 x 2048 x 1001: 68*, 80, 87 / 169*, 182, 191;
//   2 x 8192 x 1001: 66 / 152 with 4, 49* / 103* with 8, 65 / 138 with 16;
//   packed, 37 sequences of 1500 tokens of 651 channels: 146, 119*, 109 / 373, 274*, 236;  200 of 150 of 1001: 76*, 131 / 161*, 219.
template <class T, bool BACK> int launch_direct(const ScanArgs& a, cudaStream_t s) {
  constexpr int LT = BACK ? 4 : 8;
  const i64 sms = sm_count(), units = a.sequences * ((a.width + 31) / 32);
  int c = 1;
  while (c < 16 && units * 2 * c <= (a.offsets ? 12 : 4) * sms && (i64)4 * LT * c < a.tokens) c *= 2;
  if (c == 16) {
    const int rc = launch_c<T, 1, 32, LT, 1, 128, 16, 4, BACK>(a, s);
    if (rc != kNoCluster) return rc;
  }
  switch (c) {
    case 1: return launch_c<T, 1, 32, LT, 1, 128, 1, 4, BACK>(a, s);
    case 2: return launch_c<T, 1, 32, LT, 1, 128, 2, 4, BACK>(a, s);
    case 4: return launch_c<T, 1, 32, LT, 1, 128, 4, 4, BACK>(a, s);
    default: return launch_c<T, 1, 32, LT, 1, 128, 8, 4, BACK>(a, s);
  }
}
template <class T> int launch_token(const ScanArgs& a, cudaStream_t s) {
  const i64 blocks = (a.sequences * a.width + 255) / 256;
  if (blocks > 0x7fffffff) return fail_named("appy_gated_scan", "too many sequences for one launch");
  k_scan_token<T><<<(unsigned)blocks, 256, 0, s>>>(a);
  return finish("gated scan launch");
}

// Whether TMA can read, and packs of four can be stored to, this array.
bool packs(const Rows& r, const ScanArgs& a, int size) {
  if (!r.base) return true;
  const i64 v = 16 / size;
  const bool rows = r.row % v == 0 && r.row >= a.width && r.row < (1ll << 36);
  const bool seqs = a.offsets || a.sequences == 1 || (r.seq % v == 0 && r.seq > 0 && r.seq < (1ll << 36));
  return aligned(r.base, 16) && rows && seqs;
}
bool packs(const ScanArgs& a, int size) {
  return a.width % 4 == 0 && a.tokens > 0 && a.tokens < (1ll << 31) && a.sequences < (1ll << 31) && encode_tiled() && packs(a.x, a, size) && packs(a.gate, a, size) &&
         packs(a.h, a, size) && packs(a.dh, a, size) && packs(a.dx, a, size) && packs(a.dgate, a, size);
}

template <class T, bool BACK> int launch_scan(const ScanArgs& a, cudaStream_t s) {
  if (!BACK && !a.offsets && a.tokens == 1) return launch_token<T>(a, s);
  const int rc = packs(a, sizeof(T)) ? launch_packed<T, BACK>(a, s) : kNoTma;
  return rc == kNoTma ? launch_direct<T, BACK>(a, s) : rc;
}

int check_shape(const char* fn, int dtype, const void* offsets, int offsets_dtype, i64 sequences, i64 tokens, i64 width) {
  if (!element_size(dtype)) return fail_named(fn, "dtype must be APPY_F32, APPY_F16 or APPY_BF16");
  if (offsets && offsets_dtype != APPY_I32 && offsets_dtype != APPY_I64) return fail_named(fn, "offsets_dtype must be APPY_I32 or APPY_I64");
  if (sequences < 0 || tokens < 0 || width < 0) return fail_named(fn, "negative size");
  if (width > 0x3fffffff) return fail_named(fn, "width is too large");
  return APPY_OK;
}

// Of no sequences at all, every packed row is one of no sequence.
int clear_all(const char* fn, void* p, i64 row, int dtype, i64 tokens, i64 width, void* stream) {
  if (tokens == 0) return APPY_OK;
  if (!p) return fail_named(fn, "NULL argument");
  const size_t size = (size_t)element_size(dtype);
  const cudaError_t e = cudaMemset2DAsync(p, (size_t)row * size, 0, (size_t)width * size, (size_t)tokens, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? APPY_OK : appy_fail_cuda(e, "gated scan clear");
}

}  // namespace

extern "C" {

int appy_gated_scan(const void* dx, int64_t x_seq, int64_t x_row, const void* dgate, int64_t gate_seq, int64_t gate_row, int dtype,
                    const void* doffsets, int offsets_dtype, int64_t sequences, int64_t tokens, int64_t width,
                    const float* dinitial, void* dh, int64_t h_seq, int64_t h_row, float* dlast, int fill, void* stream) {
  static const char fn[] = "appy_gated_scan";
  if (int rc = check_shape(fn, dtype, doffsets, offsets_dtype, sequences, tokens, width)) return rc;
  if (width == 0) return APPY_OK;
  if (sequences == 0) return fill && doffsets ? clear_all(fn, dh, h_row, dtype, tokens, width, stream) : APPY_OK;
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
  return APPY_OP_DTYPE(dtype, { return launch_scan<T, false>(a, s); });
}

int appy_gated_scan_grad(const void* ddh, int64_t dh_seq, int64_t dh_row, const void* dx, int64_t x_seq, int64_t x_row,
                         const void* dgate, int64_t gate_seq, int64_t gate_row, const void* dh, int64_t h_seq, int64_t h_row,
                         int dtype, const void* doffsets, int offsets_dtype, int64_t sequences, int64_t tokens, int64_t width,
                         const float* dinitial, const float* dgrad_last, void* dgrad_x, int64_t gx_seq, int64_t gx_row,
                         void* dgrad_gate, int64_t gg_seq, int64_t gg_row, float* dgrad_initial, int fill, void* stream) {
  static const char fn[] = "appy_gated_scan_grad";
  if (int rc = check_shape(fn, dtype, doffsets, offsets_dtype, sequences, tokens, width)) return rc;
  if (width == 0) return APPY_OK;
  if (sequences == 0) {
    if (!fill || !doffsets) return APPY_OK;
    const int rc = clear_all(fn, dgrad_x, gx_row, dtype, tokens, width, stream);
    return rc ? rc : clear_all(fn, dgrad_gate, gg_row, dtype, tokens, width, stream);
  }
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
  return APPY_OP_DTYPE(dtype, { return launch_scan<T, true>(a, s); });
}

}  // extern "C"
