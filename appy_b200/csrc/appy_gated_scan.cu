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

const int kBlock = 256, kWarps = kBlock / 32;

// f = sigmoid(g) and 1 - f, each to a few units in the last place whichever is small: both come from
// exp(-|g|) <= 1, so neither overflows nor cancels.
APPY_DEV void sigmoid_pair(float g, float& f, float& i) {
  const float e = __expf(-fabsf(g)), r = __fdividef(1.f, 1.f + e), er = e * r;
  f = g >= 0.f ? r : er;
  i = g >= 0.f ? er : r;
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

// V channels per thread, CP threads along the channels, LT tokens per thread, C blocks per cluster.
template <class T, int V, int LT, int S, int C, bool BACK>
__global__ void __launch_bounds__(kBlock, 2) k_scan(ScanArgs a) {
  constexpr int CP = V == 1 ? 32 : 16, CH = CP * V, SUBS = kBlock / CP, PER_WARP = 32 / CP, L = SUBS * LT, NA = BACK ? 4 : 2;
  extern __shared__ __align__(16) unsigned char ring_memory[];
  __shared__ __align__(16) float warp_a[kWarps][CH], warp_b[kWarps][CH], enter[kWarps][CH];
  __shared__ float block_a[C > 1 ? 2 : 1][C][CH], block_b[C > 1 ? 2 : 1][C][CH];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = tid / CP, pc = (tid % CP) * V;
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
  if (C > 1) cg::this_cluster().sync();                      // every block of the cluster runs before its memory is written
  int stage = 0;
  for (i64 k = 0; k < steps; ++k) {
    const int n = rows_left(k, len);
    if constexpr (S > 1) {
      fetch(stage == 0 ? S - 1 : stage - 1, k + S - 1);
      feed.arrived();
    }
    float f[LT][V], u[LT][V];                      // forward: gate and (1 - gate) * x; gradient: gate and dh
    float in[BACK ? LT : 1][V], w[BACK ? LT : 1][V];          // gradient: 1 - gate and (h[t-1] - x) * gate * (1 - gate)
#pragma unroll
    for (int j = 0; j < LT; ++j) {
      float g[V], x[V];
      feed.get(stage, 0, j, g);
      feed.get(stage, 1, j, x);
      if constexpr (!BACK) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float i;
          sigmoid_pair(g[v], f[j][v], i);
          u[j][v] = i * x[v];
        }
      } else {
        float hp[V];
        feed.get(stage, 2, j, u[j]);
        feed.get(stage, 3, j, hp);
        if (!a.dh.base) {
#pragma unroll
          for (int v = 0; v < V; ++v) u[j][v] = 0.f;
        }
        if (k * L * C + tau0 + j == len - 1 && live) {
#pragma unroll
          for (int v = 0; v < V; ++v) hp[v] = a.initial ? a.initial[seq * a.width + col + v] : 0.f;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          sigmoid_pair(g[v], f[j][v], in[j][v]);
          w[j][v] = (hp[v] - x[v]) * (f[j][v] * in[j][v]);
        }
      }
    }
    if (n < LT) {                                  // tokens past the end change nothing
#pragma unroll
      for (int j = 0; j < LT; ++j) {
        if (j < n) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) f[j][v] = 1.f, u[j][v] = 0.f;
      }
    }
    if constexpr (S == 1) fetch(0, k + 1);
    // this thread's run as one map
    float A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      A[v] = 1.f;
      B[v] = 0.f;
#pragma unroll
      for (int j = 0; j < LT; ++j) {
        A[v] *= f[j][v];
        B[v] = BACK ? f[j][v] * (B[v] + u[j][v]) : f[j][v] * B[v] + u[j][v];
      }
    }
    // a warp holds PER_WARP (1 or 2) runs of its channels; its last lanes publish the warp's map
    float ea[V], eb[V];                            // map of the runs before this one in the warp
#pragma unroll
    for (int v = 0; v < V; ++v) {
      ea[v] = 1.f;
      eb[v] = 0.f;
      if (PER_WARP == 2) {
        const float pa = __shfl_up_sync(APPY_FULL_MASK, A[v], CP), pb = __shfl_up_sync(APPY_FULL_MASK, B[v], CP);
        if (lane >= CP) {
          ea[v] = pa;
          eb[v] = pb;
          B[v] = A[v] * pb + B[v];
          A[v] *= pa;
        }
      }
    }
    if (lane >= 32 - CP) {
      st_plain<float, V>(&warp_a[warp][pc], pack<float, V>(A));
      st_plain<float, V>(&warp_b[warp][pc], pack<float, V>(B));
    }
    __syncthreads();
    // the channels' threads join the warps' maps (in a cluster first the blocks') and leave each warp its state
    if constexpr (C > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      const int buf = (int)(k & 1);
      if (tid < CH) {
        float ba = 1.f, bb = 0.f;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) {
          bb = warp_a[q][tid] * bb + warp_b[q][tid];
          ba *= warp_a[q][tid];
        }
#pragma unroll
        for (int r = 0; r < C; ++r) {
          cluster.map_shared_rank(&block_a[buf][rank][tid], r)[0] = ba;
          cluster.map_shared_rank(&block_b[buf][rank][tid], r)[0] = bb;
        }
      }
      cluster.sync();
      if (tid < CH) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < C; ++r) {
          if (r == rank) s = carry;
          carry = block_a[buf][r][tid] * carry + block_b[buf][r][tid];
        }
#pragma unroll
        for (int q = 0; q < kWarps; ++q) {
          enter[q][tid] = s;
          s = warp_a[q][tid] * s + warp_b[q][tid];
        }
      }
    } else if (tid < CH) {
#pragma unroll
      for (int q = 0; q < kWarps; ++q) {
        enter[q][tid] = carry;
        carry = warp_a[q][tid] * carry + warp_b[q][tid];
      }
    }
    __syncthreads();
    float s[V];
    unpack<float, V>(ld_plain<float, V>(&enter[warp][pc]), s);
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = ea[v] * s[v] + eb[v];
#pragma unroll
    for (int j = 0; j < LT; ++j) {
      float o[V], og[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if constexpr (!BACK) {
          s[v] = f[j][v] * s[v] + u[j][v];
          o[v] = s[v];
        } else {
          const float lam = u[j][v] + s[v];
          o[v] = in[j][v] * lam;
          og[v] = w[j][v] * lam;
          s[v] = f[j][v] * lam;
        }
      }
      if (j < n) {
        st_stream<T, V>(reinterpret_cast<T*>(to + j * to_row), pack<T, V>(o));
        if constexpr (BACK) st_stream<T, V>(reinterpret_cast<T*>(to_gate + j * gate_row), pack<T, V>(og));
      }
    }
    to += to_row * L * C;
    if (BACK) to_gate += gate_row * L * C;
    stage = stage + 1 == S ? 0 : stage + 1;
  }
  if (a.final_state && owner && rank == 0) a.final_state[seq * a.width + chan0 + tid] = carry;
}

// ------------------------------------------------------------------------------------------------ host side
template <class T, int V, int LT, int S, int C, bool BACK> int launch_c(const ScanArgs& a, cudaStream_t s) {
  const char* const fn = BACK ? "appy_gated_scan_grad" : "appy_gated_scan";
  const i64 blocks = a.sequences * a.tiles * C;
  if (blocks > 0x7fffffff) return fail_named(fn, "too many sequences for one launch");
  const int dyn = Feed<T, V, LT, BACK ? 4 : 2, S>::kBytes;
  static bool ready[16] = {false};                 // per instantiation and device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 16 || !ready[dev]) {
    cudaError_t e = cudaFuncSetAttribute(k_scan<T, V, LT, S, C, BACK>, cudaFuncAttributeMaxDynamicSharedMemorySize, dyn);
    if (e == cudaSuccess && C > 8) e = cudaFuncSetAttribute(k_scan<T, V, LT, S, C, BACK>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_scan<T, V, LT, S, C, BACK>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return appy_fail_cuda(e, "gated scan launch");
  }
  return finish("gated scan launch");
}

template <class T, int V, int LT, int S, bool BACK> int launch_scan(ScanArgs a, cudaStream_t s) {
  constexpr int CP = V == 1 ? 32 : 16, CH = CP * V, L = kBlock / CP * LT;
  a.tiles = (int)((a.width + CH - 1) / CH);
  // a cluster of blocks along the tokens while there are too few (sequence, channel tile) pairs for two blocks per
  // SM and the cluster's step is not longer than the tokens
  const i64 units = a.sequences * a.tiles;
  int c = 1;
  while (c < 16 && units * c < 2 * (i64)sm_count() && (i64)L * c < a.tokens) c *= 2;
  switch (c) {
    case 1: return launch_c<T, V, LT, S, 1, BACK>(a, s);
    case 2: return launch_c<T, V, LT, S, 2, BACK>(a, s);
    case 4: return launch_c<T, V, LT, S, 4, BACK>(a, s);
    case 8: return launch_c<T, V, LT, S, 8, BACK>(a, s);
    default: return launch_c<T, V, LT, S, 16, BACK>(a, s);
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
  return APPY_OP_DTYPE(dtype, { return vec ? launch_scan<T, 4, sizeof(T) == 4 ? 4 : 8, 3, false>(a, s) : launch_scan<T, 1, 16, sizeof(T) == 4 ? 3 : 1, false>(a, s); });
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
  return APPY_OP_DTYPE(dtype, { return vec ? launch_scan<T, 4, sizeof(T) == 4 ? 2 : 4, 3, true>(a, s) : launch_scan<T, 1, 8, sizeof(T) == 4 ? 3 : 1, true>(a, s); });
}

}  // extern "C"
