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
  int tiles, cluster;
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

// V channels per thread, CP threads along the channels, LT tokens per thread, C blocks per cluster.
template <class T, int V, int LT, int C, bool BACK>
__global__ void __launch_bounds__(kBlock, 2) k_scan(ScanArgs a) {
  constexpr int CP = V == 1 ? 32 : 16, CH = CP * V, SUBS = kBlock / CP, PER_WARP = 32 / CP, L = SUBS * LT;
  __shared__ __align__(16) float warp_a[2][kWarps][CH], warp_b[2][kWarps][CH];
  __shared__ __align__(16) float block_a[C > 1 ? 2 : 1][C][CH], block_b[C > 1 ? 2 : 1][C][CH], enter[C > 1 ? 2 : 1][CH];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = tid / CP;
  const int rank = C > 1 ? blockIdx.x % C : 0;
  const i64 unit = blockIdx.x / C, seq = unit / a.tiles;
  const i64 chan0 = (unit % a.tiles) * CH, col = chan0 + (tid % CP) * V;
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
  // the state that walks along: one block keeps it in every thread for its channels, a cluster in one thread per
  // channel of every block
  const float* const start = BACK ? a.dlast : a.initial;
  float carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) carry[v] = 0.f;
  if (start) {
    if (C == 1) {
      if (live) {
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = start[seq * a.width + col + v];
      }
    } else if (tid < CH && chan0 + tid < a.width) {
      carry[0] = start[seq * a.width + chan0 + tid];
    }
  }
  const i64 steps = (len + (i64)L * C - 1) / ((i64)L * C);
  if (C > 1) cg::this_cluster().sync();            // every block of the cluster runs before its memory is written
  for (i64 k = 0; k < steps; ++k) {
    const int buf = (int)(k & 1);
    const i64 tau0 = (k * C + rank) * L + (i64)sub * LT;      // the run in walking order
    float f[LT][V], u[LT][V];                      // forward: gate and (1 - gate) * x; gradient: gate and dh
    float in[BACK ? LT : 1][V], w[BACK ? LT : 1][V];          // gradient: 1 - gate and (h[t-1] - x) * gate * (1 - gate)
    {
      Pack<T, V> xr[LT], gr[LT], hr[BACK ? LT : 1], dr[BACK ? LT : 1];
#pragma unroll
      for (int j = 0; j < LT; ++j) {
        const i64 tau = tau0 + j, t = BACK ? len - 1 - tau : tau;
        const bool on = live && tau < len;
        xr[j] = gr[j] = zero_pack<T, V>();
        if (BACK) hr[j] = dr[j] = zero_pack<T, V>();
        if (on) {
          gr[j] = ld_stream<T, V>(row_ptr<const T>(a.gate, seq_at, first, t, col));
          xr[j] = ld_stream<T, V>(row_ptr<const T>(a.x, seq_at, first, t, col));
          if (BACK) {
            if (a.dh.base) dr[j] = ld_stream<T, V>(row_ptr<const T>(a.dh, seq_at, first, t, col));
            if (t > 0) hr[j] = ld_stream<T, V>(row_ptr<const T>(a.h, seq_at, first, t - 1, col));
          }
        }
      }
#pragma unroll
      for (int j = 0; j < LT; ++j) {
        const i64 tau = tau0 + j;
        const bool on = live && tau < len;
        float x[V], g[V];
        unpack<T, V>(xr[j], x);
        unpack<T, V>(gr[j], g);
        if (!BACK) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            float i;
            sigmoid_pair(g[v], f[j][v], i);
            u[j][v] = i * x[v];
            if (!on) f[j][v] = 1.f, u[j][v] = 0.f;
          }
        } else {
          float hp[V];
          unpack<T, V>(hr[j], hp);
          unpack<T, V>(dr[j], u[j]);
          if (on && tau == len - 1 && a.initial) {
#pragma unroll
            for (int v = 0; v < V; ++v) hp[v] = a.initial[seq * a.width + col + v];
          }
#pragma unroll
          for (int v = 0; v < V; ++v) {
            sigmoid_pair(g[v], f[j][v], in[j][v]);
            w[j][v] = (hp[v] - x[v]) * (f[j][v] * in[j][v]);
            if (!on) f[j][v] = 1.f, u[j][v] = 0.f;
          }
        }
      }
    }
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
#pragma unroll
      for (int v = 0; v < V; ++v) {
        warp_a[buf][warp][(tid % CP) * V + v] = A[v];
        warp_b[buf][warp][(tid % CP) * V + v] = B[v];
      }
    }
    __syncthreads();
    float s[V];                                    // state before this warp's runs
    if (C == 1) {
#pragma unroll
      for (int q = 0; q < kWarps; ++q) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (q == warp) s[v] = carry[v];
          carry[v] = warp_a[buf][q][(tid % CP) * V + v] * carry[v] + warp_b[buf][q][(tid % CP) * V + v];
        }
      }
    } else {
      cg::cluster_group cluster = cg::this_cluster();
      if (tid < CH) {
        float ba = 1.f, bb = 0.f;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) {
          bb = warp_a[buf][q][tid] * bb + warp_b[buf][q][tid];
          ba *= warp_a[buf][q][tid];
        }
#pragma unroll
        for (int r = 0; r < C; ++r) {
          cluster.map_shared_rank(&block_a[buf][rank][tid], r)[0] = ba;
          cluster.map_shared_rank(&block_b[buf][rank][tid], r)[0] = bb;
        }
      }
      cluster.sync();
      if (tid < CH) {
#pragma unroll
        for (int r = 0; r < C; ++r) {
          if (r == rank) enter[buf][tid] = carry[0];
          carry[0] = block_a[buf][r][tid] * carry[0] + block_b[buf][r][tid];
        }
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) s[v] = enter[buf][(tid % CP) * V + v];
      for (int q = 0; q < warp; ++q) {
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = warp_a[buf][q][(tid % CP) * V + v] * s[v] + warp_b[buf][q][(tid % CP) * V + v];
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = ea[v] * s[v] + eb[v];
#pragma unroll
    for (int j = 0; j < LT; ++j) {
      const i64 tau = tau0 + j, t = BACK ? len - 1 - tau : tau;
      float o[V], og[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (!BACK) {
          s[v] = f[j][v] * s[v] + u[j][v];
          o[v] = s[v];
        } else {
          const float lam = u[j][v] + s[v];
          o[v] = in[j][v] * lam;
          og[v] = w[j][v] * lam;
          s[v] = f[j][v] * lam;
        }
      }
      if (live && tau < len) {
        st_stream<T, V>(row_ptr<T>(BACK ? a.dx : a.h, seq_at, first, t, col), pack<T, V>(o));
        if (BACK) st_stream<T, V>(row_ptr<T>(a.dgate, seq_at, first, t, col), pack<T, V>(og));
      }
    }
  }
  if (!a.final_state) return;
  if (C == 1) {
    if (sub == 0 && live) {
#pragma unroll
      for (int v = 0; v < V; ++v) a.final_state[seq * a.width + col + v] = carry[v];
    }
  } else if (rank == 0 && tid < CH && chan0 + tid < a.width) {
    a.final_state[seq * a.width + chan0 + tid] = carry[0];
  }
}

// ------------------------------------------------------------------------------------------------ host side
template <class T, int V, int LT, int C, bool BACK> int launch_c(const ScanArgs& a, cudaStream_t s) {
  const i64 blocks = a.sequences * a.tiles * C;
  if (blocks > 0x7fffffff) return fail_named(BACK ? "appy_gated_scan_grad" : "appy_gated_scan", "too many sequences for one launch");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kBlock);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_scan<T, V, LT, C, BACK>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return appy_fail_cuda(e, "gated scan launch");
  }
  return finish("gated scan launch");
}

template <class T, int V, int LT, bool BACK> int launch_scan(ScanArgs a, cudaStream_t s) {
  constexpr int CP = V == 1 ? 32 : 16, CH = CP * V, L = kBlock / CP * LT;
  a.tiles = (int)((a.width + CH - 1) / CH);
  // a cluster of blocks along the tokens while there are too few (sequence, channel tile) pairs for two blocks per
  // SM and the cluster's step is not longer than the tokens
  const i64 units = a.sequences * a.tiles;
  int c = 1;
  while (c < 8 && units * c < 2 * (i64)sm_count() && (i64)L * c < a.tokens) c *= 2;
  a.cluster = c;
  switch (c) {
    case 1: return launch_c<T, V, LT, 1, BACK>(a, s);
    case 2: return launch_c<T, V, LT, 2, BACK>(a, s);
    case 4: return launch_c<T, V, LT, 4, BACK>(a, s);
    default: return launch_c<T, V, LT, 8, BACK>(a, s);
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
  return APPY_OP_DTYPE(dtype, { return vec ? launch_scan<T, 4, 8, false>(a, s) : launch_scan<T, 1, 16, false>(a, s); });
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
  return APPY_OP_DTYPE(dtype, { return vec ? launch_scan<T, 4, 4, true>(a, s) : launch_scan<T, 1, 16, true>(a, s); });
}

}  // extern "C"
