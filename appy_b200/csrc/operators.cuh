// Shared by the language-model operators (appy_embedding.cu, appy_gated_scan.cu, appy_token_logprobs.cu): element
// types and their conversion to float32, in which every operator computes, and the host-side checks and launch
// helpers of their C entry points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "../../include/appy_sm100.h"
#include "templates/appy_device.cuh"

void appy_note_launch();
int appy_fail_cuda(cudaError_t e, const char* what);
int appy_fail_arg(const char* what);

namespace appy_op {

typedef __nv_bfloat16 bf16;
typedef __half f16;

APPY_DEV float to_f32(float v) { return v; }
APPY_DEV float to_f32(f16 v) { return __half2float(v); }
APPY_DEV float to_f32(bf16 v) { return __bfloat162float(v); }
// one rounding to nearest-even, the only one between the float32 arithmetic of an operator and its result
template <class T> APPY_DEV T from_f32(float v);
template <> APPY_DEV float from_f32<float>(float v) { return v; }
template <> APPY_DEV f16 from_f32<f16>(float v) { return __float2half_rn(v); }
template <> APPY_DEV bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }

// V elements as one 2..32-byte word, moved as raw bits and converted in registers
struct __align__(16) Raw32 { uint4 a, b; };
template <int BYTES> struct Raw { typedef typename appy_raw<BYTES>::type type; };
template <> struct Raw<32> { typedef Raw32 type; };
template <class T, int V> struct Pack {
  typename Raw<sizeof(T) * V>::type raw;
  union Bits {                                   // the same bits as elements
    typename Raw<sizeof(T) * V>::type raw;
    unsigned short h[sizeof(T) * V / 2];
    unsigned w[(sizeof(T) * V + 3) / 4];
    APPY_DEV Bits() {}
  };
};
template <class T, int V> APPY_DEV Pack<T, V> ld_stream(const T* p) {        // read once: evict-first
  return {__ldcs(reinterpret_cast<const typename Raw<sizeof(T) * V>::type*>(p))};
}
template <class T, int V> APPY_DEV Pack<T, V> ld_keep(const T* p) {          // read again soon, never written here
  return {__ldg(reinterpret_cast<const typename Raw<sizeof(T) * V>::type*>(p))};
}
template <class T, int V> APPY_DEV Pack<T, V> ld_plain(const T* p) {         // this kernel may also write there
  return {*reinterpret_cast<const typename Raw<sizeof(T) * V>::type*>(p)};
}
template <class T, int V> APPY_DEV void st_stream(T* p, Pack<T, V> v) {
  __stcs(reinterpret_cast<typename Raw<sizeof(T) * V>::type*>(p), v.raw);
}
template <class T, int V> APPY_DEV void st_plain(T* p, Pack<T, V> v) {
  *reinterpret_cast<typename Raw<sizeof(T) * V>::type*>(p) = v.raw;
}
template <class T, int V> APPY_DEV Pack<T, V> zero_pack() {
  typename Pack<T, V>::Bits u;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) * V / 2); ++i) u.h[i] = 0;
  return {u.raw};
}
// two 16-bit elements of one register to and from float32
APPY_DEV void unpack2(unsigned w, float& lo, float& hi, bf16) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}
APPY_DEV void unpack2(unsigned w, float& lo, float& hi, f16) {
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.f32.f16 %0, l;\ncvt.f32.f16 %1, h;\n}" : "=f"(lo), "=f"(hi) : "r"(w));
}
APPY_DEV unsigned pack2(float lo, float hi, bf16) {
  unsigned w;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  return w;
}
APPY_DEV unsigned pack2(float lo, float hi, f16) {
  unsigned w;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  return w;
}
template <class T, int V> APPY_DEV void unpack(Pack<T, V> k, float (&f)[V]) {
  typename Pack<T, V>::Bits u;
  u.raw = k.raw;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = __uint_as_float(u.w[i]);
  } else if constexpr (V == 1) {
    T t;
    memcpy(&t, &u.h[0], 2);
    f[0] = to_f32(t);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) unpack2(u.w[i], f[2 * i], f[2 * i + 1], T());
  }
}
template <class T, int V> APPY_DEV Pack<T, V> pack(const float (&f)[V]) {
  typename Pack<T, V>::Bits u;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) u.w[i] = __float_as_uint(f[i]);
  } else if constexpr (V == 1) {
    const T t = from_f32<T>(f[0]);
    memcpy(&u.h[0], &t, 2);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) u.w[i] = pack2(f[2 * i], f[2 * i + 1], T());
  }
  return {u.raw};
}

// ------------------------------------------------------------------------------------------------ V floats at a time
// Two float32 of one 64-bit register per instruction where V is even: kernels that issue a dozen operations per element
// are bound by that, and products and sums of pairs cost half.
template <int V> struct Vec { u64 p[V / 2]; };
template <> struct Vec<1> { float p[1]; };

APPY_DEV u64 pair(float lo, float hi) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
APPY_DEV float mul1(float a, float b) { return a * b; }
APPY_DEV float add1(float a, float b) { return a + b; }
APPY_DEV u64 mul1(u64 a, u64 b) { u64 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
APPY_DEV u64 add1(u64 a, u64 b) { u64 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
APPY_DEV float fma1(float a, float b, float c) { return fmaf(a, b, c); }
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

// ------------------------------------------------------------------------------------------------ host side
inline int sm_count() {
  static int known[16] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 16) return 148;
  if (!known[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    known[dev] = n;
  }
  return known[dev];
}
inline int finish(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return appy_fail_cuda(e, what);
  appy_note_launch();
  return APPY_OK;
}
inline int fail_named(const char* fn, const char* what) {
  char text[256];
  snprintf(text, sizeof text, "%s: %s", fn, what);
  return appy_fail_arg(text);
}
// Whether clusters as wide as `cfg` says are resident at all: 16 blocks are more than every device has to offer (one that is
// partitioned may have fewer SMs next to one another).  Not a status of an entry: the caller takes another way.
const int kNoCluster = -1001;
template <class K> bool cluster_fits(K kernel, const cudaLaunchConfig_t& cfg) {
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0) return true;
  cudaGetLastError();
  return false;
}
inline bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
inline int element_size(int dtype) { return dtype == APPY_F32 ? 4 : (dtype == APPY_F16 || dtype == APPY_BF16) ? 2 : 0; }

}  // namespace appy_op

// Runs `...` with `T` standing for the element type that `dtype` names.
#define APPY_OP_DTYPE(dtype, ...)                                          \
  [&]() -> int {                                                           \
    if ((dtype) == APPY_F32) { typedef float T; __VA_ARGS__ }              \
    if ((dtype) == APPY_F16) { typedef appy_op::f16 T; __VA_ARGS__ }       \
    typedef appy_op::bf16 T;                                               \
    __VA_ARGS__                                                            \
  }()
