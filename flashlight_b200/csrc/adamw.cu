// One AdamW step over many tensors at once (flb200_adamw_step):
//     g = grad_scale * grad          m = beta1 m + (1 - beta1) g          v = beta2 v + (1 - beta2) g^2
//     p = p - lr * (m / c1 / (sqrt(v / c2) + epsilon) + weight_decay * p),   c_i = 1 - beta_i^step
// fl::AdamOptimizer::step (flashlight/fl/optim/AdamOptimizer.cpp) is the same moments as a chain of tensor
// operators per parameter; a language model has a hundred and more parameters, most of them short.  Here the
// tensors' addresses and lengths travel as the kernel's own argument, so that a step is one launch without a
// table to copy first, and CTAs walk chunks of 2048 elements over all tensors.
//
// States of 8 bits: a warp owns a block of 256 elements.  m is kept as e4m3 times a scale per block (largest
// magnitude / 448).  Of v its square root is kept, as e4m3 likewise: e4m3 spans a factor of 2^18 between its least
// and its largest value, so v spans 2^36, and a relative error of at most 2^-4 of the root is one of the
// step's length.  A root above zero is rounded up to the least code where it would become zero: it divides, and
// m / epsilon would be a step a thousand times too long.  The step itself uses the new m and v before they are
// rounded.  All arithmetic is in fp32; the step's quotient is the approximate one (2^-22 of its length, itself a
// small part of p).
//
// HBM bounds it: 28 bytes per element in fp32, 10 with 16-bit parameters and gradients and 8-bit states.
#include <cuda_fp8.h>

#include <cmath>
#include <type_traits>

#include "common.cuh"

namespace flb200 {
namespace {

constexpr int kPer = 8;                      // consecutive elements of a lane
constexpr int kStateBlock = 32 * kPer;       // elements of a warp, and of a scale of 8-bit states
constexpr int kChunk = 256 * kPer;           // elements of a CTA's pass
static_assert(kStateBlock == FLB200_ADAMW_BLOCK, "a warp owns a block");

struct AdamwMath {
  float beta1, rest1, beta2, rest2;  // rest = 1 - beta
  float inv_c1, inv_root_c2, epsilon, lr, weight_decay, grad_scale;
};

// Kernel arguments may take 32764 bytes; a launch copies what it is given, so short lists have short tables.  Steps behind
// one another, us, with the table of 480 / 160 / 32 tensors: 8 short tensors 5.1 / 3.5 / 3.3; 30 of them 6.2 / 4.6 / 4.4;
// 100 9.5 / 7.9; 155 12.1 / 10.4; 300 18.7 with 480 alone.
template <int CAP>
struct AdamwTable {
  flb200_adamw_tensor t[CAP];
  unsigned first_chunk[CAP + 1];  // chunks of the tensors before
  unsigned vec[(CAP + 31) / 32];  // a bit per tensor: aligned for eight elements at once
  int count;
};
constexpr int kSmall = 32, kMiddle = 160, kLarge = 480;
static_assert(sizeof(AdamwTable<kLarge>) + sizeof(AdamwMath) < 32764, "kernel arguments");

// Eight elements, as they lie in memory where all of them exist and are aligned.
template <typename T>
struct alignas(16) Eight {
  uint32_t w[2 * sizeof(T)];
};
template <typename T>
__device__ __forceinline__ void read8(const T* p, Eight<T>& r) {
  if constexpr (sizeof(T) == 4) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                   "=r"(r.w[7])
                 : "l"(p));
  } else if constexpr (sizeof(T) == 2) {
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
                 : "l"(p));
  } else {
    asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
  }
}
template <typename T>
__device__ __forceinline__ void widen8(const Eight<T>& r, float* v) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = __uint_as_float(r.w[j]);
  } else {
    unpack16(*reinterpret_cast<const Vec16<T>*>(&r), v);
  }
}
// One by one, of which `live` exist.
template <typename T>
__device__ __forceinline__ void load_live(const T* p, int live, float* v) {
#pragma unroll
  for (int j = 0; j < kPer; ++j) v[j] = j < live ? Num<T>::to_f(p[j]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool whole, int live, float* v) {
  if (whole) {
    Eight<T> r;
    read8(p, r);
    widen8(r, v);
  } else {
    load_live(p, live, v);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool whole, int live, const float* v) {
  if (whole) {
    if constexpr (sizeof(T) == 4) {
      asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]),
                   "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                   : "memory");
    } else {
      store16(p, pack16<T>(v));
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < live) p[j] = Num<T>::from_f(v[j]);
  }
}

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 8-bit states: the values of eight codes over their block's scale
__device__ __forceinline__ void widen_codes(const Eight<uint8_t>& r, float scale, float* v) {
#pragma unroll
  for (int j = 0; j < kPer; j += 2) {
    const __half2_raw h =
        __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(r.w[j >> 2] >> (8 * (j & 2))), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[j] = f.x * scale;
    v[j + 1] = f.y * scale;
  }
}
__device__ __forceinline__ Eight<uint8_t> codes_live(const uint8_t* p, int live) {
  Eight<uint8_t> r{{0, 0}};
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (j < live) r.w[j >> 2] |= (uint32_t)p[j] << (8 * (j & 3));
  return r;
}
// of numbers that are not negative: their bits are in their order
__device__ __forceinline__ float warp_top(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}
// The warp's block: its scale, and the codes of its values.  kRoot: values >= 0 of which none but zero becomes zero.
template <bool kRoot>
__device__ __forceinline__ void store_codes(uint8_t* p, float* scale, bool whole, int live, const float* v) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) top = fmaxf(top, kRoot ? v[j] : fabsf(v[j]));  // (past the end: zeros)
  top = fmaxf(warp_top(top), 1e-30f);
  const float to_code = __fmul_rn(__frcp_rn(top), 448.f);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < kPer; j += 2) {
    float2 s = make_float2(v[j] * to_code, v[j + 1] * to_code);
    if (kRoot) {
      if (v[j] > 0.f) s.x = fmaxf(s.x, 0x1p-9f);
      if (v[j + 1] > 0.f) s.y = fmaxf(s.y, 0x1p-9f);
    }
    const uint32_t two = __nv_cvt_float2_to_fp8x2(s, __NV_SATFINITE, __NV_E4M3);
    w[j >> 2] |= two << (8 * (j & 2));
  }
  if (whole) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < live) p[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
  }
  if ((threadIdx.x & 31) == 0) *scale = __fmul_rn(top, 1.f / 448.f);
}

// Where a warp is: its block of 256 elements of tensor `at`, and this lane's eight of them.
struct Place {
  int at, live;
  bool exists, whole;  // of the warp; eight elements that can be read at once
  long long block, i;
};
template <int CAP>
__device__ __forceinline__ Place place_of(const AdamwTable<CAP>& table, unsigned chunk, int from) {
  Place x;
  x.at = from;  // (a CTA's chunks only grow)
  int hi = table.count;
  while (hi - x.at > 1) {  // the last tensor that begins at or before this chunk
    const int mid = (x.at + hi) >> 1;
    if (table.first_chunk[mid] <= chunk) x.at = mid;
    else hi = mid;
  }
  x.block = (long long)(chunk - table.first_chunk[x.at]) * 8 + (threadIdx.x >> 5);
  x.i = x.block * kStateBlock + (threadIdx.x & 31) * kPer;
  const long long n = table.t[x.at].n, left = n - x.i;
  x.exists = x.block * kStateBlock < n;
  x.live = left >= kPer ? kPer : (left > 0 ? (int)left : 0);
  x.whole = x.live == kPer && (table.vec[x.at >> 5] >> (x.at & 31) & 1u);
  return x;
}
template <typename TP, typename TG, typename TS>
struct Read {
  Eight<TP> p;
  Eight<TG> g;
  Eight<TS> m, v;
  float m_scale, v_scale;
};

// With 8-bit states, whose conversions are most of the work, a chunk is read while the one before it is computed
// (10^9 elements in 16 bits: 3111 us without, 2560 with).  With 32-bit states the warps that fit without those
// registers keep memory busy (134 10^6 elements: 565 us, with chunks read ahead 608).
template <typename TP, typename TG, int BITS, int CAP>
__global__ void __launch_bounds__(256, BITS == 8 ? 3 : 1)
adamw_kernel(const __grid_constant__ AdamwTable<CAP> table, const AdamwMath k) {
  chain_begin();
  using TS = std::conditional_t<BITS == 8, uint8_t, float>;
  const unsigned chunks = table.first_chunk[table.count];
  Read<TP, TG, TS> next;
  auto read = [&](const Place& x, Read<TP, TG, TS>& r) {
    const flb200_adamw_tensor& t = table.t[x.at];
    if (x.whole) {
      read8(static_cast<const TP*>(t.param) + x.i, r.p);
      read8(static_cast<const TG*>(t.grad) + x.i, r.g);
      read8(static_cast<const TS*>(t.first) + x.i, r.m);
      read8(static_cast<const TS*>(t.second) + x.i, r.v);
    }
    if (BITS == 8 && x.exists) {
      r.m_scale = t.first_scale[x.block];
      r.v_scale = t.second_scale[x.block];
    }
  };
  Place there{};
  int from = 0;
  if (BITS == 8 && blockIdx.x < chunks) {
    there = place_of(table, blockIdx.x, 0);
    read(there, next);
  }
  for (unsigned chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    Place here;
    Read<TP, TG, TS> now;
    if constexpr (BITS == 8) {
      here = there;
      now = next;
      if (chunk + gridDim.x < chunks) {
        there = place_of(table, chunk + gridDim.x, here.at);
        read(there, next);
      }
    } else {
      here = place_of(table, chunk, from);
      from = here.at;
    }
    if (!here.exists) continue;  // (all lanes of the warp)
    const flb200_adamw_tensor& t = table.t[here.at];
    const long long i = here.i, block = here.block;
    const int live = here.live;
    const bool whole = here.whole;
    float p[kPer], g[kPer], m[kPer], v[kPer];
    if constexpr (BITS == 32) {
      load8(static_cast<const TP*>(t.param) + i, whole, live, p);
      load8(static_cast<const TG*>(t.grad) + i, whole, live, g);
      load8(static_cast<const float*>(t.first) + i, whole, live, m);
      load8(static_cast<const float*>(t.second) + i, whole, live, v);
    } else {
      if (whole) {
        widen8(now.p, p);
        widen8(now.g, g);
      } else {
        load_live(static_cast<const TP*>(t.param) + i, live, p);
        load_live(static_cast<const TG*>(t.grad) + i, live, g);
        now.m = codes_live(static_cast<const uint8_t*>(t.first) + i, live);
        now.v = codes_live(static_cast<const uint8_t*>(t.second) + i, live);
      }
      widen_codes(now.m, now.m_scale, m);
      widen_codes(now.v, now.v_scale, v);
    }
    // Each operation of the moments rounds by itself (no contraction): what is kept in 8 bits then depends on
    // the formula alone.
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const float gg = __fmul_rn(g[j], k.grad_scale);
      m[j] = __fadd_rn(__fmul_rn(m[j], k.beta1), __fmul_rn(gg, k.rest1));
      const float old = BITS == 8 ? __fmul_rn(v[j], v[j]) : v[j];
      const float vv = __fadd_rn(__fmul_rn(old, k.beta2), __fmul_rn(__fmul_rn(gg, gg), k.rest2));
      const float root = __fsqrt_rn(vv);
      const float step = m[j] * k.inv_c1 * reciprocal(fmaf(root, k.inv_root_c2, k.epsilon));
      p[j] = fmaf(-k.lr, fmaf(k.weight_decay, p[j], step), p[j]);
      v[j] = BITS == 32 ? vv : root;
    }
    store8(static_cast<TP*>(t.param) + i, whole, live, p);
    if constexpr (BITS == 32) {
      store8(static_cast<float*>(t.first) + i, whole, live, m);
      store8(static_cast<float*>(t.second) + i, whole, live, v);
    } else {
      store_codes<false>(static_cast<uint8_t*>(t.first) + i, t.first_scale + block, whole, live, m);
      store_codes<true>(static_cast<uint8_t*>(t.second) + i, t.second_scale + block, whole, live, v);
    }
  }
}

bool aligned_to(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename TP, typename TG, int BITS, int CAP>
int launch_adamw(const AdamwMath& math, const flb200_adamw_tensor* tensors, int64_t* at, int64_t count,
                 cudaStream_t st) {
  AdamwTable<CAP> table;
  table.count = 0;
  table.first_chunk[0] = 0;
  for (unsigned& w : table.vec) w = 0;
  long long chunks = 0;
  for (; *at < count && table.count < CAP; ++*at) {
    const flb200_adamw_tensor& t = tensors[*at];
    const long long mine = (t.n + kChunk - 1) / kChunk;
    if (mine == 0) continue;
    if (chunks + mine > 0x7fffffffLL) break;  // (one tensor alone has fewer, the entry point sees to it)
    chunks += mine;
    if (aligned_to(t.param, kPer * sizeof(TP)) && aligned_to(t.grad, kPer * sizeof(TG)) &&
        aligned_to(t.first, kPer * BITS / 8) && aligned_to(t.second, kPer * BITS / 8))
      table.vec[table.count >> 5] |= 1u << (table.count & 31);
    table.t[table.count++] = t;
    table.first_chunk[table.count] = (unsigned)chunks;
  }
  if (chunks == 0) return FLB200_OK;
  const long long cap = 8LL * (BITS == 8 ? 1 : 4) * device_info().sm_count;
  launch_chained(adamw_kernel<TP, TG, BITS, CAP>, (unsigned)(chunks < cap ? chunks : cap), 256, 0, st, table, math);
  FLB200_AFTER_LAUNCH("adamw_step");
  return FLB200_OK;
}

template <typename TP, typename TG, int BITS>
int run_adamw(const AdamwMath& math, const flb200_adamw_tensor* tensors, int64_t count, cudaStream_t st) {
  for (int64_t at = 0; at < count;) {
    const int64_t left = count - at;
    const int rc = left <= kSmall    ? launch_adamw<TP, TG, BITS, kSmall>(math, tensors, &at, count, st)
                   : left <= kMiddle ? launch_adamw<TP, TG, BITS, kMiddle>(math, tensors, &at, count, st)
                                     : launch_adamw<TP, TG, BITS, kLarge>(math, tensors, &at, count, st);
    if (rc) return rc;
  }
  return FLB200_OK;
}
template <typename TP, typename TG>
int run_adamw_bits(int bits, const AdamwMath& math, const flb200_adamw_tensor* tensors, int64_t count,
                   cudaStream_t st) {
  return bits == 32 ? run_adamw<TP, TG, 32>(math, tensors, count, st)
                    : run_adamw<TP, TG, 8>(math, tensors, count, st);
}

}  // namespace
}  // namespace flb200

extern "C" int flb200_adamw_step(const flb200_adamw_desc* d, const flb200_adamw_tensor* tensors, int64_t count,
                                 void* stream) {
  using namespace flb200;
  FLB200_REQUIRE(d && (tensors || count == 0) && count >= 0, "adamw_step: null argument");
  FLB200_REQUIRE(d->step >= 1, "adamw_step: steps are counted from 1");
  FLB200_REQUIRE(d->beta1 >= 0 && d->beta1 < 1 && d->beta2 >= 0 && d->beta2 < 1,
                 "adamw_step: betas lie in [0, 1)");
  FLB200_REQUIRE(d->epsilon >= 0, "adamw_step: negative epsilon");
  FLB200_REQUIRE(d->state_bits == 32 || d->state_bits == 8, "adamw_step: states have 32 or 8 bits");
  const int pt = d->param_dtype, gt = d->grad_dtype;
  const bool half = pt == FLB200_F16 || pt == FLB200_BF16;
  FLB200_REQUIRE(half || pt == FLB200_F32, "adamw_step: unknown dtype %d", pt);
  FLB200_REQUIRE(gt == FLB200_F32 || gt == FLB200_F16 || gt == FLB200_BF16, "adamw_step: unknown dtype %d", gt);
  if (half && gt != pt)
    return fail(FLB200_UNSUPPORTED, "adamw_step: 16-bit parameters take gradients of their own type");
  for (int64_t i = 0; i < count; ++i) {
    const flb200_adamw_tensor& t = tensors[i];
    FLB200_REQUIRE(t.n >= 0 && t.n <= (1LL << 40), "adamw_step: bad length");
    if (t.n == 0) continue;
    FLB200_REQUIRE(t.param && t.grad && t.first && t.second, "adamw_step: null tensor");
    FLB200_REQUIRE(d->state_bits == 32 || (t.first_scale && t.second_scale),
                   "adamw_step: 8-bit states need their scales");
    const unsigned ps = half ? 2 : 4, gs = gt == FLB200_F32 ? 4 : 2, ss = d->state_bits / 8;
    FLB200_REQUIRE(aligned_to(t.param, ps) && aligned_to(t.grad, gs) && aligned_to(t.first, ss) &&
                       aligned_to(t.second, ss) && aligned_to(t.first_scale, 4) && aligned_to(t.second_scale, 4),
                   "adamw_step: tensors must be aligned to their elements");
  }
  AdamwMath k;
  k.beta1 = (float)d->beta1;
  k.rest1 = (float)(1.0 - d->beta1);
  k.beta2 = (float)d->beta2;
  k.rest2 = (float)(1.0 - d->beta2);
  k.inv_c1 = (float)(1.0 / (1.0 - std::pow(d->beta1, (double)d->step)));
  k.inv_root_c2 = (float)(1.0 / std::sqrt(1.0 - std::pow(d->beta2, (double)d->step)));
  k.epsilon = (float)d->epsilon;
  k.lr = (float)d->lr;
  k.weight_decay = (float)d->weight_decay;
  k.grad_scale = (float)d->grad_scale;
  const cudaStream_t st = as_stream(stream);
  if (pt == FLB200_BF16) return run_adamw_bits<__nv_bfloat16, __nv_bfloat16>(d->state_bits, k, tensors, count, st);
  if (pt == FLB200_F16) return run_adamw_bits<__half, __half>(d->state_bits, k, tensors, count, st);
  if (gt == FLB200_BF16) return run_adamw_bits<float, __nv_bfloat16>(d->state_bits, k, tensors, count, st);
  if (gt == FLB200_F16) return run_adamw_bits<float, __half>(d->state_bits, k, tensors, count, st);
  return run_adamw_bits<float, float>(d->state_bits, k, tensors, count, st);
}
