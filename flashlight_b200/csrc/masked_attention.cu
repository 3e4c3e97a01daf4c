// Attention over the interval of keys that each query sees, with capped scores and a distance bias, forward and
// gradient; f16 or bf16, head dimensions up to 128, key heads shared by several query heads:
//     u = scale q.k / cap    z = cap tanh(u)  (cap 0: scale q.k)    s = z - slope_h |i - j|
//     P = exp(s - lse) over j in [lo_i, hi_i), 0 elsewhere          o = P v
//     dP = do v^T    D = rowsum(do o)    dS = P (dP - D) (1 - tanh(u)^2)
//     dq = scale dS k    dk = scale dS^T q    dv = P^T do           (dk, dv summed over the heads that share them)
// flashlight/fl/autograd/Functions.cpp:1828-1891 is the chain of whole-tensor operators for this, its mask an
// additive tensor.  One interval per query says all that a causal mask, documents packed into a row, a prefix and
// padding say together.  Without documents it is a formula; with them flb200_attention_mask makes a table of it once per
// batch, with what the kernels below need to know
// of blocks of 128: which key blocks a query block meets, and whether all of a block is seen.
//
// The scores of a 128 x 128 block live in tensor memory only.  tanh(u) = 1 - 2 r, r = 1 / (1 + e^2u), from the
// approximate exponential and reciprocal: its absolute error is below 2^-21 (the approximate tanh is 2^-11 off, at a
// cap of 50 an error of 2 % in P), and 1 - tanh(u)^2 = 4 r (1 - r) comes with it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

#include "common.cuh"
#include "flb200.h"
#include "packed.cuh"
#include "tc_core.cuh"
#include "tc_gemm.cuh"

namespace flb200 {
namespace {

using namespace tc;

constexpr int kBlock = 128;        // queries and keys of a block
constexpr int kBox = 128 * 128;    // bytes of [128 rows][64 16-bit values], one TMA box
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kFwdThreads = 320;   // warps 0..7: two threads per row; 8: TMA; 9: MMA

// ------------------------------------------------------------------------------------------ the mask
// rows: [lo, hi) of each query ([batch][q_len]; hi <= lo: it sees nothing).  q_blocks: of each block of queries the
// least lo and the greatest hi of those that see something, and the greatest lo and the least hi of all (an
// empty row makes that pair empty).  k_blocks: the query blocks [first, last) that may see a block of keys.
__host__ __device__ inline int blocks_of(long long n) { return (int)((n + kBlock - 1) / kBlock); }
struct MaskView {
  const int2* rows;  // null: no documents, what follows is computed
  const int4* q_blocks;
  const int2* k_blocks;
  const int* prefix;
  int causal, q_len, k_len;

  __device__ __forceinline__ int seen_by_all(int batch) const {
    return prefix ? min(max(prefix[batch], 0), k_len) : 0;
  }
  __device__ __forceinline__ int end_of(int i, int all) const {  // of row i's interval, without documents
    return causal ? max(i + k_len - q_len + 1, all) : k_len;
  }
  __device__ __forceinline__ int2 row(int batch, int i) const {
    if (rows) return rows[(long long)batch * q_len + i];
    return make_int2(0, end_of(i, seen_by_all(batch)));
  }
  __device__ __forceinline__ int4 q_block(int batch, int b) const {
    if (rows) return q_blocks[(long long)batch * blocks_of(q_len) + b];
    const int all = seen_by_all(batch);
    return make_int4(0, end_of(min(q_len, (b + 1) * kBlock) - 1, all), 0, end_of(b * kBlock, all));
  }
  __device__ __forceinline__ int2 k_block(int batch, int j) const {
    if (rows) return k_blocks[(long long)batch * blocks_of(k_len) + j];
    // the first block with a query at or behind the block's first key; all where the prefix reaches into it
    const int behind = j * kBlock - (k_len - q_len);
    return make_int2(causal && behind > 0 && seen_by_all(batch) <= j * kBlock ? behind / kBlock : 0, blocks_of(q_len));
  }
};
inline size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }
size_t mask_bytes(long long batch, long long q_len, long long k_len) {
  return round16(batch * blocks_of(q_len) * sizeof(int4)) + round16(batch * blocks_of(k_len) * sizeof(int2)) +
         batch * q_len * sizeof(int2);
}
MaskView mask_view(const void* mask, long long batch, long long q_len, long long k_len) {
  const char* p = static_cast<const char*>(mask);
  MaskView v{};
  v.q_len = (int)q_len;
  v.k_len = (int)k_len;
  if (!mask) return v;
  v.q_blocks = reinterpret_cast<const int4*>(p);
  p += round16(batch * blocks_of(q_len) * sizeof(int4));
  v.k_blocks = reinterpret_cast<const int2*>(p);
  p += round16(batch * blocks_of(k_len) * sizeof(int2));
  v.rows = reinterpret_cast<const int2*>(p);
  return v;
}

__device__ __forceinline__ int warp_running_max(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = max(v, u);
  }
  return v;
}
// Of the CTA's 1024 threads, the maximum of `carry` and the values of those before this one; carry becomes that of all.
__device__ __forceinline__ int max_before(int v, int* carry, int* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_running_max(v);
  __syncthreads();  // scratch may still be read from the call before
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  const int warps = max(warp_running_max(scratch[lane]), *carry);
  const int ahead = __shfl_sync(0xffffffffu, warps, (warp + 31) & 31), mine = __shfl_up_sync(0xffffffffu, v, 1);
  const int before = warp > 0 ? ahead : *carry;
  *carry = __shfl_sync(0xffffffffu, warps, 31);
  return lane > 0 ? max(before, mine) : before;
}

// One CTA per row of the batch: a query's document is the run of equal ids around its position, and the ends of the
// runs are a running maximum from the left and one from the right.
constexpr int kRun = 4;  // positions of a thread
__global__ void __launch_bounds__(1024)
attention_mask_kernel(const int* __restrict__ documents, const int* __restrict__ prefix, int q_len, int k_len,
                      int causal, int4* __restrict__ q_blocks, int2* __restrict__ k_blocks, int2* __restrict__ rows) {
  chain_begin();
  __shared__ int scratch[32];
  const int b = blockIdx.x, off = k_len - q_len, step = 1024 * kRun;
  const int nq = blocks_of(q_len), nk = blocks_of(k_len);
  const int* ids = documents + (long long)b * k_len;
  const int seen_by_all = prefix ? min(max(prefix[b], 0), k_len) : 0;
  rows += (long long)b * q_len;
  q_blocks += (long long)b * nq;
  k_blocks += (long long)b * nk;
  int carry = 0;
  for (int p0 = 0; p0 < k_len; p0 += step) {
    int start[kRun], id[kRun], last = 0;
    const int p = p0 + threadIdx.x * kRun;
    int before = p > 0 && p < k_len ? ids[p - 1] : 0;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      id[j] = p + j < k_len ? ids[p + j] : 0;
      if (p + j < k_len && (p + j == 0 || id[j] != before)) last = p + j;
      start[j] = last;
      before = id[j];
    }
    const int left = max_before(last, &carry, scratch);
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      const int i = p + j - off;
      if (p + j < k_len && i >= 0)
        rows[i] = id[j] < 0 ? make_int2(0, 0)
                            : make_int2(max(start[j], left), causal ? p + j + 1 : k_len);
    }
  }
  if (!causal || seen_by_all > 0) {  // the runs' ends count
    int from_right = 0;  // k_len - end, running
    const int last0 = (k_len - 1) / step * step;
    for (int p0 = last0; p0 >= 0; p0 -= step) {
      // thread t looks at positions from the right: the chunk's last kRun positions are thread 0's
      const int p = p0 + step - 1 - threadIdx.x * kRun;
      int end[kRun], id[kRun], last = 0;
      int behind = p + 1 < k_len ? ids[p + 1] : 0;
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        id[j] = p - j < k_len ? ids[p - j] : 0;
        if (p - j < k_len && p - j + 1 < k_len && id[j] != behind) last = k_len - (p - j + 1);
        end[j] = last;
        behind = id[j];
      }
      const int right = max_before(last, &from_right, scratch);
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        const int i = p - j - off;
        if (p - j < k_len && i >= 0 && id[j] >= 0) {
          const int e = k_len - max(end[j], right);
          rows[i].y = causal ? min(e, max(p - j + 1, seen_by_all)) : e;
        }
      }
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < nq; i += 32) {
    int lo_min = 0x7fffffff, hi_max = 0, lo_max = 0, hi_min = 0x7fffffff;
    for (int r = i * kBlock + lane; r < min(q_len, (i + 1) * kBlock); r += 32) {
      const int2 x = rows[r];
      if (x.y > x.x) {
        lo_min = min(lo_min, x.x);
        hi_max = max(hi_max, x.y);
        lo_max = max(lo_max, x.x);
        hi_min = min(hi_min, x.y);
      } else {
        lo_max = 0x7fffffff;
        hi_min = 0;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      lo_min = min(lo_min, __shfl_xor_sync(0xffffffffu, lo_min, o));
      hi_max = max(hi_max, __shfl_xor_sync(0xffffffffu, hi_max, o));
      lo_max = max(lo_max, __shfl_xor_sync(0xffffffffu, lo_max, o));
      hi_min = min(hi_min, __shfl_xor_sync(0xffffffffu, hi_min, o));
    }
    if (lane == 0) q_blocks[i] = make_int4(lo_min, hi_max, lo_max, hi_min);
  }
  __syncthreads();
  for (int j = threadIdx.x; j < nk; j += 1024) {
    int first = nq, last = 0;
    for (int i = 0; i < nq; ++i) {
      const int4 q = q_blocks[i];
      if (q.x < (j + 1) * kBlock && q.y > j * kBlock) {
        first = min(first, i);
        last = i + 1;
      }
    }
    k_blocks[j] = make_int2(first, last);
  }
}

// ------------------------------------------------------------------------------------------ common parts
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (fmaxf and max.f32 would drop a NaN)
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// 2^z of two numbers below 2^7 on the FMA pipe: Cody and Waite's reduction to [-1/2, 1/2], a polynomial of degree 4 (the
// one of the least relative error, 2.6e-6, from Remez' exchange), and a product with the power of two that has the
// integer for its exponent.  At -127 that power's bits are zero, so what is smaller gives zero; a NaN stays one, through
// the clamp and the product (added to a NaN's bits the exponent would make a finite number of it).
__device__ __forceinline__ void exp2_by_fma(F2 z, float& a, float& b) {
  float z0, z1, t0, t1;
  unpair(z, z0, z1);
  z = pair(max_or_nan(z0, -127.f), max_or_nan(z1, -127.f));
  const F2 t = z + pair(12582912.f);  // 1.5 * 2^23: the nearest integer is in the low bits
  const F2 f = z + fused(t, pair(-1.f), pair(12582912.f));
  F2 p = fused(f, pair(0.009570102207362652f), pair(0.05591785907745361f));
  p = fused(p, f, pair(0.240247443318367f));
  p = fused(p, f, pair(0.6931217908859253f));
  p = fused(p, f, pair(0.9999992847442627f));
  unpair(t, t0, t1);
  p = p * pair(__uint_as_float((__float_as_uint(t0) << 23) + 0x3f800000u),
               __uint_as_float((__float_as_uint(t1) << 23) + 0x3f800000u));
  unpair(p, a, b);
}
// One pair of a row's exponentials in this many is made so in the forward pass, the others by the special function unit
// (0: all).  At 64 dimensions that unit is the busiest, but with a distance bias, whose arithmetic is the FMA pipe's; at
// 128 it is the tensor pipe.  us with none, one in eight, in four, in two:
//   16 heads of 8192 causal positions of 64, forward 199, 193, 183, 206; gradient 514, 538, 528, 571
//   16 heads of 2 x 4096 of 64, a cap, forward 239, 234, 232; gradient 556, 550, 551
//   12 in documents of 3000 of 64 with a distance bias, forward 105, 107, 106; gradient 201, 202, 208
//   16 of 8192 of 128, forward 266, 266, 267, 284; 2 x 1500, a cap, 54, 53, 53; gradient 127, 126, 126
// The gradient, whose chains leave that unit idle half the time, makes none so.
constexpr int forward_by_fma(int D, bool bias) { return D == 64 && !bias ? 4 : 0; }
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
#define FLB200_R32(r)                                                                                       \
  "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),           \
      "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), \
      "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),            \
      "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),            \
      "+r"(r[30]), "+r"(r[31])
// 32 columns of this thread's lane; the registers may be used after wait_ld and settle only
__device__ __forceinline__ void ld32_begin(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void settle(uint32_t* r) { asm volatile("" : FLB200_R32(r)); }
__device__ __forceinline__ void ld16_begin(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void settle16(uint32_t* r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]));
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] += A[tmem] B[smem]: a row of A per lane, two 16-bit k per column
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// A tile of 128 rows and D columns is D / 64 boxes.  As a K-major operand (a row per m or n) k advances 32 bytes per 16
// inside a box, rows 128 bytes; as an MN-major one (a row per k) k advances 2048 bytes per 16.
template <int D>
__device__ __forceinline__ uint64_t k_major(const char* tile) { return umma_desc(smem_u32(tile), 16, 1024, 2); }
template <int D>
__device__ __forceinline__ uint64_t mn_major(const char* tile) { return umma_desc(smem_u32(tile), kBox, 1024, 2); }
__device__ __forceinline__ uint32_t k_step(int kk) { return (uint32_t)((kk >> 2) * kBox + (kk & 3) * 32); }

template <int D>
__device__ __forceinline__ void load_tile(const CUtensorMap* map, uint64_t* bar, char* to, int row0, int head,
                                          int batch) {
#pragma unroll
  for (int x = 0; x < D; x += 64) {
    int c[4] = {x, row0, head, batch};
    tma_load(map, bar, to + x / 64 * kBox, 4, c);
  }
}

struct OutTensor {  // element (batch b, row t, head h, d) at b * batch + t * row + h * head + d
  void* p;
  long long batch, row, head;
  int wide;  // 16 elements of a row are a sector of 32 bytes
};
template <typename T>
__device__ __forceinline__ void store_32(T* to, const Vec16<T>& a, const Vec16<T>& b) {
  const uint4 x = *reinterpret_cast<const uint4*>(&a), y = *reinterpret_cast<const uint4*>(&b);
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(x.x), "r"(x.y), "r"(x.z),
               "r"(x.w), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w)
               : "memory");
}
// 16 columns from c0 on of a row, of which those in front of head_dim exist.  rest (its row, or null; as wide as o) gets
// what the rounding took: out + rest is right to 2^-16, which D is taken from.  (From out alone D carries a rounding
// of |do||o|, and the scores' gradient half as much error again.)
template <typename T>
__device__ __forceinline__ void store16_of(const OutTensor& o, int b, int t, int h, int c0, int head_dim,
                                           const uint32_t* v, float factor, T* rest) {
  T* to = static_cast<T*>(o.p) + b * o.batch + t * o.row + h * o.head + c0;
  float x[16];
  Vec16<T> r[2];
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(v[e]) * factor;
  r[0] = pack16<T>(x);
  r[1] = pack16<T>(x + 8);
  if (o.wide) {
    if (c0 < head_dim) store_32(to, r[0], r[1]);
  } else {
    if (c0 < head_dim) store16(to, r[0]);
    if (c0 + 8 < head_dim) store16(to + 8, r[1]);
  }
  if (rest) {
    float y[16];
    unpack16(r[0], y);
    unpack16(r[1], y + 8);
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = x[e] - y[e];
    r[0] = pack16<T>(y);
    r[1] = pack16<T>(y + 8);
    if (o.wide) {
      if (c0 < head_dim) store_32(rest + c0, r[0], r[1]);
    } else {
      if (c0 < head_dim) store16(rest + c0, r[0]);
      if (c0 + 8 < head_dim) store16(rest + c0 + 8, r[1]);
    }
  }
}

struct AttnShape {
  int q_len, k_len, heads, group, head_dim;  // group: query heads per key head
  MaskView mask;
  const float* slopes;
  float to_log2;     // scale * log2 e (no cap)
  float cap_log2;    // cap * log2 e
  float to_2u_log2;  // 2 scale / cap * log2 e
  float scale;
  int* status;
};

// ------------------------------------------------------------------------------------------ forward
// One CTA takes 128 queries of a head and walks the keys' blocks, two CTAs to an SM: while one is at its softmax the
// tensor pipe is at the other's products.
//     S = Q K_j^T    columns 0 ..       P, 16 bits, the A operand of
//     O += P V_j     columns 128 ..     (kept over j)
// At 128 dimensions P lies over S.  At 64 it has columns 192 .. of its own, and the next S is made as soon as all have
// read this one.
// Two threads share a row, half of the columns each, and agree on its maximum through shared memory.  P is exp2 of
// the scores less a reference that is raised, and O rescaled, only where a row's maximum passed it by more than
// 2^8: rarely behind the first blocks.  P up to 2^8 loses nothing in either type.
// The output is divided by the sum of P less what the largest P of each 64 lost in its rounding.  Where few keys have
// most of a row's weight, that is most of what P's rounding does to the output and, through D, to the gradient (scores
// three times as wide as usual: 2.1e-3 of the output -> 1.9e-3 in bf16, of dq 2.6e-3 -> 2.5e-3, where the
// roundings of dS and of dq alone are 2.4e-3).  Over all of P it gives the same at 15 % of the time, so at 5 or less.
// Sixteen warps of softmax on an SM, for each scheduler four, hide each other's waits for tensor memory and
// exponentials; eight (a thread per row) left it idle half the time.
template <int D>
struct FwdSmem {
  static constexpr int kTile = D / 64 * kBox, kStages = D == 64 ? 2 : 1;
  static constexpr int kExchange = 2 * 2 * 128 * 4;  // two buffers of a float per row and half
  static constexpr int kTotal = kTile + 2 * kStages * kTile + kExchange + 1024 + 256;
  static_assert(2 * kTotal <= 227 * 1024, "two CTAs to an SM");
};
struct AttnFwdArgs {
  AttnShape s;
  OutTensor out;
  void* rest;  // [batch][q_len][heads][head_dim]: what out's rounding took, or null
  float* lse;  // [batch][heads][q_len], or null
  // Few queries behind many keys: `splits` CTAs share a query block's keys, each leaves its rows' output and lse (in
  // powers of 2) in fp32, [split][batch][heads][q_len][D] and [split][batch][heads][q_len], and join_splits_kernel joins
  // them.
  int splits, ctas;  // ctas: of one split
  float* part;
  float* part_lse;
};

template <int D, typename T, bool CAP, bool BIAS>
__global__ void __maxnreg__(96)
masked_forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const AttnFwdArgs a) {
  chain_begin();
  using SM = FwdSmem<D>;
  constexpr int kStages = SM::kStages, kTile = SM::kTile;
  constexpr bool kApart = D == 64;                  // P beside S
  constexpr int kByFma = forward_by_fma(D, BIAS);
  constexpr uint32_t kP = kApart ? 192 : 0;         // its first column
  extern __shared__ __align__(1024) char smem_raw[];
  char* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  char *sQ = base, *sK = base + kTile, *sV = sK + kStages * kTile;
  float* exchange = reinterpret_cast<float*>(sV + kStages * kTile);  // [2][2 halves][128 rows]
  uint64_t* bars = reinterpret_cast<uint64_t*>(exchange + 512);
  uint64_t *bar_q = bars, *k_full = bars + 1, *k_empty = k_full + kStages, *v_full = k_empty + kStages,
           *v_empty = v_full + kStages, *bar_s = v_empty + kStages, *bar_p = bar_s + 1, *bar_o = bar_p + 1,
           *bar_read = bar_o + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_read + 1);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int nq = blocks_of(a.s.q_len), off = a.s.k_len - a.s.q_len;
  const int all_heads = a.ctas / nq, split = blockIdx.x / a.ctas, cta = blockIdx.x - split * a.ctas;
  const int i = nq - 1 - cta / all_heads;  // of all heads the longest of a causal mask first
  const int bh = cta % all_heads, batch = bh / a.s.heads, head = bh - batch * a.s.heads;
  const int4 info = a.s.mask.q_block(batch, i);
  int begin = info.y > info.x ? info.x / kBlock : 0;
  int blocks = info.y > info.x ? blocks_of(info.y) - begin : 0;
  if (a.splits > 1) {
    const int each = (blocks + a.splits - 1) / a.splits;
    begin += split * each;
    blocks = max(0, min(each, blocks - split * each));
  }

  const int kv = head / a.s.group;
  auto load = [&](int j, uint32_t s, bool k, bool v) {
    if (k) {
      mbar_expect_tx(&k_full[s], kTile);
      load_tile<D>(&map_k, &k_full[s], sK + s * kTile, j * kBlock, kv, batch);
    }
    if (v) {
      mbar_expect_tx(&v_full[s], kTile);
      load_tile<D>(&map_v, &v_full[s], sV + s * kTile, j * kBlock, kv, batch);
    }
  };
  if (warp == 8 && elect_one()) {
    mbar_init(bar_q, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(bar_s, 1);
    mbar_init(bar_p, 8);
    mbar_init(bar_o, 1);
    mbar_init(bar_read, 8);
    *failed = 0;
    fence_barrier_init();
    if (blocks > 0) {  // (the first copies run while tensor memory is allocated)
      mbar_expect_tx(bar_q, kTile);
      load_tile<D>(&map_q, bar_q, sQ, i * kBlock, head, batch);
      load(begin, 0, true, true);
    }
  }
  if (warp == 9) tmem_alloc(tmem_slot, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t phase, int code) {
    if (*failed == 0 && !mbar_wait(bar, phase)) *failed = code;
    tc_fence_after();
  };

  if (warp == 8) {
    if (blocks > 1 && elect_one()) {
      uint32_t s = kStages == 1 ? 0 : 1, round = kStages == 1 ? 1 : 0;
      for (int j = begin + 1; j < begin + blocks; ++j) {
        if (round > 0) wait(&k_empty[s], (round - 1) & 1, 1);
        load(j, s, true, false);
        if (round > 0) wait(&v_empty[s], (round - 1) & 1, 2);
        load(j, s, false, true);
        if (++s == kStages) { s = 0; ++round; }
      }
    }
  } else if (warp == 9) {
    if (blocks > 0 && elect_one()) {
      constexpr int kOperand = std::is_same<T, __half>::value ? kOperandF16 : kOperandBf16;
      const uint32_t id_s = umma_idesc_f16(kOperand, kBlock, 0, 0), id_o = umma_idesc_f16(kOperand, D, 0, 1);
      const uint64_t dQ = k_major<D>(sQ), dK = k_major<D>(sK), dV = mn_major<D>(sV);
      uint32_t ks = 0, k_round = 0, vs = 0, v_round = 0;
      auto scores = [&] {
        wait(&k_full[ks], k_round & 1, 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16(tmem, umma_desc_advance(dQ, k_step(kk)), umma_desc_advance(dK, ks * kTile + k_step(kk)), id_s,
                   kk > 0);
        umma_commit(bar_s);
        umma_commit(&k_empty[ks]);
        if (++ks == kStages) { ks = 0; ++k_round; }
      };
      wait(bar_q, 0, 3);
      scores();
      for (int it = 0; it < blocks; ++it) {
        if (kApart && it + 1 < blocks) {
          wait(bar_read, it & 1, 7);
          scores();
        }
        wait(&v_full[vs], v_round & 1, 6);
        wait(bar_p, it & 1, 5);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)  // K = 128 keys
          umma_f16_ts(tmem + 128, tmem + kP + 8 * kk, umma_desc_advance(dV, vs * kTile + kk * 2048), id_o,
                      (it > 0 || kk > 0) ? 1u : 0u);
        umma_commit(bar_o);
        umma_commit(&v_empty[vs]);
        if (++vs == kStages) { vs = 0; ++v_round; }
        if (!kApart && it + 1 < blocks) scores();  // (behind the product that reads P, in the pipe's order)
      }
    }
  } else {
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const int q = i * kBlock + row;
    const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_addr = lane_addr + 64u * half, p_addr = lane_addr + kP + 32u * half;
    const uint32_t o_addr = lane_addr + 128u + (uint32_t)(D / 2 * half);
    int2 seen = make_int2(0, 0);
    if (q < a.s.q_len) seen = a.s.mask.row(batch, q);
    const float slope = BIAS ? a.s.slopes[head] * kLog2e : 0.f;
    float ref = -1e30f, sum = 0.f;  // in powers of 2; a row that has seen nothing yet is far below all scores
    float lost = 0.f;               // of the largest P, by rounding
    for (int it = 0; it < blocks; ++it) {
      const int key0 = (begin + it) * kBlock + 64 * half;  // this thread's 64 keys
      uint32_t s[2][32];
      wait(bar_s, it & 1, 8);
      ld32_begin(s_addr, s[0]);
      ld32_begin(s_addr + 32, s[1]);
      wait_ld();
      settle(s[0]);
      settle(s[1]);
      if (kApart && it + 1 < blocks) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive(bar_read);
      }
      // The scores in powers of 2.  (Without cap and bias they stay as they are: the factor is positive and comes
      // with the subtraction below.)
      if constexpr (CAP || BIAS) {
        const float apart = (float)(q + off - key0);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            F2 z = pair(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
            if (CAP) {
              float z0, z1;
              unpair(z * pair(a.s.to_2u_log2), z0, z1);
              z = fused(pair(rcp(1.f + ex2(z0)), rcp(1.f + ex2(z1))), pair(-2.f * a.s.cap_log2), pair(a.s.cap_log2));
            } else {
              z = z * pair(a.s.to_log2);
            }
            if (BIAS)
              z = fused(pair(fabsf(apart - (float)(32 * c + e)), fabsf(apart - (float)(32 * c + e + 1))), pair(-slope),
                        z);
            float z0, z1;
            unpair(z, z0, z1);
            s[c][e] = __float_as_uint(z0);
            s[c][e + 1] = __float_as_uint(z1);
          }
      }
      // (blocks that all rows see whole need no test per element)
      const bool whole = info.z <= key0 && info.w >= key0 + 64;
      if (!whole) {
        const unsigned width = (unsigned)max(seen.y - seen.x, 0);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if ((unsigned)(key0 + 32 * c + e - seen.x) >= width) s[c][e] = 0xff800000u;  // -infinity
      }
      float mx4[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx4[c] = __uint_as_float(s[c >> 1][16 * (c & 1)]);
#pragma unroll
        for (int e = 1; e < 16; ++e) mx4[c] = fmaxf(mx4[c], __uint_as_float(s[c >> 1][16 * (c & 1) + e]));
      }
      float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      if constexpr (!CAP && !BIAS) mx *= a.s.to_log2;
      float* met = exchange + (it & 1) * 256 + row;
      met[128 * half] = mx;
      const float mine = mx;
      // the two warps that share these rows (behind it P may lie over the scores, which both have read)
      asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
      mx = fmaxf(mx, met[128 * (half ^ 1)]);
      if (kApart && it > 0) wait(bar_o, (it - 1) & 1, 9);  // the last P has been read
      const bool raise = mx > ref + 8.f;
      if (__any_sync(0xffffffffu, raise)) {
        const float next = raise ? mx : ref, alpha = raise ? ex2(ref - next) : 1.f;
        ref = next;
        sum *= alpha;
        lost *= alpha;
        if (it > 0) {
          if (!kApart) wait(bar_o, (it - 1) & 1, 9);
#pragma unroll 1
          for (int c = 0; c < D / 2; c += 16) {
            uint32_t o[16];
            ld16_begin(o_addr + c, o);
            wait_ld();
            settle16(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            st16(o_addr + c, o);
          }
        }
      }
      F2 sum2 = pair(0.f);
      const auto exponentials = [&](auto mixed) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            F2 z = pair(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
            if constexpr (CAP || BIAS) z = z + pair(-ref);
            else z = fused(z, pair(a.s.to_log2), pair(-ref));
            float p0, p1;
            if (kByFma > 0 && decltype(mixed)::value && (e / 2) % (kByFma + !kByFma) == 0) {
              exp2_by_fma(z, p0, p1);
            } else {
              unpair(z, p0, p1);
              p0 = ex2(p0);
              p1 = ex2(p1);
            }
            sum2 = sum2 + pair(p0, p1);
            p[e / 2] = pack2<T>(p0, p1);
          }
          st16(p_addr + 16 * c, p);
        }
      };
      if (whole) exponentials(std::true_type{});
      else exponentials(std::false_type{});  // (what is not seen is zero to the bit)
      float s0, s1;
      unpair(sum2, s0, s1);
      sum += s0 + s1;
      const float largest = ex2(mine - ref);
      lost += largest - Num<T>::to_f(Num<T>::from_f(largest));
      wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive(bar_p);
    }
    // (the exchange's other buffer was last read before the last block's barrier)
    float* met = exchange + (blocks & 1) * 256 + row;
    met[128 * half] = sum;
    asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
    sum = half == 0 ? sum + met[128] : met[0] + sum;
    met = exchange + ((blocks + 1) & 1) * 256 + row;
    met[128 * half] = lost;
    asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
    lost = half == 0 ? lost + met[128] : met[0] + lost;
    if (blocks > 0) wait(bar_o, (blocks - 1) & 1, 10);
    const float inv = sum > 0.f ? 1.f / (sum - lost) : sum;  // (a sum that is not a number shows in the output)
    const long long part_row = ((long long)split * all_heads + bh) * a.s.q_len + q;
    const long long rest_at = (((long long)batch * a.s.q_len + q) * a.s.heads + head) * a.s.head_dim;
#pragma unroll 1
    for (int c = 0; c < D / 2; c += 16) {
      uint32_t o[16];
      __syncwarp();  // the lanes past the end store nothing, and are back for the next load
      if (blocks > 0) {
        ld16_begin(o_addr + c, o);
        wait_ld();
        settle16(o);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = 0;
      }
      if (q >= a.s.q_len) continue;
      if (a.splits > 1) {
        float4* to = reinterpret_cast<float4*>(a.part + (part_row * D + D / 2 * half + c));
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          to[e / 4] = make_float4(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv,
                                  __uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
      } else {
        store16_of<T>(a.out, batch, q, head, D / 2 * half + c, a.s.head_dim, o, inv,
                      a.rest ? static_cast<T*>(a.rest) + rest_at : nullptr);
      }
    }
    if (half == 0 && q < a.s.q_len) {
      const float lse = sum == 0.f ? -INFINITY : ref + log2f(sum);
      if (a.splits > 1) a.part_lse[part_row] = lse;
      else if (a.lse) a.lse[(long long)bh * a.s.q_len + q] = lse * kLn2;
    }
  }
  if (*failed)  // copies and contractions under way when a wait ran out have ended after this
    for (const long long t0 = clock64(); clock64() - t0 < 100000;) {
    }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *failed != 0 && a.s.status) atomicExch(a.s.status, *failed);
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// A warp joins a row's splits: o = sum_s w_s o_s / sum_s w_s with w_s = 2^(lse_s - max lse).  Four columns a lane at 128.
template <int D, typename T>
__global__ void __launch_bounds__(256)
join_splits_kernel(const AttnFwdArgs a, long long rows) {
  chain_begin();
  constexpr int kPer = D / 32;
  const long long r = (blockIdx.x * 256LL + threadIdx.x) >> 5;  // [batch][heads][q_len]
  const int lane = threadIdx.x & 31;
  if (r >= rows) return;
  float top = -1e30f;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_lse[s * rows + r]);
  float o[kPer], sum = 0.f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) o[e] = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float w = ex2(a.part_lse[s * rows + r] - top);
    sum += w;
    const float* from = a.part + (s * rows + r) * D + kPer * lane;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = fmaf(w, from[e], o[e]);
  }
  const long long bh = r / a.s.q_len, b = bh / a.s.heads;
  const int q = (int)(r - bh * a.s.q_len), h = (int)(bh - b * a.s.heads), c0 = kPer * lane;
  const float inv = sum > 0.f ? 1.f / sum : sum;
  T* to = static_cast<T*>(a.out.p) + b * a.out.batch + q * a.out.row + h * a.out.head;
  T* rest = a.rest ? static_cast<T*>(a.rest) + ((b * a.s.q_len + q) * a.s.heads + h) * a.s.head_dim : nullptr;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if (c0 + e >= a.s.head_dim) continue;
    const float x = o[e] * inv;
    const T t = Num<T>::from_f(x);
    to[c0 + e] = t;
    if (rest) rest[c0 + e] = Num<T>::from_f(x - Num<T>::to_f(t));
  }
  if (lane == 0 && a.lse) a.lse[r] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// ------------------------------------------------------------------------------------------ gradient
// Two kinds of CTA in one launch, alike but for what their rows are.  A tile of 128 rows stays in shared memory, the
// other side comes by in blocks of 128 columns, in units of 64, each unit some four warps' (a thread per row):
//     dK, dV   rows = keys K_j V_j     columns = queries Q_i dO_i of all heads that share the key head
//     dQ       rows = queries Q_i dO_i columns = keys K_j V_j
//     S = rows1 cols1^T, dP = rows2 cols2^T     (128 x 64 each, columns 128 k .. of tensor memory)
//     P and dS over the same columns, 16 bits, A operands of
//     dV += P cols2, dK += dS cols1   or   dQ += dS cols1     (the last 2 D columns)
// What bounds a unit is its chain from contraction to P and dS to contraction, so as many units are under way as tensor
// memory holds: three at 64 dimensions (or one in each of two CTAs, see launch_backward), two at 128.
// dS in f16.  dS is P (dP - D), P about one over the number of keys seen: with the small dO of a training step it falls
// below 2^-14, where f16 loses bits (750 keys and a dO of 1e-4: dS of 25 of f16's least numbers).  So f16 keeps it times
// a power of two, 2^shift, which brings the norm of dO to [1, 2) where it is below: of a query's own for dQ, of the
// call's greatest for dK, whose sums run over queries.  It goes into the exponent that P is made from (dQ), or into D and a
// fused product (dK); the sums are multiplied by 2^-shift in fp32.  A load a row and the maximum at a CTA's start are 1 to
// 4 % of the gradient's time (16 heads of 8192 of 64: 560 -> 568 us; 8 x 512, 12 heads: 39 -> 41).
// Nothing is added across CTAs: the result does not depend on their order.  The price is that S and dP are made
// twice, 7 contractions where sums in device memory need 5; those would cost 4 bytes a value per key block.
template <int D, int UNITS>
struct BwdSmem {
  static constexpr int kUnits = UNITS;  // under way: four warps, and 128 columns of tensor memory, each
  static constexpr int kTmem = UNITS == 1 ? 256 : 512;
  static_assert(128 * UNITS + 2 * D <= kTmem, "tensor memory");
  // (the unit that is issued behind the last of a block lies up to kUnits / 2 blocks further)
  static constexpr int kTile = D / 64 * kBox, kStages = UNITS == 3 ? 3 : 2;
  static constexpr int kThreads = (4 * kUnits + 2) * 32, kTma = 4 * kUnits, kMma = kTma + 1;  // (the last two warps)
  static constexpr int kColumns = kUnits * 2 * 64 * 16;  // two buffers of lse, D and interval per query column
  static constexpr int kTotal = 2 * kTile + 2 * kStages * kTile + kColumns + 1024 + 256;
};
constexpr int kTops = 1152;  // CTAs that leave a maximum, at most; a multiple of 128
struct AttnBwdArgs {
  AttnShape s;
  const float* lse;   // [batch][heads][q_len]
  const float* dsum;  // the same of D
  const float* shift; // the same of dQ's shift (f16)
  const float* tops;  // [top_count <= kTops]: their greatest is that of |dO|^2 (f16)
  int top_count;
  OutTensor dq, dk, dv;
  int kv_ctas;        // the first of the grid: dK and dV
};

// The power of two that brings a norm below one, given squared, to [1, 2); 0 for others and what is not a number.
__device__ __forceinline__ float shift_of(float norm2) {
  if (!(norm2 > 0.f && norm2 < 1.f)) return 0.f;
  return (float)(-(((int)(__float_as_uint(norm2) >> 23) - 127) >> 1));
}

template <int D, int UNITS, typename T, bool CAP, bool BIAS, bool KV>
__device__ __forceinline__ void
backward_body(const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, const CUtensorMap& map_do,
              const AttnBwdArgs& a, int cta) {
  using SM = BwdSmem<D, UNITS>;
  constexpr int kStages = SM::kStages, kTile = SM::kTile, kUnits = SM::kUnits;
  constexpr uint32_t kSums = SM::kTmem - 2 * D;  // first column of the sums
  constexpr bool kShift = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) char smem_raw[];
  char* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  char *sR1 = base, *sR2 = base + kTile, *sC1 = base + 2 * kTile, *sC2 = sC1 + kStages * kTile;
  float2* columns = reinterpret_cast<float2*>(sC2 + kStages * kTile);      // [kUnits][2][64] lse, D
  int2* intervals = reinterpret_cast<int2*>(columns + kUnits * 128);       // [kUnits][2][64]
  uint64_t* bars = reinterpret_cast<uint64_t*>(intervals + kUnits * 128);
  uint64_t *bar_r = bars, *full = bars + 1, *empty = full + kStages, *bar_s = empty + kStages,
           *bar_p = bar_s + kUnits, *bar_a = bar_p + kUnits;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_a + 1);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* tops = reinterpret_cast<float*>(tmem_slot + 2);  // [4 kUnits] of the call's greatest |dO|^2, a warp's part each

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int nq = blocks_of(a.s.q_len), nk = blocks_of(a.s.k_len), off = a.s.k_len - a.s.q_len;
  const int per_head = KV ? nk : nq, heads = KV ? a.s.heads / a.s.group : a.s.heads;
  const int all_heads = (KV ? a.kv_ctas : (int)gridDim.x - a.kv_ctas) / per_head;
  // (of all heads the longest of a causal mask first)
  const int block = KV ? cta / all_heads : per_head - 1 - cta / all_heads;
  const int bh = cta % all_heads, batch = bh / heads, head = bh - batch * heads;
  int first, count, total;  // column blocks, and how many there are over all heads
  int4 info = make_int4(0, 0, 0, 0);
  if (KV) {
    const int2 r = a.s.mask.k_block(batch, block);
    first = r.x;
    count = max(r.y - r.x, 0);
    total = count * a.s.group;
  } else {
    info = a.s.mask.q_block(batch, block);
    first = info.y > info.x ? info.x / kBlock : 0;
    count = info.y > info.x ? blocks_of(info.y) - first : 0;
    total = count;
  }

  auto load = [&](uint32_t s, int b, int h) {
    mbar_expect_tx(&full[s], 2 * kTile);
    load_tile<D>(KV ? &map_q : &map_k, &full[s], sC1 + s * kTile, b * kBlock, h, batch);
    load_tile<D>(KV ? &map_do : &map_v, &full[s], sC2 + s * kTile, b * kBlock, h, batch);
  };
  const int first_head = KV ? head * a.s.group : head / a.s.group;  // of the columns
  if (warp == SM::kTma && elect_one()) {
    mbar_init(bar_r, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int w = 0; w < kUnits; ++w) {
      mbar_init(&bar_s[w], 1);
      mbar_init(&bar_p[w], 4);
    }
    mbar_init(bar_a, 1);
    *failed = 0;
    fence_barrier_init();
    if (total > 0) {  // (the first copies run while tensor memory is allocated)
      mbar_expect_tx(bar_r, 2 * kTile);
      load_tile<D>(KV ? &map_k : &map_q, bar_r, sR1, block * kBlock, head, batch);
      load_tile<D>(KV ? &map_v : &map_do, bar_r, sR2, block * kBlock, head, batch);
      load(0, first, first_head);
    }
  }
  if (warp == SM::kMma) tmem_alloc(tmem_slot, SM::kTmem);
  if (kShift && KV && warp < 4 * kUnits) {
    float top = 0.f;
#pragma unroll
    for (int k = warp; k < kTops / 128; k += 4 * kUnits) {
      const int at = 32 * k + lane;
      if (4 * at >= a.top_count) continue;
      const float4 x = reinterpret_cast<const float4*>(a.tops)[at];
      top = fmaxf(top, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)));
    }
    top = warp_max(top);
    if (lane == 0) tops[warp] = top;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t phase, int code) {
    if (*failed == 0 && !mbar_wait(bar, phase)) *failed = code;
    tc_fence_after();
  };

  if (warp == SM::kTma) {
    if (total > 1 && elect_one()) {
      uint32_t s = 1, round = 0;
      int in_head = 1, h = first_head;
      for (int it = 1; it < total; ++it) {
        if (in_head == count) { in_head = 0; ++h; }
        if (round > 0) wait(&empty[s], (round - 1) & 1, 1);
        load(s, first + in_head++, h);
        if (++s == kStages) { s = 0; ++round; }
      }
    }
  } else if (warp == SM::kMma) {
    if (total > 0 && elect_one()) {
      constexpr int kOperand = std::is_same<T, __half>::value ? kOperandF16 : kOperandBf16;
      const uint32_t id_s = umma_idesc_f16(kOperand, 64, 0, 0), id_a = umma_idesc_f16(kOperand, D, 0, 1);
      const uint64_t dR1 = k_major<D>(sR1), dR2 = k_major<D>(sR2), dC1 = k_major<D>(sC1), dC2 = k_major<D>(sC2);
      const uint64_t mC1 = mn_major<D>(sC1), mC2 = mn_major<D>(sC2);
      const int units = 2 * total;
      uint32_t next_s = 0, next_round = 0;  // of the block whose scores come next
      auto scores = [&](int u, int w) {     // rows 64 (u % 2) .. of its block's tiles
        if ((u & 1) == 0) wait(&full[next_s], next_round & 1, 3);
        const uint32_t at = next_s * kTile + (u & 1) * 8192;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16(tmem + 128 * w, umma_desc_advance(dR1, k_step(kk)), umma_desc_advance(dC1, at + k_step(kk)), id_s,
                   kk > 0);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16(tmem + 128 * w + 64, umma_desc_advance(dR2, k_step(kk)), umma_desc_advance(dC2, at + k_step(kk)),
                   id_s, kk > 0);
        umma_commit(&bar_s[w]);
        if ((u & 1) && ++next_s == kStages) { next_s = 0; ++next_round; }
      };
      wait(bar_r, 0, 2);
      for (int u = 0; u < kUnits && u < units; ++u) scores(u, u);
      uint32_t s = 0;
      int w = 0, k = 0;  // unit u is the k-th of its warps w
      for (int u = 0; u < units; ++u) {
        wait(&bar_p[w], k & 1, 4);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {  // K = 64 columns
          const uint32_t at = s * kTile + (u & 1) * 8192 + kk * 2048, add = (u > 0 || kk > 0) ? 1u : 0u;
          if (KV) umma_f16_ts(tmem + kSums, tmem + 128 * w + 8 * kk, umma_desc_advance(mC2, at), id_a, add);
          umma_f16_ts(tmem + kSums + D, tmem + 128 * w + 64 + 8 * kk, umma_desc_advance(mC1, at), id_a, add);
        }
        if (u & 1) {
          umma_commit(u + 1 < units ? &empty[s] : bar_a);
          if (++s == kStages) s = 0;
        }
        if (u + kUnits < units) scores(u + kUnits, w);  // (behind the products that read P and dS, in the pipe's order)
        if (++w == kUnits) { w = 0; ++k; }
      }
    }
  } else {
    const int w = warp >> 2;                    // of the units, every kUnits-th from w on
    const int row = (warp & 3) * 32 + lane;
    const int mine = block * kBlock + row;      // key or query
    const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_addr = lane_addr + 128u * w;
    const int tid = threadIdx.x & 127;          // in the unit's four warps
    const long long rows0 = (long long)(KV ? batch * a.s.heads + head * a.s.group : bh) * a.s.q_len;
    // (a row that sees nothing, and what lies past the end: lse of infinity makes P zero)
    auto lse_of = [&](long long at) {
      const float l = a.lse[at];
      return l == -INFINITY ? INFINITY : l * kLog2e;
    };
    float my_lse = INFINITY, my_d = 0.f, slope = 0.f;
    float shift = 0.f, up = 1.f;  // up: 2^shift, of all columns (KV)
    if (kShift && KV && total > 0) {
      float top = tops[0];
#pragma unroll
      for (int at = 1; at < 4 * kUnits; ++at) top = fmaxf(top, tops[at]);
      shift = shift_of(top);
      up = exp2f(shift);
    }
    int2 seen = make_int2(0, 0);
    if (!KV && mine < a.s.q_len) {
      my_lse = lse_of(rows0 + mine);
      my_d = a.dsum[rows0 + mine];
      if (kShift) {
        shift = a.shift[rows0 + mine];
        my_lse -= shift;
      }
      seen = a.s.mask.row(batch, mine);
    }
    if (BIAS && !KV) slope = a.s.slopes[head] * kLog2e;
    // of a unit's columns, where they are queries: lse, D and the interval, a thread per column
    struct Column { float2 ld; int2 seen; };
    auto column = [&](int u, int in_head, int hq) {
      Column c{make_float2(INFINITY, 0.f), make_int2(0, 0)};
      const int q = (first + in_head) * kBlock + 64 * (u & 1) + tid;
      if (tid < 64 && q < a.s.q_len) {
        const long long at = rows0 + (long long)hq * a.s.q_len + q;
        c.seen = a.s.mask.row(batch, q);
        c.ld = make_float2(lse_of(at), kShift ? up * a.dsum[at] : a.dsum[at]);
      }
      return c;
    };
    auto keep = [&](int buffer, const Column& c) {
      if (tid < 64) {
        columns[(2 * w + buffer) * 64 + tid] = c.ld;
        intervals[(2 * w + buffer) * 64 + tid] = c.seen;
      }
    };
    // the block of unit u within its head, and the head
    int in_head = w >> 1, hq = 0;
    auto settle_head = [&] {
      while (in_head >= count) { in_head -= count; ++hq; }
    };
    if (total > 0) settle_head();
    if (KV && w < 2 * total) keep(0, column(w, in_head, hq));
    for (int u = w, k = 0; u < 2 * total; u += kUnits, ++k) {
      const int col0 = (first + in_head) * kBlock + 64 * (u & 1);
      const float2* cols = columns + (2 * w + (k & 1)) * 64;
      const int2* seen_by = intervals + (2 * w + (k & 1)) * 64;
      bool whole;
      Column ahead;
      const int this_in = in_head, this_hq = hq;
      in_head += ((u + kUnits) >> 1) - (u >> 1);
      settle_head();
      if (KV) {
        asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory");  // the columns are there
        const int4 q = a.s.mask.q_block(batch, first + this_in);
        whole = q.z <= block * kBlock && q.w >= (block + 1) * kBlock;
        if (BIAS) slope = a.s.slopes[head * a.s.group + this_hq] * kLog2e;
        if (u + kUnits < 2 * total) ahead = column(u + kUnits, in_head, hq);
      } else {
        whole = info.z <= col0 && info.w >= col0 + 64;
      }
      wait(&bar_s[w], k & 1, 5);
      const float apart = (float)(KV ? mine - col0 - off : mine + off - col0);  // of this row and column col0
      // 32 columns at a time: P and dS lie over columns that have been read
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t sr[32], dr[32];
        ld32_begin(s_addr + 32 * c, sr);
        ld32_begin(s_addr + 64 + 32 * c, dr);
        wait_ld();
        settle(sr);
        settle(dr);
        uint32_t p[16], ds[16];
        // two columns at a time; `whole` tests no element
        const auto columns_of = [&](auto tested) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const int col = 32 * c + e;
            float4 x;  // lse and D of both columns
            if (KV) x = *reinterpret_cast<const float4*>(cols + col);
            F2 less = KV ? pair(-x.x, -x.z) : pair(-my_lse);
            if (BIAS)
              less = fused(pair(fabsf(apart - (float)col), fabsf(apart - (float)(col + 1))), pair(-slope), less);
            F2 z = pair(__uint_as_float(sr[e]), __uint_as_float(sr[e + 1])), flat;
            if (CAP) {
              float z0, z1;
              unpair(z * pair(a.s.to_2u_log2), z0, z1);
              const F2 r = pair(rcp(1.f + ex2(z0)), rcp(1.f + ex2(z1)));
              z = fused(r, pair(-2.f * a.s.cap_log2), pair(a.s.cap_log2)) + less;
              flat = r * fused(r, pair(-4.f), pair(4.f));
            } else {
              z = fused(z, pair(a.s.to_log2), less);
            }
            float p0, p1, d0, d1;
            unpair(z, p0, p1);
            p0 = ex2(p0);
            p1 = ex2(p1);
            const F2 less_d = KV ? pair(-x.y, -x.w) : pair(-my_d);
            F2 d = pair(__uint_as_float(dr[e]), __uint_as_float(dr[e + 1]));
            if constexpr (kShift && KV) d = fused(d, pair(up), less_d);
            else d = d + less_d;
            d = d * pair(p0, p1);
            if (CAP) d = d * flat;
            unpair(d, d0, d1);
            if constexpr (decltype(tested)::value) {  // what is not seen counts nothing, whatever its score
              bool sees0, sees1;
              if (KV) {
                const int4 r = *reinterpret_cast<const int4*>(seen_by + col);
                sees0 = mine >= r.x && mine < r.y;
                sees1 = mine >= r.z && mine < r.w;
              } else {
                sees0 = col0 + col >= seen.x && col0 + col < seen.y;
                sees1 = col0 + col + 1 >= seen.x && col0 + col + 1 < seen.y;
              }
              if (!sees0) p0 = d0 = 0.f;
              if (!sees1) p1 = d1 = 0.f;
            }
            p[e / 2] = pack2<T>(p0, p1);
            ds[e / 2] = pack2<T>(d0, d1);
          }
        };
        if (whole) columns_of(std::false_type{});
        else columns_of(std::true_type{});
        if (KV) st16(s_addr + 16 * c, p);
        st16(s_addr + 64 + 16 * c, ds);
      }
      wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive(&bar_p[w]);
      // (the other buffer was last read before this unit's barrier)
      if (KV && u + kUnits < 2 * total) keep((k + 1) & 1, ahead);
    }
    if (total > 0) wait(bar_a, 0, 6);
    // dV and dK, 2 D columns of sums, or dQ, the last D: 16 columns at a time, in turn
    const int rows = KV ? a.s.k_len : a.s.q_len;
    const float down = kShift ? a.s.scale * exp2f(-shift) : a.s.scale;
#pragma unroll 1
    for (int c = (KV ? 0 : D) + 16 * w; c < 2 * D; c += 16 * kUnits) {
      uint32_t o[16];
      __syncwarp();
      if (total > 0) {
        ld16_begin(lane_addr + kSums + c, o);
        wait_ld();
        settle16(o);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = 0;
      }
      if (mine < rows)
        store16_of<T>(KV ? (c < D ? a.dv : a.dk) : a.dq, batch, mine, head, c & (D - 1), a.s.head_dim, o,
                      c < D ? 1.f : down, nullptr);
    }
  }
  if (*failed)
    for (const long long t0 = clock64(); clock64() - t0 < 100000;) {
    }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *failed != 0 && a.s.status) atomicExch(a.s.status, *failed);
  if (warp == SM::kMma) {
    tc_fence_after();
    tmem_dealloc(tmem, SM::kTmem);
  }
}

template <int D, int UNITS, typename T, bool CAP, bool BIAS>
__global__ void __launch_bounds__(BwdSmem<D, UNITS>::kThreads, UNITS == 1 ? 2 : 1)
masked_backward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                       const AttnBwdArgs a) {
  chain_begin();
  if ((int)blockIdx.x < a.kv_ctas)
    backward_body<D, UNITS, T, CAP, BIAS, true>(map_q, map_k, map_v, map_do, a, blockIdx.x);
  else
    backward_body<D, UNITS, T, CAP, BIAS, false>(map_q, map_k, map_v, map_do, a, blockIdx.x - a.kv_ctas);
}

// D = rowsum(dO * (O + rest)): LANES lanes per row, one 16-byte load of each.  Results in [batch][heads][q_len].  In f16
// also each row's shift, and each CTA's greatest |dO|^2 of its rows; there CTAs take several runs of rows each, so that
// these are few.
template <typename T, int LANES>
__global__ void __launch_bounds__(256)
masked_dsum_kernel(const OutTensor o, const T* __restrict__ rest, const OutTensor go, float* __restrict__ dsum,
                   float* __restrict__ shift, float* __restrict__ tops, long long rows, int q_len, int heads,
                   int head_dim) {
  constexpr bool kShift = std::is_same<T, __half>::value;
  chain_begin();
  const int c = 8 * (int)(threadIdx.x % LANES);
  float top = 0.f;
  for (long long r0 = blockIdx.x * (256LL / LANES); r0 < rows; r0 += gridDim.x * (256LL / LANES)) {
    const long long r = r0 + threadIdx.x / LANES;
    float acc = 0.f, norm2 = 0.f;
    long long bt = 0, b = 0;
    int h = 0;
    if (r < rows) {
      bt = r / heads;
      h = (int)(r - bt * heads);
      b = bt / q_len;
      if (c < head_dim) {
        const long long i = bt - b * q_len;
        float x[8], g[8];
        unpack16(load16(static_cast<const T*>(o.p) + b * o.batch + i * o.row + h * o.head + c), x);
        unpack16(load16(static_cast<const T*>(go.p) + b * go.batch + i * go.row + h * go.head + c), g);
        if (rest) {
          float y[8];
          unpack16(load16(rest + r * head_dim + c), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] += y[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) acc = fmaf(x[e], g[e], acc);
        if (kShift)
#pragma unroll
          for (int e = 0; e < 8; ++e) norm2 = fmaf(g[e], g[e], norm2);
      }
    }
#pragma unroll
    for (int k = 1; k < LANES; k <<= 1) {
      acc += __shfl_xor_sync(0xffffffffu, acc, k);
      if (kShift) norm2 += __shfl_xor_sync(0xffffffffu, norm2, k);
    }
    if (r < rows && c == 0) {
      const long long at = (b * heads + h) * q_len + bt - b * q_len;
      dsum[at] = acc;
      if (kShift) shift[at] = shift_of(norm2);
    }
    if (kShift && norm2 < INFINITY) top = fmaxf(top, norm2);
  }
  if constexpr (kShift) {
    __shared__ float met[8];
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0) met[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < 8; ++w) top = fmaxf(top, met[w]);
      tops[blockIdx.x] = top;
      for (unsigned at = gridDim.x; blockIdx.x == 0 && at % 4 != 0; ++at) tops[at] = 0.f;  // (read four at a time)
    }
  }
}

// ------------------------------------------------------------------------------------------ host
int head_map(CUtensorMap* m, const flb200_head_tensor& t, long long batch, long long heads, long long len,
             long long head_dim, int operand) {
  const uint64_t dims[4] = {(uint64_t)head_dim, (uint64_t)len, (uint64_t)heads, (uint64_t)batch};
  const uint64_t strides[3] = {(uint64_t)t.row * 2, (uint64_t)t.head * 2, (uint64_t)t.batch * 2};
  const uint32_t box[4] = {64, kBlock, 1, 1};
  return make_tensor_map(m, t.data, 4, dims, strides, box, kMapKMajor, nullptr, operand);
}
int configure(const void* kernel, int smem) {
  static std::mutex mu;
  static std::set<std::pair<int, const void*>> done;
  int dev = 0;
  FLB200_CUDA_CHECK(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({dev, kernel})) return FLB200_OK;
  FLB200_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  done.insert({dev, kernel});
  return FLB200_OK;
}
OutTensor out_of(const flb200_head_tensor& t, long long head_dim) {
  const bool wide = (reinterpret_cast<uintptr_t>(t.data) & 31) == 0 &&
                    (t.batch | t.row | t.head | head_dim) % 16 == 0;
  return OutTensor{t.data, t.batch, t.row, t.head, wide ? 1 : 0};
}

// Of how many parts each query block's keys are: as many as fill the SMs' two places each, of four blocks at least.  One
// query of 8 heads of 128 behind 8000 keys: 102 us in one part, 24 in parts of two blocks, 19 of four, 23 of eight; 77
// behind 2000: 20, 12.6, 12.9, 15; 512 of 512: 8 in one part (as the rule leaves it), 12.5 in parts of two.
int splits_of(const flb200_attention_desc* d) {
  const long long ctas = d->batch * d->heads * blocks_of(d->q_len), places = 2LL * device_info().sm_count;
  const long long s = std::min(places / ctas, (long long)blocks_of(d->k_len) / 4);
  return s < 2 ? 1 : (int)s;
}
// CTAs of the gradient's first pass.  In f16, where each leaves a maximum that every CTA of dK and dV reads, about as
// many as the SMs hold at once.
unsigned dsum_ctas(const flb200_attention_desc* d) {
  const long long lanes = d->head_dim <= 64 ? 8 : 16, ctas = (d->batch * d->heads * d->q_len * lanes + 255) / 256;
  return (unsigned)(d->dtype == FLB200_F16 ? std::min(ctas, (long long)kTops) : ctas);
}
int padded_dim(const flb200_attention_desc* d) { return d->head_dim <= 64 ? 64 : 128; }

AttnShape shape_of(const flb200_attention_desc* d, const float* slopes, const void* mask) {
  AttnShape s{};
  s.q_len = (int)d->q_len;
  s.k_len = (int)d->k_len;
  s.heads = (int)d->heads;
  s.group = (int)(d->heads / d->kv_heads);
  s.head_dim = (int)d->head_dim;
  s.mask = mask_view(mask, d->batch, d->q_len, d->k_len);
  s.mask.causal = d->causal ? 1 : 0;
  s.mask.prefix = mask ? nullptr : d->prefix;
  s.slopes = slopes;
  s.scale = d->scale;
  s.to_log2 = d->scale * kLog2e;
  s.cap_log2 = d->softcap * kLog2e;
  s.to_2u_log2 = d->softcap > 0.f ? 2.f * d->scale / d->softcap * kLog2e : 0.f;
  s.status = status_ptr();
  return s;
}
int check_attention(const char* name, const flb200_attention_desc* d) {
  FLB200_REQUIRE(d, "%s: null descriptor", name);
  FLB200_REQUIRE(d->batch >= 1 && d->q_len >= 1 && d->k_len >= d->q_len && d->heads >= 1 && d->kv_heads >= 1 &&
                     d->heads % d->kv_heads == 0 && d->head_dim >= 1,
                 "%s: bad extents", name);
  FLB200_REQUIRE(d->causal || !d->prefix, "%s: a prefix belongs to a causal mask", name);
  FLB200_REQUIRE(d->scale > 0.f && d->scale < 1e30f, "%s: the scale must be positive", name);
  FLB200_REQUIRE(d->softcap >= 0.f && d->softcap < 1e30f && (d->softcap == 0.f || d->scale / d->softcap < 1e30f),
                 "%s: the cap must be positive, or 0 for none", name);
  if (!flb200_masked_attention_supported(d))
    return fail(FLB200_UNSUPPORTED, "%s: built for f16 and bf16 and head dimensions that are multiples of 8 up to 128",
                name);
  return FLB200_OK;
}
// 16-byte rows that TMA can address
int check_tensor(const char* name, const flb200_head_tensor* t) {
  FLB200_REQUIRE(t && t->data, "%s: null tensor", name);
  FLB200_REQUIRE(aligned16(t->data) && t->batch > 0 && t->row > 0 && t->head > 0 && t->batch % 8 == 0 &&
                     t->row % 8 == 0 && t->head % 8 == 0,
                 "%s: tensors need 16-byte aligned rows and positive strides", name);
  return FLB200_OK;
}

template <int D, typename T, bool CAP, bool BIAS>
int launch_forward(const flb200_attention_desc* d, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                   AttnFwdArgs a, cudaStream_t st) {
  const auto kernel = masked_forward_kernel<D, T, CAP, BIAS>;
  if (int rc = configure(reinterpret_cast<const void*>(kernel), FwdSmem<D>::kTotal)) return rc;
  a.ctas = (int)(d->batch * d->heads * blocks_of(d->q_len));
  launch_chained(kernel, (unsigned)(a.ctas * a.splits), kFwdThreads, FwdSmem<D>::kTotal, st, mq, mk, mv, a);
  FLB200_AFTER_LAUNCH("masked_attention_forward");
  count_tc_launch();
  if (a.splits > 1) {
    const long long rows = d->batch * d->heads * d->q_len;
    launch_chained(join_splits_kernel<D, T>, (unsigned)((rows + 7) / 8), 256, 0, st, a, rows);
    FLB200_AFTER_LAUNCH("masked_attention_join");
  }
  return FLB200_OK;
}
template <int D, int UNITS, typename T, bool CAP, bool BIAS>
int launch_backward_as(const flb200_attention_desc* d, const CUtensorMap& mq, const CUtensorMap& mk,
                       const CUtensorMap& mv, const CUtensorMap& mg, AttnBwdArgs a, cudaStream_t st) {
  using SM = BwdSmem<D, UNITS>;
  const auto kernel = masked_backward_kernel<D, UNITS, T, CAP, BIAS>;
  if (int rc = configure(reinterpret_cast<const void*>(kernel), SM::kTotal)) return rc;
  a.kv_ctas = (int)(d->batch * d->kv_heads * blocks_of(d->k_len));
  const unsigned grid = (unsigned)(a.kv_ctas + d->batch * d->heads * blocks_of(d->q_len));
  launch_chained(kernel, grid, SM::kThreads, SM::kTotal, st, mq, mk, mv, mg, a);
  FLB200_AFTER_LAUNCH("masked_attention_backward");
  count_tc_launch();
  return FLB200_OK;
}
template <int D, typename T, bool CAP, bool BIAS>
int launch_backward(const flb200_attention_desc* d, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                    const CUtensorMap& mg, const AttnBwdArgs& a, cudaStream_t st) {
  if constexpr (D == 64) {
    // Short rows are bound by what a CTA does before its first and after its last unit, which a second CTA on the SM
    // fills; long ones by the units under way, of which one CTA holds three and two CTAs one each.  12 heads of 8 x 512,
    // documents of 128: 27 us with two CTAs, 37 with one; 16 of 2 x 4096 315 and 301, in documents of 1000
    // 144 and 155; 16 of 8192 570 and 516, in documents of 1000 149 and 155.
    if (d->k_len <= 4096) return launch_backward_as<D, 1, T, CAP, BIAS>(d, mq, mk, mv, mg, a, st);
    return launch_backward_as<D, 3, T, CAP, BIAS>(d, mq, mk, mv, mg, a, st);
  } else {
    return launch_backward_as<D, 2, T, CAP, BIAS>(d, mq, mk, mv, mg, a, st);
  }
}
// f(std::integral_constant<int, D>, T, cap, bias)
template <class F>
int dispatch(const flb200_attention_desc* d, bool bias, const F& f) {
  const auto by_flags = [&](auto dim, auto type) {
    using std::false_type;
    using std::true_type;
    if (d->softcap > 0.f) return bias ? f(dim, type, true_type{}, true_type{}) : f(dim, type, true_type{}, false_type{});
    return bias ? f(dim, type, false_type{}, true_type{}) : f(dim, type, false_type{}, false_type{});
  };
  const auto by_type = [&](auto dim) {
    return d->dtype == FLB200_F16 ? by_flags(dim, __half{}) : by_flags(dim, __nv_bfloat16{});
  };
  return d->head_dim <= 64 ? by_type(std::integral_constant<int, 64>{}) : by_type(std::integral_constant<int, 128>{});
}

}  // namespace
}  // namespace flb200

using namespace flb200;

extern "C" {

size_t flb200_attention_mask_bytes(int64_t batch, int64_t q_len, int64_t k_len) {
  return batch < 1 || q_len < 1 || k_len < 1 ? 0 : mask_bytes(batch, q_len, k_len);
}

int flb200_attention_mask(int64_t batch, int64_t q_len, int64_t k_len, int causal, const int32_t* documents,
                          const int32_t* prefix, void* mask, void* stream) {
  FLB200_REQUIRE(batch >= 1 && q_len >= 1 && k_len >= q_len && k_len < (1 << 24) && batch < 65536,
                 "attention_mask: bad extents");
  FLB200_REQUIRE(documents, "attention_mask: null documents");
  FLB200_REQUIRE(mask && aligned16(mask), "attention_mask: the mask must be 16-byte aligned");
  FLB200_REQUIRE(causal || !prefix, "attention_mask: a prefix belongs to a causal mask");
  const MaskView v = mask_view(mask, batch, q_len, k_len);
  launch_chained(attention_mask_kernel, (unsigned)batch, 1024, 0, as_stream(stream), documents, prefix, (int)q_len,
                 (int)k_len, causal ? 1 : 0, const_cast<int4*>(v.q_blocks), const_cast<int2*>(v.k_blocks),
                 const_cast<int2*>(v.rows));
  FLB200_AFTER_LAUNCH("attention_mask");
  return FLB200_OK;
}

int flb200_masked_attention_supported(const flb200_attention_desc* d) {
  return d && flb200_has_tensor_core_path() && (d->dtype == FLB200_BF16 || d->dtype == FLB200_F16) &&
                 d->head_dim % 8 == 0 && d->head_dim <= 128 && d->k_len < (1 << 24) &&
                 d->batch * d->heads * ((d->k_len + 127) / 128) < (1LL << 30)
             ? 1
             : 0;
}

size_t flb200_masked_attention_forward_workspace_bytes(const flb200_attention_desc* d) {
  if (!d || d->batch < 1 || d->heads < 1 || d->q_len < 1 || d->k_len < 1) return 0;
  const long long splits = splits_of(d);
  return splits < 2 ? 0 : (size_t)(splits * d->batch * d->heads * d->q_len * (padded_dim(d) + 1)) * sizeof(float);
}

int flb200_masked_attention_forward(const flb200_attention_desc* d, const flb200_head_tensor* q,
                                    const flb200_head_tensor* k, const flb200_head_tensor* v, const float* slopes,
                                    const void* mask, const flb200_head_tensor* out, void* rest, float* lse,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_attention("masked_attention_forward", d)) return rc;
  FLB200_REQUIRE(!mask || aligned16(mask), "masked_attention_forward: the mask must be 16-byte aligned");
  FLB200_REQUIRE(!rest || aligned16(rest), "masked_attention_forward: rest must be 16-byte aligned");
  for (const flb200_head_tensor* t : {q, k, v, out})
    if (int rc = check_tensor("masked_attention_forward", t)) return rc;
  const int operand = operand_of(d->dtype);
  CUtensorMap mq, mk, mv;
  if (int rc = head_map(&mq, *q, d->batch, d->heads, d->q_len, d->head_dim, operand)) return rc;
  if (int rc = head_map(&mk, *k, d->batch, d->kv_heads, d->k_len, d->head_dim, operand)) return rc;
  if (int rc = head_map(&mv, *v, d->batch, d->kv_heads, d->k_len, d->head_dim, operand)) return rc;
  AttnFwdArgs a{};
  a.s = shape_of(d, slopes, mask);
  a.out = out_of(*out, d->head_dim);
  a.rest = rest;
  if (reinterpret_cast<uintptr_t>(rest) & 31) a.out.wide = 0;
  a.splits = splits_of(d);
  const size_t need = flb200_masked_attention_forward_workspace_bytes(d);
  if (need) {
    if (!workspace || !aligned16(workspace) || workspace_bytes < need)
      return fail(FLB200_WORKSPACE_TOO_SMALL, "masked_attention_forward: workspace %zu < %zu", workspace_bytes, need);
    a.part = static_cast<float*>(workspace);
    a.part_lse = a.part + a.splits * d->batch * d->heads * d->q_len * padded_dim(d);
  }
  a.lse = lse;
  return dispatch(d, slopes != nullptr, [&](auto dim, auto type, auto cap, auto bias) {
    return launch_forward<decltype(dim)::value, decltype(type), decltype(cap)::value, decltype(bias)::value>(
        d, mq, mk, mv, a, as_stream(stream));
  });
}

size_t flb200_masked_attention_backward_workspace_bytes(const flb200_attention_desc* d) {
  if (!d || d->batch < 1 || d->heads < 1 || d->q_len < 1) return 0;
  const size_t rows = (size_t)(d->batch * d->heads * d->q_len);
  return (d->dtype == FLB200_F16 ? 2 * rows + 4 + kTops : rows) * sizeof(float);  // (4: tops on 16 bytes)
}

int flb200_masked_attention_backward(const flb200_attention_desc* d, const flb200_head_tensor* q,
                                     const flb200_head_tensor* k, const flb200_head_tensor* v,
                                     const flb200_head_tensor* out, const void* rest,
                                     const flb200_head_tensor* grad_out, const float* lse, const float* slopes, const void* mask,
                                     const flb200_head_tensor* grad_q, const flb200_head_tensor* grad_k,
                                     const flb200_head_tensor* grad_v, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  if (reinterpret_cast<uintptr_t>(workspace) & 3)
    return fail(FLB200_WORKSPACE_TOO_SMALL, "masked_attention_backward: the workspace must be 4-byte aligned");
  if (int rc = check_attention("masked_attention_backward", d)) return rc;
  FLB200_REQUIRE(lse, "masked_attention_backward: null lse");
  FLB200_REQUIRE(!mask || aligned16(mask), "masked_attention_backward: the mask must be 16-byte aligned");
  FLB200_REQUIRE(!rest || aligned16(rest), "masked_attention_backward: rest must be 16-byte aligned");
  for (const flb200_head_tensor* t : {q, k, v, out, grad_out, grad_q, grad_k, grad_v})
    if (int rc = check_tensor("masked_attention_backward", t)) return rc;
  const size_t need = flb200_masked_attention_backward_workspace_bytes(d);
  if (!workspace || workspace_bytes < need)
    return fail(FLB200_WORKSPACE_TOO_SMALL, "masked_attention_backward: workspace %zu < %zu", workspace_bytes, need);
  const cudaStream_t st = as_stream(stream);
  const int operand = operand_of(d->dtype);
  CUtensorMap mq, mk, mv, mg;
  if (int rc = head_map(&mq, *q, d->batch, d->heads, d->q_len, d->head_dim, operand)) return rc;
  if (int rc = head_map(&mk, *k, d->batch, d->kv_heads, d->k_len, d->head_dim, operand)) return rc;
  if (int rc = head_map(&mv, *v, d->batch, d->kv_heads, d->k_len, d->head_dim, operand)) return rc;
  if (int rc = head_map(&mg, *grad_out, d->batch, d->heads, d->q_len, d->head_dim, operand)) return rc;
  float* dsum = static_cast<float*>(workspace);
  const long long rows = d->batch * d->heads * d->q_len;
  float* shift = dsum + rows;  // (these two in f16)
  float* tops = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(shift + rows) + 15) & ~(uintptr_t)15);
  const auto row_sums = [&](auto type, auto lanes) {
    using T = decltype(type);
    launch_chained(masked_dsum_kernel<T, decltype(lanes)::value>, dsum_ctas(d), 256, 0, st,
                   out_of(*out, d->head_dim), static_cast<const T*>(rest), out_of(*grad_out, d->head_dim), dsum,
                   shift, tops, rows, (int)d->q_len, (int)d->heads, (int)d->head_dim);
  };
  const auto by_lanes = [&](auto type) {
    if (d->head_dim <= 64) row_sums(type, std::integral_constant<int, 8>{});
    else row_sums(type, std::integral_constant<int, 16>{});
  };
  if (d->dtype == FLB200_F16) by_lanes(__half{});
  else by_lanes(__nv_bfloat16{});
  FLB200_AFTER_LAUNCH("masked_attention_dsum");
  AttnBwdArgs a{};
  a.s = shape_of(d, slopes, mask);
  a.lse = lse;
  a.dsum = dsum;
  a.shift = shift;
  a.tops = tops;
  a.top_count = (int)dsum_ctas(d);
  a.dq = out_of(*grad_q, d->head_dim);
  a.dk = out_of(*grad_k, d->head_dim);
  a.dv = out_of(*grad_v, d->head_dim);
  return dispatch(d, slopes != nullptr, [&](auto dim, auto type, auto cap, auto bias) {
    return launch_backward<decltype(dim)::value, decltype(type), decltype(cap)::value, decltype(bias)::value>(
        d, mq, mk, mv, mg, a, st);
  });
}

}  // extern "C"
