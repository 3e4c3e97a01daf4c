// categoricalCrossEntropy(logSoftmax(linear(x))) over a large vocabulary and its gradient without the scores in
// memory (the chain of flashlight/fl/autograd/Functions.cpp:1255-1309, 1044-1154):
//     z[r][v] = sum_i x[r][i] w[i][v] + bias[v]      lse[r] = log sum_v exp z[r][v]      loss[r] = lse[r] - z[r][t_r]
//     G[r][v] = g_r (exp(z[r][v] - lse[r]) - [v = t_r])      dx = G w^T      dw = x^T G      dbias[v] = sum_r G[r][v]
// The scores of a tile live in tensor memory only (tc_kernel.cuh, tc_pair.cuh).  Forward, an epilogue warp keeps
// the running maximum and sum of its 32 rows over the tile's columns and stores one pair per row and tile;
// what follows joins them, in tile order.  Of the scores the targets' own and lse are kept.  The gradient makes the
// scores once more, a piece of the vocabulary at a time: G in the tensors' 16-bit type into scratch, then the two
// products from it.  dx is summed in fp32 over pieces (and over splits of a piece where its tiles are few) and
// rounded once; dbias comes from G before its rounding.
//
// Rounding of G.  G is at most g_r, and where the vocabulary is large most of it is tiny; so what is stored is
// G / max_r |g_r|, in f16 times 2^15 (f16 keeps 11 bits down to 2^-14: a probability of 2^-29 of the largest weight),
// and the factor is applied to the fp32 sums.  Each entry is then off by at most 2^-9 (bf16) or 2^-12 (f16) of itself.
//
// Bound by the tensor pipe: 2 R d V operations forward, 6 R d V backward, of which a third is the scores again (to
// keep them would cost R V values each way and the memory this operator is there to save).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>

#include "common.cuh"
#include "flb200.h"
#include "tc_gemm.cuh"
#include "tc_pair.cuh"

namespace flb200 {
namespace {

using namespace tc;

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// e^x, x being a difference from a row's maximum
__device__ __forceinline__ float exp_below(float x) { return exp2_of(x * kLog2e); }
// element (row r, column c) of an epilogue warp's staged 32 x 32 chunk (epi_stage_write)
__device__ __forceinline__ float staged(const float* stage, int r, int c) {
  return stage[r * 32 + (((c >> 2) ^ (r & 7)) << 2) + (c & 3)];
}

// The warp's staged chunk to rows m_first.. and columns nb.. of a row-major matrix of T; ADD: onto what is there.
// vec: rows are aligned to four elements.
template <typename T, bool ADD>
__device__ __forceinline__ void store_staged(const float* stage, int lane, T* out, long long ld, int m_first, int M,
                                             int nb, int N, bool vec) {
  if (vec && nb + 32 <= N) {
    T* to = out + (long long)(m_first + (lane >> 3)) * ld + nb + 4 * (lane & 7);
#pragma unroll
    for (int k = 0; k < 8; ++k, to += 4 * ld) {
      if (m_first + 4 * k + (lane >> 3) >= M) continue;
      float4 v = epi_stage_read(stage, lane, k);
      if constexpr (ADD) {
        const float4 old = *reinterpret_cast<const float4*>(to);
        v.x += old.x; v.y += old.y; v.z += old.z; v.w += old.w;
      }
      epi_store4(to, v);
    }
  } else if (nb + lane < N) {  // a row's 32 columns per store
    const int rows = min(32, M - m_first);
    T* to = out + (long long)m_first * ld + nb + lane;
    for (int r = 0; r < rows; ++r, to += ld) {
      float v = staged(stage, r, lane);
      if constexpr (ADD) v += *to;
      *to = Num<T>::from_f(v);
    }
  }
}

// ------------------------------------------------------------------------------------------ the three products
// M = rows, N = columns of the piece of the vocabulary that begins at col0
struct ScoreArgs {
  const float* bias;       // of the piece, or null
  bool bias_vec;
  const int32_t* targets;  // of the rows
  int col0;
  float* target_score;     // forward: [M]
  float2* partial;         // forward: (maximum, sum) [tiles * groups of this piece][M]
  const struct RowInfo* rows;  // gradient: [M]
  void* grad;              // gradient: [M][grad_ld] of T
  long long grad_ld;
  float* column_sum;       // gradient: [groups of 32 rows][grad_ld], or null
};

template <int BN>
struct ScoreProblem : GemmProblem<BN> {
  ScoreArgs s;
  __device__ __forceinline__ void add_bias(int nb, const float* v, float* z) const {
    if (!s.bias) {
#pragma unroll
      for (int j = 0; j < 32; ++j) z[j] = v[j];
    } else if (s.bias_vec && nb + 32 <= this->N) {
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(s.bias + nb + j));
        z[j] = v[j] + b.x; z[j + 1] = v[j + 1] + b.y; z[j + 2] = v[j + 2] + b.z; z[j + 3] = v[j + 3] + b.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) z[j] = nb + j < this->N ? v[j] + __ldg(s.bias + nb + j) : v[j];
    }
  }
};

// (kGroups: how many groups of epilogue warps share a tile's 32-column chunks)
template <int BN>
struct LseProblem : ScoreProblem<BN> {
  static constexpr int kGroups = BN >= 128 ? 2 : 1;
  // A warp meets its chunks of a tile from left to right; between them its rows' maxima and sums wait in its
  // staging tile.  The maximum starts at the lowest finite value: a chunk of -inf alone then counts zeros.
  __device__ __forceinline__ void store(const typename GemmProblem<BN>::Tile& t, int row, int c0, const float* v,
                                        float* stage, int lane) const {
    const int m = t.m0 + row, nb = t.n0 + c0;
    const ScoreArgs& s = this->s;
    float z[32];
    this->add_bias(nb, v, z);
    const int live = this->N - nb;  // columns that exist
    float top = -FLT_MAX, sum = 0.f;
    float2* kept = reinterpret_cast<float2*>(stage) + lane;
    if (c0 >= 32 * kGroups) {
      top = kept->x;
      sum = kept->y;
    }
    float mx = top;
    if (live >= 32) {
#pragma unroll
      for (int j = 0; j < 32; ++j) mx = fmaxf(mx, z[j]);
      sum *= exp_below(top - mx);
#pragma unroll
      for (int j = 0; j < 32; ++j) sum += exp_below(z[j] - mx);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) mx = j < live ? fmaxf(mx, z[j]) : mx;
      sum *= exp_below(top - mx);
#pragma unroll
      for (int j = 0; j < 32; ++j) sum += j < live ? exp_below(z[j] - mx) : 0.f;
    }
    const int rel = m < this->M ? s.targets[m] - s.col0 - nb : -1;
    if (rel >= 0 && rel < 32 && rel < live) {
      float score = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j) score = j == rel ? z[j] : score;
      s.target_score[m] = score;
    }
    if (c0 + 32 * kGroups < BN && nb + 32 * kGroups < this->N) {
      *kept = make_float2(mx, sum);
    } else if (m < this->M) {
      const int part = t.n0 / BN * kGroups + (c0 / 32) % kGroups;
      s.partial[(long long)part * this->M + m] = make_float2(mx, sum);
    }
  }
};

// What a row of the gradient's scores needs, one 16-byte load: lse log2 e, what G is stored with (0 where the row does
// not count) and the target.
struct RowInfo {
  float lse_log2, weight;
  int target, unused;
};

// A lane has 32 columns of its row, 64 bytes of G: it stores them itself, whole sectors of 32 bytes.  Only the
// columns' sums pass through the staging tile.  (Staged like the other products' results, with three loads per row
// and a test per element, a tile of 256 columns took 16700 clocks, two and a half times its contraction over 768.)
template <int BN, typename T>
struct GradScoreProblem : ScoreProblem<BN> {
  __device__ __forceinline__ void store(const typename GemmProblem<BN>::Tile& t, int row, int c0, const float* v,
                                        float* stage, int lane) const {
    const int m = t.m0 + row, nb = t.n0 + c0, m_first = m - lane;
    const ScoreArgs& s = this->s;
    if (m_first >= this->M) return;  // (the whole warp)
    RowInfo info{0.f, 0.f, -1, 0};
    if (m < this->M) {
      const int4 r = __ldg(reinterpret_cast<const int4*>(s.rows + m));
      info = RowInfo{__int_as_float(r.x), __int_as_float(r.y), r.z, 0};
    }
    const float less = -info.lse_log2;
    float z[32];
    if (!s.bias) {
#pragma unroll
      for (int j = 0; j < 32; ++j) z[j] = fmaf(v[j], kLog2e, less);
    } else if (s.bias_vec && nb + 32 <= this->N) {
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(s.bias + nb + j));
        z[j] = fmaf(v[j] + b.x, kLog2e, less);
        z[j + 1] = fmaf(v[j + 1] + b.y, kLog2e, less);
        z[j + 2] = fmaf(v[j + 2] + b.z, kLog2e, less);
        z[j + 3] = fmaf(v[j + 3] + b.w, kLog2e, less);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        z[j] = fmaf(nb + j < this->N ? v[j] + __ldg(s.bias + nb + j) : v[j], kLog2e, less);
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) z[j] = info.weight * exp2_of(z[j]);
    if (info.weight == 0.f) {  // zeros whatever the row's scores
#pragma unroll
      for (int j = 0; j < 32; ++j) z[j] = 0.f;
    }
    const int rel = info.target - s.col0 - nb;
    if (rel >= 0 && rel < 32) {
#pragma unroll
      for (int j = 0; j < 32; ++j) z[j] = j == rel ? z[j] - info.weight : z[j];
    }
    const bool whole = nb + 32 <= this->N;
    T* out = static_cast<T*>(s.grad);
    if (whole && m < this->M) {
      T* to = out + (long long)m * s.grad_ld + nb;
#pragma unroll
      for (int j = 0; j < 32; j += 16) {
        const Vec16<T> lo = pack16<T>(z + j), hi = pack16<T>(z + j + 8);
        const uint4 a = *reinterpret_cast<const uint4*>(&lo), b = *reinterpret_cast<const uint4*>(&hi);
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + j), "r"(a.x), "r"(a.y),
                     "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                     : "memory");
      }
    }
    if (whole && !s.column_sum) return;
    epi_stage_write(stage, lane, z);
    if (!whole)
      store_staged<T, false>(stage, lane, out, s.grad_ld, m_first, this->M, nb, this->N, true);
    if (s.column_sum) {
      // four columns of every fourth row, then the four lanes that have the same columns; rows past the end are zeros
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float4 x = epi_stage_read(stage, lane, k);
        sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
      }
#pragma unroll
      for (int o = 8; o < 32; o <<= 1) {
        sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
        sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
        sum.z += __shfl_xor_sync(0xffffffffu, sum.z, o);
        sum.w += __shfl_xor_sync(0xffffffffu, sum.w, o);
      }
      if (lane < 8)  // (rows of sums are as long as whole chunks)
        *reinterpret_cast<float4*>(s.column_sum + (long long)(m_first >> 5) * s.grad_ld + nb + 4 * lane) = sum;
    }
    __syncwarp();  // the staging tile is rewritten by the next chunk
  }
};

// dx: fp32 sums [split][M][N], ADD onto those of the pieces before.  dw: rows of the result in its type.
template <int BN, typename T, bool ADD>
struct SumProblem : GemmProblem<BN> {
  T* out;
  long long ld, split_stride;
  const float* factor;  // or null
  bool vec;
  // rows of `stride` elements; `by`: factor, `aligned`: rows are aligned to four elements
  void set(void* to, long long stride, long long splits_apart, const float* by, bool aligned) {
    out = static_cast<T*>(to);
    ld = stride;
    split_stride = splits_apart;
    factor = by;
    vec = aligned;
  }
  __device__ __forceinline__ void store(const typename GemmProblem<BN>::Tile& t, int row, int c0, const float* v,
                                        float* stage, int lane) const {
    const int nb = t.n0 + c0, m_first = t.m0 + row - lane;
    if (m_first >= this->M) return;
    if (factor) {
      const float f = *factor;
      float w[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) w[j] = f * v[j];
      epi_stage_write(stage, lane, w);
    } else {
      epi_stage_write(stage, lane, v);
    }
    store_staged<T, ADD>(stage, lane, out + t.split * split_stride, ld, m_first, this->M, nb, this->N, vec);
    __syncwarp();
  }
};

struct Product {  // D[M][N] over K, 16-bit operands
  long long M, N, K;
  Launch plan;
  int operand;
  int n_fast = 0;  // pair tiles of one pair of row tiles behind one another: for a large row operand and few columns
  CUtensorMap ma, mb;
  OperandPlan pa, pb;
};

// Tiles of 64 columns at least: a stage's box of an MN-major operand.
Launch plan_product(long long M, long long N, long long K, bool a_mn, bool b_mn, int operand, bool split) {
  Launch l = plan_launch(M, N, (K + 63) / 64, 1, a_mn, b_mn, operand, split);
  if (l.bn < 64) l.bn = 64;
  return l;
}

template <template <int> class Problem, int BN, class Fill>
int launch_as(const char* name, const Product& p, const Fill& fill, cudaStream_t st) {
  Problem<BN> g;
  static_cast<GemmProblem<BN>&>(g) = GemmProblem<BN>{};
  g.operand = p.operand;
  g.a = make_coords(p.pa);
  g.b = make_coords(p.pb);
  g.a_mn_major = p.pa.mn_major;
  g.b_mn_major = p.pb.mn_major;
  g.M = (int)p.M;
  g.N = (int)p.N;
  g.k_iters = (int)((p.K + 63) / 64);
  g.splits = p.plan.splits;
  g.iters_per_split = p.plan.iters_per_split;
  g.tiles_m = (int)((p.M + kBM - 1) / kBM);
  g.tiles_n = (int)((p.N + BN - 1) / BN);
  g.Z = 1;
  g.pair_n_fast = p.n_fast;
  fill(g);
  const long long tiles = (long long)g.tiles_m * g.tiles_n * g.splits;
  FLB200_REQUIRE(tiles < 0x7fffffffLL, "%s: too many tiles", name);
  if constexpr (BN == 256) {
    if (p.plan.pairs)
      return launch_pair_problem<Problem<BN>, BN>(name, p.ma, p.mb, g,
                                                  (long long)((g.tiles_m + 1) / 2) * g.tiles_n * g.splits, st);
  }
  constexpr int kSub = BN <= 128 ? 2 : 1;
  return launch_problem_as<Problem<BN>, BN, stages_for(BN), 0, kSub>(name, p.ma, p.mb, g, tiles, st);
}
template <template <int> class Problem, class Fill>
int launch_product(const char* name, const Product& p, const Fill& fill, cudaStream_t st) {
  if (p.plan.bn == 64) return launch_as<Problem, 64>(name, p, fill, st);
  if (p.plan.bn == 128) return launch_as<Problem, 128>(name, p, fill, st);
  return launch_as<Problem, 256>(name, p, fill, st);
}
template <int BN> using GradScoreBf16 = GradScoreProblem<BN, __nv_bfloat16>;
template <int BN> using GradScoreF16 = GradScoreProblem<BN, __half>;
template <int BN> using SumFirst = SumProblem<BN, float, false>;
template <int BN> using SumNext = SumProblem<BN, float, true>;
template <typename T>
struct Result16 {
  template <int BN> using Of = SumProblem<BN, T, false>;
};

// ------------------------------------------------------------------------------------------ around the products
// dst [rows][dst_ld] = src [rows][src_ld] of 16-bit values, `cols` of each row and zeros behind them: the copy of
// a matrix whose rows TMA cannot address.
__global__ void __launch_bounds__(256)
pad_rows_kernel(const uint16_t* __restrict__ src, long long src_ld, uint16_t* __restrict__ dst, int dst_ld,
                int cols, long long rows) {
  chain_begin();
  const int row_quads = dst_ld / 8;
  const long long total = rows * row_quads;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const long long r = i / row_quads;
    const int c = 8 * (int)(i - r * row_quads);
    alignas(16) uint16_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? src[r * src_ld + c + j] : (uint16_t)0;
    *reinterpret_cast<uint4*>(dst + r * dst_ld + c) = *reinterpret_cast<const uint4*>(v);
  }
}

__device__ __forceinline__ bool counts(int target, int ignore, long long classes) {
  return target != ignore && target >= 0 && target < classes;
}

// What a call's rows add up to.
struct LossSums {
  double loss;
  int count, bad;
};
// (a lane each of one warp)
__device__ __forceinline__ LossSums sum_of_warp(LossSums s) {
  s.loss = warp_sum(s.loss);
  s.count = __reduce_add_sync(0xffffffffu, s.count);
  s.bad = __reduce_or_sync(0xffffffffu, s.bad);
  return s;
}
__device__ __forceinline__ void write_loss(const LossSums& s, int reduction, float* loss, int32_t* count,
                                           int32_t* bad) {
  if (count) *count = s.count;
  if (bad) *bad = s.bad;
  if (reduction == FLB200_REDUCE_MEAN) loss[0] = (float)(s.loss / (double)s.count);
  else if (reduction == FLB200_REDUCE_SUM) loss[0] = (float)s.loss;
}

// Joins the tiles' (maximum, sum) of 32 rows per CTA: a warp has all of them, or where a call has few, `few` rows (a power
// of two) of 32 / few parts at once; the 32 warps' shares meet in shared memory (with eight warps 13 us for 4096 rows of
// 250 parts, so 7; four rows of 784 parts 10.5 with a lane per row).  Then the rows' losses, and what they add up to:
// of all rows where there is one CTA, else finish_loss_kernel adds the CTAs'.
constexpr int kJoin = 32;
__global__ void __launch_bounds__(32 * kJoin)
join_lse_kernel(const float2* __restrict__ partial, int parts, const float* __restrict__ target_score,
                const int32_t* __restrict__ targets, int ignore, long long classes, int rows, int reduction,
                float* __restrict__ lse, float* __restrict__ loss, int32_t* __restrict__ count,
                int32_t* __restrict__ bad, LossSums* __restrict__ sums, int few) {
  chain_begin();
  __shared__ float2 met[kJoin][32];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int r = few < 32 && lane >= few ? rows : blockIdx.x * 32 + lane;  // this lane's row in what follows the parts
  float top = -FLT_MAX, sum = 0.f;
  const int at = blockIdx.x * 32 + (lane & (few - 1)), at_once = 32 / few;
  if (at < rows) {
#pragma unroll 4
    for (int p = g * at_once + lane / few; p < parts; p += kJoin * at_once) {
      const float2 x = partial[(long long)p * rows + at];
      const float mx = fmaxf(top, x.x);
      sum = sum * exp_below(top - mx) + x.y * exp_below(x.x - mx);
      top = mx;
    }
  }
  for (int o = few; o < 32; o <<= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, top, o), more = __shfl_xor_sync(0xffffffffu, sum, o);
    const float mx = fmaxf(top, other);
    sum = sum * exp_below(top - mx) + more * exp_below(other - mx);
    top = mx;
  }
  met[g][lane] = make_float2(top, sum);
  for (int half = kJoin / 2; half > 0; half >>= 1) {
    __syncthreads();
    if (g < half) {
      const float2 x = met[g + half][lane];
      const float mx = fmaxf(top, x.x);
      sum = sum * exp_below(top - mx) + x.y * exp_below(x.x - mx);
      top = mx;
      met[g][lane] = make_float2(top, sum);
    }
  }
  if (g > 0) return;
  LossSums all{0.0, 0, 0};
  if (r < rows) {
    const float l = top + logf(sum);
    lse[r] = l;
    const int t = targets[r];
    float mine = 0.f;
    if (counts(t, ignore, classes)) {
      mine = l - target_score[r];
      all.count = 1;
    } else if (t != ignore) {
      all.bad = 1;
    }
    if (reduction == FLB200_REDUCE_NONE) loss[r] = mine;
    all.loss = mine;
  }
  all = sum_of_warp(all);
  if (lane == 0) {
    if (gridDim.x == 1) write_loss(all, reduction, loss, count, bad);
    else sums[blockIdx.x] = all;
  }
}
__global__ void __launch_bounds__(32)
finish_loss_kernel(const LossSums* __restrict__ sums, int n, int reduction, float* __restrict__ loss,
                   int32_t* __restrict__ count, int32_t* __restrict__ bad) {
  chain_begin();
  LossSums all{0.0, 0, 0};
  for (int i = threadIdx.x; i < n; i += 32) {
    const LossSums x = sums[i];
    all.loss += x.loss;
    all.count += x.count;
    all.bad |= x.bad;
  }
  all = sum_of_warp(all);
  if (threadIdx.x == 0) write_loss(all, reduction, loss, count, bad);
}

// Each row's RowInfo, its weight step * g_r / max |g| over the finite g, zero where the row does not count; factor =
// max |g| / step.  A g that is not finite is its row's weight itself: the row's entries are then not finite in any type,
// and the others' are as without it.
__global__ void __launch_bounds__(1024)
row_weights_kernel(const float* __restrict__ grad_loss, const int32_t* __restrict__ targets,
                   const int32_t* __restrict__ count, const float* __restrict__ lse, int reduction, int ignore,
                   long long classes, int rows, float step, RowInfo* __restrict__ info,
                   float* __restrict__ factor) {
  chain_begin();
  __shared__ float scratch[32];
  float top = 0.f, all = 0.f;  // all: what every row has, where the loss is reduced
  if (reduction == FLB200_REDUCE_NONE) {  // (one CTA)
    for (int r = threadIdx.x; r < rows; r += 1024)
      if (counts(targets[r], ignore, classes) && isfinite(grad_loss[r])) top = fmaxf(top, fabsf(grad_loss[r]));
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = top;
    __syncthreads();
    top = warp_max(scratch[threadIdx.x & 31]);
  } else {
    all = grad_loss[0];
    if (reduction == FLB200_REDUCE_MEAN) all = *count > 0 ? all / (float)*count : 0.f;
    top = isfinite(all) ? all : 1.f;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *factor = top / step;
  for (int r = blockIdx.x * 1024 + threadIdx.x; r < rows; r += gridDim.x * 1024) {
    float w = 0.f;
    if (counts(targets[r], ignore, classes)) {
      const float g = reduction != FLB200_REDUCE_NONE ? all : grad_loss[r];
      if (!isfinite(g)) w = g;
      else if (reduction != FLB200_REDUCE_NONE) w = step;
      else w = top > 0.f ? step * (g / top) : 0.f;
    }
    info[r] = RowInfo{lse[r] * kLog2e, w, targets[r], 0};
  }
}

// out [n] = factor * sum of `splits` slabs; vec: n is a multiple of 4 and out aligned to four elements
template <typename T>
__global__ void __launch_bounds__(256)
finish_sums_kernel(const float* __restrict__ slabs, int splits, long long n, const float* __restrict__ factor,
                   T* __restrict__ out, int vec) {
  chain_begin();
  const float f = *factor;
  for (long long i = 4 * (blockIdx.x * 256LL + threadIdx.x); i < n; i += 1024LL * gridDim.x) {
    if (vec) {
      float4 s = *reinterpret_cast<const float4*>(slabs + i);
      for (int k = 1; k < splits; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(slabs + k * n + i);
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
      }
      epi_store4(out + i, make_float4(f * s.x, f * s.y, f * s.z, f * s.w));
    } else {
      for (long long e = i; e < n && e < i + 4; ++e) {
        float s = 0.f;
        for (int k = 0; k < splits; ++k) s += slabs[k * n + e];
        out[e] = Num<T>::from_f(f * s);
      }
    }
  }
}

// out[c] = factor * sum over groups of sums[group][c]
__global__ void __launch_bounds__(256)
finish_columns_kernel(const float* __restrict__ sums, int groups, long long ld, int cols,
                      const float* __restrict__ factor, float* __restrict__ out) {
  chain_begin();
  __shared__ float met[8][33];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < cols)
    for (int k = g; k < groups; k += 8) s += sums[k * ld + c];
  met[g][lane] = s;
  __syncthreads();
  if (g > 0 || c >= cols) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += met[k][lane];
  out[c] = *factor * s;
}

// ------------------------------------------------------------------------------------------ host
constexpr long long kPieceBytes = 128LL << 20;  // of G: the vocabulary is taken in pieces of that

struct Shape {
  long long rows, dim, classes;
  long long x_ld, w_ld;  // of what the products read (copies where the tensors' rows are not 16-byte aligned)
  bool copy_x, copy_w;
  long long piece;       // columns of a piece, a multiple of 256 (forward: all, unless w is copied)
  int operand;
};
long long up(long long n, long long to) { return (n + to - 1) / to * to; }

Shape shape_of(const flb200_linear_cce_desc* d, const void* x, const void* w, bool backward) {
  Shape s{};
  s.rows = d->rows;
  s.dim = d->features;
  s.classes = d->classes;
  s.operand = operand_of(d->dtype);
  s.copy_x = s.dim % 8 != 0 || !aligned16(x);
  s.copy_w = s.classes % 8 != 0 || !aligned16(w);
  s.x_ld = s.copy_x ? up(s.dim, 64) : s.dim;
  s.piece = std::max<long long>(2048, kPieceBytes / (2 * s.rows) / 256 * 256);
  // (a piece of w that is copied is no larger either)
  if (s.copy_w) s.piece = std::min(s.piece, std::max<long long>(2048, kPieceBytes / (2 * s.dim) / 256 * 256));
  if (!backward && !s.copy_w) s.piece = s.classes;
  s.piece = std::min(s.piece, up(s.classes, 256));
  s.w_ld = s.copy_w ? s.piece : s.classes;
  return s;
}

// Scratch, carved in order; with a null base it only adds up.
struct Carve {
  char* base;
  size_t at = 0;
  template <typename T>
  T* take(long long n) {
    T* p = base ? reinterpret_cast<T*>(base + at) : nullptr;
    at = (at + (size_t)n * sizeof(T) + 255) & ~(size_t)255;
    return p;
  }
};
struct ForwardScratch {
  float2* partial;
  float* target_score;
  LossSums* sums;
  uint16_t *x, *w;
  ForwardScratch(Carve& c, const Shape& s) {
    // parts: two per 256 or 128 columns or one per 64, and a short one per piece
    const long long pieces = (s.classes + s.piece - 1) / s.piece;
    partial = c.take<float2>(((s.classes + 63) / 64 + 2 * pieces) * s.rows);
    target_score = c.take<float>(s.rows);
    sums = c.take<LossSums>((s.rows + 31) / 32);
    x = c.take<uint16_t>(s.copy_x ? s.rows * s.x_ld : 0);
    w = c.take<uint16_t>(s.copy_w ? s.dim * s.w_ld : 0);
  }
};
Launch plan_dx(const Shape& s, long long cols) {
  return plan_product(s.rows, s.dim, cols, false, false, s.operand, true);
}
// The splits of K that have something to add when it is cut into `splits` runs of whole stages.
int fit_splits(long long K, int splits, int* stages_each) {
  const long long stages = (K + 63) / 64, each = (stages + splits - 1) / splits;
  *stages_each = (int)each;
  return (int)((stages + each - 1) / each);
}
struct BackwardScratch {
  RowInfo* rows;
  float *factor, *dx, *column_sum;
  uint16_t *grad, *x, *w;
  int dx_splits;
  BackwardScratch(Carve& c, const Shape& s, bool need_x, bool need_bias) {
    rows = c.take<RowInfo>(s.rows);
    factor = c.take<float>(1);
    grad = c.take<uint16_t>(s.rows * s.piece);
    int stages;
    dx_splits = fit_splits(std::min(s.piece, s.classes), std::min(16, plan_dx(s, std::min(s.piece, s.classes)).splits),
                           &stages);
    dx = c.take<float>(need_x ? dx_splits * s.rows * s.dim : 0);
    column_sum = c.take<float>(need_bias ? (s.rows + 31) / 32 * s.piece : 0);
    x = c.take<uint16_t>(s.copy_x ? s.rows * s.x_ld : 0);
    w = c.take<uint16_t>(s.copy_w ? s.dim * s.w_ld : 0);
  }
};

int pad_rows(const void* src, long long src_ld, uint16_t* dst, long long dst_ld, long long cols, long long rows,
             cudaStream_t st) {
  launch_chained(pad_rows_kernel, grid_for(rows * (dst_ld / 8), 256), 256, 0, st,
                 static_cast<const uint16_t*>(src), src_ld, dst, (int)dst_ld, (int)cols, rows);
  FLB200_AFTER_LAUNCH("linear_cce_pad");
  return FLB200_OK;
}

// The operands of a call's products: x, and the piece of w that begins at col0.
struct Operands {
  const void *x, *w;  // of a piece
};
int operands_of(const Shape& s, const void* x, const void* w, uint16_t* x_copy, uint16_t* w_copy, long long col0,
                long long cols, Operands* o, cudaStream_t st) {
  if (s.copy_x && col0 == 0)
    if (int rc = pad_rows(x, s.dim, x_copy, s.x_ld, s.dim, s.rows, st)) return rc;
  o->x = s.copy_x ? x_copy : x;
  const uint16_t* from = static_cast<const uint16_t*>(w) + col0;
  if (s.copy_w)
    if (int rc = pad_rows(from, s.classes, w_copy, s.w_ld, cols, s.dim, st)) return rc;
  o->w = s.copy_w ? w_copy : from;
  return FLB200_OK;
}

int score_product(const Shape& s, const Operands& o, long long cols, Product* p) {
  p->M = s.rows;
  p->N = cols;
  p->K = s.dim;
  p->operand = s.operand;
  p->plan = plan_product(s.rows, cols, s.dim, false, true, s.operand, false);
  if (int rc = matrix_operand(false, s.x_ld, o.x, s.rows, s.dim, kBM, s.operand, &p->ma, &p->pa)) return rc;
  return matrix_operand(true, s.w_ld, o.w, cols, s.dim, p->plan.b_box_rows(), s.operand, &p->mb, &p->pb);
}

int check_desc(const char* name, const flb200_linear_cce_desc* d) {
  FLB200_REQUIRE(d, "%s: null descriptor", name);
  FLB200_REQUIRE(d->reduction >= FLB200_REDUCE_NONE && d->reduction <= FLB200_REDUCE_SUM,
                 "unknown reduction method for categorical cross entropy (%s: %d)", name, d->reduction);
  FLB200_REQUIRE(d->rows >= 1 && d->features >= 1 && d->classes >= 1, "%s: bad extents", name);
  if (!flb200_linear_cce_supported(d))
    return fail(FLB200_UNSUPPORTED, "%s: built for 16-bit tensors of fewer than 2^31 elements a side", name);
  return FLB200_OK;
}

}  // namespace
}  // namespace flb200

using namespace flb200;

extern "C" {

int flb200_linear_cce_supported(const flb200_linear_cce_desc* d) {
  return d && flb200_has_tensor_core_path() && (d->dtype == FLB200_BF16 || d->dtype == FLB200_F16) &&
                 d->rows < (1LL << 24) && d->features < (1LL << 24) && d->classes < (1LL << 30)
             ? 1
             : 0;
}

size_t flb200_linear_cce_workspace_bytes(const flb200_linear_cce_desc* d, const void* x, const void* w, int which) {
  if (!d || d->rows < 1 || d->features < 1 || d->classes < 1 || !flb200_linear_cce_supported(d)) return 0;
  const Shape s = shape_of(d, x, w, which != 0);
  Carve c{nullptr};
  if (which == 0) ForwardScratch(c, s);
  else BackwardScratch(c, s, true, true);
  return c.at;
}

int flb200_linear_cce_forward(const flb200_linear_cce_desc* d, const void* x, const void* w, const float* bias,
                              const int32_t* targets, float* loss, float* lse, int32_t* count_out,
                              int32_t* bad_target_flag, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_desc("linear_cce_forward", d)) return rc;
  FLB200_REQUIRE(x && w && targets && loss && lse, "linear_cce_forward: null tensor");
  const size_t need = flb200_linear_cce_workspace_bytes(d, x, w, 0);
  if (!workspace || !aligned16(workspace) || workspace_bytes < need)
    return fail(FLB200_WORKSPACE_TOO_SMALL, "linear_cce_forward: workspace %zu < %zu", workspace_bytes, need);
  const cudaStream_t st = as_stream(stream);
  const Shape s = shape_of(d, x, w, false);
  Carve carve{static_cast<char*>(workspace)};
  const ForwardScratch scratch(carve, s);
  int parts = 0;
  for (long long col0 = 0; col0 < s.classes; col0 += s.piece) {
    const long long cols = std::min(s.piece, s.classes - col0);
    Operands o;
    if (int rc = operands_of(s, x, w, scratch.x, scratch.w, col0, cols, &o, st)) return rc;
    Product p;
    if (int rc = score_product(s, o, cols, &p)) return rc;
    const int groups = p.plan.bn >= 128 ? 2 : 1;
    // the last tile may have no chunk for the second group
    const long long tiles = (cols + p.plan.bn - 1) / p.plan.bn;
    const bool short_last = groups == 2 && cols - (tiles - 1) * p.plan.bn <= 32;
    ScoreArgs a{};
    a.bias = bias ? bias + col0 : nullptr;
    a.bias_vec = bias && aligned16(bias);
    a.targets = targets;
    a.col0 = (int)col0;
    a.target_score = scratch.target_score;
    a.partial = scratch.partial + (long long)parts * s.rows;
    if (int rc = launch_product<LseProblem>("linear_cce_lse", p, [&](auto& g) { g.s = a; }, st)) return rc;
    parts += (int)(tiles * groups) - (short_last ? 1 : 0);
  }
  const int blocks = (int)((s.rows + 31) / 32);
  int few = 1;
  while (few < 32 && few < s.rows) few *= 2;
  launch_chained(join_lse_kernel, blocks, 32 * kJoin, 0, st, scratch.partial, parts, scratch.target_score, targets,
                 d->ignore_index, s.classes, (int)s.rows, d->reduction, lse, loss, count_out, bad_target_flag,
                 scratch.sums, few);
  FLB200_AFTER_LAUNCH("linear_cce_join");
  if (blocks == 1) return FLB200_OK;
  launch_chained(finish_loss_kernel, 1, 32, 0, st, scratch.sums, blocks, d->reduction, loss, count_out,
                 bad_target_flag);
  FLB200_AFTER_LAUNCH("linear_cce_loss");
  return FLB200_OK;
}

int flb200_linear_cce_backward(const flb200_linear_cce_desc* d, const void* x, const void* w, const float* bias,
                               const float* lse, const float* grad_loss, const int32_t* targets,
                               const int32_t* count, void* grad_x, void* grad_w, int grad_w_dtype, float* grad_bias,
                               void* workspace, size_t workspace_bytes, void* stream) {
  // (G lies at multiples of 256 bytes in it, and is stored 32 bytes at a time)
  if (reinterpret_cast<uintptr_t>(workspace) & 31)
    return fail(FLB200_WORKSPACE_TOO_SMALL, "linear_cce_backward: the workspace must be 32-byte aligned");
  if (int rc = check_desc("linear_cce_backward", d)) return rc;
  FLB200_REQUIRE(x && w && lse && grad_loss && targets, "linear_cce_backward: null tensor");
  FLB200_REQUIRE(d->reduction != FLB200_REDUCE_MEAN || count, "linear_cce_backward: MEAN needs count");
  FLB200_REQUIRE(!grad_w || grad_w_dtype == d->dtype || grad_w_dtype == FLB200_F32,
                 "linear_cce_backward: the weights' gradient is of their type or f32");
  const size_t need = flb200_linear_cce_workspace_bytes(d, x, w, 1);
  if (!workspace || workspace_bytes < need)
    return fail(FLB200_WORKSPACE_TOO_SMALL, "linear_cce_backward: workspace %zu < %zu", workspace_bytes, need);
  const cudaStream_t st = as_stream(stream);
  const Shape s = shape_of(d, x, w, true);
  Carve carve{static_cast<char*>(workspace)};
  const BackwardScratch scratch(carve, s, true, true);
  const bool bf16 = d->dtype == FLB200_BF16;
  const bool at_once = s.piece >= s.classes && scratch.dx_splits == 1;  // one product makes dx
  const unsigned row_ctas = d->reduction == FLB200_REDUCE_NONE ? 1u : (unsigned)((s.rows + 1023) / 1024);
  launch_chained(row_weights_kernel, row_ctas, 1024, 0, st, grad_loss, targets, count, lse, d->reduction, d->ignore_index,
                 s.classes, (int)s.rows, bf16 ? 1.f : 32768.f, scratch.rows, scratch.factor);
  FLB200_AFTER_LAUNCH("linear_cce_weights");
  for (long long col0 = 0; col0 < s.classes; col0 += s.piece) {
    const long long cols = std::min(s.piece, s.classes - col0);
    Operands o;
    if (int rc = operands_of(s, x, w, scratch.x, scratch.w, col0, cols, &o, st)) return rc;
    Product p;
    if (int rc = score_product(s, o, cols, &p)) return rc;
    ScoreArgs a{};
    a.bias = bias ? bias + col0 : nullptr;
    a.bias_vec = bias && aligned16(bias);
    a.targets = targets;
    a.col0 = (int)col0;
    a.rows = scratch.rows;
    a.grad = scratch.grad;
    a.grad_ld = s.piece;
    a.column_sum = grad_bias ? scratch.column_sum : nullptr;
    const auto fill = [&](auto& g) { g.s = a; };
    if (int rc = bf16 ? launch_product<GradScoreBf16>("linear_cce_grad", p, fill, st)
                      : launch_product<GradScoreF16>("linear_cce_grad", p, fill, st))
      return rc;
    if (grad_x) {
      Product q;
      q.M = s.rows; q.N = s.dim; q.K = cols;
      q.operand = s.operand;
      q.n_fast = 1;  // (G once from memory: 4096 x 768 of 16384 columns read 295 MB without)
      q.plan = plan_dx(s, std::min(s.piece, s.classes));
      // (a last, short piece may have fewer splits: it adds to the sums of the first of them)
      q.plan.splits = fit_splits(cols, scratch.dx_splits, &q.plan.iters_per_split);
      if (int rc = matrix_operand(false, s.piece, scratch.grad, s.rows, cols, kBM, s.operand, &q.ma, &q.pa)) return rc;
      if (int rc = matrix_operand(false, s.w_ld, o.w, s.dim, cols, q.plan.b_box_rows(), s.operand, &q.mb, &q.pb))
        return rc;
      const bool vec = s.dim % 4 == 0;
      const auto sums = [&](auto& g) { g.set(scratch.dx, s.dim, s.rows * s.dim, nullptr, vec); };
      const auto result = [&](auto& g) { g.set(grad_x, s.dim, 0, scratch.factor, vec && aligned16(grad_x)); };
      if (int rc = at_once    ? (bf16 ? launch_product<Result16<__nv_bfloat16>::Of>("linear_cce_dx", q, result, st)
                                      : launch_product<Result16<__half>::Of>("linear_cce_dx", q, result, st))
                   : col0 == 0 ? launch_product<SumFirst>("linear_cce_dx", q, sums, st)
                               : launch_product<SumNext>("linear_cce_dx", q, sums, st))
        return rc;
    }
    if (grad_w) {
      Product q;
      q.M = s.dim; q.N = cols; q.K = s.rows;
      q.operand = s.operand;
      q.plan = plan_product(q.M, q.N, q.K, true, true, s.operand, false);
      if (int rc = matrix_operand(true, s.x_ld, o.x, s.dim, s.rows, kBM, s.operand, &q.ma, &q.pa)) return rc;
      if (int rc = matrix_operand(true, s.piece, scratch.grad, cols, s.rows, q.plan.b_box_rows(), s.operand, &q.mb,
                                  &q.pb))
        return rc;
      const long long bytes = grad_w_dtype == FLB200_F32 ? 4 : 2;
      const auto result = [&](auto& g) {
        g.set(static_cast<char*>(grad_w) + col0 * bytes, s.classes, 0, scratch.factor,
              s.classes % 4 == 0 && aligned16(grad_w));
      };
      if (int rc = grad_w_dtype == FLB200_F32
                       ? launch_product<SumFirst>("linear_cce_dw", q, result, st)
                       : (bf16 ? launch_product<Result16<__nv_bfloat16>::Of>("linear_cce_dw", q, result, st)
                               : launch_product<Result16<__half>::Of>("linear_cce_dw", q, result, st)))
        return rc;
    }
    if (grad_bias) {
      launch_chained(finish_columns_kernel, (unsigned)((cols + 31) / 32), 256, 0, st, scratch.column_sum,
                     (int)((s.rows + 31) / 32), s.piece, (int)cols, scratch.factor, grad_bias + col0);
      FLB200_AFTER_LAUNCH("linear_cce_dbias");
    }
  }
  if (grad_x && !at_once) {
    const long long n = s.rows * s.dim;
    const int vec = n % 4 == 0 && aligned16(grad_x);
    if (bf16)
      launch_chained(finish_sums_kernel<__nv_bfloat16>, grid_for(n, 1024), 256, 0, st, scratch.dx, scratch.dx_splits, n,
                     scratch.factor, static_cast<__nv_bfloat16*>(grad_x), vec);
    else
      launch_chained(finish_sums_kernel<__half>, grid_for(n, 1024), 256, 0, st, scratch.dx, scratch.dx_splits, n,
                     scratch.factor, static_cast<__half*>(grad_x), vec);
    FLB200_AFTER_LAUNCH("linear_cce_dx_sum");
  }
  return FLB200_OK;
}

}  // extern "C"
