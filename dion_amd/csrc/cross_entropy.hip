// Cross entropy of rows of logits over the vocabulary, and its gradient.
//
//   z = cap tanh(x / cap)  (z = x without a cap),   lse = log sum_v exp z_v,   loss = lse - z_target + zl lse^2
//   dloss/dx_v = (p_v (1 + 2 zl lse) - [v = target]) (1 - (z_v / cap)^2),   p_v = exp(z_v - lse)
//
// Rows whose target is the ignored one have no loss and a gradient of zero, and their logits are not read; any other target
// outside the vocabulary gives NaN.  The sum runs beside its maximum, so that one pass over a row is enough; both are fp32, the
// gradient is rounded once.  All of it is bound by HBM: a read of the logits, and a write of their gradient.
#include "../../include/dion_amd.h"
#include "model_ops.h"
#include "prof.h"
#include <algorithm>

namespace {

constexpr float QUIET_NAN = __builtin_nanf("");
constexpr float LOG2E = 1.44269504088896340736f;
// How a kernel takes the logits' cap.
enum Cap : int {
  NONE,    // z = x
  SMALL,   // bf16 logits and at most SMALL_CAP: z by a reciprocal alone, and no maximum
  WIDE,    // any other cap: z as exact as x
};
// Up to this cap no maximum is looked for in bf16 logits: they lie between -cap and cap, and the sum of exp(z - cap), at least
// exp(-80), serves like that of exp(z - maximum).
constexpr float SMALL_CAP = 40.f;
constexpr float NO_MAX = -__builtin_inff();
constexpr int COUNT_BLOCKS = 64;   // partial counts of the rows that count: one a lane where they are added up
constexpr int SLICES = 64;         // slices of a row at most: one a lane where their sums are joined

struct CeArgs {
  const void* x;
  long long ld, rows;
  int vocab;
  DaIndex targets;
  long long ignore;
  float cap, inv_cap, exp_scale, z_loss;   // exp_scale: 2 log2(e) / cap
  int reduction;        // DION_AMD_REDUCE_*
  const float* counts;  // [COUNT_BLOCKS] partial counts, for the mean; null: a workgroup counts the rows by itself
  float* losses;        // [rows]
  float* lse;           // [rows + 1], or null: the last is the number of rows that count
  // rows in slices
  int slices, slice;    // number of slices, elements of one (a multiple of the vectors')
  int parts;            // number of slices that the statistics were taken in
  float2* partial;      // [rows][parts] maximum and sum of every slice
  float* target_logit;  // [rows]: kept for the launch behind, which may write the gradient over it
  // gradient
  const float* known_lse;   // [rows]: the rows' normalisers, if they have been left before
  const float* known_count; // the number of rows that count, likewise
  const float* dloss;   // upstream gradient: one, or one a row (no reduction); null: scale alone
  float scale;
  void* dx;
  long long ldd;
};

__device__ __forceinline__ float fast_exp(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }

// z = cap tanh(x / cap), or z = x, and the derivative dz/dx.
//
// With r = 1 / (1 + exp(2 u)), u = x / cap: tanh u = 1 - 2 r and 1 - tanh^2 u = 4 r (1 - r).  That z is off by up to some 2^-22 of the
// cap, however small it is itself, since the terms are of the cap's size.  A SMALL cap leaves it at that, 1e-5 at the most, and
// exp(z - ref) is then one multiply-add and one exponential of r: of 2048 rows of bf16 logits of deviation 2 the losses are 8.8e-7,
// 1.7e-6 and 2.4e-6 off in the root mean square with caps of 15, 30 and 40, and 4.5e-7 if they are taken as WIDE, which costs half as much
// again where the arithmetic bounds a kernel (8192 rows of 50304 classes with the gradient 380 and 560 us).  WIDE caps and fp32
// logits take the series of the tangent up to u^11 where |u| < 0.3, off by a few 2^-24 of z itself whatever the cap, and subtract before
// they scale.
template <Cap CAP>
struct Capped {
  float r = 0.f, z = 0.f, slope = 1.f;   // of a SMALL cap r alone, unless z or the slope is asked for
  __device__ __forceinline__ Capped(const CeArgs& a, float x) {
    if (CAP == NONE) {
      z = x;
      return;
    }
    r = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * a.exp_scale));
    z = fmaf(-2.f * a.cap, r, a.cap);
    slope = 4.f * fmaf(-r, r, r);
    if (CAP == WIDE) {
      const float u = x * a.inv_cap, q = u * u;
      float p = fmaf(q, -1382.f / 155925.f, 62.f / 2835.f);
      p = fmaf(q, p, -17.f / 315.f);
      p = fmaf(q, p, 2.f / 15.f);
      p = fmaf(q, p, -1.f / 3.f);
      p = fmaf(u * q, p, u);
      if (fabsf(u) < 0.3f) {
        z = a.cap * p;
        slope = fmaf(-p, p, 1.f);
      }
    }
  }
};
template <Cap CAP>
__device__ __forceinline__ float capped(const CeArgs& a, float x) { return Capped<CAP>(a, x).z; }

// exp(z - ref), ref fixed for a row.
template <Cap CAP>
struct Exponential {
  float ref, shift, scale;
  __device__ __forceinline__ Exponential(const CeArgs& a, float ref) : ref(ref), shift((a.cap - ref) * LOG2E), scale(-2.f * LOG2E * a.cap) {}
  __device__ __forceinline__ float operator()(const Capped<CAP>& c) const {
    if (CAP == SMALL) return __builtin_amdgcn_exp2f(fmaf(scale, c.r, shift));
    return fast_exp(c.z - ref);
  }
};

// Maxima and the sums of exp(z - maximum) that belong to them.  A maximum of -inf (nothing but masked classes so far) is never
// subtracted: exp would see -inf - -inf.
__device__ __forceinline__ float reference(float m) { return m == NO_MAX ? 0.f : m; }

// Joins those of the lanes of a wavefront.
__device__ __forceinline__ void wave_join(float& m, float& s, int log2_group = 6) {
  const float all = da_group_max(m, log2_group);
  s = da_group_sum(s * fast_exp(m - reference(all)), log2_group);
  m = all;
}

// Joins those of the threads of a workgroup, and adds up n.
template <int THREADS>
__device__ __forceinline__ void block_join(float& m, float& s, float& n) {
  wave_join(m, s);
  n = da_group_sum(n);
  if constexpr (THREADS > DA_WAVE) {
    constexpr int WAVES = THREADS / DA_WAVE, LOG2 = WAVES == 4 ? 2 : 4;
    static_assert(WAVES == 4 || WAVES == 16);
    __shared__ float part[3][WAVES];
    const int wave = threadIdx.x / DA_WAVE, lane = threadIdx.x % DA_WAVE;
    if (lane == 0) { part[0][wave] = m; part[1][wave] = s; part[2][wave] = n; }
    __syncthreads();
    m = part[0][lane % WAVES];
    s = part[1][lane % WAVES];
    n = part[2][lane % WAVES];
    wave_join(m, s, LOG2);
    n = da_group_sum(n, LOG2);
  }
}

// Rows that are not ignored, as partial counts.  (There are fewer rows than 2^24: fp32 holds their numbers exactly.)
__global__ __launch_bounds__(256) void ce_count_kernel(DaIndex targets, long long rows, long long ignore, float* counts) {
  __shared__ float part[4];
  float n = 0.f;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows; i += (long long)gridDim.x * 256)
    n += da_index(targets, i) != ignore ? 1.f : 0.f;
  n = da_group_sum(n);
  if (threadIdx.x % DA_WAVE == 0) part[threadIdx.x / DA_WAVE] = n;
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// A thread's share of the rows that count, which a gradient of the mean needs: to be summed over a wavefront where there are partial
// counts, else over `threads` threads.
__device__ __forceinline__ float count_share(const CeArgs& a, int threads) {
  if (a.reduction != DION_AMD_REDUCE_MEAN || !a.dx) return 0.f;
  if (a.counts) return a.counts[threadIdx.x % DA_WAVE];
  float n = 0.f;
  for (int i = threadIdx.x % threads; i < a.rows; i += threads) n += da_index(a.targets, i) != a.ignore ? 1.f : 0.f;
  return n;
}

__device__ __forceinline__ float row_loss(const CeArgs& a, float lse, float zt, bool known) {
  return known ? fmaf(a.z_loss * lse, lse, lse - zt) : QUIET_NAN;
}

// Factors of a row's gradient: dx = (wp exp(z - lse) - w [target]) dz/dx.
struct Weights {
  float w, wp;
};
__device__ __forceinline__ Weights weights(const CeArgs& a, long long row, float lse, bool known, float count) {
  float w = a.scale;
  if (a.dloss) w *= a.dloss[a.reduction == DION_AMD_REDUCE_NONE ? row : 0];
  if (a.reduction == DION_AMD_REDUCE_MEAN) w /= count;
  if (!known) w = QUIET_NAN;
  return {w, w * fmaf(2.f * a.z_loss, lse, 1.f)};
}

// Gradient of N classes from `first` on, in place of their logits.
template <Cap CAP, int N>
__device__ __forceinline__ void gradient(const CeArgs& a, float (&x)[N], int first, long long target, const Exponential<CAP>& e, Weights g) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Capped<CAP> c(a, x[i]);
    float d = g.wp * e(c);
    if ((unsigned long long)(target - first) < N && first + i == target) d -= g.w;
    x[i] = CAP == NONE ? d : d * c.slope;
  }
}

// ---- a row in the registers of one workgroup: loss and gradient from one read
//
// A thread holds up to VECS vectors of 16 bytes of the row (24 at the most: 113 registers, 119 with a wide cap), and one element of its
// end where that is no whole vector.  The maximum and the sum are each thread's own until the one exchange between the wavefronts.
//
// 16384 rows of 50304 bf16 classes, a tenth of them ignored: 550-580 us for 2.92 GiB (5.4-5.7 TB/s; read twice, 2000 with the plain
// two passes).  19 cycles a lane and element without a cap; a small one in bf16 takes 36 and a wide one half as many again, where the
// arithmetic bounds it (8192 rows of 50304 classes 390 and 560 us: 4.2 and 3.0 TB/s).  Two workgroups a compute unit take turns at memory and arithmetic; rows of more than 8192 vectors leave room for one (4.0 TB/s with 18992
// vectors: 2048 rows of 151936 bf16 classes in 312 us, 383 if they are read twice).
template <typename T, Cap CAP, int THREADS, int VECS>
__global__ __launch_bounds__(THREADS) void ce_row_kernel(CeArgs a) {
  constexpr int N = 16 / sizeof(T);
  const long long row = blockIdx.x;
  const long long target = da_index(a.targets, row);
  const T* x = static_cast<const T*>(a.x) + row * a.ld;
  T* dx = static_cast<T*>(a.dx) + row * a.ldd;
  const int vecs = a.vocab / N, rest = a.vocab - vecs * N, end = vecs * N + (int)threadIdx.x;
  if (target == a.ignore) {
    const float zero[N] = {};
    if (a.dx) {
      for (int v = threadIdx.x; v < vecs; v += THREADS) da_store(dx + v * N, 0, zero);
      if ((int)threadIdx.x < rest) st_from_float(dx + end, 0.f);
    }
    if (threadIdx.x == 0) {
      a.losses[row] = 0.f;
      if (a.lse) a.lse[row] = 0.f;
    }
    return;
  }
  const bool known = target >= 0 && target < a.vocab;
  DaVec<T, N> raw[VECS];
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    const int v = j * THREADS + (int)threadIdx.x;
    if (vecs) raw[j].raw = *reinterpret_cast<const typename DaVec<T, N>::raw_t*>(x + (v < vecs ? v : 0) * N);
  }
  const bool ends = (int)threadIdx.x < rest;
  const float last = ends ? ld_as_float(x + end) : NO_MAX;
  const float xt = ld_as_float(x + (known ? target : 0));
  const float share = count_share(a, THREADS);

  float m = a.cap;
  if (CAP != SMALL) {
    m = last;
    if (vecs) {
#pragma unroll
      for (int j = 0; j < VECS; ++j) {   // (a vector in place of one behind the row's end changes no maximum)
        float z[N];
        raw[j].get(z);
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, z[i]);
      }
    }
    m = capped<CAP>(a, m);   // (it rises with its argument)
  }
  const Exponential<CAP> from_max(a, reference(m));
  float s = ends ? from_max({a, last}) : 0.f;
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    if (j * THREADS + (int)threadIdx.x < vecs) {
      float z[N];
      raw[j].get(z);
#pragma unroll
      for (int i = 0; i < N; ++i) s += from_max({a, z[i]});
    }
  }
  float count = a.counts ? 0.f : share;
  block_join<THREADS>(m, s, count);
  if (a.counts) count = da_group_sum(share);
  const float lse = m + logf(s);
  if (threadIdx.x == 0) {
    a.losses[row] = row_loss(a, lse, capped<CAP>(a, xt), known);
    if (a.lse) a.lse[row] = lse;
  }
  if (!a.dx) return;
  const Weights g = weights(a, row, lse, known, count);
  const Exponential<CAP> from_lse(a, lse);
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    const int v = j * THREADS + (int)threadIdx.x;
    if (v < vecs) {
      float z[N];
      raw[j].get(z);
      gradient<CAP>(a, z, v * N, target, from_lse, g);
      da_store(dx + v * N, 0, z);
    }
  }
  if (ends) {
    float z[1] = {last};
    gradient<CAP>(a, z, end, target, from_lse, g);
    st_from_float(dx + end, z[0]);
  }
}

// ---- rows in slices: the loss alone, rows too long for the registers, and few rows that have to share the chip
//
// Statistics: a thread requests its next four vectors before it works on four.  2047 rows of 50257 bf16 classes with a cap, 206 MB in
// 46-50 us (with 256 threads in place of 1024, and without the request ahead, 43-57); 8192 of 50304 without one 134 us (6.1
// TB/s).  16 rows of 128000 fp32 classes in 7 slices: 4.6 us and 2.2 for the join, from one workgroup a row 73.
constexpr int SLICE_THREADS = 1024, SLICE_VECS = 4;

// Maximum and sum of one slice of a row; of a row in one slice also its loss.
template <typename T, Cap CAP>
__global__ __launch_bounds__(SLICE_THREADS) void ce_slice_kernel(CeArgs a) {
  constexpr int N = 16 / sizeof(T);
  const long long row = blockIdx.x / a.slices;
  const int slice = blockIdx.x % a.slices;
  const long long target = da_index(a.targets, row);
  if (target == a.ignore) {
    if (threadIdx.x == 0 && slice == 0) {
      a.losses[row] = 0.f;
      if (a.lse) a.lse[row] = 0.f;
    }
    return;
  }
  const T* x = static_cast<const T*>(a.x) + row * a.ld;
  const int begin = slice * a.slice, end = slice + 1 < a.slices ? begin + a.slice : a.vocab;
  const int vecs = (end - begin) / N;
  float top = NO_MAX, m = CAP == SMALL ? a.cap : capped<CAP>(a, top), s = 0.f;   // top: before the cap
  constexpr int STEP = SLICE_THREADS * SLICE_VECS;
  DaVec<T, N> next[SLICE_VECS];
  auto request = [&](int base) {
#pragma unroll
    for (int j = 0; j < SLICE_VECS; ++j) {
      const int v = base + j * SLICE_THREADS + (int)threadIdx.x;
      next[j].raw = *reinterpret_cast<const typename DaVec<T, N>::raw_t*>(x + begin + (v < vecs ? v : 0) * N);
    }
  };
  if (vecs) request(0);
  for (int base = 0; base < vecs; base += STEP) {
    DaVec<T, N> here[SLICE_VECS];
#pragma unroll
    for (int j = 0; j < SLICE_VECS; ++j) here[j] = next[j];
    if (base + STEP < vecs) request(base + STEP);
    float z[SLICE_VECS][N];
#pragma unroll
    for (int j = 0; j < SLICE_VECS; ++j) here[j].get(z[j]);
    if (CAP != SMALL) {
#pragma unroll
      for (int j = 0; j < SLICE_VECS; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, z[j][i]);   // (a repeated vector changes no maximum)
      const float nm = capped<CAP>(a, top);
      s *= fast_exp(m - reference(nm));
      m = nm;
    }
    const Exponential<CAP> from_max(a, reference(m));
#pragma unroll
    for (int j = 0; j < SLICE_VECS; ++j) {
      if (base + j * SLICE_THREADS + (int)threadIdx.x < vecs) {
#pragma unroll
        for (int i = 0; i < N; ++i) s += from_max({a, z[j][i]});
      }
    }
  }
  if (vecs * N + (int)threadIdx.x < end - begin) {
    const float z = capped<CAP>(a, ld_as_float(x + begin + vecs * N + threadIdx.x)), nm = fmaxf(m, z);
    s = s * fast_exp(m - reference(nm)) + fast_exp(z - reference(nm));
    m = nm;
  }
  float none = 0.f;
  block_join<SLICE_THREADS>(m, s, none);
  if (threadIdx.x) return;
  const bool known = target >= 0 && target < a.vocab;
  const float zt = capped<CAP>(a, ld_as_float(x + (known ? target : 0)));
  if (a.slices > 1) {
    a.partial[row * a.slices + slice] = make_float2(m, s);
    if (slice == 0) a.target_logit[row] = zt;
    return;
  }
  const float lse = m + logf(s);
  a.losses[row] = row_loss(a, lse, zt, known);
  if (a.lse) a.lse[row] = lse;
}

// The normaliser of a row from its slices' sums, by one wavefront.
__device__ __forceinline__ float joined_lse(const CeArgs& a, long long row) {
  const int lane = threadIdx.x % DA_WAVE;
  float m = NO_MAX, s = 0.f;
  if (lane < a.parts) {
    const float2 p = a.partial[row * a.parts + lane];
    m = p.x;
    s = p.y;
  }
  wave_join(m, s);
  return m + logf(s);
}

// Loss of the rows in slices, where no gradient does it: a wavefront a row.
__global__ __launch_bounds__(256) void ce_finish_kernel(CeArgs a) {
  const long long row = (long long)blockIdx.x * 4 + threadIdx.x / DA_WAVE;
  if (row >= a.rows) return;
  const long long target = da_index(a.targets, row);
  if (target == a.ignore) return;
  const float lse = joined_lse(a, row);
  if (threadIdx.x % DA_WAVE) return;
  a.losses[row] = row_loss(a, lse, a.target_logit[row], target >= 0 && target < a.vocab);
  if (a.lse) a.lse[row] = lse;
}

constexpr int GRAD_THREADS = 256, GRAD_VECS = 4;

// Gradient of one slice of a row, from the normaliser of an earlier call or from the slices' sums.  A thread has all its vectors under
// way at once, and a compute unit four workgroups at different points of their work: 8192 rows of 50304 bf16 classes 286 us (5.8 TB/s),
// with a cap 296; in slices of twice as many vectors, half of them at a time, 303 and 332, half of them ahead 314 and 319, all of
// them at once 306 and 309; 512 threads 295 and 292.
template <typename T, Cap CAP>
__global__ __launch_bounds__(GRAD_THREADS) void ce_grad_kernel(CeArgs a) {
  constexpr int N = 16 / sizeof(T);
  const long long row = blockIdx.x / a.slices;
  const int slice = blockIdx.x % a.slices;
  const long long target = da_index(a.targets, row);
  const int begin = slice * a.slice, end = slice + 1 < a.slices ? begin + a.slice : a.vocab;
  const int vecs = (end - begin) / N, tail = vecs * N + (int)threadIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ld + begin;
  T* dx = static_cast<T*>(a.dx) + row * a.ldd + begin;
  const bool ignored = target == a.ignore, known = target >= 0 && target < a.vocab, ends = tail < end - begin;
  DaVec<T, N> raw[GRAD_VECS] = {};
  float last[1] = {0.f};
  float lse = 0.f;
  Weights g{0.f, 0.f};
  if (!ignored) {
#pragma unroll
    for (int j = 0; j < GRAD_VECS; ++j) {
      const int v = j * GRAD_THREADS + (int)threadIdx.x;
      if (v < vecs) raw[j].raw = *reinterpret_cast<const typename DaVec<T, N>::raw_t*>(x + v * N);
    }
    if (ends) last[0] = ld_as_float(x + tail);
    lse = a.known_lse ? a.known_lse[row] : joined_lse(a, row);
    const float count = a.known_count ? *a.known_count : da_group_sum(count_share(a, DA_WAVE));   // (by every wavefront)
    g = weights(a, row, lse, known, count);
    if (!a.known_lse && slice == 0 && threadIdx.x == 0) {
      a.losses[row] = row_loss(a, lse, a.target_logit[row], known);
      if (a.lse) a.lse[row] = lse;
    }
  }
  const Exponential<CAP> from_lse(a, lse);
#pragma unroll
  for (int j = 0; j < GRAD_VECS; ++j) {
    const int v = j * GRAD_THREADS + (int)threadIdx.x;
    if (v >= vecs) break;
    float z[N];
    raw[j].get(z);
    if (!ignored) gradient<CAP>(a, z, begin + v * N, target, from_lse, g);
    da_store(dx + v * N, 0, z);
  }
  if (ends) {
    if (!ignored) gradient<CAP>(a, last, begin + tail, target, from_lse, g);
    st_from_float(dx + tail, last[0]);
  }
}

// Sum or mean of the rows' losses: one workgroup, in a fixed order, in fp64.
__global__ __launch_bounds__(1024) void ce_sum_kernel(CeArgs a, float* out) {
  __shared__ double part[16];
  __shared__ int counts[16];
  double sum = 0.0;
  int n = 0;
  constexpr int AHEAD = 8;
  for (long long base = threadIdx.x; base < a.rows; base += 1024 * AHEAD) {
    long long at[AHEAD], t[AHEAD];
    float l[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      at[i] = base + 1024 * i < a.rows ? base + 1024 * i : base;
      l[i] = a.losses[at[i]];
    }
    da_indices(a.targets, at, t);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (base + 1024 * i >= a.rows) break;
      sum += (double)l[i];
      n += t[i] != a.ignore;
    }
  }
  for (int d = DA_WAVE / 2; d > 0; d >>= 1) {
    sum += __shfl_xor(sum, d);
    n += __shfl_xor(n, d);
  }
  if (threadIdx.x % DA_WAVE == 0) {
    part[threadIdx.x / DA_WAVE] = sum;
    counts[threadIdx.x / DA_WAVE] = n;
  }
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) {
    sum += part[w];
    n += counts[w];
  }
  *out = (float)(a.reduction == DION_AMD_REDUCE_MEAN ? sum / (double)n : sum);
  if (a.lse) a.lse[a.rows] = (float)n;
}

// ---- host

constexpr long long MAX_VOCAB = 0x7fffffffll - 65536;
constexpr long long MAX_ROWS = 1ll << 22;   // a launch has fewer than 2^32 threads

// How the rows of a call are taken.
struct Form {
  int threads, vecs;   // of ce_row_kernel, 0: in slices
  int slices, slice;   // number of slices of a row and elements of one
};

// `slices` equal ones, whole vectors but for the row's end.
void cut(Form& f, long long vocab, int n, int slices) {
  const long long vecs = vocab / n, per = (vecs + slices - 1) / slices;
  f.slices = per ? (int)((vecs + per - 1) / per) : 1;
  f.slice = (int)(f.slices > 1 ? per * n : vocab);
}

// Few rows are cut into slices of 2048 vectors or more, as many as give every compute unit a workgroup; without a gradient of 4096,
// since a row in one slice needs no launch to join it (100 rows of 50304 bf16 classes 12.5 us, 14.7 with 2048 and 15.9 with two
// workgroups a compute unit; 400 rows 22.6, 22.6 and 26.3; with the gradient 64 rows 17.5, 16.8 and 17.4).
// Without a gradient, rows of up to 2048 vectors go to the workgroups of 256 threads that hold them: 20000 rows of 10000 bf16 classes
// 73 us (5.5 TB/s), in workgroups of 1024 147; of 16384 classes 115 and 158; of 32000, held by 1024, 213 and 217, but 8192 of 50304 138
// and 134 (all with the sum behind).  With one, rows
// are in slices if they are a quarter of the compute units or fewer: 64 rows of 50304 bf16 classes 17 us either way, 100 18.4 in
// registers and 21 in slices.
Form plan_form(long long rows, long long vocab, int dtype, bool grad) {
  const int n = dtype == DA_BF16 ? 8 : 4;
  const long long vecs = vocab / n, cus = da_cu_count();
  Form f{};
  cut(f, vocab, n, (int)std::max(1ll, std::min({cus / std::max(1ll, rows), (long long)SLICES, vecs / (grad ? 2048 : 4096)})));
  if (!grad && (vecs > 256 * 8 || f.slices > 1)) return f;   // (without a gradient there is nothing to hold a long row for)
  if (vecs > 24 * 1024 || (rows * 4 <= cus && vecs >= 4096)) return f;
  f.threads = vecs <= 64 * 8 ? 64 : vecs <= 256 * 8 ? 256 : 1024;
  f.vecs = (int)((vecs + f.threads - 1) / f.threads);
  return f;
}

struct Plan {
  size_t losses, lse, target_logit, partial, bytes;   // offsets; the counts come first
};
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
Plan plan(long long rows, long long vocab, int dtype) {
  const Form f = plan_form(rows, vocab, dtype, true);   // (without a gradient there are no more slices)
  Plan p{};
  p.losses = COUNT_BLOCKS * sizeof(float);
  p.lse = p.losses + round256((size_t)rows * sizeof(float));
  p.target_logit = p.lse + round256(((size_t)rows + 1) * sizeof(float));
  p.partial = p.target_logit + round256((size_t)rows * sizeof(float));
  p.bytes = p.partial + round256(f.slices > 1 ? (size_t)rows * f.slices * sizeof(float2) : 0) + 256;
  return p;
}

int check_args(const void* logits, int dtype, long long ld, const void* targets, int index_bits, long long rows, long long vocab,
               float softcap, int reduction) {
  if (rows < 0 || vocab <= 0 || ld < vocab || (index_bits != 32 && index_bits != 64)) return DA_ERR_ARG;
  if (softcap != 0.f && !(softcap >= 1e-30f && softcap <= 1e30f)) return DA_ERR_ARG;   // (its reciprocal is needed)
  if (reduction != DION_AMD_REDUCE_NONE && reduction != DION_AMD_REDUCE_SUM && reduction != DION_AMD_REDUCE_MEAN) return DA_ERR_ARG;
  if (!da_float_dtype(dtype)) return DA_ERR_DTYPE;
  if (rows >= MAX_ROWS || vocab > MAX_VOCAB) return DA_ERR_LIMIT;
  if (rows && (!logits || !targets)) return DA_ERR_ARG;
  if (!da_aligned(logits, da_esize(dtype)) || !da_aligned(targets, index_bits / 8)) return DA_ERR_ALIGN;
  return DA_OK;
}

// More rows than a workgroup of the others counts in passing.
constexpr long long COUNT_FROM = 256;

void launch_count(CeArgs& a, float* counts, hipStream_t s) {
  if (a.reduction != DION_AMD_REDUCE_MEAN || a.rows <= COUNT_FROM) return;
  a.counts = counts;
  hipLaunchKernelGGL(ce_count_kernel, dim3(COUNT_BLOCKS), dim3(256), 0, s, a.targets, a.rows, a.ignore, counts);
}

#define DA_CE(LAUNCH)                                                                                                        \
  do {                                                                                                                       \
    if (dtype == DA_BF16 && a.cap > SMALL_CAP) LAUNCH(bf16_t, WIDE);                                                         \
    else if (dtype == DA_BF16 && a.cap > 0.f) LAUNCH(bf16_t, SMALL);                                                         \
    else if (dtype == DA_BF16) LAUNCH(bf16_t, NONE);                                                                         \
    else if (a.cap > 0.f) LAUNCH(float, WIDE);                                                                               \
    else LAUNCH(float, NONE);                                                                                                \
  } while (0)
#define DA_CE_SLICES(kernel, threads) hipLaunchKernelGGL(kernel, dim3((unsigned)(a.rows * a.slices)), dim3(threads), 0, s, a)
#define DA_CE_STATS(T, CAP) DA_CE_SLICES((ce_slice_kernel<T, CAP>), SLICE_THREADS)
#define DA_CE_GRAD(T, CAP) DA_CE_SLICES((ce_grad_kernel<T, CAP>), GRAD_THREADS)
#define DA_CE_ROW_OF(T, CAP, THREADS, VECS)                                                                                  \
  hipLaunchKernelGGL((ce_row_kernel<T, CAP, THREADS, VECS>), dim3((unsigned)a.rows), dim3(THREADS), 0, s, a)
#define DA_CE_ROW(T, CAP)                                                                                                    \
  do {                                                                                                                       \
    if (f.threads == 64) {                                                                                                   \
      if (f.vecs <= 2) DA_CE_ROW_OF(T, CAP, 64, 2);                                                                          \
      else if (f.vecs <= 4) DA_CE_ROW_OF(T, CAP, 64, 4);                                                                     \
      else DA_CE_ROW_OF(T, CAP, 64, 8);                                                                                      \
    } else if (f.threads == 256) {                                                                                           \
      if (f.vecs <= 4) DA_CE_ROW_OF(T, CAP, 256, 4);                                                                         \
      else DA_CE_ROW_OF(T, CAP, 256, 8);                                                                                     \
    } else {                                                                                                                 \
      if (f.vecs <= 4) DA_CE_ROW_OF(T, CAP, 1024, 4);                                                                        \
      else if (f.vecs <= 8) DA_CE_ROW_OF(T, CAP, 1024, 8);                                                                   \
      else if (f.vecs <= 16) DA_CE_ROW_OF(T, CAP, 1024, 16);                                                                 \
      else DA_CE_ROW_OF(T, CAP, 1024, 24);                                                                                   \
    }                                                                                                                        \
  } while (0)

int grad_slices(long long vocab, int dtype) {
  constexpr int MOST = GRAD_THREADS * GRAD_VECS;
  return (int)std::max(1ll, (vocab / (dtype == DA_BF16 ? 8 : 4) + MOST - 1) / MOST);
}

void launch_grad(CeArgs& a, int dtype, const float* lse, hipStream_t s) {
  Form f{};
  cut(f, a.vocab, dtype == DA_BF16 ? 8 : 4, grad_slices(a.vocab, dtype));
  a.slices = f.slices;
  a.slice = f.slice;
  a.known_lse = lse;
  DA_CE(DA_CE_GRAD);
}

constexpr long long MAX_BLOCKS = 1ll << 24;   // of 256 threads

}  // namespace

extern "C" {

size_t dion_amd_cross_entropy_workspace_bytes(long long rows, long long vocab, int dtype) {
  if (rows < 0 || rows >= MAX_ROWS || vocab <= 0 || vocab > MAX_VOCAB || !da_float_dtype(dtype)) return 0;
  return plan(rows, vocab, dtype).bytes;
}

int dion_amd_cross_entropy(const void* logits, int dtype, long long ld, const void* targets, int index_bits, long long rows,
                           long long vocab, long long ignore_index, float softcap, float z_loss, int reduction, float* loss,
                           float* lse, void* dlogits, long long ldd, float grad_scale, void* workspace, size_t workspace_bytes,
                           void* stream) {
  int rc = check_args(logits, dtype, ld, targets, index_bits, rows, vocab, softcap, reduction);
  if (rc) return rc;
  if (!workspace || (!loss && (rows || reduction != DION_AMD_REDUCE_NONE)) || (dlogits && ldd < vocab)) return DA_ERR_ARG;
  if (!da_aligned(loss, 4) || !da_aligned(lse, 4) || !da_aligned(dlogits, da_esize(dtype)) || !da_aligned(workspace, 256)) return DA_ERR_ALIGN;
  const Plan p = plan(rows, vocab, dtype);
  if (workspace_bytes < p.bytes) return DA_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Form f = plan_form(rows, vocab, dtype, dlogits != nullptr);
  if (rows * f.slices >= MAX_BLOCKS || (dlogits && !f.threads && rows * grad_slices(vocab, dtype) >= MAX_BLOCKS)) return DA_ERR_LIMIT;
  CeArgs a{};
  a.x = logits; a.ld = ld; a.rows = rows; a.vocab = (int)vocab;
  a.targets = {targets, index_bits == 64};
  a.ignore = ignore_index;
  a.cap = softcap; a.inv_cap = softcap > 0.f ? 1.f / softcap : 0.f; a.exp_scale = 2.f * LOG2E * a.inv_cap; a.z_loss = z_loss;
  a.reduction = reduction;
  a.losses = reduction == DION_AMD_REDUCE_NONE ? loss : reinterpret_cast<float*>(ws + p.losses);
  a.lse = lse;
  a.slices = a.parts = f.slices; a.slice = f.slice;
  a.partial = reinterpret_cast<float2*>(ws + p.partial);
  a.target_logit = reinterpret_cast<float*>(ws + p.target_logit);
  a.scale = grad_scale;
  a.dx = dlogits; a.ldd = ldd;
  DaProfScope prof(DA_PROF_LOSS, (double)rows * vocab * da_esize(dtype) * (dlogits ? 2 : 1), s);
  if (rows) {
    if (dlogits) launch_count(a, reinterpret_cast<float*>(ws), s);
    if (f.threads) {
      DA_CE(DA_CE_ROW);
    } else {
      if (dlogits && !a.lse) a.lse = reinterpret_cast<float*>(ws + p.lse);
      DA_CE(DA_CE_STATS);
      if (dlogits) launch_grad(a, dtype, f.slices > 1 ? nullptr : a.lse, s);
      else if (f.slices > 1) hipLaunchKernelGGL(ce_finish_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
    }
  }
  if (reduction != DION_AMD_REDUCE_NONE) hipLaunchKernelGGL(ce_sum_kernel, dim3(1), dim3(1024), 0, s, a, loss);
  return da_launch_status();
}

int dion_amd_cross_entropy_grad(const void* logits, int dtype, long long ld, const void* targets, int index_bits, long long rows,
                                long long vocab, long long ignore_index, float softcap, float z_loss, int reduction,
                                const float* lse, const float* dloss, void* dlogits, long long ldd, void* stream) {
  int rc = check_args(logits, dtype, ld, targets, index_bits, rows, vocab, softcap, reduction);
  if (rc) return rc;
  if (rows == 0) return DA_OK;
  if (!lse || !dloss || !dlogits || ldd < vocab) return DA_ERR_ARG;
  if (!da_aligned(lse, 4) || !da_aligned(dloss, 4) || !da_aligned(dlogits, da_esize(dtype))) return DA_ERR_ALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows * grad_slices(vocab, dtype) >= MAX_BLOCKS) return DA_ERR_LIMIT;
  CeArgs a{};
  a.x = logits; a.ld = ld; a.rows = rows; a.vocab = (int)vocab;
  a.targets = {targets, index_bits == 64};
  a.ignore = ignore_index;
  a.cap = softcap; a.inv_cap = softcap > 0.f ? 1.f / softcap : 0.f; a.exp_scale = 2.f * LOG2E * a.inv_cap; a.z_loss = z_loss;
  a.reduction = reduction;
  a.dloss = dloss;
  a.scale = 1.f;
  a.dx = dlogits; a.ldd = ldd;
  DaProfScope prof(DA_PROF_LOSS, 2.0 * rows * vocab * da_esize(dtype), s);
  a.known_count = lse + rows;
  launch_grad(a, dtype, lse, s);
  return da_launch_status();
}

}  // extern "C"
