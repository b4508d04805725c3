// RMS norm of every query and key head with the position rotation in the same pass, and its gradient.
//
//   r = 1 / sqrt(mean_i x_i^2 + eps),   n_i = x_i r w_i,   y = R(pos) n
//
// R turns the pairs of the first `rotary` channels -- (i, i + rotary / 2), or (2i, 2i + 1) if interleaved -- by the angle whose cosine
// and sine are row `pos` of the tables; the other channels pass.  With dn = R^T dy and c = sum_i dn_i w_i x_i / dim:
//
//   dx_i = r (dn_i w_i - x_i r^2 c),            dw_i = sum over rows of dn_i x_i r
//
// One pass over the data each way, bound by HBM; nothing but the inputs is kept for the gradient.  Norms and sums are fp32, the
// result is rounded once.  A position outside the tables gives a row of NaN.
#include "../../include/dion_amd.h"
#include "model_ops.h"
#include "prof.h"
#include <algorithm>

namespace {

constexpr float QUIET_NAN = __builtin_nanf("");
constexpr int MAX_DIM = 1024;

// One of the two tensors, as the kernels see it (strides in elements, last dimension contiguous).
struct Heads {
  const void* x;
  const void* dy;
  void* y;          // result: y, or dx
  const void* gain;
  float* partial;   // gradient: [blocks][dim] sums of the gain's gradient, or null
  long long xb, xt, xh, db, dt, dh, yb, yt, yh;
  int heads;
  int blocks;       // workgroups of this tensor: the queries' come first
  unsigned items;   // tokens * heads
  DaDivisor by_heads;
};

struct QkArgs {
  Heads t[2];       // queries, keys
  long long tokens; // batch * length
  int length, dim, half, interleaved, gain_dtype;
  DaDivisor by_length;
  const float *cos, *sin;
  long long ld_table;
  int table_rows;
  DaIndex positions;   // null: the place in the sequence
  long long pos_batch;
  float eps, inv_dim;
  int turn_lanes, lanes, log2_group;   // lanes with turned pairs, lanes of a head, and of the group that it takes
};

// Where a head is (offsets in elements), and the angles of its token.
struct Place {
  long long x, d, y;
  unsigned b, t;
};
struct Angle {
  long long row;   // offset of its row of the tables
  bool known;
};

__device__ __forceinline__ Place find_head(const QkArgs& a, const Heads& h, unsigned item) {
  const unsigned token = h.by_heads.quotient(item), head = item - token * h.by_heads.by;
  const unsigned b = a.by_length.quotient(token), t = token - b * a.by_length.by;
  return {b * h.xb + t * h.xt + head * h.xh, b * h.db + t * h.dt + head * h.dh, b * h.yb + t * h.yt + head * h.yh, b, t};
}
__device__ __forceinline__ Angle find_angle(const QkArgs& a, const Place& p) {
  const long long pos = a.positions.p ? da_index(a.positions, p.b * a.pos_batch + p.t) : p.t;
  const bool known = a.half == 0 || (pos >= 0 && pos < a.table_rows);
  return {(known ? pos : 0) * a.ld_table, known};
}

__device__ __forceinline__ float gain_at(const QkArgs& a, const void* g, int i) {
  if (!g) return 1.f;
  return a.gain_dtype == DA_BF16 ? bf2f(static_cast<const bf16_t*>(g)[i]) : static_cast<const float*>(g)[i];
}

// ---- heads in vectors
//
// A head is taken by a group of lanes.  A lane holds PAIRS channel pairs: of the turned channels, where one vector of PAIRS channels
// comes from the first half and one from the second (or both side by side, if interleaved); or of the others, which are not turned.
// So a rotation stays inside a lane, and the head's sums take log2(group) steps between neighbouring lanes.  Vectors at the end of a
// range that is no multiple of them are moved back (RAGGED): the sums leave what another lane counts, and the results that two lanes
// hold are the same bits, stored by both (7680 tokens of 40 heads of 80 channels, 40 of them turned, bf16: 23 us and 44 for the
// gradient, 30 and 56 with the shared elements stored one by one by one of them).

// Where this lane's channels are.
template <int PAIRS, bool INTER, bool RAGGED>
struct Lane {
  int first, second;   // first channel of either vector
  int table;           // column of the tables, -1: not turned
  int skip1, skip2;    // elements at the front of the vectors that are another lane's
  bool none;           // a lane without channels reads the group's first, and leaves them
  __device__ __forceinline__ Lane(const QkArgs& a, int lane) : none(RAGGED && lane >= a.lanes) {
    if (none) lane = 0;
    int skip;
    if (lane < a.turn_lanes) {
      const int at = RAGGED ? min(lane * PAIRS, a.half - PAIRS) : lane * PAIRS;
      first = INTER ? 2 * at : at;
      second = INTER ? first + PAIRS : at + a.half;
      table = at;
      skip = lane * PAIRS - at;
      skip1 = INTER ? min(2 * skip, PAIRS) : skip;
      skip2 = INTER ? 2 * skip - skip1 : skip;
    } else {
      const int l = lane - a.turn_lanes, rest = a.dim - 2 * a.half;
      const int at = RAGGED ? min(l * 2 * PAIRS, rest - 2 * PAIRS) : l * 2 * PAIRS;
      first = 2 * a.half + at;
      second = first + PAIRS;
      table = -1;
      skip = l * 2 * PAIRS - at;
      skip1 = min(skip, PAIRS);
      skip2 = skip - skip1;
    }
    if (none) skip1 = skip2 = PAIRS;
  }
};

// The 2 PAIRS channels of a lane as they lie in memory, and as pairs (u, v).
template <typename T, int PAIRS>
struct Raw {
  DaVec<T, PAIRS> x[2];
  template <typename L>
  __device__ __forceinline__ void load(const T* head, const L& at) {
    x[0].raw = *reinterpret_cast<const typename DaVec<T, PAIRS>::raw_t*>(head + at.first);
    x[1].raw = *reinterpret_cast<const typename DaVec<T, PAIRS>::raw_t*>(head + at.second);
  }
  template <bool INTER>
  __device__ __forceinline__ void pairs(float (&u)[PAIRS], float (&v)[PAIRS]) const {
    float e[2][PAIRS];
    x[0].get(e[0]);
    x[1].get(e[1]);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      u[i] = INTER ? e[2 * i / PAIRS][2 * i % PAIRS] : e[0][i];
      v[i] = INTER ? e[2 * i / PAIRS][2 * i % PAIRS + 1] : e[1][i];
    }
  }
};
template <typename T, int PAIRS, bool INTER, typename L>
__device__ __forceinline__ void load_pairs(const T* head, const L& at, float (&u)[PAIRS], float (&v)[PAIRS]) {
  Raw<T, PAIRS> raw;
  raw.load(head, at);
  raw.template pairs<INTER>(u, v);
}
// SHARED: elements that two lanes hold are stored by both, the same bits.
template <bool SHARED, typename T, int PAIRS, bool INTER, typename L>
__device__ __forceinline__ void store_pairs(T* head, const L& at, const float (&u)[PAIRS], const float (&v)[PAIRS]) {
  float x[2][PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    x[INTER ? 2 * i / PAIRS : 0][INTER ? 2 * i % PAIRS : i] = u[i];
    x[INTER ? 2 * i / PAIRS : 1][INTER ? 2 * i % PAIRS + 1 : i] = v[i];
  }
  if (SHARED && at.none) return;
  da_store(head + at.first, SHARED ? 0 : at.skip1, x[0]);
  da_store(head + at.second, SHARED ? 0 : at.skip2, x[1]);
}
// Zero in place of the channels that another lane counts.
template <int PAIRS, bool INTER, typename L>
__device__ __forceinline__ void leave(const L& at, float (&u)[PAIRS], float (&v)[PAIRS]) {
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    const int iu = INTER ? 2 * i : i, iv = INTER ? 2 * i + 1 : i + PAIRS;   // element, over both vectors
    if (iu < PAIRS ? iu < at.skip1 : iu - PAIRS < at.skip2) u[i] = 0.f;
    if (iv < PAIRS ? iv < at.skip1 : iv - PAIRS < at.skip2) v[i] = 0.f;
  }
}
// The squares of a lane's own channels.
template <int PAIRS, bool INTER, bool RAGGED, typename L>
__device__ __forceinline__ float own_square(const L& at, const float (&x)[PAIRS], const float (&y)[PAIRS]) {
  float u[PAIRS], v[PAIRS], sum = 0.f;
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    u[i] = x[i];
    v[i] = y[i];
  }
  if (RAGGED) leave<PAIRS, INTER>(at, u, v);
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) sum = fmaf(u[i], u[i], fmaf(v[i], v[i], sum));
  return sum;
}
// The gain of a lane's channels, as pairs.
template <int PAIRS, bool INTER, typename L>
__device__ __forceinline__ void load_gain(const QkArgs& a, const void* gain, const L& at, float (&u)[PAIRS], float (&v)[PAIRS]) {
  if (gain && a.gain_dtype == DA_BF16) load_pairs<bf16_t, PAIRS, INTER>(static_cast<const bf16_t*>(gain), at, u, v);
  else if (gain) load_pairs<float, PAIRS, INTER>(static_cast<const float*>(gain), at, u, v);
  else
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) u[i] = v[i] = 1.f;
}
// Cosines and sines of a token for a lane's pairs, if they are turned.
template <int PAIRS, typename L>
__device__ __forceinline__ void load_angles(const QkArgs& a, const Angle& angle, const L& at, float (&c)[PAIRS], float (&s)[PAIRS]) {
  if (at.table < 0) return;
  da_load(a.cos + angle.row + at.table, c);
  da_load(a.sin + angle.row + at.table, s);
}
// Pairs turned by their angles, or back.
template <int PAIRS, bool BACK>
__device__ __forceinline__ void turn(float (&u)[PAIRS], float (&v)[PAIRS], const float (&c)[PAIRS], const float (&s)[PAIRS]) {
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    const float sine = BACK ? -s[i] : s[i], x = u[i], y = v[i];
    u[i] = fmaf(x, c[i], -(y * sine));
    v[i] = fmaf(y, c[i], x * sine);
  }
}

// 32768 tokens of 24 heads of 64 channels, bf16, from one projection's output: 41 us for 192 MiB read and written (4.9 TB/s, as a
// large copy).  A lane that takes two or four heads of a token for one set of angles and addresses is no faster.
template <typename T, int PAIRS, bool INTER, bool RAGGED>
__global__ __launch_bounds__(256) void qk_heads_kernel(QkArgs a) {
  const int which = (int)blockIdx.x >= a.t[0].blocks;
  const Heads& h = a.t[which];
  const unsigned block = blockIdx.x - (which ? a.t[0].blocks : 0);
  const unsigned item = (block * 256u + threadIdx.x) >> a.log2_group;
  if (item >= h.items) return;
  const Lane<PAIRS, INTER, RAGGED> at(a, threadIdx.x & ((1 << a.log2_group) - 1));
  const Place p = find_head(a, h, item);
  float u[PAIRS], v[PAIRS], c[PAIRS] = {}, s[PAIRS] = {}, gu[PAIRS], gv[PAIRS];
  load_pairs<T, PAIRS, INTER>(static_cast<const T*>(h.x) + p.x, at, u, v);
  const Angle angle = find_angle(a, p);
  load_angles<PAIRS>(a, angle, at, c, s);
  load_gain<PAIRS, INTER>(a, h.gain, at, gu, gv);
  const float square = own_square<PAIRS, INTER, RAGGED>(at, u, v);
  const float r = angle.known ? rsqrtf(fmaf(da_group_sum(square, a.log2_group), a.inv_dim, a.eps)) : QUIET_NAN;
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    u[i] = u[i] * r * gu[i];
    v[i] = v[i] * r * gv[i];
  }
  if (at.table >= 0) turn<PAIRS, false>(u, v, c, s);
  store_pairs<true, T, PAIRS, INTER>(static_cast<T*>(h.y) + p.y, at, u, v);
}

// The gain's gradient is summed by the lanes over the items of a workgroup, then over its lanes of the same channels, and by the
// kernel behind over the workgroups: an order that depends on the sizes alone.
//
// 16384 tokens of 40 heads of 128 channels, bf16, with gains and positions: 99 us for 491 MiB (5.2 TB/s), and 5 for the last sums.
// Without gains 93, in workgroups that take one head after another 98.
template <typename T, int PAIRS, bool INTER, bool RAGGED, bool GAIN>
__global__ __launch_bounds__(256) void qk_heads_grad_kernel(QkArgs a) {
  const int which = (int)blockIdx.x >= a.t[0].blocks;
  const Heads& h = a.t[which];
  const unsigned block = blockIdx.x - (which ? a.t[0].blocks : 0);
  const Lane<PAIRS, INTER, RAGGED> at(a, threadIdx.x & ((1 << a.log2_group) - 1));
  float gu[PAIRS], gv[PAIRS], du_sum[PAIRS] = {}, dv_sum[PAIRS] = {};
  load_gain<PAIRS, INTER>(a, h.gain, at, gu, gv);
  // with gains, the head behind is requested before this one is worked on; without, a lane has one.  (Its angles are not: they come
  // from the caches, and 16 registers fewer are worth more, 4096 tokens 29.8 us in place of 32.4.)
  struct Item {
    Raw<T, PAIRS> x, d;
    Angle angle;
    long long y;
  };
  auto request = [&](unsigned i, Item& it) {
    const Place p = find_head(a, h, i < h.items ? i : h.items - 1);
    it.x.load(static_cast<const T*>(h.x) + p.x, at);
    it.d.load(static_cast<const T*>(h.dy) + p.d, at);
    it.angle = find_angle(a, p);
    it.y = p.y;
  };
  const unsigned step = (h.blocks * 256u) >> a.log2_group;
  unsigned item = (block * 256u + threadIdx.x) >> a.log2_group;
  Item next;
  request(item, next);
  for (; item < h.items; item += step) {
    const Item it = next;
    float c[PAIRS] = {}, s[PAIRS] = {};
    load_angles<PAIRS>(a, it.angle, at, c, s);
    if (GAIN) request(item + step, next);
    float u[PAIRS], v[PAIRS], du[PAIRS], dv[PAIRS];
    it.x.template pairs<INTER>(u, v);
    it.d.template pairs<INTER>(du, dv);
    if (at.table >= 0) turn<PAIRS, true>(du, dv, c, s);
    float own_u[PAIRS], own_v[PAIRS], wu[PAIRS], wv[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      own_u[i] = u[i];
      own_v[i] = v[i];
      wu[i] = du[i] * gu[i];
      wv[i] = dv[i] * gv[i];
    }
    if (RAGGED) {   // both factors: what another lane counts may be infinite
      leave<PAIRS, INTER>(at, own_u, own_v);
      leave<PAIRS, INTER>(at, wu, wv);
    }
    float square = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      square = fmaf(own_u[i], own_u[i], fmaf(own_v[i], own_v[i], square));
      dot = fmaf(wu[i], own_u[i], fmaf(wv[i], own_v[i], dot));
    }
    square = da_group_sum(square, a.log2_group);
    dot = da_group_sum(dot, a.log2_group);
    const float r = it.angle.known ? rsqrtf(fmaf(square, a.inv_dim, a.eps)) : QUIET_NAN;
    const float m = r * r * (dot * a.inv_dim);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      if (GAIN) {
        du_sum[i] = fmaf(du[i] * own_u[i], r, du_sum[i]);
        dv_sum[i] = fmaf(dv[i] * own_v[i], r, dv_sum[i]);
      }
      u[i] = r * fmaf(-u[i], m, du[i] * gu[i]);
      v[i] = r * fmaf(-v[i], m, dv[i] * gv[i]);
    }
    store_pairs<true, T, PAIRS, INTER>(static_cast<T*>(h.y) + it.y, at, u, v);
    if (!GAIN) return;
  }
  if (!GAIN || !h.partial) return;
  __shared__ float sums[4][2][PAIRS][DA_WAVE];
  const int wave = threadIdx.x / DA_WAVE;
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    for (int d = 1 << a.log2_group; d < DA_WAVE; d <<= 1) {
      du_sum[i] += __shfl_xor(du_sum[i], d);
      dv_sum[i] += __shfl_xor(dv_sum[i], d);
    }
    sums[wave][0][i][threadIdx.x % DA_WAVE] = du_sum[i];
    sums[wave][1][i][threadIdx.x % DA_WAVE] = dv_sum[i];
  }
  __syncthreads();
  if ((int)threadIdx.x >= 1 << a.log2_group) return;
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    du_sum[i] = (sums[0][0][i][threadIdx.x] + sums[1][0][i][threadIdx.x]) + (sums[2][0][i][threadIdx.x] + sums[3][0][i][threadIdx.x]);
    dv_sum[i] = (sums[0][1][i][threadIdx.x] + sums[1][1][i][threadIdx.x]) + (sums[2][1][i][threadIdx.x] + sums[3][1][i][threadIdx.x]);
  }
  store_pairs<false, float, PAIRS, INTER>(h.partial + (long long)block * a.dim, at, du_sum, dv_sum);
}

// ---- heads too narrow for vectors: one wavefront a head, a lane takes whole pairs and then the channels that are not turned
//
// Bound by instructions, an element a load and most lanes idle: 32768 tokens of 32 heads of 24 channels, 12 of them turned, bf16, 267 us
// (0.4 TB/s) and 817 for the gradient (0.2 TB/s); of 12 heads of 64 with 56 turned 108 and 337, where vectors (64 turned) take 18 and 28.
template <typename T>
__global__ __launch_bounds__(256) void qk_narrow_kernel(QkArgs a) {
  const int which = (int)blockIdx.x >= a.t[0].blocks;
  const Heads& h = a.t[which];
  const int lane = threadIdx.x % DA_WAVE;
  const unsigned item = (blockIdx.x - (which ? a.t[0].blocks : 0)) * 4 + threadIdx.x / DA_WAVE;
  if (item >= h.items) return;
  const Place at = find_head(a, h, item);
  const Angle angle = find_angle(a, at);
  const T* x = static_cast<const T*>(h.x) + at.x;
  T* y = static_cast<T*>(h.y) + at.y;
  float sum = 0.f;
  for (int i = lane; i < a.dim; i += DA_WAVE) {
    const float v = ld_as_float(x + i);
    sum = fmaf(v, v, sum);
  }
  const float r = angle.known ? rsqrtf(fmaf(da_group_sum(sum), a.inv_dim, a.eps)) : QUIET_NAN;
  const float* cs = a.cos + angle.row;
  const float* sn = a.sin + angle.row;
  for (int p = lane; p < a.half; p += DA_WAVE) {
    const int i = a.interleaved ? 2 * p : p, j = a.interleaved ? 2 * p + 1 : p + a.half;
    const float u = ld_as_float(x + i) * r * gain_at(a, h.gain, i), v = ld_as_float(x + j) * r * gain_at(a, h.gain, j);
    st_from_float(y + i, fmaf(u, cs[p], -(v * sn[p])));
    st_from_float(y + j, fmaf(v, cs[p], u * sn[p]));
  }
  for (int i = 2 * a.half + lane; i < a.dim; i += DA_WAVE) st_from_float(y + i, ld_as_float(x + i) * r * gain_at(a, h.gain, i));
}

template <typename T>
__global__ __launch_bounds__(256) void qk_narrow_grad_kernel(QkArgs a) {
  extern __shared__ float sums[];   // [4][dim], if there is a gain
  const int which = (int)blockIdx.x >= a.t[0].blocks;
  const Heads& h = a.t[which];
  const unsigned block = blockIdx.x - (which ? a.t[0].blocks : 0);
  const int lane = threadIdx.x % DA_WAVE, wave = threadIdx.x / DA_WAVE;
  float* mine = sums + wave * a.dim;   // a lane always meets the same channels
  if (h.partial)
    for (int i = lane; i < a.dim; i += DA_WAVE) mine[i] = 0.f;
  __syncthreads();
  for (unsigned item = block * 4 + wave; item < h.items; item += h.blocks * 4) {
    const Place at = find_head(a, h, item);
    const Angle angle = find_angle(a, at);
    const T* x = static_cast<const T*>(h.x) + at.x;
    const T* dy = static_cast<const T*>(h.dy) + at.d;
    T* dx = static_cast<T*>(h.y) + at.y;
    const float* cs = a.cos + angle.row;
    const float* sn = a.sin + angle.row;
    float square = 0.f, dot = 0.f;
    for (int p = lane; p < a.half; p += DA_WAVE) {
      const int i = a.interleaved ? 2 * p : p, j = a.interleaved ? 2 * p + 1 : p + a.half;
      const float u = ld_as_float(x + i), v = ld_as_float(x + j), du = ld_as_float(dy + i), dv = ld_as_float(dy + j);
      square = fmaf(u, u, fmaf(v, v, square));
      dot = fmaf(fmaf(du, cs[p], dv * sn[p]) * gain_at(a, h.gain, i), u, dot);
      dot = fmaf(fmaf(dv, cs[p], -(du * sn[p])) * gain_at(a, h.gain, j), v, dot);
    }
    for (int i = 2 * a.half + lane; i < a.dim; i += DA_WAVE) {
      const float u = ld_as_float(x + i);
      square = fmaf(u, u, square);
      dot = fmaf(ld_as_float(dy + i) * gain_at(a, h.gain, i), u, dot);
    }
    const float r = angle.known ? rsqrtf(fmaf(da_group_sum(square), a.inv_dim, a.eps)) : QUIET_NAN;
    const float c = r * r * (da_group_sum(dot) * a.inv_dim);
    auto channel = [&](int i, float u, float dn) {
      if (h.partial) mine[i] = fmaf(dn * u, r, mine[i]);
      st_from_float(dx + i, r * fmaf(-u, c, dn * gain_at(a, h.gain, i)));
    };
    for (int p = lane; p < a.half; p += DA_WAVE) {
      const int i = a.interleaved ? 2 * p : p, j = a.interleaved ? 2 * p + 1 : p + a.half;
      const float u = ld_as_float(x + i), v = ld_as_float(x + j), du = ld_as_float(dy + i), dv = ld_as_float(dy + j);
      channel(i, u, fmaf(du, cs[p], dv * sn[p]));
      channel(j, v, fmaf(dv, cs[p], -(du * sn[p])));
    }
    for (int i = 2 * a.half + lane; i < a.dim; i += DA_WAVE) channel(i, ld_as_float(x + i), ld_as_float(dy + i));
  }
  if (!h.partial) return;
  __syncthreads();
  for (int i = threadIdx.x; i < a.dim; i += 256)
    h.partial[(long long)block * a.dim + i] = (sums[i] + sums[a.dim + i]) + (sums[2 * a.dim + i] + sums[3 * a.dim + i]);
}

// Sums of the workgroups' partial sums, in a fixed order: a workgroup takes 16 channels of one tensor, each group of 16 lanes every
// 64th partial sum.  Bound by latency: 768 partial sums of 90 channels take 3.9 us, of which a launch is 2.5; with 64 channels a
// workgroup, and so a quarter of the loads under way, 5.
struct GainArgs {
  const float* partial[2];
  void* out[2];
  int blocks[2];
  int dim, slices, gain_dtype;
};
constexpr int GAIN_CHANNELS = 16, GAIN_GROUPS = 1024 / GAIN_CHANNELS, GAIN_AHEAD = 3;

__global__ __launch_bounds__(1024) void qk_gain_kernel(GainArgs a) {
  __shared__ float part[16][GAIN_CHANNELS];
  const int which = (int)blockIdx.x >= a.slices, lane = threadIdx.x % DA_WAVE, wave = threadIdx.x / DA_WAVE;
  const int i = (blockIdx.x - which * a.slices) * GAIN_CHANNELS + threadIdx.x % GAIN_CHANNELS;
  void* out = a.out[which];
  if (!out) return;
  const int blocks = a.blocks[which];
  const float* partial = a.partial[which] + (i < a.dim ? i : 0);
  float sum = 0.f;
  for (int base = threadIdx.x / GAIN_CHANNELS; base < blocks; base += GAIN_GROUPS * GAIN_AHEAD) {
    float x[GAIN_AHEAD];
#pragma unroll
    for (int j = 0; j < GAIN_AHEAD; ++j) {
      const int b = base + j * GAIN_GROUPS;
      x[j] = partial[(long long)(b < blocks ? b : base) * a.dim];
    }
#pragma unroll
    for (int j = 0; j < GAIN_AHEAD; ++j)
      if (base + j * GAIN_GROUPS < blocks) sum += x[j];
  }
#pragma unroll
  for (int d = GAIN_CHANNELS; d < DA_WAVE; d *= 2) sum += __shfl_xor(sum, d);
  if (lane < GAIN_CHANNELS) part[wave][lane] = sum;
  __syncthreads();
  if ((int)threadIdx.x >= GAIN_CHANNELS || i >= a.dim) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) sum += part[w][lane];
  if (a.gain_dtype == DA_BF16) static_cast<bf16_t*>(out)[i] = f2bf(sum);
  else static_cast<float*>(out)[i] = sum;
}

// ---- host

// Workgroups of a gradient with gains at most, each of which leaves a partial sum of their gradients: as many as a compute unit holds.
// (138 registers; 16384 tokens of 40 heads of 128: 102 us; in 128 registers, 4 a compute unit 106; without the request ahead 102, but
// of 4096 tokens 30.5 in place of 29.8.)
constexpr int GRAD_BLOCKS_PER_CU = 3;

// How the heads are taken: `pairs` channel pairs a lane (0: by the kernels for narrow heads).
struct Form {
  int pairs;
  bool ragged;
};

// Lanes, items and workgroups of both tensors.
Form arrange(QkArgs& a, int dtype, bool grad, bool gains) {
  Form f{dtype == DA_BF16 ? 8 : 4, false};   // 16 bytes of a vector
  const int rest = a.dim - 2 * a.half;
  if ((a.half && a.half < f.pairs) || (rest && rest < 2 * f.pairs)) f.pairs = 0;
  if (f.pairs) {
    a.turn_lanes = (a.half + f.pairs - 1) / f.pairs;
    a.lanes = a.turn_lanes + (rest + 2 * f.pairs - 1) / (2 * f.pairs);
    a.log2_group = 0;
    while (1 << a.log2_group < a.lanes) ++a.log2_group;
    f.ragged = a.lanes != 1 << a.log2_group || a.half % f.pairs || rest % (2 * f.pairs);
    if (a.log2_group > 6) f.pairs = 0;
  }
  const long long cap = (long long)GRAD_BLOCKS_PER_CU * da_cu_count();
  for (int w = 0; w < 2; ++w) {
    Heads& h = a.t[w];
    h.by_heads = da_divisor((unsigned)std::max(1, h.heads));
    h.items = (unsigned)(a.tokens * h.heads);
    const long long threads = (long long)h.items << (f.pairs ? a.log2_group : 6);
    long long blocks = (threads + 255) / 256;
    if (grad && (gains || !f.pairs)) {   // both tensors' share of the cap by their heads
      const long long mine = std::max(1ll, cap * h.heads / std::max(1, a.t[0].heads + a.t[1].heads));
      blocks = std::min(blocks, mine);
    }
    h.blocks = (int)blocks;
  }
  return f;
}

// Checks what both directions share and fills the kernels' arguments.
int fill(QkArgs& a, const dion_amd_heads* q, const dion_amd_heads* k, int batch, int length, int dim, int rotary, int interleaved,
         int dtype, int gain_dtype, const float* cos, const float* sin, long long ld_table, int table_rows, const void* positions,
         int index_bits, long long pos_batch, float eps, bool grad) {
  if (!q || !k || batch < 0 || length < 0 || dim <= 0 || rotary < 0 || rotary > dim || rotary % 2) return DA_ERR_ARG;
  if (q->heads < 0 || k->heads < 0) return DA_ERR_ARG;
  if (!da_float_dtype(dtype) || !da_float_dtype(gain_dtype)) return DA_ERR_DTYPE;
  if (dim > MAX_DIM) return DA_ERR_LIMIT;
  if (rotary && (!cos || !sin || ld_table < rotary / 2 || table_rows <= 0)) return DA_ERR_ARG;
  if (positions && index_bits != 32 && index_bits != 64) return DA_ERR_ARG;
  if (!da_aligned(cos, 4) || !da_aligned(sin, 4) || !da_aligned(positions, positions ? index_bits / 8 : 1)) return DA_ERR_ALIGN;
  const dion_amd_heads* in[2] = {q, k};
  const size_t e = da_esize(dtype), ge = da_esize(gain_dtype);
  for (int w = 0; w < 2; ++w) {
    const dion_amd_heads& s = *in[w];
    Heads& h = a.t[w];
    h.heads = s.heads;
    const bool empty = s.heads == 0 || batch == 0 || length == 0;
    if (!empty && (!s.x || !s.y || (grad && !s.dy))) return DA_ERR_ARG;
    if (!da_aligned(s.x, e) || !da_aligned(s.y, e) || !da_aligned(s.dy, e) || !da_aligned(s.gain, ge) || !da_aligned(s.dgain, ge))
      return DA_ERR_ALIGN;
    if (grad && s.dgain && !s.gain) return DA_ERR_ARG;
    h.x = s.x; h.dy = s.dy; h.y = s.y; h.gain = s.gain;
    h.xb = s.x_batch; h.xt = s.x_token; h.xh = s.x_head;
    h.db = s.dy_batch; h.dt = s.dy_token; h.dh = s.dy_head;
    h.yb = s.y_batch; h.yt = s.y_token; h.yh = s.y_head;
  }
  a.tokens = (long long)batch * length;
  a.length = length; a.dim = dim; a.half = rotary / 2; a.interleaved = interleaved; a.gain_dtype = gain_dtype;
  a.cos = cos; a.sin = sin; a.ld_table = ld_table; a.table_rows = table_rows;
  a.positions = {positions, index_bits == 64};
  a.pos_batch = pos_batch;
  a.eps = eps;
  a.inv_dim = 1.f / (float)dim;
  a.by_length = da_divisor((unsigned)(length > 0 ? length : 1));
  if (a.tokens * (q->heads + k->heads) >= (1ll << 26) - 8) return DA_ERR_LIMIT;   // a launch has fewer than 2^32 threads, both ends rounded up
  return DA_OK;
}

// One of the eight forms of the vector kernels.
#define DA_QK_FORMS(LAUNCH)                                                                                                 \
  do {                                                                                                                     \
    if (dtype == DA_BF16 && interleaved) { if (f.ragged) LAUNCH(bf16_t, 8, true, true); else LAUNCH(bf16_t, 8, true, false); }      \
    else if (dtype == DA_BF16) { if (f.ragged) LAUNCH(bf16_t, 8, false, true); else LAUNCH(bf16_t, 8, false, false); }     \
    else if (interleaved) { if (f.ragged) LAUNCH(float, 4, true, true); else LAUNCH(float, 4, true, false); }              \
    else { if (f.ragged) LAUNCH(float, 4, false, true); else LAUNCH(float, 4, false, false); }                             \
  } while (0)

}  // namespace

extern "C" {

int dion_amd_qk_norm_rope(const dion_amd_heads* q, const dion_amd_heads* k, int batch, int length, int dim, int rotary,
                          int interleaved, int dtype, int gain_dtype, const float* cos, const float* sin, long long ld_table,
                          int table_rows, const void* positions, int index_bits, long long pos_batch, float eps, void* stream) {
  QkArgs a{};
  const int rc = fill(a, q, k, batch, length, dim, rotary, interleaved, dtype, gain_dtype, cos, sin, ld_table, table_rows,
                      positions, index_bits, pos_batch, eps, false);
  if (rc) return rc;
  const Form f = arrange(a, dtype, false, false);
  const dim3 grid((unsigned)(a.t[0].blocks + a.t[1].blocks));
  if (grid.x == 0) return DA_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  DaProfScope prof(DA_PROF_QK_NORM, 2.0 * a.tokens * (q->heads + k->heads) * dim * da_esize(dtype), s);
  if (f.pairs == 0) {
    if (dtype == DA_BF16) hipLaunchKernelGGL(qk_narrow_kernel<bf16_t>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(qk_narrow_kernel<float>, grid, dim3(256), 0, s, a);
    return da_launch_status();
  }
#define DA_QK(T, PAIRS, INTER, RAGGED) hipLaunchKernelGGL((qk_heads_kernel<T, PAIRS, INTER, RAGGED>), grid, dim3(256), 0, s, a)
  DA_QK_FORMS(DA_QK);
#undef DA_QK
  return da_launch_status();
}

size_t dion_amd_qk_norm_rope_grad_workspace_bytes(int batch, int length, int dim, int heads) {
  if (batch < 0 || length < 0 || dim <= 0 || heads < 0 || dim > MAX_DIM) return 0;
  // (one partial sum a workgroup; either tensor has at least one)
  return ((size_t)GRAD_BLOCKS_PER_CU * da_cu_count() + 2) * dim * sizeof(float);
}

int dion_amd_qk_norm_rope_grad(const dion_amd_heads* q, const dion_amd_heads* k, int batch, int length, int dim, int rotary,
                               int interleaved, int dtype, int gain_dtype, const float* cos, const float* sin,
                               long long ld_table, int table_rows, const void* positions, int index_bits, long long pos_batch,
                               float eps, void* workspace, size_t workspace_bytes, void* stream) {
  QkArgs a{};
  int rc = fill(a, q, k, batch, length, dim, rotary, interleaved, dtype, gain_dtype, cos, sin, ld_table, table_rows, positions,
                index_bits, pos_batch, eps, true);
  if (rc) return rc;
  const bool gains = q->dgain || k->dgain;
  if (gains) {
    if (!workspace) return DA_ERR_ARG;
    if (!da_aligned(workspace, 256)) return DA_ERR_ALIGN;
    if (workspace_bytes < dion_amd_qk_norm_rope_grad_workspace_bytes(batch, length, dim, q->heads + k->heads))
      return DA_ERR_WORKSPACE;
  }
  const Form f = arrange(a, dtype, true, gains);
  if (gains) {
    float* partial = static_cast<float*>(workspace);
    if (q->dgain) a.t[0].partial = partial;
    if (k->dgain) a.t[1].partial = partial + (long long)a.t[0].blocks * dim;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  DaProfScope prof(DA_PROF_QK_NORM, 3.0 * a.tokens * (q->heads + k->heads) * dim * da_esize(dtype), s);
  const dim3 grid((unsigned)(a.t[0].blocks + a.t[1].blocks));
  if (grid.x && f.pairs == 0) {
    const size_t lds = gains ? (size_t)4 * dim * sizeof(float) : 0;
    if (dtype == DA_BF16) hipLaunchKernelGGL(qk_narrow_grad_kernel<bf16_t>, grid, dim3(256), lds, s, a);
    else hipLaunchKernelGGL(qk_narrow_grad_kernel<float>, grid, dim3(256), lds, s, a);
  } else if (grid.x) {
#define DA_QK(T, PAIRS, INTER, RAGGED)                                                                                      \
  do {                                                                                                                     \
    if (gains) hipLaunchKernelGGL((qk_heads_grad_kernel<T, PAIRS, INTER, RAGGED, true>), grid, dim3(256), 0, s, a);        \
    else hipLaunchKernelGGL((qk_heads_grad_kernel<T, PAIRS, INTER, RAGGED, false>), grid, dim3(256), 0, s, a);             \
  } while (0)
    DA_QK_FORMS(DA_QK);
#undef DA_QK
  }
  rc = da_launch_status();
  if (rc || !gains) return rc;
  GainArgs ga{{a.t[0].partial, a.t[1].partial}, {q->dgain, k->dgain}, {a.t[0].blocks, a.t[1].blocks}, dim,
              (dim + GAIN_CHANNELS - 1) / GAIN_CHANNELS, gain_dtype};
  hipLaunchKernelGGL(qk_gain_kernel, dim3(2 * ga.slices), dim3(1024), 0, s, ga);
  return da_launch_status();
}

}  // extern "C"
