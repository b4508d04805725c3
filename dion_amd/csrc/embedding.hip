// Embedding lookup with a scale, and the dense gradient of the table.
//
//   out[t] = r(scale * W[tok_t])                       dW[v] = r(scale * sum of g[t] over the t with tok_t = v  (+ dW[v]))
//
// Both are bound by HBM: the lookup reads one row and writes one row a token, the gradient reads one row a token and writes every
// row of the table once.  Sums are formed in fp32 in an order that depends on the tokens alone, on all of them: the same bits every time.
#include "../../include/dion_amd.h"
#include "model_ops.h"
#include "prof.h"
#include <algorithm>

namespace {

constexpr float QUIET_NAN = __builtin_nanf("");

// ---- lookup: a lane takes 8 columns of two tokens' rows.  A token outside the table gives a row of NaN.
//
// 65536 tokens of 768 columns, fp32 to bf16: 39 us (152 MB with every named row read once: 3.9 TB/s).  The L2s of the eight XCDs fetch
// the rows of frequent tokens one each, 114 MiB in place of 52: 5.9 TB/s between them and the memory.  One row a lane 42 us, four 39.5;
// 4 columns a lane, at 2 to 8 rows, 42 to 46; the columns dealt to the XCDs, so that a row's part is fetched once, 49.
constexpr int UNITS = 2;

template <typename W, typename O, int COLS>
__global__ __launch_bounds__(256) void embedding_kernel(const W* w, long long ldw, long long vocab, int dim, DaDivisor lanes,
                                                        DaIndex tokens, long long count, O* out, long long ldo, float scale) {
  unsigned t[UNITS];
  int c[UNITS], shared;
  bool known[UNITS];
  long long at[UNITS], v[UNITS];
  float x[UNITS][COLS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const unsigned unit = (blockIdx.x * UNITS + u) * 256u + threadIdx.x;
    t[u] = lanes.quotient(unit);
    c[u] = da_column<COLS>((int)(unit - t[u] * lanes.by), dim, shared);   // (what two lanes hold is stored by both: 763 columns 38.0 us, 39.4 by one)
    at[u] = t[u] < count ? t[u] : 0;
  }
  da_indices(tokens, at, v);
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    known[u] = v[u] >= 0 && v[u] < vocab;
    da_load(w + (known[u] ? v[u] : 0) * ldw + c[u], x[u]);
  }
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    if (t[u] >= count) return;
#pragma unroll
    for (int i = 0; i < COLS; ++i) x[u][i] = known[u] ? scale * x[u][i] : QUIET_NAN;
    da_store(out + t[u] * ldo + c[u], 0, x[u]);
  }
}

// ---- index of the gradient: the positions of every token id, in order
//
// Ids are dealt to B bins (a power of two) by their low bits, so that the frequent ids of a text, which tokenizers put side by
// side, fall into different ones.  A workgroup of the index owns one bin.  For few tokens it looks at all of them: it counts those of
// lower bins -- the place where its own positions begin, so that no workgroup waits for another -- and lists its own.  For many
// tokens a launch before has sorted each part of 1024 tokens or more by bin; the workgroup gathers its run of every part, and the places of
// the runs in their parts add up to the place where it begins.  Sorting the positions of a bin by id is then a counting sort in LDS,
// stable because each wavefront takes a contiguous run of tokens and ranks its lanes in order.
//
// A frequent id keeps the one workgroup of its bin busy while the others are done: the gradient of 65536 tokens of 768 bf16 columns takes
// 51 us, 82 if a fifth of them are one id, 198 if all are.  Tables of more ids than 256 bins hold (262144) have more bins and no sorted
// parts, so that the work is bins times tokens: 131072 tokens of 64 columns 49 us with 262144 ids and 135 with 262145, 2^20 tokens of 16
// columns and as many ids 1.1 ms.
constexpr int IDX_THREADS = 1024, IDX_WAVES = IDX_THREADS / DA_WAVE;
constexpr int IDX_ROWS = 1024;   // ids of a bin at most: one per thread in the scan
constexpr int IDX_AHEAD = 4;     // rounds of 64 tokens requested before the first is looked at
constexpr int IDX_LIST = 256;    // own positions a wavefront keeps; a wavefront with more looks at its tokens again
constexpr int PART_BITS = 8, PART_BINS = 1 << PART_BITS;   // bins of the sorted parts
constexpr int PARTS = 256;       // parts at most: a part is a multiple of 1024 tokens

struct IndexArgs {
  DaIndex tokens;
  int vocab, padding;         // padding: id whose tokens are left out, -1 for none
  int count;
  int log2_bins, rows;        // rows: ids of a bin
  int2* range;                // [bins][rows]: first entry of `order` and number of entries of id r * bins + b
  int2* order;                // (position, id) by (bin, id, position)
  int* kept;                  // number of entries
  int part, parts;            // tokens of a part, number of parts
  int2* parted;               // (position, id), every part sorted by bin; a part's tokens that do not count are left out
  int* offsets;               // [parts][PART_BINS + 1] where a part's bins begin
};

// Token i, or -1 if it does not count.
__device__ __forceinline__ int token_at(const IndexArgs& a, int i) {
  int v, high = 0;
  if (a.tokens.wide) {
    const int2 w = static_cast<const int2*>(a.tokens.p)[i];
    v = w.x;
    high = w.y;
  } else {
    v = static_cast<const int*>(a.tokens.p)[i];
  }
  return high == 0 && (unsigned)v < (unsigned)a.vocab && v != a.padding ? v : -1;
}

// The lanes whose key equals this lane's (keys of `bits` bits), among `active` ones.
__device__ __forceinline__ unsigned long long same_key(int key, int bits, unsigned long long active) {
  unsigned long long same = active;
  for (int b = 0; b < bits; ++b) {
    const unsigned long long ones = __ballot((key >> b) & 1);
    same &= (key >> b) & 1 ? ones : ~ones;
  }
  return same;
}

// Inclusive sum over the threads of a workgroup of IDX_THREADS, and the sum of all; scan: IDX_WAVES words.
__device__ __forceinline__ int block_scan(int v, int* scan, int& all) {
  const int wave = threadIdx.x / DA_WAVE, lane = threadIdx.x % DA_WAVE;
  for (int d = 1; d < DA_WAVE; d <<= 1) {
    const int up = __shfl_up(v, d);
    if (lane >= d) v += up;
  }
  if (lane == DA_WAVE - 1) scan[wave] = v;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < IDX_WAVES; ++w) {
    const int s = scan[w];
    if (w < wave) v += s;
    all += s;
  }
  __syncthreads();
  return v;
}

// Zeros for the whole table, by the workgroups behind those of the index: that work waits for memory, not for bandwidth, and the
// rows that tokens name (the fewer, as a rule) are written over by the launch behind.
struct FillArgs {
  void* dw;
  long long ldw;         // 0: the rows lie without gaps, and the table is one row of `dim` elements
  long long dim;
  long long lanes;       // 16-byte pieces of a row, or elements of one too short for that
  long long begin, end;  // pieces of the table to fill in this launch
};
constexpr int FILL = 8;  // pieces a thread

template <typename W>
__device__ __forceinline__ void fill(const FillArgs& f, long long block) {
  constexpr int COLS = 16 / sizeof(W);
  const float zero[COLS] = {};
#pragma unroll
  for (int i = 0; i < FILL; ++i) {
    const long long unit = f.begin + (block * FILL + i) * IDX_THREADS + threadIdx.x;
    if (unit >= f.end) return;
    const long long v = f.ldw ? unit / f.lanes : 0, lane = unit - v * f.lanes;
    W* row = static_cast<W*>(f.dw) + v * f.ldw;
    if (f.dim < COLS) st_from_float(row + lane, 0.f);
    else da_store(row + (lane * COLS < f.dim - COLS ? lane * COLS : f.dim - COLS), 0, zero);   // (the last one moved back)
  }
}

// One part sorted by bin, stable.
template <typename W>
__global__ __launch_bounds__(IDX_THREADS) void embedding_part_kernel(IndexArgs a, FillArgs f) {
  if ((int)blockIdx.x >= a.parts) {
    fill<W>(f, (int)blockIdx.x - a.parts);
    return;
  }
  __shared__ int cnt[IDX_WAVES][PART_BINS];
  __shared__ int scan[IDX_WAVES];
  const int wave = threadIdx.x / DA_WAVE, lane = threadIdx.x % DA_WAVE;
  for (int i = threadIdx.x; i < IDX_WAVES * PART_BINS; i += IDX_THREADS) (&cnt[0][0])[i] = 0;
  __syncthreads();
  const int run = a.part / IDX_WAVES, start = blockIdx.x * a.part;
  const int begin = start + wave * run < a.count ? start + wave * run : a.count;
  const int end = begin + run < a.count ? begin + run : a.count;
  for (int base = begin; base < end; base += DA_WAVE) {
    const int v = base + lane < end ? token_at(a, base + lane) : -1;
    if (v >= 0) atomicAdd(&cnt[wave][v & (PART_BINS - 1)], 1);
  }
  __syncthreads();
  int total = 0, here[IDX_WAVES];
#pragma unroll
  for (int w = 0; w < IDX_WAVES; ++w) {
    here[w] = threadIdx.x < PART_BINS ? cnt[w][threadIdx.x] : 0;
    total += here[w];
  }
  int all;
  int at = block_scan(total, scan, all) - total;
  if (threadIdx.x < PART_BINS) {
    a.offsets[(long long)blockIdx.x * (PART_BINS + 1) + threadIdx.x] = at;
    if (threadIdx.x == 0) a.offsets[(long long)blockIdx.x * (PART_BINS + 1) + PART_BINS] = all;
#pragma unroll
    for (int w = 0; w < IDX_WAVES; ++w) {
      cnt[w][threadIdx.x] = at;
      at += here[w];
    }
  }
  __syncthreads();
  const unsigned long long before = (1ull << lane) - 1;
  for (int base = begin; base < end; base += DA_WAVE) {
    const int v = base + lane < end ? token_at(a, base + lane) : -1;
    const int bin = v & (PART_BINS - 1);
    const unsigned long long same = same_key(bin, PART_BITS, __ballot(v >= 0));
    if (v < 0) continue;
    const int place = __hip_atomic_load(&cnt[wave][bin], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    a.parted[start + place + __popcll(same & before)] = make_int2(base + lane, v);
    if ((same & before) == 0)
      __hip_atomic_store(&cnt[wave][bin], place + __popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
}

// The bin of this workgroup.  row_range(row, first entry, entries) is called by one thread for every id, in any order;
// put(entry, position, row) for every token of the bin.
template <bool PARTED, typename Range, typename Put>
__device__ __forceinline__ void index_bin(const IndexArgs& a, int* lds, Range&& row_range, Put&& put) {
  int* cnt = lds;                                 // [IDX_WAVES][rows]: own tokens by wavefront and id, then their places
  int* list = cnt + IDX_WAVES * a.rows;           // [IDX_WAVES][IDX_LIST][2]: position, row
  int* scan = list + IDX_WAVES * IDX_LIST * 2;    // [IDX_WAVES]
  int* lower = scan + IDX_WAVES;                  // [IDX_WAVES] tokens of lower bins
  int* part_items = lower + IDX_WAVES;            // [PARTS] own tokens of every part
  int* part_at = part_items + PARTS;              // [PARTS] where they begin
  const int wave = threadIdx.x / DA_WAVE, lane = threadIdx.x % DA_WAVE;
  const int bin = blockIdx.x, mask = (1 << a.log2_bins) - 1;
  for (int i = threadIdx.x; i < IDX_WAVES * a.rows; i += IDX_THREADS) cnt[i] = 0;

  int bin_start = 0;
  if (PARTED) {
    int from = 0;
    if (threadIdx.x < a.parts) {
      const int* off = a.offsets + (long long)threadIdx.x * (PART_BINS + 1) + bin;
      from = off[0];
      part_items[threadIdx.x] = off[1] - from;
      part_at[threadIdx.x] = threadIdx.x * a.part + from;
    }
    block_scan(from, scan, bin_start);
  }
  __syncthreads();

  // this wavefront's run: of parts, or of tokens
  const int items = PARTED ? a.parts : a.count, unit = PARTED ? 1 : DA_WAVE;
  const int per = ((items + IDX_WAVES - 1) / IDX_WAVES + unit - 1) / unit * unit;
  const long long first = (long long)wave * per;
  const int begin = first < items ? (int)first : items;
  const int end = first + per < items ? (int)(first + per) : items;
  int* my_cnt = cnt + wave * a.rows;
  int* my_list = list + wave * IDX_LIST * 2;

  const unsigned long long before = (1ull << lane) - 1;
  // 64 tokens at a time in order.  f(position, id, counts, own): the lanes whose tokens count at all, and those of this bin
  auto each = [&](auto&& f) {
    if (PARTED) {
      // runs of up to 64 items come one a round from IDX_AHEAD parts at a time, longer ones by themselves
      for (int p0 = begin; p0 < end; p0 += IDX_AHEAD) {
        int n[IDX_AHEAD], longest = 0;
        const int2* run[IDX_AHEAD];
#pragma unroll
        for (int k = 0; k < IDX_AHEAD; ++k) {
          const int p = p0 + k < end ? p0 + k : end - 1;
          n[k] = p0 + k < end ? __builtin_amdgcn_readfirstlane(part_items[p]) : 0;
          run[k] = a.parted + __builtin_amdgcn_readfirstlane(part_at[p]);
          longest = n[k] > longest ? n[k] : longest;
        }
        if (longest <= DA_WAVE) {
          int2 e[IDX_AHEAD];
#pragma unroll
          for (int k = 0; k < IDX_AHEAD; ++k) e[k] = lane < n[k] ? run[k][lane] : make_int2(0, -1);
#pragma unroll
          for (int k = 0; k < IDX_AHEAD; ++k)
            if (n[k]) {
              const unsigned long long there = __ballot(e[k].y >= 0);
              f(e[k].x, e[k].y, there, there);
            }
          continue;
        }
        for (int k = 0; k < IDX_AHEAD && p0 + k < end; ++k) {
          const int p = p0 + k, items = __builtin_amdgcn_readfirstlane(part_items[p]);
          const int2* from = a.parted + __builtin_amdgcn_readfirstlane(part_at[p]);
          for (int base = 0; base < items; base += DA_WAVE * IDX_AHEAD) {
            int2 e[IDX_AHEAD];
#pragma unroll
            for (int j = 0; j < IDX_AHEAD; ++j) {
              const int i = base + j * DA_WAVE + lane;
              e[j] = from[i < items ? i : items - 1];
              if (i >= items) e[j].y = -1;
            }
#pragma unroll
            for (int j = 0; j < IDX_AHEAD; ++j)
              if (base + j * DA_WAVE < items) {
                const unsigned long long there = __ballot(e[j].y >= 0);
                f(e[j].x, e[j].y, there, there);
              }
          }
        }
      }
    } else {
      int2 next[IDX_AHEAD];   // low and high half
      auto request = [&](int base) {
        if (a.tokens.wide) {
#pragma unroll
          for (int i = 0; i < IDX_AHEAD; ++i) {
            const int at = base + i * DA_WAVE + lane;
            next[i] = static_cast<const int2*>(a.tokens.p)[at < end ? at : end - 1];
          }
        } else {
#pragma unroll
          for (int i = 0; i < IDX_AHEAD; ++i) {
            const int at = base + i * DA_WAVE + lane;
            next[i] = make_int2(static_cast<const int*>(a.tokens.p)[at < end ? at : end - 1], 0);
          }
        }
      };
      if (begin < end) request(begin);
      for (int base = begin; base < end; base += DA_WAVE * IDX_AHEAD) {
        int2 v[IDX_AHEAD];
#pragma unroll
        for (int i = 0; i < IDX_AHEAD; ++i) v[i] = next[i];
        if (base + DA_WAVE * IDX_AHEAD < end) request(base + DA_WAVE * IDX_AHEAD);
#pragma unroll
        for (int i = 0; i < IDX_AHEAD; ++i) {
          const int at = base + i * DA_WAVE + lane;
          const unsigned long long counts = __ballot(at < end && v[i].y == 0 && (unsigned)v[i].x < (unsigned)a.vocab && v[i].x != a.padding);
          f(at, v[i].x, counts, __ballot((v[i].x & mask) == bin) & counts);
        }
      }
    }
  };
  int below = 0, own = 0;
  each([&](int position, int v, unsigned long long counts, unsigned long long m) {
    if (!PARTED) below += __popcll(__ballot((v & mask) < bin) & counts);
    if (m == 0) return;
    if (m >> lane & 1) {
      const int row = v >> a.log2_bins;
      atomicAdd(my_cnt + row, 1);
      const int at = own + __popcll(m & before);
      if (at < IDX_LIST) {
        my_list[at * 2] = position;
        my_list[at * 2 + 1] = row;
      }
    }
    own += __popcll(m);
  });
  if (!PARTED && lane == 0) lower[wave] = below;
  __syncthreads();
  if (!PARTED)
    for (int w = 0; w < IDX_WAVES; ++w) bin_start += lower[w];

  // places: exclusive sums over the ids of the bin, then over the wavefronts
  int total = 0, here[IDX_WAVES];
#pragma unroll
  for (int w = 0; w < IDX_WAVES; ++w) {
    here[w] = threadIdx.x < a.rows ? cnt[w * a.rows + threadIdx.x] : 0;
    total += here[w];
  }
  int all;
  int start = bin_start + block_scan(total, scan, all) - total;
  if (bin == mask && threadIdx.x == 0 && a.kept) *a.kept = bin_start + all;   // (the last bin's tokens end the list)
  if (threadIdx.x < a.rows) {
    row_range((int)threadIdx.x, start, total);
#pragma unroll
    for (int w = 0; w < IDX_WAVES; ++w) {
      cnt[w * a.rows + threadIdx.x] = start;
      start += here[w];
    }
  }
  __syncthreads();

  // up to 64 own tokens in the order of the lanes: those of one id take the next places of their wavefront
  const int row_bits = 32 - __clz(a.rows);
  auto place = [&](bool mine, int row, int position) {
    const unsigned long long same = same_key(row, row_bits, __ballot(mine));
    if (!mine) return;
    const int at = __hip_atomic_load(my_cnt + row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    put(at + __popcll(same & before), position, row);
    if ((same & before) == 0)
      __hip_atomic_store(my_cnt + row, at + __popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  if (own <= IDX_LIST) {
    for (int base = 0; base < own; base += DA_WAVE) {
      const int i = base + lane;
      const bool mine = i < own;
      place(mine, mine ? my_list[i * 2 + 1] : 0, mine ? my_list[i * 2] : 0);
    }
  } else {
    each([&](int position, int v, unsigned long long, unsigned long long m) {
      if (m) place(m >> lane & 1, m >> lane & 1 ? v >> a.log2_bins : 0, position);
    });
  }
}

// (8 wavefronts a SIMD, 64 registers: a workgroup of zeros fits beside the one of the index)
template <bool PARTED, typename W>
__global__ __launch_bounds__(IDX_THREADS, 8) void embedding_index_kernel(IndexArgs a, FillArgs f) {
  if ((int)blockIdx.x >> a.log2_bins) {
    fill<W>(f, (int)blockIdx.x - (1 << a.log2_bins));
    return;
  }
  extern __shared__ int lds[];
  const int bin = blockIdx.x;
  index_bin<PARTED>(
      a, lds, [&](int row, int start, int n) { a.range[(long long)bin * a.rows + row] = make_int2(start, n); },
      [&](int at, int position, int row) { a.order[at] = make_int2(position, (row << a.log2_bins) + bin); });
}

// ---- rows of the gradient
//
// The sorted list is cut into pieces of equal length, whatever rows they belong to, so that every lane has the same work under any
// distribution of the tokens.  A lane sums its columns of one piece, requesting BATCH rows before it adds the first, and stores a
// row of the table whenever the id changes.  A row that crosses a border of pieces leaves partial sums (fp32): at the front of every
// piece it comes into from the left, at the back of the piece it begins in.  The launch behind joins them in order.
//
// Bound by HBM.  65536 tokens of 768 bf16 columns and 50304 ids: 27.6 us for 127 MiB read and written (4.8 TB/s), of a gradient of
// 51 us: sorting the parts 7.3 and the index 11.4, both beside 74 MiB of zeros, the join 5.0 (all latency), three gaps between launches.
// The rows of g are read once and pass by the caches (non-temporal), which keep the zeros until they are written over: 59.7 -> 52.8.
// Rows requested 16 at a time were slower than 8.
constexpr int BATCH = 8;

struct RowArgs {
  const int2* range;
  const int2* order;
  const int* kept;
  int log2_bins, rows, lanes;
  int piece, pieces;   // entries of a piece (a multiple of BATCH), number of pieces
  const void* g;
  long long ldg;
  void* dw;
  long long ldw;
  float* partial;   // [pieces][2][dim]: front, back
  int dim, accumulate;
  float scale;
  DaDivisor by_lanes;
};

template <typename W, int COLS>
__device__ __forceinline__ void store_row(const RowArgs& a, long long v, int c, int skip, const float (&sum)[COLS]) {
  W* dst = static_cast<W*>(a.dw) + v * a.ldw + c;
  float y[COLS];
  if (a.accumulate) da_load(dst, y);
#pragma unroll
  for (int i = 0; i < COLS; ++i) y[i] = a.accumulate ? fmaf(sum[i], a.scale, y[i]) : sum[i] * a.scale;
  da_store(dst, a.accumulate ? skip : 0, y);   // (what two lanes hold is stored by both, but added by one)
}

// Entries of the list come two to a 16-byte load; the list is padded to whole pieces.
__device__ __forceinline__ void load_entries(const int2* order, int4 (&e)[BATCH / 2]) {
#pragma unroll
  for (int i = 0; i < BATCH / 2; ++i) e[i] = reinterpret_cast<const int4*>(order)[i];
}

template <typename G, typename W, int COLS>
__global__ __launch_bounds__(256) void embedding_rows_kernel(RowArgs a) {
  const unsigned unit = blockIdx.x * 256u + threadIdx.x;
  const unsigned piece = a.by_lanes.quotient(unit);
  if (piece >= (unsigned)a.pieces) return;
  const int first = (int)piece * a.piece;
  int4 e[BATCH / 2];
  load_entries(a.order + first, e);   // (past the last entry: not used)
  int id = first > 0 ? a.order[first - 1].y : -1;
  const int kept = *a.kept;
  if (first >= kept) return;
  const int last = first + a.piece < kept ? first + a.piece : kept;
  int skip;
  const int c = da_column<COLS>((int)(unit - piece * a.lanes), a.dim, skip);
  const G* g = static_cast<const G*>(a.g) + c;
  bool from_left = id == e[0].y;
  id = e[0].y;
  float* front = a.partial + (long long)piece * 2 * a.dim + c;
  float sum[COLS] = {};
  for (int base = first; base < last; base += BATCH) {
    float x[BATCH][COLS];
    int ids[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int position = i % 2 ? e[i / 2].z : e[i / 2].x;
      ids[i] = i % 2 ? e[i / 2].w : e[i / 2].y;
      da_load<true>(g + (base + i < last ? position : 0) * a.ldg, x[i]);
    }
    if (base + BATCH < last) load_entries(a.order + base + BATCH, e);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (base + i >= last) break;
      if (ids[i] != id) {
        if (from_left) da_store(front, 0, sum);
        else store_row<W, COLS>(a, id, c, skip, sum);
        from_left = false;
        id = ids[i];
#pragma unroll
        for (int k = 0; k < COLS; ++k) sum[k] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < COLS; ++k) sum[k] += x[i][k];
    }
  }
  if (from_left) da_store(front, 0, sum);
  else if (last < kept && a.order[last].y == id) da_store(front + a.dim, 0, sum);
  else store_row<W, COLS>(a, id, c, skip, sum);
}

// The whole gradient of a short call in one launch: the workgroup of a bin sorts its tokens in LDS and writes its rows, a wavefront a
// row.  With few tokens three launches are mostly their own latency: 128 tokens of 256 columns take 6.6 us in place of 13.6, 512 tokens
// of 768 columns and 50304 ids 20.7 in place of 20.9, 1000 tokens 23.5 in place of 21.5.
constexpr int SMALL_COUNT = 512;
constexpr int SMALL_ROW = 32;   // tokens of a row from which all wavefronts of the workgroup take a share of them

template <typename G, typename W, int COLS>
__global__ __launch_bounds__(IDX_THREADS) void embedding_small_kernel(IndexArgs a, RowArgs r) {
  extern __shared__ int lds[];
  __shared__ int position[SMALL_COUNT];
  __shared__ int2 range[IDX_ROWS];
  __shared__ float part[IDX_WAVES - 1][DA_WAVE][COLS];
  __shared__ int long_rows[SMALL_COUNT / SMALL_ROW], n_long;
  if (threadIdx.x == 0) n_long = 0;   // (seen by all behind the index's first barrier)
  // (entries of a bin are consecutive and at most SMALL_COUNT, so that their places modulo it are distinct)
  index_bin<false>(
      a, lds,
      [&](int row, int start, int n) {
        range[row] = make_int2(start, n);
        if (n > SMALL_ROW) long_rows[atomicAdd(&n_long, 1)] = row;
      },
      [&](int at, int pos, int) { position[at % SMALL_COUNT] = pos; });
  __syncthreads();
  const G* g = static_cast<const G*>(r.g);
  const int wave = threadIdx.x / DA_WAVE, lane = threadIdx.x % DA_WAVE;
  constexpr int ROWS = COLS == 8 ? 4 : 8;   // requested at a time
  auto add = [&](float (&sum)[COLS], int c, int begin, int end) {
#pragma unroll ROWS
    for (int i = begin; i < end; ++i) {
      float x[COLS];
      da_load(g + position[i % SMALL_COUNT] * r.ldg + c, x);
#pragma unroll
      for (int k = 0; k < COLS; ++k) sum[k] += x[k];
    }
  };
  for (int row = wave; row < a.rows; row += IDX_WAVES) {
    const int v = (row << a.log2_bins) + (int)blockIdx.x;
    const int2 e = range[row];
    if (v >= a.vocab || e.y > SMALL_ROW || (r.accumulate && e.y == 0)) continue;
    for (int at = lane; at < r.lanes; at += DA_WAVE) {
      int skip;
      const int c = da_column<COLS>(at, r.dim, skip);
      float sum[COLS] = {};
      add(sum, c, e.x, e.x + e.y);
      store_row<W, COLS>(r, v, c, skip, sum);
    }
  }
  for (int i = 0; i < n_long; ++i) {
    const int row = long_rows[i];
    const int2 e = range[row];
    const int per = (e.y + IDX_WAVES - 1) / IDX_WAVES, begin = wave * per < e.y ? wave * per : e.y, end = begin + per < e.y ? begin + per : e.y;
    for (int base = 0; base < r.lanes; base += DA_WAVE) {
      const int at = base + lane < r.lanes ? base + lane : r.lanes - 1;
      int skip;
      const int c = da_column<COLS>(at, r.dim, skip);
      float sum[COLS] = {};
      add(sum, c, e.x + begin, e.x + end);
      if (wave)
#pragma unroll
        for (int k = 0; k < COLS; ++k) part[wave - 1][lane][k] = sum[k];
      __syncthreads();
      if (wave == 0) {
#pragma unroll 1
        for (int w = 0; w < IDX_WAVES - 1; ++w)
#pragma unroll
          for (int k = 0; k < COLS; ++k) sum[k] += part[w][lane][k];
        if (base + lane < r.lanes) store_row<W, COLS>(r, (row << a.log2_bins) + (int)blockIdx.x, c, skip, sum);
      }
      __syncthreads();
    }
  }
}

// Rows that cross borders: the workgroup of the piece where one begins joins its partial sums, 64 lanes of columns, each wavefront
// a contiguous quarter of them.
template <typename W, int COLS>
__global__ __launch_bounds__(256) void embedding_join_kernel(RowArgs a, int slices) {
  __shared__ float part[3][DA_WAVE][COLS];
  const int piece = blockIdx.x / slices;
  const int first = piece * a.piece, next = first + a.piece;   // (there is a piece behind)
  const int kept = *a.kept, id = a.order[next].y, before = a.order[next - 1].y;
  if (next >= kept || before != id) return;
  const int2 range = a.range[(long long)(id & ((1 << a.log2_bins) - 1)) * a.rows + (id >> a.log2_bins)];
  if (range.x < first) return;   // it began further left
  const int lane = threadIdx.x % DA_WAVE, wave = threadIdx.x / DA_WAVE;
  const int column = blockIdx.x % slices * DA_WAVE + lane;
  int skip;
  const int c = da_column<COLS>(column < a.lanes ? column : a.lanes - 1, a.dim, skip);
  // partial sum 0 is the back of this piece, i > 0 the front of piece + i
  const int n = (range.x + range.y - 1) / a.piece - piece + 1, quarter = (n + 3) / 4;
  const int begin = wave * quarter, end = begin + quarter < n ? begin + quarter : n;
  const float* src = a.partial + (long long)piece * 2 * a.dim + c;
  float sum[COLS] = {};
  if (column < a.lanes) {
#pragma unroll 4
    for (int i = begin; i < end; ++i) {
      float x[COLS];
      da_load(src + (i ? (long long)i * 2 * a.dim : a.dim), x);
#pragma unroll
      for (int k = 0; k < COLS; ++k) sum[k] += x[k];
    }
  }
  if (wave)
#pragma unroll
    for (int k = 0; k < COLS; ++k) part[wave - 1][lane][k] = sum[k];
  __syncthreads();
  if (wave || column >= a.lanes) return;
#pragma unroll
  for (int w = 0; w < 3; ++w)
#pragma unroll
    for (int k = 0; k < COLS; ++k) sum[k] += part[w][lane][k];
  store_row<W, COLS>(a, id, c, skip, sum);
}

// ---- host

// Tokens from which the parts are sorted first.  Without that launch and with it, 50304 ids: 18000 tokens of 64 columns 21.1 and
// 22.5 us, 26000 24.8 and 24.1, 65536 40 and 32; of 768 columns 26000 34.5 and 35.5, 32000 38.0 and 38.8, 65536 63 and 55.
constexpr long long PART_FROM = 24000;

struct GradPlan {
  int log2_bins, rows;
  int cols, lanes;              // columns of a lane, lanes of a row
  int piece, pieces;
  int part, parts;              // 0 parts: the index looks at all tokens
  size_t range, order, kept, partial, parted, offsets, bytes;   // offsets in the workspace, and its size
};

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Bins: as many as fill the chip with one workgroup each, more where a bin would hold more ids than the scan has threads.
GradPlan plan_grad(long long count, long long vocab, int dim, int g_dtype) {
  GradPlan p{};
  const int wide = g_dtype == DA_BF16 ? 8 : 4;   // 16 bytes of the gradient
  p.cols = dim >= wide ? wide : 1;
  p.lanes = da_lanes(dim, p.cols);
  p.log2_bins = 8;
  while (vocab > (long long)IDX_ROWS << p.log2_bins) ++p.log2_bins;
  const long long bins = 1ll << p.log2_bins;
  p.rows = (int)((vocab + bins - 1) / bins);
  p.range = 0;
  // Pieces of 32 entries while they give the chip 8 wavefronts a compute unit, shorter ones below: 65536 tokens of 768 columns took
  // 56 us with 32, 58 with 16 and 62 with 8, 9973 of 1021 in fp32 53, 51 and 50.
  p.piece = 32;
  while (p.piece > BATCH && count * p.lanes / p.piece < 256 * 8 * DA_WAVE) p.piece /= 2;
  p.pieces = (int)((count + p.piece - 1) / p.piece);
  p.order = round256((size_t)(bins * p.rows) * sizeof(int2));
  p.kept = p.order + round256((size_t)p.pieces * p.piece * sizeof(int2));
  p.partial = p.kept + 256;
  // (the sorted parts are read before the first partial sum is written: they share their place)
  p.parted = p.partial;
  size_t parted = 0;
  if (p.log2_bins == PART_BITS && count > PART_FROM) {
    p.part = 1024 * (int)((count + 1024 * PARTS - 1) / (1024 * PARTS));
    p.parts = (int)((count + p.part - 1) / p.part);
    p.offsets = p.parted + round256((size_t)count * sizeof(int2));
    parted = p.offsets + (size_t)p.parts * (PART_BINS + 1) * sizeof(int);
  }
  const size_t sums = p.partial + (size_t)p.pieces * 2 * dim * sizeof(float);
  p.bytes = round256(sums > parted ? sums : parted);
  return p;
}

size_t index_lds(int rows) {
  return ((size_t)IDX_WAVES * rows + (size_t)IDX_WAVES * IDX_LIST * 2 + 2 * IDX_WAVES + 2 * PARTS) * sizeof(int);
}

template <typename G, typename W, int COLS>
int set_lds() {
  static DaOncePerDevice once;
  return once.run([] {
    for (const void* k : {reinterpret_cast<const void*>(embedding_index_kernel<false, W>), reinterpret_cast<const void*>(embedding_index_kernel<true, W>),
                          reinterpret_cast<const void*>(embedding_small_kernel<G, W, COLS>), reinterpret_cast<const void*>(embedding_small_kernel<G, W, 1>)}) {
      const hipError_t e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)index_lds(IDX_ROWS));
      if (e != hipSuccess) return (int)e;
    }
    return (int)DA_OK;
  });
}

constexpr long long MAX_BLOCKS = 1ll << 22;   // of 1024 threads: a launch has fewer than 2^32

template <typename G, typename W, int COLS>
int run_grad(const GradPlan& p, const IndexArgs& ia, const RowArgs& ra, long long vocab, hipStream_t s) {
  const int rc = set_lds<G, W, COLS>();
  if (rc) return rc;
  const int bins = 1 << p.log2_bins, slices = (p.lanes + DA_WAVE - 1) / DA_WAVE;
  if (ia.count <= SMALL_COUNT) {
    IndexArgs small = ia;
    small.kept = nullptr;
    if (p.cols == 1) hipLaunchKernelGGL((embedding_small_kernel<G, W, 1>), dim3(bins), dim3(IDX_THREADS), index_lds(p.rows), s, small, ra);
    else hipLaunchKernelGGL((embedding_small_kernel<G, W, COLS>), dim3(bins), dim3(IDX_THREADS), index_lds(p.rows), s, small, ra);
    return da_launch_status();
  }
  // the table's zeros: a third beside the sorting of the parts, where there is that launch, the rest beside the index
  const bool dense = ra.ldw == ra.dim;
  FillArgs fill{ra.dw, dense ? 0 : ra.ldw, dense ? vocab * ra.dim : ra.dim, 0, 0, 0};
  constexpr int FILL_COLS = 16 / sizeof(W);
  fill.lanes = fill.dim >= FILL_COLS ? (fill.dim + FILL_COLS - 1) / FILL_COLS : fill.dim;
  const long long units = ra.accumulate ? 0 : (dense ? 1 : vocab) * fill.lanes, span = (long long)FILL * IDX_THREADS;
  const long long early = p.parts ? units / 3 : 0;
  const long long early_blocks = (early + span - 1) / span, late_blocks = (units - early + span - 1) / span;
  const long long row_blocks = ((long long)p.pieces * p.lanes + 255) / 256;
  if (bins + late_blocks >= MAX_BLOCKS || row_blocks >= MAX_BLOCKS * 4 || (long long)p.pieces * slices >= MAX_BLOCKS * 4) return DA_ERR_LIMIT;
  if (p.parts) {
    fill.end = early;
    hipLaunchKernelGGL(embedding_part_kernel<W>, dim3((unsigned)(p.parts + early_blocks)), dim3(IDX_THREADS), 0, s, ia, fill);
  }
  fill.begin = early;
  fill.end = units;
  const dim3 index((unsigned)(bins + late_blocks));
  if (p.parts) hipLaunchKernelGGL((embedding_index_kernel<true, W>), index, dim3(IDX_THREADS), index_lds(p.rows), s, ia, fill);
  else hipLaunchKernelGGL((embedding_index_kernel<false, W>), index, dim3(IDX_THREADS), index_lds(p.rows), s, ia, fill);
  static_assert(SMALL_COUNT >= 32, "there is more than one piece from here on");
  const dim3 rows((unsigned)row_blocks), join((unsigned)((p.pieces - 1) * slices));
  if (p.cols == 1) hipLaunchKernelGGL((embedding_rows_kernel<G, W, 1>), rows, dim3(256), 0, s, ra);
  else hipLaunchKernelGGL((embedding_rows_kernel<G, W, COLS>), rows, dim3(256), 0, s, ra);
  if (p.cols == 1) hipLaunchKernelGGL((embedding_join_kernel<W, 1>), join, dim3(256), 0, s, ra, slices);
  else hipLaunchKernelGGL((embedding_join_kernel<W, COLS>), join, dim3(256), 0, s, ra, slices);
  return da_launch_status();
}

bool sizes_ok(long long count, long long vocab, int dim) { return count >= 0 && vocab > 0 && dim > 0; }
constexpr long long MAX_COUNT = 1ll << 25;

}  // namespace

extern "C" {

int dion_amd_embedding(const void* W, int w_dtype, long long ldw, long long vocab, int dim, const void* tokens, int index_bits,
                       long long count, void* out, int out_dtype, long long ldo, float scale, void* stream) {
  if (!sizes_ok(count, vocab, dim) || ldw < dim || ldo < dim || (index_bits != 32 && index_bits != 64)) return DA_ERR_ARG;
  if (!da_float_dtype(w_dtype) || !da_float_dtype(out_dtype)) return DA_ERR_DTYPE;
  if (count > MAX_COUNT || vocab > MAX_COUNT) return DA_ERR_LIMIT;
  if (count == 0) return DA_OK;
  if (!W || !tokens || !out) return DA_ERR_ARG;
  if (!da_aligned(W, da_esize(w_dtype)) || !da_aligned(out, da_esize(out_dtype)) || !da_aligned(tokens, index_bits / 8))
    return DA_ERR_ALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const DaIndex idx{tokens, index_bits == 64};
  DaProfScope prof(DA_PROF_EMBEDDING, (double)count * dim * (da_esize(w_dtype) + da_esize(out_dtype)), s);
  const int cols = dim >= 8 ? 8 : 1, lanes = da_lanes(dim, cols);
  if (count * lanes >= (1ll << 32) - 256 * UNITS) return DA_ERR_LIMIT;
  const dim3 grid((unsigned)((count * lanes + 256 * UNITS - 1) / (256 * UNITS)));
  const DaDivisor by_lanes = da_divisor((unsigned)lanes);
#define DA_LOOKUP(WT, OT)                                                                                                  \
  do {                                                                                                                     \
    if (cols > 1) hipLaunchKernelGGL((embedding_kernel<WT, OT, 8>), grid, dim3(256), 0, s, static_cast<const WT*>(W),     \
                                      ldw, vocab, dim, by_lanes, idx, count, static_cast<OT*>(out), ldo, scale);              \
    else hipLaunchKernelGGL((embedding_kernel<WT, OT, 1>), grid, dim3(256), 0, s, static_cast<const WT*>(W), ldw, vocab,   \
                            dim, by_lanes, idx, count, static_cast<OT*>(out), ldo, scale);                                    \
  } while (0)
  if (w_dtype == DA_BF16 && out_dtype == DA_BF16) DA_LOOKUP(bf16_t, bf16_t);
  else if (w_dtype == DA_BF16) DA_LOOKUP(bf16_t, float);
  else if (out_dtype == DA_BF16) DA_LOOKUP(float, bf16_t);
  else DA_LOOKUP(float, float);
#undef DA_LOOKUP
  return da_launch_status();
}

size_t dion_amd_embedding_grad_workspace_bytes(long long count, long long vocab, int dim) {
  if (!sizes_ok(count, vocab, dim) || count > MAX_COUNT || vocab > MAX_COUNT) return 0;
  return std::max(plan_grad(count, vocab, dim, DA_BF16).bytes, plan_grad(count, vocab, dim, DA_F32).bytes);
}

int dion_amd_embedding_grad(const void* G, int g_dtype, long long ldg, const void* tokens, int index_bits, long long count,
                            void* dW, int w_dtype, long long ldw, long long vocab, int dim, long long padding, float scale,
                            int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
  if (!sizes_ok(count, vocab, dim) || ldw < dim || ldg < dim || (index_bits != 32 && index_bits != 64)) return DA_ERR_ARG;
  if (!da_float_dtype(g_dtype) || !da_float_dtype(w_dtype)) return DA_ERR_DTYPE;
  if (count > MAX_COUNT || vocab > MAX_COUNT) return DA_ERR_LIMIT;
  if (!dW || (count && (!G || !tokens)) || !workspace) return DA_ERR_ARG;
  if (!da_aligned(G, da_esize(g_dtype)) || !da_aligned(dW, da_esize(w_dtype)) || !da_aligned(tokens, index_bits / 8) ||
      !da_aligned(workspace, 256))
    return DA_ERR_ALIGN;
  const GradPlan p = plan_grad(count, vocab, dim, g_dtype);
  if (workspace_bytes < p.bytes) return DA_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  DaProfScope prof(DA_PROF_EMBEDDING, (double)count * dim * da_esize(g_dtype) + (double)vocab * dim * da_esize(w_dtype), s);

  const IndexArgs ia{{tokens, index_bits == 64}, (int)vocab, padding >= 0 && padding < vocab ? (int)padding : -1, (int)count,
                     p.log2_bins, p.rows, reinterpret_cast<int2*>(ws + p.range), reinterpret_cast<int2*>(ws + p.order),
                     reinterpret_cast<int*>(ws + p.kept), p.part, p.parts, reinterpret_cast<int2*>(ws + p.parted),
                     reinterpret_cast<int*>(ws + p.offsets)};
  const RowArgs ra{ia.range, ia.order, ia.kept, p.log2_bins, p.rows, p.lanes, p.piece, p.pieces, G, ldg, dW, ldw,
                   reinterpret_cast<float*>(ws + p.partial), dim, accumulate, scale, da_divisor((unsigned)p.lanes)};
  if (g_dtype == DA_BF16 && w_dtype == DA_BF16) return run_grad<bf16_t, bf16_t, 8>(p, ia, ra, vocab, s);
  if (g_dtype == DA_BF16) return run_grad<bf16_t, float, 8>(p, ia, ra, vocab, s);
  if (w_dtype == DA_BF16) return run_grad<float, bf16_t, 4>(p, ia, ra, vocab, s);
  return run_grad<float, float, 4>(p, ia, ra, vocab, s);
}

}  // extern "C"
