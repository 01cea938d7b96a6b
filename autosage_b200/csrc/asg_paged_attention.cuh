// Attention of one new token per sequence over a paged cache: what its kernels share.
//
// The work is a flat list of units: a unit is kUnit consecutive tokens of one item, an item is one row
// (sequence) with the query heads of one group (up to GT heads that share a key head).  The list runs over
// rows, inside a row over items, inside an item over tokens, and each item is preceded by kStart empty units
// that stand for the cost of starting one (its query, its first pages, its result).  CTA c of G takes the
// entries [c S, (c + 1) S), S = ceil(total / G), so every CTA does the same work whatever the lengths are,
// one long row fills the GPU, and an item is cut only where a CTA's share ends.  A piece that is a whole item
// is normalised and stored at once; the others leave (max, sum, accumulator) in the workspace, at most two
// per CTA (the piece it begins with and the piece it ends with), and join_kernel puts them together in the
// order of the tokens, so results do not depend on timing.  Nothing waits on another CTA.
//
// Long sums.  A piece of more than an engine's kLeg units is computed in legs of that many; each ends like a piece, and what it
// has summed is added to what the legs before it left in the CTA's record.  Added up in one accumulator, the rounding
// of one sum after the other builds up: 2^20 tokens of equal weight and value in one piece were off by 1.5e-3 in float16
// (the tensor core cuts its sums off) and by 5e-4 in float32.
//
// Softmax: scores are kept in units of log2 (scale * log2(e) is a factor of q or of the score), each warp keeps a running
// maximum m, sum l and accumulator o of its tokens:
//   m' = max(m, s),  o' = o 2^(m - m') + 2^(s - m') v,  l' = l 2^(m - m') + 2^(s - m').
// m moves only when a score exceeds it by more than kSlack: weights up to 2^kSlack do no harm in float32, and most
// tiles then need neither the maximum over their lanes nor the rescaling (each of them a third of a tile's work).  Where such a
// weight makes a sum of very large values infinite, the piece is computed once more without slack (unsound()).
// With 8-bit pages the key scale multiplies the score and the value scale the weight; codes are never
// multiplied out in memory.
#pragma once

#include <math_constants.h>

#include <atomic>

#include "asg_paged.cuh"

namespace asg {
namespace paged {

constexpr int kRings = 4;                  // warps, or groups of warps, of a CTA; each takes every fourth tile of a piece
constexpr int kUnit = 64;                  // tokens per unit: one 16-token tile for each ring
constexpr int kTile = kUnit / kRings;
// Cost of starting an item, in units (where the GPU has more than a unit a CTA).  3 against 1, measured in turn: 75.4 against 81.8 us
// for 48 rows of up to 16384 e4m3 tokens of 4 x 128, 113 against 128 for 64 of up to 8192 int8 of 8 x 128, 42.8 against 46.0 for 192
// windows of 1024 bfloat16 of 1 x 256, 17.2 against 19.6 for 13 rows of up to 5001 int8; within 1 % on float16, float32 and single rows.
constexpr int kStart = 3;
constexpr float kSlack = 6.f;
constexpr float kNoScore = -3.402823466e38f; // m before the first score: every finite score is above it
constexpr int kMaxCtasPerSm = 4;           // bounds the workspace; no kernel is launched with more

struct AttentionArgs {
  const int64_t* crow;
  const int64_t* col;
  const int64_t* lengths;
  const void* q;
  void* out;
  float* lse;
  asg_page_pool key, value;
  long long q_token_stride, q_head_stride;
  long long n_cols, n_pages, window;
  int n_rows, page_size, n_heads, n_kv_heads, dim;
  int group;        // query heads per key head
  int subgroups;    // items per key head: ceil(group / GT)
  int type;         // of q and out
  float scale_log2; // scale * log2(e)
  bool q_fours;     // the query's rows start on four features' bytes
  bool join;        // the join kernel follows
  bool same_strides;  // of the pages of keys and values: one offset serves both
  bool out_vector;  // four neighbours of out can be stored at once
  int partial_pitch;
  float* partial;   // [G][2][GT][partial_pitch] accumulators of unfinished pieces
  float2* stats;    // [G][2][GT] their (m, l)
  int4* pieces;     // [G] (row, item, n, 0): CTA c starts an item that it does not finish, cut into n pieces; n = 0: none
};

size_t workspace_bytes_for(int ctas, int gt, int dim);

#ifdef __CUDACC__

// 64-bit quotients that mostly have 32-bit operands (a 64-bit division is some hundred instructions)
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if ((static_cast<unsigned long long>(a) | static_cast<unsigned long long>(b)) >> 32 == 0)
    return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}

// Tokens [first, last) of a row that are seen, and where its pages start in col.  Whatever the arrays hold,
// nothing outside them is addressed: crow is cut to [0, n_cols], lengths to what the pages hold.
struct RowSpan {
  long long first, last, pages_begin;
  __device__ __forceinline__ int units() const { return static_cast<int>((last - first + kUnit - 1) / kUnit); }
};
__device__ __forceinline__ RowSpan row_span(const AttentionArgs& a, int row) {
  const long long n_cols = a.n_cols;
  const long long lo = a.crow[row], hi = a.crow[row + 1], n = a.lengths[row];
  RowSpan s;
  s.pages_begin = lo < 0 ? 0 : (lo > n_cols ? n_cols : lo);
  const long long end = hi < s.pages_begin ? s.pages_begin : (hi > n_cols ? n_cols : hi);
  const long long held = (end - s.pages_begin) * a.page_size;
  s.last = n < 0 ? 0 : (n > held ? held : n);
  s.first = a.window > 0 && s.last > a.window ? s.last - a.window : 0;
  return s;
}

// Where a CTA's share begins.  The host has seen to it that entries have 31-bit numbers where crow is what it should be.
// Rows of any other crow may overlap and list more than 2^32 entries; sums of entries are unsigned and wrap then, several
// threads may find the share's first entry among their rows, and one of them is chosen: the span that all go by is
// one that row_span has cut, so nothing is addressed that should not be, and what is computed is nobody's.
struct Share {
  int pos, end;   // entries of the list
  int row_begin;  // entry at which the row begins
  int per_cta;
  int row;
  int start;      // empty units before each item
  RowSpan span;   // of the row
};

// Every thread sums the units of its rows, a block scan finds the row that holds the share's first entry.
template <int WARPS>
__device__ __forceinline__ Share locate_share(const AttentionArgs& a, int items_per_row) {
  __shared__ unsigned warp_units[WARPS], warp_rows[WARPS];
  __shared__ RowSpan found_span;
  __shared__ int found_row;
  __shared__ unsigned found_begin, claimed;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per_thread = (a.n_rows + WARPS * 32 - 1) / (WARPS * 32);
  const long long r0 = static_cast<long long>(tid) * per_thread;
  unsigned units = 0, rows = 0;
  for (long long r = r0; r < r0 + per_thread && r < a.n_rows; ++r) {
    const int here = row_span(a, static_cast<int>(r)).units();
    units += here;
    rows += here > 0;
  }
  unsigned units_scan = units, rows_scan = rows;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned u = __shfl_up_sync(kFull, units_scan, o), r = __shfl_up_sync(kFull, rows_scan, o);
    if (lane >= o) {
      units_scan += u;
      rows_scan += r;
    }
  }
  if (lane == 31) {
    warp_units[warp] = units_scan;
    warp_rows[warp] = rows_scan;
  }
  if (tid == 0) {
    found_row = -1;
    claimed = 0;
  }
  __syncthreads();
  unsigned units_before = units_scan - units, rows_before = rows_scan - rows, all_units = 0, all_rows = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) {
      units_before += warp_units[w];
      rows_before += warp_rows[w];
    }
    all_units += warp_units[w];
    all_rows += warp_rows[w];
  }
  Share s;
  const unsigned items = static_cast<unsigned>(items_per_row);
  s.start = all_units * items > gridDim.x ? kStart : 0;
  const unsigned total = min((all_units + s.start * all_rows) * items, 0x7fffffffu);
  s.per_cta = static_cast<int>((total + gridDim.x - 1) / gridDim.x);
  s.pos = static_cast<int>(min(static_cast<long long>(s.per_cta) * blockIdx.x, static_cast<long long>(total)));
  s.end = static_cast<int>(min(static_cast<long long>(s.pos) + s.per_cta, static_cast<long long>(total)));
  const unsigned pos = static_cast<unsigned>(s.pos);
  unsigned at = (units_before + s.start * rows_before) * items;
  // one thread has the entry among its rows
  if (s.pos < s.end && pos - at < (units + s.start * rows) * items && atomicExch(&claimed, 1u) == 0) {
    long long r = r0;
    RowSpan span = row_span(a, static_cast<int>(r));
    while (r + 1 < a.n_rows) {
      const unsigned n = span.units(), here = n > 0 ? (n + s.start) * items : 0;
      if (pos - at < here) break;
      at += here;
      span = row_span(a, static_cast<int>(++r));
    }
    found_row = static_cast<int>(r);
    found_begin = at;
    found_span = span;
  }
  __syncthreads();
  s.row = found_row;
  s.row_begin = static_cast<int>(found_begin);
  s.span = found_span;
  return s;
}

// First row after `row` that has units (there is one), looked for by all lanes together.
__device__ __forceinline__ int next_row(const AttentionArgs& a, int row) {
  for (int base = row + 1; base < a.n_rows; base += 32) {
    const int r = base + lane_id();
    const bool some = r < a.n_rows && row_span(a, r).units() > 0;
    const unsigned who = __ballot_sync(kFull, some);
    if (who != 0) return base + __ffs(who) - 1;
  }
  return a.n_rows;
}

__device__ __forceinline__ float load_wide(const void* p, long long i, int type) {
  if (type == ASG_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == ASG_TYPE_BF16) return __bfloat162float(static_cast<const BF16*>(p)[i]);
  return __half2float(static_cast<const F16*>(p)[i]);
}
__device__ __forceinline__ void store_wide(void* p, long long i, int type, float v) {
  if (type == ASG_TYPE_F32) static_cast<float*>(p)[i] = v;
  else if (type == ASG_TYPE_BF16) static_cast<BF16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<F16*>(p)[i] = __float2half_rn(v);
}

// 2^(m - top) as the factor of a part with maximum m and sum l; a part without tokens counts nothing,
// one that holds a NaN keeps it.
__device__ __forceinline__ float part_factor(float m, float l, float top) {
  return m == -CUDART_INF_F && l == 0.f ? 0.f : exp2f(m - top);
}
__device__ __forceinline__ float log_sum(float top, float sum) {
  return sum == 0.f ? -CUDART_INF_F : (top + log2f(sum)) * 0.6931471805599453f;
}

// Four neighbours, or what is left of them, of a result row.
__device__ __forceinline__ void store_four(const AttentionArgs& a, long long row, int d, float4 v) {
  const long long at = row * a.dim + d;
  if (a.out_vector) {
    if (a.type == ASG_TYPE_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = v;
    } else {
      uint2 two;
      if (a.type == ASG_TYPE_BF16) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
        two = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
      } else {
        const __half2 x = __floats2half2_rn(v.x, v.y), y = __floats2half2_rn(v.z, v.w);
        two = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
      }
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = two;
    }
    return;
  }
  const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (d + i < a.dim) store_wide(a.out, at + i, a.type, x[i]);
}

// The rings' parts of one piece lie in shared memory: ring w's accumulators o[w * ring_stride + g * PITCH + d] and
// ml[w * GT + g] = (m, l).  Puts them together with the record of the legs before (`more`) and stores the result (`whole`: the
// item is complete) or a partial record.  A thread writes and reads the same parts of a record.  All threads call it
// between barriers.
template <int THREADS, int GT, int DIM, int PITCH>
__device__ __forceinline__ void store_piece(const AttentionArgs& a, int row, int kv_head, int sub, int slot, bool more, bool whole,
                                            const float* o, int ring_stride, const float2* ml) {
  __shared__ float4 factors[GT];
  __shared__ float factors_before[GT];
  static_assert(kRings == 4, "one float4 of factors per head");
  const int heads = min(GT, a.group - sub * GT);
  const long long first_row = static_cast<long long>(row) * a.n_heads + kv_head * a.group + sub * GT;
  const long long first_record = (static_cast<long long>(blockIdx.x) * 2 + slot) * GT;
  const int tid = threadIdx.x;
  if (tid < heads) {
    float2 part[kRings];
    float top = -CUDART_INF_F, sum = 0.f, f[kRings];
#pragma unroll
    for (int w = 0; w < kRings; ++w) {
      part[w] = ml[w * GT + tid];
      top = fmaxf(top, part[w].x);
    }
    float2 before = make_float2(-CUDART_INF_F, 0.f);
    if (more) before = a.stats[first_record + tid];
    top = fmaxf(top, before.x);
    const float f_before = part_factor(before.x, before.y, top);
    sum = f_before * before.y;
#pragma unroll
    for (int w = 0; w < kRings; ++w) {
      f[w] = part_factor(part[w].x, part[w].y, top);
      sum += f[w] * part[w].y;
    }
    float scale = 1.f;
    if (whole) {
      scale = sum == 0.f ? 0.f : 1.f / sum;
      if (a.lse != nullptr) a.lse[first_row + tid] = log_sum(top, sum);
    } else {
      a.stats[first_record + tid] = make_float2(top, sum);
    }
    factors[tid] = make_float4(f[0] * scale, f[1] * scale, f[2] * scale, f[3] * scale);
    factors_before[tid] = f_before * scale;
  }
  __syncthreads();
  constexpr int kFours = DIM / 4;
  for (int i = tid; i < heads * kFours; i += THREADS) {
    const int g = i / kFours, d = i % kFours * 4;
    if (d >= a.dim) continue;
    const float4 f = factors[g];
    const float* at = o + g * PITCH + d;
    const float4 x0 = *reinterpret_cast<const float4*>(at), x1 = *reinterpret_cast<const float4*>(at + ring_stride),
                 x2 = *reinterpret_cast<const float4*>(at + 2 * ring_stride), x3 = *reinterpret_cast<const float4*>(at + 3 * ring_stride);
    float4 v = make_float4(f.x * x0.x + f.y * x1.x + f.z * x2.x + f.w * x3.x, f.x * x0.y + f.y * x1.y + f.z * x2.y + f.w * x3.y,
                                 f.x * x0.z + f.y * x1.z + f.z * x2.z + f.w * x3.z, f.x * x0.w + f.y * x1.w + f.z * x2.w + f.w * x3.w);
    float4* record = reinterpret_cast<float4*>(a.partial + (first_record + g) * a.partial_pitch + d);
    if (more) {
      const float4 x = *record;
      const float fb = factors_before[g];
      v = make_float4(v.x + fb * x.x, v.y + fb * x.y, v.z + fb * x.z, v.w + fb * x.w);
    }
    if (whole) store_four(a, first_row + g, d, v);
    else *record = v;
  }
}

// Rows that see nothing: block `block` of `blocks` clears its share of them.
__device__ __forceinline__ void clear_empty_rows(const AttentionArgs& a, int block, int blocks) {
  for (long long r = block; r < a.n_rows; r += blocks) {
    if (row_span(a, static_cast<int>(r)).units() > 0) continue;
    for (int i = threadIdx.x; i < a.n_heads * a.dim; i += blockDim.x)
      store_wide(a.out, r * a.n_heads * a.dim + i, a.type, 0.f);
    if (a.lse != nullptr)
      for (int h = threadIdx.x; h < a.n_heads; h += blockDim.x) a.lse[r * a.n_heads + h] = -CUDART_INF_F;
  }
}

// One piece of a CTA's share, or a leg of it.
struct Piece {
  RowSpan span;
  int row, item, kv_head, sub;
  int entry;          // of the list at which the item's tokens begin
  int units, u0, u1;  // of the item; the leg's
  int from, to;       // the piece's
  __device__ __forceinline__ long long first() const { return span.first + static_cast<long long>(u0) * kUnit; }
  __device__ __forceinline__ long long last() const { return u1 == units ? span.last : span.first + static_cast<long long>(u1) * kUnit; }
  __device__ __forceinline__ bool any() const { return u0 < u1; }
};

// Walks through a share.
struct Walk {
  Share s;
  RowSpan span;
  int units, at;  // of the row's items; entry inside the item
  int began;      // entry inside the item at which the piece begins
  int item, items_per_row;
  __device__ __forceinline__ void begin(int items, const Share& share) {
    s = share;
    items_per_row = items;
    if (s.pos >= s.end) return;
    span = s.span;
    units = s.row < 0 ? 0 : span.units();
    const unsigned into = static_cast<unsigned>(s.pos) - static_cast<unsigned>(s.row_begin);
    const unsigned entries = static_cast<unsigned>(units + s.start);
    // crow is not what it should be: rows that overlap can list more than 2^31 entries, whose numbers are then wrong
    if (units <= 0 || into / entries >= static_cast<unsigned>(items)) {
      s.pos = s.end;
      return;
    }
    item = static_cast<int>(into / entries);
    at = began = static_cast<int>(into - item * entries);
  }
  // The next leg, of at most `leg` units, that has tokens, or one without (all lanes of a warp).
  __device__ __forceinline__ Piece next(const AttentionArgs& a, int leg) {
    Piece p;
    while (s.pos < s.end) {
      const int entries = units + s.start, to = min(entries, at + (s.end - s.pos));
      p.span = span;
      p.row = s.row;
      p.item = item;
      p.units = units;
      p.entry = s.pos - at + s.start;
      const int stop = min(to, max(at, s.start) + leg);
      p.u0 = max(at - s.start, 0);
      p.u1 = max(stop - s.start, 0);
      p.from = max(began - s.start, 0);
      p.to = max(to - s.start, 0);
      s.pos += stop - at;
      at = stop;
      if (stop == to) {
        at = began = 0;
        if (s.pos < s.end && ++item == items_per_row) {
          item = 0;
          s.row = next_row(a, s.row);
          if (s.row >= a.n_rows) s.pos = s.end;
          else span = row_span(a, s.row);
          units = span.units();
        }
      }
      if (p.any()) {
        p.kv_head = p.item / a.subgroups;
        p.sub = p.item - p.kv_head * a.subgroups;
        return p;
      }
    }
    p.u0 = p.u1 = 0;
    return p;
  }
};

// The copies of a ring: where they come from and how far they are.  Lane l looks after token l % 16 of the next
// tile: the page of the table it lies in, its place there, and the page's id, loaded one tile ahead.
struct Source {
  const char* keys;
  const char* values;
  const int64_t* ids;                 // of the page that holds the piece's first token
  long long page_bytes, token_bytes;  // of the keys' pages
  int kv_head, count, tile;
  int nth, place;
  int step_pages, step_place;         // kUnit tokens on
  long long id;

  __device__ __forceinline__ void start(const AttentionArgs& a, const Piece& p, int ring, int item_bytes) {
    keys = static_cast<const char*>(a.key.data) + p.kv_head * a.key.head_stride * item_bytes;
    values = static_cast<const char*>(a.value.data) + p.kv_head * a.value.head_stride * item_bytes;
    page_bytes = a.key.page_stride * item_bytes;
    token_bytes = a.key.token_stride * item_bytes;
    kv_head = p.kv_head;
    const unsigned page_size = static_cast<unsigned>(a.page_size);
    const long long first = p.first(), page0 = quotient(first, a.page_size);  // 32-bit page arithmetic from here on
    ids = a.col + p.span.pages_begin + page0;
    count = static_cast<int>(p.last() - first);
    tile = ring * kTile;
    const unsigned at = static_cast<unsigned>(first - page0 * a.page_size) + tile + (lane_id() & (kTile - 1));
    nth = static_cast<int>(at / page_size);
    place = static_cast<int>(at % page_size);
    step_pages = static_cast<int>(kUnit / page_size);
    step_place = static_cast<int>(kUnit % page_size);
    look_up();
  }
  __device__ __forceinline__ void look_up() { id = tile + (lane_id() & (kTile - 1)) < count ? ids[nth] : -1; }
  __device__ __forceinline__ void advance(const AttentionArgs& a) {
    tile += kUnit;
    nth += step_pages;
    place += step_place;
    if (place >= a.page_size) {
      place -= a.page_size;
      ++nth;
    }
    look_up();
  }
};

// bytes of global memory into shared memory, zeros if !ok (nothing is read then)
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool ok) {
  static_assert(BYTES == 4 || BYTES == 8 || BYTES == 16, "sizes of cp.async");
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(ok ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(ok ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 2^x and log2(x) of the hardware (results and arguments below the normal range count as 0)
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A part's maximum as the joins know it: minus infinity where no score has been.
__device__ __forceinline__ float published_max(float m) { return m == kNoScore ? -CUDART_INF_F : m; }

// The kernel around an Engine, which computes one ring's part of a piece:
//   kLeg                              units after which sums are put away
//   Engine(smem)                      once
//   fetch(a, piece)                   loads the piece's query; the part of the piece before is still unpublished
//   start(a, piece)                   begins to copy the piece's tokens
//   query(a)                          takes the query and clears the accumulators
//   run(a)                            the ring's tiles
//   unsound(a, piece)                 whether a sum that run() has left cannot stand (the same for all lanes of a ring)
//   drain()                           waits for the copies that were started
//   run_carefully(a)                  the ring's tiles once more, however long it takes
//   publish(smem, ml)                 its part into shared memory: float o[kHeads][kPitch] at smem + ring * kRingBytes +
//                                     kPublish, which no copy of a started piece writes before run()
// kRingBytes * kRings bytes of shared memory belong to the engine, the (m, l) pairs lie behind them.
template <typename Engine>
__global__ void __launch_bounds__(Engine::kThreads, Engine::kCtasPerSm) attention_kernel(const AttentionArgs a) {
  constexpr int GT = Engine::kHeads;
  extern __shared__ __align__(128) unsigned char smem[];
  pdl_wait_for_primary();  // launched while the kernel before on the stream ends
  pdl_release_dependents();
  // The walk and the pieces it finds live in shared memory: the loop over tiles wants the registers.  The first warp looks
  // two pieces ahead, so that the barriers of a piece are all that the others need to see the next one.
  __shared__ Walk shared_walk;
  __shared__ Piece pieces[3];
  const bool first_warp = threadIdx.x < 32, first_lane = threadIdx.x == 0;
  {
    const int items_per_row = a.n_kv_heads * a.subgroups;
    const Share share = locate_share<Engine::kThreads / 32>(a, items_per_row);
    if (first_warp) {
      Walk walk;
      walk.begin(items_per_row, share);
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const Piece p = walk.next(a, Engine::kLeg);
        if (first_lane) pieces[i] = p;
      }
      if (first_lane) shared_walk = walk;
    }
    if (a.join && first_lane) a.pieces[blockIdx.x] = make_int4(0, 0, 0, 0);
    __syncthreads();
  }
  if (pieces[0].any()) {
    Engine engine(smem);
    const float* o = reinterpret_cast<const float*>(smem + Engine::kPublish);
    float2* ml = reinterpret_cast<float2*>(smem + kRings * Engine::kRingBytes);
    engine.fetch(a, pieces[0]);
    engine.start(a, pieces[0]);
    engine.query(a);
    for (int now = 0;;) {
      const int next = now == 2 ? 0 : now + 1, after = next == 2 ? 0 : next + 1;
      if (first_warp) {
        Walk walk = shared_walk;
        __syncwarp();  // all lanes have their copy before the first one replaces it
        const Piece p = walk.next(a, Engine::kLeg);
        if (first_lane) {
          pieces[after] = p;
          shared_walk = walk;
        }
      }
      engine.run(a);
      const bool more = pieces[next].any();
      if (more) {
        engine.fetch(a, pieces[next]);
        engine.start(a, pieces[next]);
      }
      if (engine.unsound(a, pieces[now])) {  // (looked at while the copies are under way)
        engine.drain();
        engine.fetch(a, pieces[now]);
        engine.start(a, pieces[now]);
        engine.query(a);
        engine.run_carefully(a);
        if (more) {
          engine.fetch(a, pieces[next]);
          engine.start(a, pieces[next]);
        }
      }
      engine.publish(smem, ml);
      if (more) engine.query(a);
      __syncthreads();
      const Piece& p = pieces[now];
      const bool ends = p.u1 == p.to, whole = p.from == 0 && p.to == p.units;
      const int slot = p.from > 0 ? 0 : 1;  // (legs of a whole item: the record of the item that the CTA does not finish is still free)
      if (slot == 1 && ends && !whole && first_lane)  // the CTA of the item's last unit is the one of its last piece
        a.pieces[blockIdx.x] = make_int4(p.row, p.item, (p.entry + p.units - 1) / shared_walk.s.per_cta - static_cast<int>(blockIdx.x) + 1, 0);
      store_piece<Engine::kThreads, GT, Engine::kDim, Engine::kPitch>(a, p.row, p.kv_head, p.sub, slot, p.u0 > p.from, whole && ends, o,
                                                                                 Engine::kRingBytes / 4, ml);
      __syncthreads();  // the buffers are free again
      if (!more) break;
      now = next;
    }
  }
  if (!a.join) clear_empty_rows(a, blockIdx.x, gridDim.x);  // otherwise the join kernel does, while this one runs
}

// Host: launch of one instance.
template <typename Engine>
int launch_engine(const AttentionArgs& args, int ctas, cudaStream_t stream) {
  constexpr int smem = kRings * (Engine::kRingBytes + Engine::kHeads * static_cast<int>(sizeof(float2)));
  static_assert(Engine::kRingBytes >= Engine::kPublish + Engine::kHeads * Engine::kPitch * 4 && Engine::kRingBytes % 128 == 0, "ring region");
  static_assert(Engine::kCtasPerSm <= kMaxCtasPerSm && Engine::kCtasPerSm * (smem + 1024) <= 228 * 1024, "shared memory");
  auto kernel = attention_kernel<Engine>;
  if (smem > 48 * 1024) {  // once per device
    static std::atomic<unsigned long long> known{0};
    int device = 0;
    ASG_CUDA(cudaGetDevice(&device));
    const unsigned long long bit = 1ull << (device & 63);
    if ((known.load(std::memory_order_relaxed) & bit) == 0) {
      ASG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      if (device < 64) known.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  ASG_CUDA(launch_overlapped(kernel, ctas, Engine::kThreads, static_cast<size_t>(smem), stream, args));
  return ASG_OK;
}

#endif  // __CUDACC__

// What a family of engines would launch for given sizes; `launch` null: the family does not take them.
struct Choice {
  int gt = 0;          // query heads per item
  int ctas_per_sm = 0;
  int (*launch)(const AttentionArgs&, int ctas, cudaStream_t) = nullptr;
};
Choice choose_general(const AttentionArgs& a, int cache_type);  // asg_paged_general.cu
Choice choose_tensor16(const AttentionArgs& a, int cache_type); // asg_paged_tensor16.cu
Choice choose_tensor8(const AttentionArgs& a, int cache_type);  // asg_paged_tensor8.cu

template <typename Engine>
inline Choice made() {
  Choice c;
  c.gt = Engine::kHeads;
  c.ctas_per_sm = Engine::kCtasPerSm;
  c.launch = launch_engine<Engine>;
  return c;
}

}  // namespace paged
}  // namespace asg
