// Paged attention on the tensor cores: 16-bit queries with 16-bit pages, any query with 8-bit pages.
//
// A decoding step multiplies each key with the few query heads of its group, so it is bound by the bytes of
// the cache; what the kernel has to do is keep enough of them in flight and stay out of their way.  The
// tiles are far too thin for tcgen05 (its smallest tile is 64 or 128 rows on a side that here holds 1 to 16
// query heads, or 8 columns against 128 tokens whose rows would have to be gathered into one swizzled operand), so
// the products use the warp-level instruction m16n8k16 with the TOKENS as its 16 rows and the query heads as
// its 8 columns: half the instructions of the other orientation for groups of up to 8.
//
//   S^T[16 tokens x 8 heads] = K Q^T      A = K rows (ldmatrix), B = Q^T in registers for the whole item
//   O^T[16 d x 8 heads]     += V^T P^T    A = V columns (ldmatrix.trans), B = the weights: S^T's registers
//                                         packed to 16 bits and transposed by movmatrix, no trip to memory
// The weights enter as two 16-bit pieces (p = hi + lo, 2^-17 of p lost at most), so that the result is as
// good as one with float32 weights: the second product costs nothing while the kernel waits for memory.
// An infinite value times two pieces is not what it is times their sum (lo may be 0 or negative, and so may a weight's hi
// be 0).  Such a value leaves a sum that is not finite, and so may a large one times a weight above 1 (kSlack); a ring
// that ends a piece with such a sum goes through it again, holds weights to 1 and multiplies them in float32 with single
// values on the FMA pipe (run_carefully), which costs nothing where all is finite.
//
// Each warp works alone (with more than 8 heads, two warps share a ring): 16-token tiles, a ring of kStages tiles in
// shared memory filled by cp.async 16 bytes at a time (rows swizzled or padded, so ldmatrix is free of bank
// conflicts), page ids fetched one tile ahead of the copies that need them.  The warps of a CTA meet only at the end
// of a piece.
//
// 8-bit pages.  Codes stay codes in shared memory and become f16 numbers in registers, exactly:
//   int8   0x6400 | (c + 128) is the number 1024 + c + 128; subtract 1152
//   e4m3   the hardware's conversion of two at a time
// A byte-wise ldmatrix hands a lane four neighbouring features of a token (K) or two features of two tokens
// (V, transposed in 16-bit units); the order of features inside a k-step or of output rows inside a block
// is free, so Q and O are simply laid out to match.  f16 holds codes whole but not every scale, so
//   - a query head is multiplied by the power of two that brings its largest feature into [1, 2) (features
//     below 2^-14 of that lose what lies below 2^-24 of it), undone in the factor of its scores;
//   - the accumulator is held 2^-d times its value, 2^d about the largest 2^(s_t - m) |c_t| so far with value scales
//     c_t: its weights, 2^(s_t - m) of the sum times c_t 2^-d, are small numbers whatever the scales are.  d is
//     a whole number, so that taking 2^-d back in the end rounds nothing.
//
// float32 queries with 8-bit pages (WIDE).  Codes are exact in f16, so only the query and the weights need their 24
// bits: a feature x enters as h1 + 2^-12 h2, h1 = f16(x), h2 = f16(2^12 (x - h1)), which is x to 2^-24, each with
// sums of its own; weights are hi + lo as before (2^-23 of a weight, 2^-33 of the largest).  The tensor core cuts its sums
// off rather than rounding them, so nothing is added up in it over more than two steps: its results are added
// in float32 by the FMA pipe.  (64 rows of up to 8192 tokens of 8 x 128 int8: 132 us, on the FMA pipe alone 308.)
#pragma once

#include "asg_paged_attention.cuh"

namespace asg {
namespace paged {

#ifdef __CUDACC__

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename H>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<BF16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<F16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two floats as two 16-bit numbers (first in the low half), and what they lose.
template <typename H> __device__ __forceinline__ uint32_t pack2(float a, float b, float& rest_a, float& rest_b);
template <>
__device__ __forceinline__ uint32_t pack2<BF16>(float a, float b, float& rest_a, float& rest_b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  const float2 f = __bfloat1622float2(h);
  rest_a = a - f.x;
  rest_b = b - f.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<F16>(float a, float b, float& rest_a, float& rest_b) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  rest_a = a - f.x;
  rest_b = b - f.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Four codes as four f16 numbers: bytes 0 and 1 in `a`, 2 and 3 in `b`.
__device__ __forceinline__ void decode_neighbours(uint32_t x, uint32_t& a, uint32_t& b, INT8) {
  const uint32_t lifted = x ^ 0x80808080u;
  const uint32_t u = __byte_perm(lifted, 0x64646464u, 0x4140), v = __byte_perm(lifted, 0x64646464u, 0x4342);
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));
  const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&u), bias), q = __hsub2(*reinterpret_cast<const __half2*>(&v), bias);
  a = *reinterpret_cast<const uint32_t*>(&p);
  b = *reinterpret_cast<const uint32_t*>(&q);
}
__device__ __forceinline__ void decode_neighbours(uint32_t x, uint32_t& a, uint32_t& b, E4M3) {
  asm("{\n\t.reg .b16 low, high;\n\tmov.b32 {low, high}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, low;\n\tcvt.rn.f16x2.e4m3x2 %1, high;\n\t}"
      : "=r"(a), "=r"(b) : "r"(x));
}
// Bytes 0 and 2 in `a`, 1 and 3 in `b`.
template <typename T>
__device__ __forceinline__ void decode_alternate(uint32_t x, uint32_t& a, uint32_t& b, T type) {
  decode_neighbours(__byte_perm(x, 0u, 0x3120), a, b, type);
}

// T: type of the pages; DP: features, padded; SHARE: warps that share a ring's tiles, each with 8 query heads of its own;
// WIDE: the query is float32.
template <typename T, int DP, int SHARE, int STAGES, int CTAS, bool WIDE = false>
struct Tensor {
  static constexpr int kThreads = kRings * SHARE * 32;
  static constexpr int kHeads = 8 * SHARE;
  static constexpr int kCtasPerSm = CTAS;
  static constexpr int kStages = STAGES;
  static constexpr int kLeg = 128;  // 2 x 128 sums cut off by 2^-23 at most (mean 2^-24): 3e-5
  static constexpr bool kCoded = TypeOf<T>::coded;
  static constexpr int kRowBytes = DP * static_cast<int>(sizeof(T));
  // Rows of 128 bytes: the 16-byte piece c of row r lies at place c ^ (r mod 8); other rows are padded by 16 bytes.
  // Either way the eight rows that an ldmatrix reads lie in different banks.
  static constexpr bool kSwizzled = kRowBytes == 128;
  static constexpr int kRowPitch = kSwizzled ? kRowBytes : kRowBytes + 16;
  static constexpr int kChunks = kRowBytes / 16;                    // 16-byte pieces of a row
  static constexpr int kValues = kTile * kRowPitch;                 // offset of the V tile in a stage
  static constexpr int kExtras = 2 * kTile * kRowPitch;             // then the scales (key, value), then the mask of seen tokens
  static constexpr int kStageAlign = kSwizzled ? 128 : 16;
  static constexpr int kStageBytes = (kExtras + (kCoded ? 2 * kTile * 4 : 0) + 4 + kStageAlign - 1) / kStageAlign * kStageAlign;
  static constexpr int kDim = DP;
  static constexpr int kPitch = DP + 4;                             // of the published accumulators: no bank conflicts
  static constexpr int kPublish = (kStages - 1) * kStageBytes;      // the next piece's first copies go to the stages before it
  static constexpr int kNeed = kPublish + (kStageBytes > kHeads * kPitch * 4 ? kStageBytes : kHeads * kPitch * 4);
  static constexpr int kRingBytes = (kNeed + 127) / 128 * 128;
  static constexpr int kSteps = DP / 16;
  using H = typename std::conditional<kCoded, F16, T>::type;        // type of the products
  // f16 weights are held 2^8 above their value: the pieces of small weights stay clear of f16's smallest step, and
  // with kSlack there are still two powers of two to its largest number
  static constexpr float kLift = std::is_same<H, F16>::value ? 8.f : 0.f;
  static_assert(kSlack + 8.f <= 15.f, "weights in f16");

  static_assert(!WIDE || kCoded, "float32 queries go with 8-bit pages");
  // d stays in range of float32 exponents: larger scales overflow anyway, smaller ones count little, and a weight (2^14 at
  // most) times 2^-d is finite, so that a weight of 0 makes 0 of every value scale
  static constexpr float kLeastD = -112.f, kMostD = 120.f;
  static __device__ __forceinline__ float power_of_two(float n) { return __int_as_float((127 + static_cast<int>(n)) << 23); }

  uint32_t q[kSteps][2];
  uint32_t q2[WIDE ? kSteps : 1][2];  // second pieces
  float o[kSteps][4];
  float dots[2][4];         // the next tile's scores: two sums to be added (WIDE: of the first and of the second pieces)
  uint32_t high[2], low[2]; // this tile's weights
  float m[2], l[2];  // of heads 2 (lane % 4) + {0, 1} of the warp's eight
  float d[2];        // 8-bit pages: the accumulator's power of two, 2^-d, ...
  float held[2];
  float unit[2];     // ... and what undoes the query's power of two
  int lane, ring, part;
  uint32_t base;     // shared address of the ring's region
  Source s;

  __device__ __forceinline__ explicit Tensor(unsigned char* smem)
      : lane(threadIdx.x & 31), ring((threadIdx.x >> 5) % kRings), part((threadIdx.x >> 5) / kRings),
        base(smem_u32(smem) + ring * kRingBytes) {}

  // All lanes of the ring's warps.
  __device__ __forceinline__ void meet() const {
    if constexpr (SHARE == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + ring), "n"(SHARE * 32) : "memory");
  }

  // Feature that a lane's register holds in step `step`: entry 0 or 1 of the pair `half`.
  static __device__ __forceinline__ int query_feature(int step, int lane, int half, int entry) {
    return kCoded ? 16 * step + 4 * (lane & 3) + 2 * half + entry : 16 * step + 8 * half + 2 * (lane & 3) + entry;
  }
  static __device__ __forceinline__ int output_feature(int step, int lane, int half) {
    return kCoded ? 16 * step + 2 * (lane >> 2) + half : 16 * step + 8 * half + (lane >> 2);
  }

  // The four query features that a lane holds in a step, as they lie in memory (16 bits each; 8-bit pages: four
  // neighbours, 16-bit pages: two pairs of neighbours).
  static __device__ __forceinline__ uint2 load_query(const AttentionArgs& a, const uint16_t* row, bool ok, int step, int lane) {
    const int d0 = query_feature(step, lane, 0, 0), d1 = query_feature(step, lane, 1, 0);
    uint2 x = make_uint2(0u, 0u);
    if (a.q_fours) {  // whole pairs lie inside or outside the head
      if constexpr (kCoded) {
        if (ok && d0 < a.dim) x = *reinterpret_cast<const uint2*>(row + d0);
      } else {
        if (ok && d0 < a.dim) x.x = *reinterpret_cast<const uint32_t*>(row + d0);
        if (ok && d1 < a.dim) x.y = *reinterpret_cast<const uint32_t*>(row + d1);
      }
    } else if (ok) {
      if (d0 < a.dim) x.x = row[d0] | static_cast<uint32_t>(row[d0 + 1]) << 16;
      if (d1 < a.dim) x.y = row[d1] | static_cast<uint32_t>(row[d1 + 1]) << 16;
    }
    return x;
  }
  static __device__ __forceinline__ float2 widen(uint32_t pair, bool bf16) {
    return bf16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&pair)) : __half22float2(*reinterpret_cast<const __half2*>(&pair));
  }

  __device__ __forceinline__ void fetch(const AttentionArgs& a, const Piece& p) {
    const int first = p.sub * kHeads + 8 * part, h = lane >> 2;  // of the group's heads
    const bool ok = first + h < a.group;
    const long long from = p.row * a.q_token_stride + (static_cast<long long>(p.kv_head) * a.group + first + h) * a.q_head_stride;
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      if constexpr (WIDE) {  // four neighbours, held in the registers of both pieces until query()
        const float* row = static_cast<const float*>(a.q) + from;
        const int d = query_feature(step, lane, 0, 0);
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (ok && d < a.dim) {
          if (a.q_fours) x = *reinterpret_cast<const uint4*>(row + d);
          else x = make_uint4(__float_as_uint(row[d]), __float_as_uint(row[d + 1]), __float_as_uint(row[d + 2]), __float_as_uint(row[d + 3]));
        }
        q[step][0] = x.x;
        q[step][1] = x.y;
        q2[step][0] = x.z;
        q2[step][1] = x.w;
      } else {
        const uint2 x = load_query(a, static_cast<const uint16_t*>(a.q) + from, ok, step, lane);
        q[step][0] = x.x;
        q[step][1] = x.y;
      }
    }
  }

  // The fetched features of pair `half` of a step as floats.
  __device__ __forceinline__ float2 fetched(int step, int half, bool bf16) const {
    if constexpr (WIDE)
      return half == 0 ? make_float2(__uint_as_float(q[step][0]), __uint_as_float(q[step][1]))
                       : make_float2(__uint_as_float(q2[step][0]), __uint_as_float(q2[step][1]));
    else
      return widen(q[step][half], bf16);
  }

  __device__ __forceinline__ void query(const AttentionArgs& a) {
    if constexpr (kCoded) {
      const bool bf16 = a.type == ASG_TYPE_BF16;
      float top = 0.f;
#pragma unroll
      for (int step = 0; step < kSteps; ++step)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float2 x = fetched(step, half, bf16);
          top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
        }
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
      // top in [2^power, 2^(power + 1)), cut to powers whose inverse is a normal number: 2^127 becomes 2, an infinity stays one
      const int power = min(max((__float_as_int(top) >> 23) - 127, -126), 126);
      const float down = __int_as_float((127 - power) << 23), up = __int_as_float((127 + power) << 23);
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        const float2 x = fetched(step, 0, bf16), y = fetched(step, 1, bf16);
        float rest[4], none0, none1;
        q[step][0] = pack2<F16>(x.x * down, x.y * down, rest[0], rest[1]);
        q[step][1] = pack2<F16>(y.x * down, y.y * down, rest[2], rest[3]);
        if constexpr (WIDE) {
          q2[step][0] = pack2<F16>(rest[0] * 4096.f, rest[1] * 4096.f, none0, none1);
          q2[step][1] = pack2<F16>(rest[2] * 4096.f, rest[3] * 4096.f, none0, none1);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        unit[i] = a.scale_log2 * __shfl_sync(kFull, up, 4 * (2 * (lane & 3) + i));
        d[i] = kLeastD;
        held[i] = power_of_two(-kLeastD);
      }
    }
#pragma unroll
    for (int step = 0; step < kSteps; ++step)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[step][i] = 0.f;
    m[0] = m[1] = kNoScore;
    l[0] = l[1] = 0.f;
  }

  // Copies the tile at token `tile` to a stage, given where the lane's token lies; the ring's warps take every SHARE-th
  // of its rows.
  __device__ __forceinline__ void copy(const AttentionArgs& a, int stage, int tile, long long id, int place) {
    if (tile < s.count) {
      const bool held = id >= 0 && id < a.n_pages;
      const unsigned seen = __ballot_sync(kFull, held) & 0xffffu;
      const long long offset = held ? id * s.page_bytes + place * s.token_bytes : 0;
      const int offset_low = static_cast<int>(offset), offset_high = static_cast<int>(offset >> 32);
      const uint32_t at = base + stage * kStageBytes;
      constexpr int kLines = 32 / kChunks;  // rows that one copy of all lanes covers
      const int chunk = lane % kChunks * 16, line0 = part * kLines + lane / kChunks;
      const uint32_t to = at + line0 * kRowPitch, piece = kSwizzled ? chunk ^ (line0 & 7) * 16 : chunk;
      const bool inside = chunk < a.dim * static_cast<int>(sizeof(T));
#pragma unroll
      for (int n = 0; n < kTile / kLines / SHARE; ++n) {
        const int line = n * kLines * SHARE + line0;
        const unsigned low = static_cast<unsigned>(__shfl_sync(kFull, offset_low, line));
        const int high = __shfl_sync(kFull, offset_high, line);
        const long long from = (static_cast<long long>(high) << 32 | low) + chunk;
        // zeros for a token that is not seen and for features past the head's end
        const bool ok = inside && (seen >> line & 1u) != 0;
        const int rows = n * kLines * SHARE;  // (a multiple of a power of two above line0: the bits do not meet)
        const uint32_t here = to + rows * kRowPitch + (kSwizzled ? piece ^ (rows & 7) * 16 : piece);
        copy_async<16>(here, s.keys + from, ok);
        copy_async<16>(here + kValues, s.values + from, ok);
      }
      if (part == 0) {
        if constexpr (kCoded) {
          const asg_page_pool& pool = lane < kTile ? a.key : a.value;
          const float* from = pool.scales + s.kv_head * pool.scale_head_stride;
          if (held) from += id * pool.scale_page_stride + place * pool.scale_token_stride;
          copy_async<4>(at + kExtras + lane * 4, from, held);
        }
        if (lane == 0) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + kStageBytes - 4), "r"(seen) : "memory");
      }
    }
    copy_commit();
  }

  __device__ __forceinline__ void start(const AttentionArgs& a, const Piece& p) {
    s.start(a, p, ring, static_cast<int>(sizeof(T)));
    const int first = s.tile;
    long long id[kStages - 1];  // the page ids of all tiles are asked for before the first is needed
    int place[kStages - 1];
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      id[i] = s.id;
      place[i] = s.place;
      s.advance(a);
    }
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) copy(a, i, first + i * kUnit, id[i], place[i]);
  }

  // A tile's products with V are issued together with the next tile's products with K: the two chains hide one
  // another's latency, and the softmax between them is all that a warp ever waits for alone.
  __device__ __forceinline__ void run(const AttentionArgs& a) {
    const int tiles = s.count <= ring * kTile ? 0 : (s.count - ring * kTile + kUnit - 1) / kUnit;
    if (tiles > 0) {
      copy_wait<kStages - 2>();
      meet();  // the first tile has arrived for all lanes
      clear_dots();
#pragma unroll
      for (int step = 0; step < kSteps; step += 2) score_steps(base, step);
      int stage = 0, fill = kStages - 1;
#pragma unroll 1
      for (int i = 1; i < tiles; ++i) {
        const uint32_t at = base + stage * kStageBytes;
        weigh(a, at);
        stage = stage + 1 == kStages ? 0 : stage + 1;
        const uint32_t next = base + stage * kStageBytes;
        copy_wait<kStages - 3>();
        meet();  // the next tile has arrived, and all lanes have left the one before this, whose stage is filled now
        copy(a, fill, s.tile, s.id, s.place);
        s.advance(a);
        fill = fill + 1 == kStages ? 0 : fill + 1;
        clear_dots();
#pragma unroll
        for (int step = 0; step < kSteps; step += 2) {
          score_steps(next, step);
          value_steps(at, step);
        }
      }
      const uint32_t at = base + stage * kStageBytes;
      weigh(a, at);
#pragma unroll
      for (int step = 0; step < kSteps; step += 2) value_steps(at, step);
    }
    copy_wait<0>();
    meet();
  }

  // What the accumulators of head h are multiplied with in the end.
  __device__ __forceinline__ float undo(int h) const {
    constexpr float lower = kLift == 0.f ? 1.f : 1.f / 256.f;
    static_assert(kLift == 0.f || kLift == 8.f, "2^-kLift");
    return kCoded ? lower * power_of_two(d[h]) : lower;
  }

  // Whether a sum of the piece's heads is not finite: 0 times it is not 0.
  __device__ __forceinline__ bool unsound(const AttentionArgs& a, const Piece& p) const {
    bool any = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float back = undo(h);
      float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        zero[step & 1] = fmaf(kCoded ? o[step][h] * back : o[step][h], 0.f, zero[step & 1]);
        zero[2 + (step & 1)] = fmaf(kCoded ? o[step][2 + h] * back : o[step][2 + h], 0.f, zero[2 + (step & 1)]);
      }
      any = any || (p.sub * kHeads + 8 * part + 2 * (lane & 3) + h < a.group && (zero[0] + zero[1]) + (zero[2] + zero[3]) != 0.f);
    }
    if constexpr (SHARE == 1) {
      any = __any_sync(kFull, any);
    } else {
      int ring_any;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
                   : "=r"(ring_any) : "r"(static_cast<int>(any)), "r"(1 + ring), "n"(SHARE * 32) : "memory");
      any = ring_any != 0;
    }
    return any;
  }

  __device__ __forceinline__ void drain() const {
    copy_wait<0>();
    meet();
  }

  __device__ __forceinline__ void run_carefully(const AttentionArgs& a) {
    const int tiles = s.count <= ring * kTile ? 0 : (s.count - ring * kTile + kUnit - 1) / kUnit;
    int stage = 0, fill = kStages - 1;
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
      copy_wait<kStages - 2>();
      meet();  // the tile has arrived, and all lanes have left the one before it, whose stage is filled now
      copy(a, fill, s.tile, s.id, s.place);
      s.advance(a);
      const uint32_t at = base + stage * kStageBytes;
      clear_dots();
#pragma unroll
      for (int step = 0; step < kSteps; step += 2) score_steps(at, step);
      weigh<true>(a, at);
      add_values(at);
      stage = stage + 1 == kStages ? 0 : stage + 1;
      fill = fill + 1 == kStages ? 0 : fill + 1;
    }
    copy_wait<0>();
    meet();
  }

  // The tile's products with V one by one: `high` and `low` hold the weights of heads 2 (lane % 4) and the next one, of tokens
  // lane / 4 and lane / 4 + 8, as floats.
  __device__ __forceinline__ void add_values(uint32_t at) {
    unsigned seen;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(seen) : "r"(at + kStageBytes - 4));
#pragma unroll 1
    for (int t = 0; t < kTile; ++t) {
      const int owner = (t & 7) * 4 + (lane & 3);
      const float w0 = __uint_as_float(__shfl_sync(kFull, t < 8 ? high[0] : high[1], owner));
      const float w1 = __uint_as_float(__shfl_sync(kFull, t < 8 ? low[0] : low[1], owner));
      if ((seen >> t & 1u) == 0) continue;
#pragma unroll
      for (int step = 0; step < kSteps; ++step)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int byte = output_feature(step, lane, half) * static_cast<int>(sizeof(T));
          const uint32_t from = place_of(at + kValues, t, 0);
          const float v = load_value((kSwizzled ? from ^ (byte & ~15) : from + (byte & ~15)) + (byte & 15));
          o[step][2 * half] = fmaf(w0, v, o[step][2 * half]);
          o[step][2 * half + 1] = fmaf(w1, v, o[step][2 * half + 1]);
        }
    }
  }
  static __device__ __forceinline__ float load_value(uint32_t from) {
    uint16_t bits;
    if constexpr (sizeof(T) == 1) {
      asm volatile("{\n\t.reg .b32 x;\n\tld.shared.u8 x, [%1];\n\tcvt.u16.u32 %0, x;\n\t}" : "=h"(bits) : "r"(from));
      T code;
      code.code = static_cast<decltype(code.code)>(bits);
      return to_float(code);
    } else {
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(from));
      return to_float(*reinterpret_cast<const T*>(&bits));
    }
  }

  // Raises `before` to the largest score of a head in the tile (the lanes of equal lane % 4 hold its tokens) and
  // returns the factor of what has been added up so far.
  static __device__ __forceinline__ float raise(float x0, float x1, float& before) {
    float top = fmaxf(x0, x1);
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 4));
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 8));
    top = fmaxf(top, __shfl_xor_sync(kFull, top, 16));
    top = fmaxf(top, before);
    const float shrink = fast_exp2(before - top);
    before = top;
    return shrink;
  }

  // Where piece `chunk` (0 or 1) of a row of the tile at `tile` lies, and the piece `bytes` (a multiple of 32) further on.
  static __device__ __forceinline__ uint32_t place_of(uint32_t tile, int row, int chunk) {
    return tile + row * kRowPitch + (kSwizzled ? (chunk ^ (row & 7)) * 16 : chunk * 16);
  }
  static __device__ __forceinline__ uint32_t further(uint32_t place, int bytes) { return kSwizzled ? place ^ bytes : place + bytes; }

  __device__ __forceinline__ void clear_dots() {
#pragma unroll
    for (int i = 0; i < 4; ++i) dots[0][i] = dots[1][i] = 0.f;
  }

  // Steps `step` and `step` + 1 (32 features) of the products with K.
  __device__ __forceinline__ void score_steps(uint32_t at, int step) {
    const uint32_t line = place_of(at, lane & 15, lane >> 4);
    if constexpr (!kCoded) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t k[4];
        ldmatrix_x4(k, further(line, (step + i) * 32));
        mma16816<H>(dots[i], k, q[step + i][0], q[step + i][1]);
      }
    } else {
      uint32_t c[4];
      ldmatrix_x4(c, further(line, step * 16));
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t k[4];
        decode_neighbours(c[2 * i], k[0], k[2], T{});
        decode_neighbours(c[2 * i + 1], k[1], k[3], T{});
        if constexpr (WIDE) {
          mma16816<H>(sum, k, q[step + i][0], q[step + i][1]);
          mma16816<H>(dots[1], k, q2[step + i][0], q2[step + i][1]);
        } else {
          mma16816<H>(dots[i], k, q[step + i][0], q[step + i][1]);
        }
      }
      if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) dots[0][i] += sum[i];
      }
    }
  }

  // The same features of the products with V.
  __device__ __forceinline__ void value_steps(uint32_t at, int step) {
    if constexpr (!kCoded) {
      const uint32_t line = place_of(at + kValues, (lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t v[4];
        ldmatrix_x4_trans(v, further(line, (step + i) * 32));
        mma16816<H>(o[step + i], v, high[0], high[1]);
        mma16816<H>(o[step + i], v, low[0], low[1]);
      }
    } else {
      const uint32_t line = place_of(at + kValues, lane & 15, lane >> 4);
      uint32_t c[4];
      ldmatrix_x4_trans(c, further(line, step * 16));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t v[4];
        decode_alternate(c[2 * i], v[0], v[1], T{});
        decode_alternate(c[2 * i + 1], v[2], v[3], T{});
        if constexpr (WIDE) {
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816<H>(sum, v, low[0], low[1]);
          mma16816<H>(sum, v, high[0], high[1]);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[step + i][j] += sum[j];
        } else {
          mma16816<H>(o[step + i], v, high[0], high[1]);
          mma16816<H>(o[step + i], v, low[0], low[1]);
        }
      }
    }
  }

  // Scores to weights, in two pieces or (WHOLE) as they are and at most 1.
  template <bool WHOLE = false>
  __device__ __forceinline__ void weigh(const AttentionArgs& a, uint32_t at) {
    // this lane's scores: tokens lane / 4 and lane / 4 + 8, heads 2 (lane % 4) + {0, 1}
    unsigned seen;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(seen) : "r"(at + kStageBytes - 4));
    float key_scale[2] = {1.f, 1.f}, value_scale[2] = {1.f, 1.f};
    if constexpr (kCoded) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int token = (lane >> 2) + 8 * t;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(key_scale[t]) : "r"(at + kExtras + token * 4));
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(value_scale[t]) : "r"(at + kExtras + (kTile + token) * 4));
      }
    }
    float x[2][2], w[2][2], u[2][2];  // [token][head]: scores, weights of the sum and of the accumulator
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[t][h] = dots[0][2 * t + h] + (WIDE ? dots[1][2 * t + h] * 0x1p-12f : dots[1][2 * t + h]);
        x[t][h] = kCoded ? x[t][h] * key_scale[t] * unit[h] : x[t][h] * a.scale_log2;  // (a key of zeros scores 0 whatever its scale)
      }
    if (seen != 0xffffu) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if ((seen >> ((lane >> 2) + 8 * t) & 1u) == 0) x[t][0] = x[t][1] = -CUDART_INF_F;
    }
    auto powers = [&]() {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          w[t][h] = fast_exp2(x[t][h] - (m[h] - kLift));
          u[t][h] = kCoded ? w[t][h] * held[h] * value_scale[t] : w[t][h];
        }
    };
    powers();
    float largest = fmaxf(fmaxf(w[0][0], w[0][1]), fmaxf(w[1][0], w[1][1]));
    if constexpr (WHOLE) largest *= 64.f;  // (no slack)
    if constexpr (kCoded) {
      const float other = fmaxf(fmaxf(fabsf(u[0][0]), fabsf(u[0][1])), fmaxf(fabsf(u[1][0]), fabsf(u[1][1])));
      largest = fmaxf(largest, other);
    }
    constexpr float limit = kLift == 0.f ? 64.f : 16384.f;
    static_assert(kSlack == 6.f, "2^kSlack, 2^(kSlack + kLift)");
    if (__any_sync(kFull, largest > limit)) {
      float shrink[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float before = m[h];
        shrink[h] = raise(x[0][h], x[1][h], m[h]);
        l[h] *= shrink[h];
        if constexpr (kCoded) {
          float largest = kNoScore;  // log2 of the tile's largest weight of the accumulator, against the new m
          raise(x[0][h] + fast_log2(fabsf(value_scale[0])), x[1][h] + fast_log2(fabsf(value_scale[1])), largest);
          const float faded = d[h] - (m[h] - before);
          const float next = fminf(fmaxf(ceilf(fmaxf(largest - m[h], faded)), kLeastD), kMostD);
          shrink[h] *= fast_exp2(fminf(d[h] - next, 126.f));
          d[h] = next;
          held[h] = power_of_two(-next);
        }
      }
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        o[step][0] *= shrink[0];
        o[step][1] *= shrink[1];
        o[step][2] *= shrink[0];
        o[step][3] *= shrink[1];
      }
      powers();
    }
    l[0] += w[0][0] + w[1][0];
    l[1] += w[0][1] + w[1][1];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (WHOLE) {
        high[t] = __float_as_uint(u[t][0]);
        low[t] = __float_as_uint(u[t][1]);
        continue;
      }
      float rest0, rest1, none0, none1;
      high[t] = transpose_8x8(pack2<H>(u[t][0], u[t][1], rest0, rest1));
      low[t] = transpose_8x8(pack2<H>(rest0, rest1, none0, none1));
    }
  }

  __device__ __forceinline__ void publish(unsigned char* smem, float2* ml) {
    float* to = reinterpret_cast<float*>(smem + ring * kRingBytes + kPublish);
    constexpr float lower = kLift == 0.f ? 1.f : 1.f / 256.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int head = 8 * part + 2 * (lane & 3) + h;
      float sum = l[h];
      sum += __shfl_xor_sync(kFull, sum, 4);
      sum += __shfl_xor_sync(kFull, sum, 8);
      sum += __shfl_xor_sync(kFull, sum, 16);
      if (lane < 4) ml[ring * kHeads + head] = make_float2(published_max(m[h]), sum * lower);
      const float back = undo(h);
#pragma unroll
      for (int step = 0; step < kSteps; ++step)
#pragma unroll
        for (int half = 0; half < 2; ++half) to[head * kPitch + output_feature(step, lane, half)] = o[step][2 * half + h] * back;
    }
  }
};

// Stages of a ring and CTAs per SM: one tile is being used with the next, the others are in flight.  As many CTAs as registers and
// shared memory hold, each with as few stages as that leaves: warps hide more than tiles in flight do.  (64 rows of up to 8192
// tokens, measured in turn: float16 8 x 128 178 us with 3 stages and 2 CTAs, 246 with 6 and 1; bfloat16 8 x 64 99 with 3 and 4, 103
// with 4 and 3; int8 8 x 128 120 with 4 and 3, 144 with 6 and 2.)
template <typename T, int SHARE, bool WIDE>
inline Choice choose_padded(const AttentionArgs& a) {
  if constexpr (WIDE) {
    if (a.dim <= 64) return made<Tensor<T, 64, SHARE, 4, SHARE == 1 ? 3 : 2, true>>();
    if (a.dim <= 128) return made<Tensor<T, 128, SHARE, 4, SHARE == 1 ? 2 : 1, true>>();
    return made<Tensor<T, 256, SHARE, 3, 1, true>>();
  } else if constexpr (sizeof(T) == 1) {
    if (a.dim <= 64) return made<Tensor<T, 64, SHARE, 4, SHARE == 1 ? 4 : 2>>();
    if (a.dim <= 128) return made<Tensor<T, 128, SHARE, 4, SHARE == 1 ? 3 : 2>>();
    return made<Tensor<T, 256, SHARE, 3, SHARE == 1 ? 2 : 1>>();
  } else {
    if (a.dim <= 64) return made<Tensor<T, 64, SHARE, 3, SHARE == 1 ? 4 : 2>>();
    if (a.dim <= 128) return made<Tensor<T, 128, SHARE, 3, 2>>();
    return made<Tensor<T, 256, SHARE, 3, 1>>();
  }
}
template <typename T, bool WIDE = false>
inline Choice choose_tensor(const AttentionArgs& a) {
  const int item = static_cast<int>(sizeof(T));
  if (a.dim * item % 16 != 0 || !rows_aligned(a.key, item, 16) || !rows_aligned(a.value, item, 16)) return Choice{};
  if (!a.same_strides) return Choice{};
  return a.group <= 8 ? choose_padded<T, 1, WIDE>(a) : choose_padded<T, 2, WIDE>(a);
}

#endif  // __CUDACC__

}  // namespace paged
}  // namespace asg
