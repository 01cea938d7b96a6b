// Paged attention on the FMA pipe: every type, head size and alignment, float32 products throughout.
//
// A warp takes batches of TB tokens, one token with all 32 lanes or (heads of up to 64 features) two side by side with 16
// lanes each; a lane holds E features of the query, key, value and accumulator rows.  The scores of a batch are
// partial sums spread over the LANES lanes of a token; a reduce-scatter (each step halves the number of values and
// the lanes they are spread over) leaves one whole score per lane for about one shuffle a score, and exponentials
// are taken once, by the lane that owns the score.  The weights come back to their token's lanes by one shuffle each.
//
// Every warp has a ring of kStages batches in shared memory.  Where a lane's E features of a row are one aligned
// vector (VEC), cp.async brings them there, several batches ahead; a lane copies what it will read itself.
// Otherwise the lanes load element by element and store into the ring.
#include "asg_paged_attention.cuh"

namespace asg {
namespace paged {

template <typename T, int E, int LANES, int GT, bool VEC, int STAGES, int CTAS>
struct General {
  static constexpr int kThreads = kRings * 32;
  static constexpr int kHeads = GT;
  static constexpr int kCtasPerSm = CTAS;
  static constexpr int kStages = STAGES;
  // 1024 sums rounded by 2^-24 at most: 6e-5, one-sided only where all values are alike.  (Legs of 32 units: 2.6 % on 64 rows of up
  // to 8192 tokens of 4 x 128 with 32 query heads, whose shares are then two legs.)
  static constexpr int kLeg = 64;
  static constexpr bool kCoded = TypeOf<T>::coded;
  static constexpr int TB = E == 8 || GT == 8 ? 4 : 8;  // tokens per batch
  static constexpr int kBatches = kTile / TB;           // of a tile
  static constexpr int kSide = 32 / LANES;              // tokens side by side
  static constexpr int kSteps = TB / kSide;
  static constexpr int N = kSteps * GT;                 // scores per batch and token's lanes: 4 ... LANES
  static constexpr int kShift = N == LANES ? 0 : 2 * N == LANES ? 1 : 4 * N == LANES ? 2 : 3;
  static_assert(N << kShift == LANES && (LANES == 32 || LANES == 16), "reduce-scatter sizes");
  static constexpr int kDim = LANES * E;
  static constexpr int kPitch = kDim;
  static constexpr int kLaneBytes = E * static_cast<int>(sizeof(T));
  static constexpr int kRowBytes = LANES * kLaneBytes;
  static constexpr int kValues = TB * kRowBytes;
  static constexpr int kExtras = 2 * TB * kRowBytes;  // the scales of a batch (key, value), then the mask of its seen tokens
  static constexpr int kStageBytes = (kExtras + (kCoded ? 2 * TB * 4 : 0) + 4 + 15) / 16 * 16;
  static constexpr int kPublish = (kStages - 1) * kStageBytes;
  static constexpr int kNeed = kPublish + (kStageBytes > GT * kPitch * 4 ? kStageBytes : GT * kPitch * 4);
  static constexpr int kRingBytes = (kNeed + 127) / 128 * 128;

  float q[GT][E], o[GT][E];
  float m, l;  // of the head that this lane owns scores of: head (place >> kShift) % GT
  int lane, place, side, ring;  // lane of the warp, of its token; which of the tokens side by side
  unsigned char* region;
  Source s;
  float slack = kSlack;
  int batch;                              // of the tile that is copied next
  bool held;                              // of the lane's token of that tile
  long long key_offset, value_offset;     // in bytes
  long long scale_id;
  int scale_place;

  __device__ __forceinline__ explicit General(unsigned char* smem)
      : lane(threadIdx.x & 31), place(threadIdx.x % LANES), side((threadIdx.x & 31) / LANES), ring(threadIdx.x >> 5),
        region(smem + (threadIdx.x >> 5) * kRingBytes) {}

  __device__ __forceinline__ int feature(int e) const { return VEC ? place * E + e : e * LANES + place; }

  __device__ __forceinline__ void fetch(const AttentionArgs& a, const Piece& p) {
    const int head = p.kv_head * a.group + p.sub * GT, heads = min(GT, a.group - p.sub * GT);
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = feature(e);
        q[g][e] = g < heads && d < a.dim ? load_wide(a.q, p.row * a.q_token_stride + (head + g) * a.q_head_stride + d, a.type) : 0.f;
      }
  }

  __device__ __forceinline__ void query(const AttentionArgs& a) {
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        q[g][e] *= a.scale_log2;
        o[g][e] = 0.f;
      }
    m = kNoScore;
    l = 0.f;
  }

  // Where the lane's token of a tile lies.
  __device__ __forceinline__ void locate(const AttentionArgs& a, long long id, int place) {
    constexpr int item = static_cast<int>(sizeof(T));
    held = id >= 0 && id < a.n_pages;
    key_offset = held ? id * s.page_bytes + place * s.token_bytes : 0;
    value_offset = held ? id * a.value.page_stride * item + place * a.value.token_stride * item : 0;
    scale_id = id;
    scale_place = place;
  }

  // Copies batch `batch` of the tile at token `tile`, located before, to a stage.
  __device__ __forceinline__ void copy(const AttentionArgs& a, int stage, int tile, int batch) {
    if (tile + batch * TB < s.count) {
      const unsigned seen = __ballot_sync(kFull, held) >> (batch * TB) & ((1u << TB) - 1u);
      unsigned char* at = region + stage * kStageBytes;
      const int key_low = static_cast<int>(key_offset), key_high = static_cast<int>(key_offset >> 32);
      const int value_low = static_cast<int>(value_offset), value_high = static_cast<int>(value_offset >> 32);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int t = i * kSide + side, from = batch * TB + t;
        const long long k = static_cast<long long>(__shfl_sync(kFull, key_high, from)) << 32 |
                            static_cast<unsigned>(__shfl_sync(kFull, key_low, from));
        const long long v = a.same_strides ? k : static_cast<long long>(__shfl_sync(kFull, value_high, from)) << 32 |
                                                     static_cast<unsigned>(__shfl_sync(kFull, value_low, from));
        const bool ok = (seen >> t & 1u) != 0;
        unsigned char* to = at + i * 32 * kLaneBytes + lane * kLaneBytes;  // token t, this lane's features
        if constexpr (VEC) {
          constexpr int kStep = kLaneBytes < 16 ? kLaneBytes : 16;
#pragma unroll
          for (int b = 0; b < kLaneBytes; b += kStep) {
            copy_async<kStep>(smem_u32(to) + b, s.keys + k + place * kLaneBytes + b, ok && place * E < a.dim);
            copy_async<kStep>(smem_u32(to) + kValues + b, s.values + v + place * kLaneBytes + b, ok && place * E < a.dim);
          }
        } else {
          const T* keys = reinterpret_cast<const T*>(s.keys + k);
          const T* values = reinterpret_cast<const T*>(s.values + v);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const bool in = ok && feature(e) < a.dim;
            reinterpret_cast<T*>(to)[e] = in ? keys[feature(e)] : T{};
            reinterpret_cast<T*>(to + kValues)[e] = in ? values[feature(e)] : T{};
          }
        }
      }
      if constexpr (kCoded) {
        // lanes of the batch's tokens: their key scales; sixteen lanes on: their value scales
        const int token = (lane & (kTile - 1)) - batch * TB;
        if (token >= 0 && token < TB) {
          const asg_page_pool& pool = lane < kTile ? a.key : a.value;
          const float* from = pool.scales + s.kv_head * pool.scale_head_stride;
          if (held) from += scale_id * pool.scale_page_stride + scale_place * pool.scale_token_stride;
          copy_async<4>(smem_u32(at + kExtras) + ((lane < kTile ? 0 : TB) + token) * 4, from, held);
        }
      }
      if (lane == 0) *reinterpret_cast<unsigned*>(at + kStageBytes - 4) = seen;
    }
    copy_commit();
  }

  __device__ __forceinline__ void start(const AttentionArgs& a, const Piece& p) {
    s.start(a, p, ring, static_cast<int>(sizeof(T)));
    constexpr int kLast = (kStages - 1) / kBatches;  // tile of the batch after the first copies
    const int first = s.tile;
    long long id[kLast + 1];  // the page ids of all tiles are asked for before the first is needed
    int place[kLast + 1];
#pragma unroll
    for (int i = 0; i <= kLast; ++i) {
      id[i] = s.id;
      place[i] = s.place;
      if (i < kLast) s.advance(a);
    }
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (i % kBatches == 0) locate(a, id[i / kBatches], place[i / kBatches]);
      copy(a, i, first + i / kBatches * kUnit, i % kBatches);
    }
    batch = (kStages - 1) % kBatches;
  }

  __device__ __forceinline__ void run(const AttentionArgs& a) {
    const int tiles = s.count <= ring * kTile ? 0 : (s.count - ring * kTile + kUnit - 1) / kUnit;
    int stage = 0, fill = kStages - 1;
#pragma unroll 1
    for (int i = 0; i < tiles * kBatches; ++i) {
      const int first = ring * kTile + i / kBatches * kUnit + i % kBatches * TB;
      copy_wait<kStages - 2>();
      __syncwarp();  // the batch has arrived for all lanes, and all have left the stage that is filled next
      if (batch == 0) locate(a, s.id, s.place);  // the id was asked for a batch ago
      copy(a, fill, s.tile, batch);
      if (++batch == kBatches) {
        batch = 0;
        s.advance(a);
      }
      if (first < s.count) compute(region + stage * kStageBytes);
      stage = stage + 1 == kStages ? 0 : stage + 1;
      fill = fill + 1 == kStages ? 0 : fill + 1;
    }
    copy_wait<0>();
    __syncwarp();
  }

  // A sum that is not finite may be a large value times a weight above 1: the second time no weight is.
  __device__ __forceinline__ bool unsound(const AttentionArgs& a, const Piece& p) const {
    bool any = false;
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      float zero = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) zero = fmaf(o[g][e], 0.f, zero);
      any = any || (p.sub * GT + g < a.group && zero != 0.f);
    }
    return __any_sync(kFull, any);
  }
  __device__ __forceinline__ void drain() const {
    copy_wait<0>();
    __syncwarp();
  }
  __device__ __forceinline__ void run_carefully(const AttentionArgs& a) {
    slack = 0.f;
    run(a);
    slack = kSlack;
  }

  __device__ __forceinline__ void row_of(float (&x)[E], const unsigned char* at) const {
    const T* from = reinterpret_cast<const T*>(at + lane * kLaneBytes);
    Pack<T, E> p;
    if constexpr (Pack<T, E>::kVec <= 16) {
      Pack<T, E>::move(p.v, from);
    } else {
#pragma unroll
      for (int i = 0; i < kLaneBytes / 16; ++i) reinterpret_cast<uint4*>(p.v)[i] = reinterpret_cast<const uint4*>(from)[i];
    }
    to_floats(p, x);
  }

  // f over the lanes that own scores of one head (of different tokens).
  template <typename F>
  static __device__ __forceinline__ float over_tokens(float v, F f) {
#pragma unroll
    for (int step = 16; step >= 1; step >>= 1)
      if (step >= LANES || step >= GT << kShift) v = f(v, __shfl_xor_sync(kFull, v, step));
    return v;
  }

  __device__ __forceinline__ void compute(const unsigned char* at) {
    float x[N];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float k[E];
      row_of(k, at + i * 32 * kLaneBytes);
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) sum = fmaf(q[g][e], k[e], sum);
        x[i * GT + g] = sum;
      }
    }
    // reduce-scatter: afterwards the lane at place P of its token's lanes holds the whole score of index P >> kShift
    int n = N;
#pragma unroll
    for (int step = LANES / 2; step >= 1; step >>= 1) {
      if (n > 1) {
        n >>= 1;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          if (i < n) {
            const bool upper = (lane & step) != 0;
            const float keep = upper ? x[i + n] : x[i];
            const float send = upper ? x[i] : x[i + n];
            x[i] = keep + __shfl_xor_sync(kFull, send, step);
          }
        }
      } else {
        x[0] += __shfl_xor_sync(kFull, x[0], step);
      }
    }
    const int token = (place >> kShift) / GT * kSide + side;  // and head (place >> kShift) % GT
    const unsigned seen = *reinterpret_cast<const unsigned*>(at + kStageBytes - 4);
    const bool in = (seen >> token & 1u) != 0;
    float weight_scale = 1.f;
    if constexpr (kCoded) {
      x[0] *= reinterpret_cast<const float*>(at + kExtras)[token];
      weight_scale = reinterpret_cast<const float*>(at + kExtras)[TB + token];
    }
    const float score = in ? x[0] : -CUDART_INF_F;
    if (__any_sync(kFull, score > m + slack)) {
      const float top = fmaxf(over_tokens(score, [](float a, float b) { return fmaxf(a, b); }), m);
      const float shrink = exp2f(m - top);
      m = top;
      l *= shrink;
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        const float f = __shfl_sync(kFull, shrink, g << kShift);
#pragma unroll
        for (int e = 0; e < E; ++e) o[g][e] *= f;
      }
    }
    float w = exp2f(score - m);
    l += w;
    w = in ? w * weight_scale : 0.f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float v[E];
      row_of(v, at + kValues + i * 32 * kLaneBytes);
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        const float f = __shfl_sync(kFull, w, side * LANES + ((i * GT + g) << kShift));
#pragma unroll
        for (int e = 0; e < E; ++e) o[g][e] = fmaf(f, v[e], o[g][e]);
      }
    }
  }

  __device__ __forceinline__ void publish(unsigned char* smem, float2* ml) {
    float* buffer = reinterpret_cast<float*>(smem + ring * kRingBytes + kPublish);
    l = over_tokens(l, [](float a, float b) { return a + b; });
    const int mine = lane >> kShift;
    if (mine < GT && (lane & ((1 << kShift) - 1)) == 0) ml[ring * GT + mine] = make_float2(published_max(m), l);
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float sum = o[g][e];
        if constexpr (kSide == 2) sum += __shfl_xor_sync(kFull, sum, 16);
        if (side == 0) buffer[g * kPitch + feature(e)] = sum;
      }
  }
};

// Stages: about 100 KB per SM in flight for float32 rows.  CTAs: q and o take 2 GT E registers.
template <typename T, int E, int LANES, int GT, bool VEC>
static Choice pick() {
  constexpr int batch = (E == 8 || GT == 8 ? 4 : 8) * 2 * LANES * E * static_cast<int>(sizeof(T));  // bytes of a stage
  constexpr int ctas = GT * E >= 32 || batch >= 8192 ? 2 : 3;
  constexpr int stages = !VEC ? 2 : batch >= 8192 ? 3 : batch >= 4096 ? 4 : 6;
  return made<General<T, E, LANES, GT, VEC, stages, ctas>>();
}

// Heads per item: the group if it is small; a group of more takes several items, whose second reading of
// the keys and values comes from L2.  Features wider than 128 leave room for four heads in registers.
template <typename T, bool VEC>
static Choice choose(const AttentionArgs& a) {
  if (a.dim > 128) return a.group == 1 ? pick<T, 8, 32, 1, VEC>() : pick<T, 8, 32, 4, VEC>();
  if (a.dim > 64) {
    if (a.group == 1) return pick<T, 4, 32, 1, VEC>();
    return a.group <= 4 ? pick<T, 4, 32, 4, VEC>() : pick<T, 4, 32, 8, VEC>();
  }
  if (a.group == 1) return pick<T, 4, 16, 1, VEC>();
  return a.group <= 4 ? pick<T, 4, 16, 4, VEC>() : pick<T, 4, 16, 8, VEC>();
}

template <typename T>
static Choice choose(const AttentionArgs& a) {
  const int item = static_cast<int>(sizeof(T));
  const int lane_features = a.dim > 128 ? 8 : 4;
  const int bytes = lane_features * item < 16 ? lane_features * item : 16;
  if (a.dim % lane_features == 0 && rows_aligned(a.key, item, bytes) && rows_aligned(a.value, item, bytes))
    return choose<T, true>(a);
  return choose<T, false>(a);
}

Choice choose_general(const AttentionArgs& a, int cache_type) {
  switch (cache_type) {
    case ASG_TYPE_F32: return choose<F32>(a);
    case ASG_TYPE_BF16: return choose<BF16>(a);
    case ASG_TYPE_F16: return choose<F16>(a);
    case ASG_TYPE_E4M3: return choose<E4M3>(a);
    default: return choose<INT8>(a);
  }
}

}  // namespace paged
}  // namespace asg
