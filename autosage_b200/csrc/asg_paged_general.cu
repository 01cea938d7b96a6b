// Paged attention on the FMA pipe: every type, head size and alignment, float32 products throughout.
//
// A warp takes batches of TB tokens; lane l holds E features of the query, key, value and accumulator rows.
// The TB x GT scores of a batch are partial sums spread over 32 lanes; a reduce-scatter (each step halves
// the number of values and the lanes they are spread over) leaves one whole score per lane for about one
// shuffle a score, and exponentials are taken once, by the lane that owns the score.  The weights come back
// to all lanes by one shuffle each.
#include "asg_paged_attention.cuh"

namespace asg {
namespace paged {

template <typename T, int E, int GT, bool VEC>
struct General {
  static constexpr int kHeads = GT;
  static constexpr int kDim = 32 * E;
  static constexpr int kPitch = kDim;
  static constexpr int kCtasPerSm = GT * E >= 32 ? 3 : 4;     // registers: q and o take 2 GT E, a batch 2 TB E
  static constexpr int TB = E == 8 ? 4 : (GT == 8 ? 4 : 8);  // tokens per batch: K and V rows of a batch are in registers
  static constexpr int N = TB * GT;                          // scores per batch: 4 ... 32
  static constexpr int kShift = N == 32 ? 0 : N == 16 ? 1 : N == 8 ? 2 : 3;
  static constexpr int kWarpBytes = GT * kPitch * 4;
  static constexpr int kPublish = 0;
  static_assert(N == 32 || N == 16 || N == 8 || N == 4, "reduce-scatter sizes");

  float q[GT][E], o[GT][E];
  float m, l;  // of the head that this lane owns scores of: head (lane >> kShift) % GT
  int lane, warp;

  __device__ __forceinline__ explicit General(unsigned char*) : lane(threadIdx.x & 31), warp(threadIdx.x >> 5) {}

  static __device__ __forceinline__ int feature(int lane, int e) { return VEC ? lane * E + e : e * 32 + lane; }

  const T* keys;
  const T* values;
  const int64_t* ids;  // of the page that holds the piece's first token
  int kv_head, place0, count;

  __device__ __forceinline__ void start(const AttentionArgs& a, const Piece& p) {
    kv_head = p.kv_head;
    keys = static_cast<const T*>(a.key.data) + kv_head * a.key.head_stride;
    values = static_cast<const T*>(a.value.data) + kv_head * a.value.head_stride;
    const long long first = p.first(), page0 = quotient(first, a.page_size);  // page arithmetic in 32 bits from here on
    place0 = static_cast<int>(first - page0 * a.page_size);
    ids = a.col + p.span.pages_begin + page0;
    count = static_cast<int>(p.last() - first);
  }

  __device__ __forceinline__ void query(const AttentionArgs& a, const Piece& p) {
    const int head = p.kv_head * a.group + p.sub * GT, heads = min(GT, a.group - p.sub * GT);
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = feature(lane, e);
        q[g][e] = g < heads && d < a.dim
                      ? load_wide(a.q, p.row * a.q_token_stride + (head + g) * a.q_head_stride + d, a.type) * a.scale_log2
                      : 0.f;
        o[g][e] = 0.f;
      }
    m = -CUDART_INF_F;
    l = 0.f;
  }

  __device__ __forceinline__ void load(float (&x)[E], const T* row, bool ok, int dim) const {
    if constexpr (VEC) {
      Pack<T, E> p;
      if (ok && lane * E < dim) {
        p.load(row + lane * E);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = to_float(p.v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = ok && feature(lane, e) < dim ? to_float(row[feature(lane, e)]) : 0.f;
    }
  }

  __device__ __forceinline__ void run(const AttentionArgs& a) {
    for (int tile = warp * kTile; tile < count; tile += kUnit) {
      // lane t < kTile finds token tile + t
      int page = -1, place = 0;
      float key_scale = 0.f, value_scale = 0.f;
      if (lane < kTile && tile + lane < count) {
        const unsigned at = static_cast<unsigned>(place0) + static_cast<unsigned>(tile + lane);
        const unsigned nth = at / static_cast<unsigned>(a.page_size);
        const long long id = ids[nth];
        place = static_cast<int>(at - nth * static_cast<unsigned>(a.page_size));
        if (id >= 0 && id < a.n_pages) page = static_cast<int>(id);
        if (TypeOf<T>::coded && page >= 0) {
          key_scale = a.key.scales[page * a.key.scale_page_stride + kv_head * a.key.scale_head_stride + place * a.key.scale_token_stride];
          value_scale = a.value.scales[page * a.value.scale_page_stride + kv_head * a.value.scale_head_stride + place * a.value.scale_token_stride];
        }
      }
#pragma unroll 1
      for (int t0 = 0; t0 < kTile && tile + t0 < count; t0 += TB) {
        float k[TB][E], v[TB][E];
        bool any = false;
#pragma unroll
        for (int t = 0; t < TB; ++t) {
          const int p = __shfl_sync(kFull, page, t0 + t);
          const int in = __shfl_sync(kFull, place, t0 + t);
          any = any || p >= 0;
          load(k[t], keys + p * a.key.page_stride + in * a.key.token_stride, p >= 0, a.dim);
          load(v[t], values + p * a.value.page_stride + in * a.value.token_stride, p >= 0, a.dim);
        }
        if (!any) continue;  // only holes
        float x[N];
#pragma unroll
        for (int t = 0; t < TB; ++t)
#pragma unroll
          for (int g = 0; g < GT; ++g) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) s = fmaf(q[g][e], k[t][e], s);
            x[t * GT + g] = s;
          }
        // reduce-scatter: afterwards lane L holds the whole score of index L >> kShift
        int n = N;
#pragma unroll
        for (int step = 16; step >= 1; step >>= 1) {
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
        const int mine = lane >> kShift;  // token mine / GT, head mine % GT
        const int token = t0 + mine / GT;
        const bool seen = __shfl_sync(kFull, page, token) >= 0;
        float weight_scale = 1.f;
        if (TypeOf<T>::coded) {
          x[0] *= __shfl_sync(kFull, key_scale, token);
          weight_scale = __shfl_sync(kFull, value_scale, token);
        }
        const float s = seen ? x[0] : -CUDART_INF_F;
        float top = s;
#pragma unroll
        for (int step = 16; step >= GT << kShift; step >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, step));
        top = fmaxf(top, m);
        const float base = top == -CUDART_INF_F ? 0.f : top;
        const float shrink = exp2f(m - base);
        float w = exp2f(s - base);
        l = l * shrink + w;
        m = top;
        w = seen ? w * weight_scale : 0.f;
        if (__any_sync(kFull, shrink != 1.f)) {
#pragma unroll
          for (int g = 0; g < GT; ++g) {
            const float f = __shfl_sync(kFull, shrink, g << kShift);
#pragma unroll
            for (int e = 0; e < E; ++e) o[g][e] *= f;
          }
        }
#pragma unroll
        for (int t = 0; t < TB; ++t)
#pragma unroll
          for (int g = 0; g < GT; ++g) {
            const float f = __shfl_sync(kFull, w, (t * GT + g) << kShift);
#pragma unroll
            for (int e = 0; e < E; ++e) o[g][e] = fmaf(f, v[t][e], o[g][e]);
          }
      }
    }
  }

  __device__ __forceinline__ void publish(unsigned char* smem, float2* ml) {
    float* buffer = reinterpret_cast<float*>(smem) + warp * GT * kPitch;
    // the sum of a head is spread over the lanes that own its scores of different tokens
#pragma unroll
    for (int step = 16; step >= GT << kShift; step >>= 1) l += __shfl_xor_sync(kFull, l, step);
    const int mine = lane >> kShift;
    if (mine < GT && (lane & ((1 << kShift) - 1)) == 0) ml[warp * GT + mine] = make_float2(m, l);
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) buffer[g * kPitch + feature(lane, e)] = o[g][e];
  }
};

// Heads per item: the group if it is small; a group of more takes several items, whose second reading of
// the keys and values comes from L2.  Features wider than 128 leave room for four heads in registers.
template <typename T, bool VEC>
static Choice choose(const AttentionArgs& a) {
  if (a.dim > 128) return a.group == 1 ? made<General<T, 8, 1, VEC>>() : made<General<T, 8, 4, VEC>>();
  if (a.dim > 64) {
    if (a.group == 1) return made<General<T, 4, 1, VEC>>();
    return a.group <= 4 ? made<General<T, 4, 4, VEC>>() : made<General<T, 4, 8, VEC>>();
  }
  if (a.group == 1) return made<General<T, 2, 1, VEC>>();
  return a.group <= 4 ? made<General<T, 2, 4, VEC>>() : made<General<T, 2, 8, VEC>>();
}

template <typename T>
static Choice choose(const AttentionArgs& a) {
  const int lane_features = a.dim > 128 ? 8 : a.dim > 64 ? 4 : 2;
  const int item = TypeOf<T>::id == ASG_TYPE_F32 ? 4 : TypeOf<T>::coded ? 1 : 2;
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
