// Writing tokens into the pages of a cache, with or without quantising to 8 bits, and reading them back.
//
//   write   page row slots[t] = x[t, h, :]                       (same type), or
//           s = max_d |x_d| / Q,  code_d = nearest(x_d / s)       (Q = 448 for e4m3, 127 for int8)
//   read    x[t, h, d] = round(code_d * s)
//
// Both move every byte once and are bound by memory: a group of lanes owns the key row AND the value row
// of one (token, head), eight features a lane in 16-byte vectors, so two independent rows are in flight
// per lane and consecutive groups touch consecutive heads of a token (contiguous in the usual layouts).
//
// Rounding.  A quotient rounded to float32 first would often land exactly between two codes that the true
// quotient is not between (16-bit inputs share few mantissa bits, so near-ties are common), and the tie
// rule would then pick the wrong one.  The quotient is therefore rounded "to odd": correctly rounded by
// one multiply with 1/s and two fused multiply-adds, then its last bit is set towards the sign of the exact
// remainder x - q s.  Borders between codes have an even last bit, so rounding that value to a code gives
// the code nearest to the true quotient, for about nine instructions a value; dividing in float64 instead
// is kept for scales so small or large that 1/s or the remainder would leave float32's range.
#include "asg_paged.cuh"

namespace asg {
namespace paged {

struct CacheArgs {
  const int64_t* slots;
  long long n_tokens, n_slots;
  asg_token_rows rows[2];   // key, value
  asg_page_pool pools[2];
  int page_size, n_heads, dim;
};

constexpr int kThreads = 256;
constexpr int kPerLane = 8;  // features of a lane: 32 lanes cover kMaxDim

__device__ __forceinline__ float largest_code(E4M3) { return 448.f; }
__device__ __forceinline__ float largest_code(INT8) { return 127.f; }

// x / s, rounded to odd in float32 (see above); inv = 1 / s, s in [2^-90, 2^90].
__device__ __forceinline__ float quotient_to_odd(float x, float s, float inv) {
  const float q0 = x * inv;
  const float q = fmaf(fmaf(-q0, s, x), inv, q0);
  const float rest = fmaf(-q, s, x);
  const int bits = __float_as_int(q);
  const int step = ((__float_as_int(rest) ^ bits) < 0) ? -1 : 1;  // towards the remainder
  return __int_as_float(rest != 0.f && (bits & 1) == 0 ? bits + step : bits);
}

__device__ __forceinline__ E4M3 nearest_code(float q, E4M3) {
  E4M3 c;
  c.code = __nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
  return c;
}
__device__ __forceinline__ INT8 nearest_code(float q, INT8) {
  INT8 c;
  c.code = static_cast<int8_t>(max(-127, min(127, __float2int_rn(q))));
  return c;
}

// Feature of entry i of a lane: eight neighbours (VEC), or one in 32 (any alignment, any head size).
template <bool VEC>
__device__ __forceinline__ int feature(int lane, int i) { return VEC ? lane * kPerLane + i : i * 32 + lane; }

template <bool VEC, typename T>
__device__ __forceinline__ void load_row(Pack<T, kPerLane>& x, const T* row, int lane, int dim) {
  if constexpr (VEC) {
    if (lane * kPerLane < dim) {
      x.load(row + lane * kPerLane);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int d = feature<VEC>(lane, i);
    x.v[i] = T{};
    if (!VEC && d < dim) x.v[i] = row[d];
  }
}

template <bool VEC, typename T>
__device__ __forceinline__ void store_row(const Pack<T, kPerLane>& x, T* row, int lane, int dim) {
  if constexpr (VEC) {
    if (lane * kPerLane < dim) x.store(row + lane * kPerLane);
  } else {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (feature<VEC>(lane, i) < dim) row[feature<VEC>(lane, i)] = x.v[i];
  }
}

template <typename IN, typename CACHE, bool VEC>
__global__ void __launch_bounds__(kThreads) write_kernel(const CacheArgs a, int group) {
  const int lane = threadIdx.x & (group - 1);
  const unsigned mask = group == 32 ? kFull : ((1u << group) - 1u) << ((threadIdx.x & 31) & ~(group - 1));
  const long long n_rows = a.n_tokens * a.n_heads;
  const long long stride = static_cast<long long>(gridDim.x) * (kThreads / group);
  for (long long r = static_cast<long long>(blockIdx.x) * (kThreads / group) + threadIdx.x / group; r < n_rows; r += stride) {
    long long token;
    int head;
    split_slot(r, a.n_heads, token, head);
    const long long slot = a.slots[token];
    if (slot < 0 || slot >= a.n_slots) continue;  // the whole group leaves together
    long long page;
    int place;
    split_slot(slot, a.page_size, page, place);
    Pack<IN, kPerLane> x[2];
#pragma unroll
    for (int w = 0; w < 2; ++w)
      load_row<VEC>(x[w], static_cast<const IN*>(a.rows[w].data) + token * a.rows[w].token_stride +
                              head * a.rows[w].head_stride, lane, a.dim);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const asg_page_pool& pool = a.pools[w];
      CACHE* to = static_cast<CACHE*>(pool.data) + page * pool.page_stride + place * pool.token_stride + head * pool.head_stride;
      if constexpr (!TypeOf<CACHE>::coded) {
        store_row<VEC>(x[w], to, lane, a.dim);
      } else {
        // the largest magnitude by its bits: a NaN is above everything and is not lost
        unsigned top = 0;
        float v[kPerLane];
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
          v[i] = to_float(x[w].v[i]);
          top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
        }
        for (int o = group >> 1; o >= 1; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
        const float s = __uint_as_float(top) / largest_code(CACHE{});
        Pack<CACHE, kPerLane> c;
        if (s > 0x1p-90f && s < 0x1p90f) {
          const float inv = 1.f / s;
#pragma unroll
          for (int i = 0; i < kPerLane; ++i) c.v[i] = nearest_code(quotient_to_odd(v[i], s, inv), CACHE{});
        } else {
          // a quotient of two 24-bit numbers is never nearer to a border between codes than 2^-40 of itself
          // without lying on it: the nearest float32 of the float64 quotient, moved off the border, decides
#pragma unroll
          for (int i = 0; i < kPerLane; ++i) {
            const double wide = s == 0.f ? 0.0 : static_cast<double>(v[i]) / static_cast<double>(s);
            float q = static_cast<float>(wide);
            const double rest = wide - static_cast<double>(q);
            if (rest != 0.0 && (__float_as_int(q) & 1) == 0 && q != 0.f && !isinf(q) && rest == rest)
              q = __int_as_float(__float_as_int(q) + ((rest < 0.0) == (q < 0.f) ? 1 : -1));
            c.v[i] = nearest_code(q, CACHE{});
          }
        }
        store_row<VEC>(c, to, lane, a.dim);
        if (lane == 0)
          pool.scales[page * pool.scale_page_stride + head * pool.scale_head_stride + place * pool.scale_token_stride] = s;
      }
    }
  }
}

template <typename CACHE, typename OUT, bool VEC>
__global__ void __launch_bounds__(kThreads) read_kernel(const CacheArgs a, int group) {
  const int lane = threadIdx.x & (group - 1);
  const long long n_rows = a.n_tokens * a.n_heads;
  const long long stride = static_cast<long long>(gridDim.x) * (kThreads / group);
  for (long long r = static_cast<long long>(blockIdx.x) * (kThreads / group) + threadIdx.x / group; r < n_rows; r += stride) {
    long long token;
    int head;
    split_slot(r, a.n_heads, token, head);
    const long long slot = a.slots[token];
    const bool held = slot >= 0 && slot < a.n_slots;
    long long page = 0;
    int place = 0;
    if (held) split_slot(slot, a.page_size, page, place);
    Pack<CACHE, kPerLane> c[2];
    float s[2] = {1.f, 1.f};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const asg_page_pool& pool = a.pools[w];
      load_row<VEC>(c[w], static_cast<const CACHE*>(pool.data) + page * pool.page_stride + place * pool.token_stride +
                              head * pool.head_stride, lane, held ? a.dim : 0);
      if (TypeOf<CACHE>::coded && held)
        s[w] = pool.scales[page * pool.scale_page_stride + head * pool.scale_head_stride + place * pool.scale_token_stride];
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      Pack<OUT, kPerLane> x;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) x.v[i] = from_float<OUT>(TypeOf<CACHE>::coded ? to_float(c[w].v[i]) * s[w] : to_float(c[w].v[i]));
      store_row<VEC>(x, static_cast<OUT*>(a.rows[w].data) + token * a.rows[w].token_stride + head * a.rows[w].head_stride,
                     lane, a.dim);
    }
  }
}

// Lanes per row and blocks.  The vector form needs rows of whole 8-feature groups that start on 16 bytes
// (8 for codes); everything else takes a warp a row, one feature in 32 a lane.
struct Shape {
  bool vec;
  int group;
  unsigned blocks;
};

static Shape shape_of(const CacheArgs& a, int wide_type, int cache_type) {
  Shape s;
  s.vec = a.dim % kPerLane == 0;
  for (int w = 0; w < 2; ++w)
    s.vec = s.vec && rows_aligned(a.rows[w], type_bytes(wide_type), 16) &&
            rows_aligned(a.pools[w], type_bytes(cache_type), is_coded(cache_type) ? 8 : 16);
  s.group = 32;
  while (s.vec && s.group > 1 && s.group / 2 * kPerLane >= a.dim) s.group /= 2;
  const long long rows_per_block = kThreads / s.group;
  const long long blocks = (a.n_tokens * a.n_heads + rows_per_block - 1) / rows_per_block;
  s.blocks = static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20));
  return s;
}

template <typename IN, typename CACHE>
static int launch_write(const CacheArgs& a, cudaStream_t stream) {
  const Shape s = shape_of(a, TypeOf<IN>::id, TypeOf<CACHE>::id);
  if (s.vec) write_kernel<IN, CACHE, true><<<s.blocks, kThreads, 0, stream>>>(a, s.group);
  else write_kernel<IN, CACHE, false><<<s.blocks, kThreads, 0, stream>>>(a, s.group);
  ASG_CUDA(cudaGetLastError());
  return ASG_OK;
}
template <typename IN>
static int launch_write(const CacheArgs& a, int cache_type, cudaStream_t stream) {
  if (cache_type == ASG_TYPE_E4M3) return launch_write<IN, E4M3>(a, stream);
  if (cache_type == ASG_TYPE_INT8) return launch_write<IN, INT8>(a, stream);
  return launch_write<IN, IN>(a, stream);
}

template <typename CACHE, typename OUT>
static int launch_read(const CacheArgs& a, cudaStream_t stream) {
  const Shape s = shape_of(a, TypeOf<OUT>::id, TypeOf<CACHE>::id);
  if (s.vec) read_kernel<CACHE, OUT, true><<<s.blocks, kThreads, 0, stream>>>(a, s.group);
  else read_kernel<CACHE, OUT, false><<<s.blocks, kThreads, 0, stream>>>(a, s.group);
  ASG_CUDA(cudaGetLastError());
  return ASG_OK;
}
template <typename CACHE>
static int launch_read(const CacheArgs& a, int out_type, cudaStream_t stream) {
  if (out_type == ASG_TYPE_F32) return launch_read<CACHE, F32>(a, stream);
  if (out_type == ASG_TYPE_BF16) return launch_read<CACHE, BF16>(a, stream);
  return launch_read<CACHE, F16>(a, stream);
}

static int fill_args(CacheArgs& a, const int64_t* slots, int64_t n_tokens, const asg_token_rows* key,
                     const asg_token_rows* value, const asg_page_pool* key_pool, const asg_page_pool* value_pool,
                     int64_t n_pages, int64_t page_size, int n_heads, int head_dim, int wide_type, int cache_type) {
  if (int rc = check_pools(key_pool, value_pool, n_pages, page_size, n_heads, head_dim, wide_type, cache_type)) return rc;
  ASG_REQUIRE(n_tokens >= 0, ASG_EINVAL, "n_tokens must be non-negative");
  ASG_REQUIRE(n_tokens <= (1ll << 40), ASG_ERANGE, "n_tokens exceeds the kernel index range");
  ASG_REQUIRE(key != nullptr && value != nullptr, ASG_EINVAL, "key and value must not be null");
  ASG_REQUIRE(n_tokens == 0 || (slots != nullptr && key->data != nullptr && value->data != nullptr), ASG_EINVAL,
              "slots, key and value must not be null");
  a.slots = slots;
  a.n_tokens = n_tokens;
  a.n_slots = n_pages * page_size;
  a.rows[0] = *key;
  a.rows[1] = *value;
  a.pools[0] = *key_pool;
  a.pools[1] = *value_pool;
  a.page_size = static_cast<int>(page_size);
  a.n_heads = n_heads;
  a.dim = head_dim;
  return ASG_OK;
}

}  // namespace paged
}  // namespace asg

extern "C" {

int asg_paged_cache_write(const int64_t* slots, int64_t n_tokens, const asg_token_rows* key, const asg_token_rows* value,
                          const asg_page_pool* key_pool, const asg_page_pool* value_pool, int64_t n_pages,
                          int64_t page_size, int n_heads, int head_dim, int in_type, int cache_type, void* stream_ptr) {
  using namespace asg;
  using namespace asg::paged;
  CacheArgs a;
  if (int rc = fill_args(a, slots, n_tokens, key, value, key_pool, value_pool, n_pages, page_size, n_heads, head_dim,
                         in_type, cache_type)) return rc;
  ASG_REQUIRE(is_coded(cache_type) || cache_type == in_type, ASG_EINVAL,
              "the pages must have the type of the tokens or an 8-bit type");
  if (n_tokens == 0 || n_pages == 0) return ASG_OK;
  DeviceGuard guard(a.pools[0].data);
  ASG_CUDA(guard.status);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (in_type == ASG_TYPE_F32) return launch_write<F32>(a, cache_type, stream);
  if (in_type == ASG_TYPE_BF16) return launch_write<BF16>(a, cache_type, stream);
  return launch_write<F16>(a, cache_type, stream);
}

int asg_paged_cache_read(const int64_t* slots, int64_t n_tokens, const asg_token_rows* key, const asg_token_rows* value,
                         const asg_page_pool* key_pool, const asg_page_pool* value_pool, int64_t n_pages,
                         int64_t page_size, int n_heads, int head_dim, int out_type, int cache_type, void* stream_ptr) {
  using namespace asg;
  using namespace asg::paged;
  CacheArgs a;
  if (int rc = fill_args(a, slots, n_tokens, key, value, key_pool, value_pool, n_pages, page_size, n_heads, head_dim,
                         out_type, cache_type)) return rc;
  if (n_tokens == 0) return ASG_OK;
  DeviceGuard guard(a.rows[0].data);
  ASG_CUDA(guard.status);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  switch (cache_type) {
    case ASG_TYPE_F32: return launch_read<F32>(a, out_type, stream);
    case ASG_TYPE_BF16: return launch_read<BF16>(a, out_type, stream);
    case ASG_TYPE_F16: return launch_read<F16>(a, out_type, stream);
    case ASG_TYPE_E4M3: return launch_read<E4M3>(a, out_type, stream);
    default: return launch_read<INT8>(a, out_type, stream);
  }
}

}  // extern "C"
