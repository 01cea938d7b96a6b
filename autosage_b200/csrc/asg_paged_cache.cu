// Writing tokens into the pages of a cache, with or without quantising to 8 bits, and reading them back.
//
//   write   page row slots[t] = x[t, h, :]                       (same type), or
//           s = max_d |x_d| / Q,  code_d = nearest(x_d / s)       (Q = 448 for e4m3, 127 for int8)
//   read    x[t, h, d] = round(code_d * s)
//
// Both move every byte once and are bound by memory: a group of lanes owns the key row AND the value row
// of one (token, head), 32 bytes of the wide type a lane where the rows allow it, so two independent rows are in
// flight per lane and consecutive groups touch consecutive heads of a token (contiguous in the usual layouts).
//
// Rounding.  The quotient x / s is not rounded before the code is chosen: rounded to float32 it would often
// land exactly between two codes that the true quotient is not between, and the tie rule would then pick the wrong one.
//   16-bit x.  With t = max|x| the quotient is x Q / t times t / (Q s), which is 1 + e, |e| <= 2^-24, the same for
//     the whole row.  x Q / t is a quotient of short numbers: unless it lies ON a border b between codes it is
//     further than 2^-19 b away from it (x Q and b t are integers below 2^19 times a power of two).  So one
//     product x w with w = (1 / s) (1 + 2^-21 sign(e)) decides every code: its own error, below 2^-22, moves
//     nothing across a border, and what lies on a border goes where e sends it.  For e = 0 the quotient is
//     corrected by its remainder instead, which gives a quotient on a border exactly, and the tie rule holds.
//   float32 x.  The quotient is rounded "to odd" (Boldo and Melquiond, Emulation of FMA and correctly rounded sums, IEEE
//     Trans. Computers 2008: a value so rounded can be rounded again as if it were exact).  With y = 1 / s correctly rounded,
//     q0 = x y is within a unit in the last place of the quotient, and q = q0 + y (x - q0 s), the inner term by a fused
//     multiply-add, is the correctly rounded one (Markstein, Computation of elementary functions on the IBM RISC System/6000,
//     IBM J. Res. Dev. 1990).  All that is needed of it here is that the quotient lies between q and a neighbour: the
//     remainder x - q s is then exact, its sign names that neighbour, and of the two the one with an odd last bit is taken.
//     Borders have an even last bit, so rounding that value to a code gives the code nearest to the true quotient.
//   Scales so small or large that 1/s or a remainder would leave float32's range: division in float64.
#include "asg_paged.cuh"

namespace asg {
namespace paged {

struct CacheArgs {
  const int64_t* slots;
  long long n_tokens, n_slots;
  asg_token_rows rows[2];   // key, value
  asg_page_pool pools[2];
  int page_size, n_heads, dim;
  Divisor by_heads, by_page;
  bool small;       // rows and slots have 31-bit numbers
  bool same_rows;   // keys and values have the same strides: in the tokens, ...
  bool same_pools;  // ... in the pages and scales
};

// Where row r = (token, head) of the tokens and its place in the pages lie, in elements; one offset each for key and
// value.  `held`: the row's slot is inside the cache.
struct RowPlace {
  long long token_at[2], page_at[2], scale_at[2];
  bool held;
  __device__ __forceinline__ RowPlace(const CacheArgs& a, long long r, bool coded) {
    long long token, page = 0, slot;
    int head, place = 0;
    if (a.small) {  // a handful of instructions instead of some hundreds
      const unsigned t = divide(static_cast<unsigned>(r), a.by_heads);
      token = t;
      head = static_cast<int>(static_cast<unsigned>(r) - t * a.by_heads.d);
      slot = a.slots[t];
      held = slot >= 0 && slot < a.n_slots;
      if (held) {
        const unsigned p = divide(static_cast<unsigned>(slot), a.by_page);
        page = p;
        place = static_cast<int>(static_cast<unsigned>(slot) - p * a.by_page.d);
      }
    } else {
      token = r / a.n_heads;
      head = static_cast<int>(r - token * a.n_heads);
      slot = a.slots[token];
      held = slot >= 0 && slot < a.n_slots;
      if (held) {
        page = slot / a.page_size;
        place = static_cast<int>(slot - page * a.page_size);
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      token_at[w] = w == 1 && a.same_rows ? token_at[0] : token * a.rows[w].token_stride + head * a.rows[w].head_stride;
      const asg_page_pool& pool = a.pools[w];
      page_at[w] = w == 1 && a.same_pools ? page_at[0]
                                          : page * pool.page_stride + place * pool.token_stride + head * pool.head_stride;
      if (coded)
        scale_at[w] = w == 1 && a.same_pools
                          ? scale_at[0]
                          : page * pool.scale_page_stride + head * pool.scale_head_stride + place * pool.scale_token_stride;
    }
  }
};

constexpr int kThreads = 256;

constexpr float largest_code(E4M3) { return 448.f; }
constexpr float largest_code(INT8) { return 127.f; }

// x / s, rounded to odd in float32; inv = 1 / s, correctly rounded, s in [2^-90, 2^90].
__device__ __forceinline__ float quotient_to_odd(float x, float s, float inv) {
  const float q0 = x * inv;
  const float q = fmaf(fmaf(-q0, s, x), inv, q0);
  const float rest = fmaf(-q, s, x);
  const int bits = __float_as_int(q);
  const int step = ((__float_as_int(rest) ^ bits) < 0) ? -1 : 1;  // towards the remainder
  return __int_as_float(rest != 0.f && (bits & 1) == 0 ? bits + step : bits);
}
// The same by way of float64: a quotient of two 24-bit numbers is never nearer to a border between codes than
// 2^-40 of itself without lying on it, so 53 bits decide; they are rounded to odd too.  Cut to the largest code (a
// subnormal scale may be rounded far down); NaN, which the scale carries, becomes 0.
__device__ __noinline__ float quotient_by_double(float x, float s, float most) {
  double wide = static_cast<double>(x) / static_cast<double>(s);
  wide = wide != wide ? 0.0 : fmin(fmax(wide, -static_cast<double>(most)), static_cast<double>(most));
  const float q = static_cast<float>(wide);
  const double rest = wide - static_cast<double>(q);
  const int bits = __float_as_int(q);
  if (!(fabs(rest) > 0.0) || (bits & 1) != 0 || q == 0.f || isinf(q)) return q;
  return __int_as_float(bits + ((rest < 0.0) == (q < 0.f) ? 1 : -1));
}

// Four quotients to their nearest codes, ties to even.  (int8: added to 1.5 * 2^23 they are rounded to whole numbers, whose
// last eight bits are the code; magnitudes are at most 127 and a rounding error.)
__device__ __forceinline__ uint32_t nearest_codes(float a, float b, float c, float d, E4M3) {
  const uint32_t low = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t high = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return __byte_perm(low, high, 0x5410);
}
__device__ __forceinline__ uint32_t nearest_codes(float a, float b, float c, float d, INT8) {
  constexpr float middle = 12582912.f;
  const uint32_t low = __byte_perm(__float_as_uint(a + middle), __float_as_uint(b + middle), 0x0040);
  const uint32_t high = __byte_perm(__float_as_uint(c + middle), __float_as_uint(d + middle), 0x0040);
  return __byte_perm(low, high, 0x5410);
}

// P features a lane, next to one another, as one aligned vector of 32 bytes of the wide type, or (SPLIT) as two of 16 of
// which the second may lie past the row's end; P = 0: eight, one in 32 each, for any alignment and head size.
constexpr int lane_features(int p) { return p == 0 ? 8 : p; }

template <int P, bool SPLIT, typename T>
__device__ __forceinline__ void load_row(Pack<T, lane_features(P)>& x, const T* row, int lane, int dim) {
  constexpr int N = lane_features(P);
  if constexpr (P == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = i * 32 + lane < dim ? row[i * 32 + lane] : T{};
  } else {
    constexpr int kParts = SPLIT ? 2 : 1;
    using Part = Pack<T, N / kParts>;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      Part part;
      const int d = lane * P + i * (P / kParts);
      if (d < dim) {
        part.load(row + d);
      } else {
#pragma unroll
        for (int j = 0; j < N / kParts; ++j) part.v[j] = T{};
      }
#pragma unroll
      for (int j = 0; j < N / kParts; ++j) x.v[i * (N / kParts) + j] = part.v[j];
    }
  }
}

template <int P, bool SPLIT, typename T>
__device__ __forceinline__ void store_row(const Pack<T, lane_features(P)>& x, T* row, int lane, int dim) {
  constexpr int N = lane_features(P);
  if constexpr (P == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * 32 + lane < dim) row[i * 32 + lane] = x.v[i];
  } else {
    constexpr int kParts = SPLIT ? 2 : 1;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int d = lane * P + i * (P / kParts);
      Pack<T, N / kParts> part;
#pragma unroll
      for (int j = 0; j < N / kParts; ++j) part.v[j] = x.v[i * (N / kParts) + j];
      if (d < dim) part.store(row + d);
    }
  }
}

// The largest magnitude of a row, by its bits: a NaN is above everything and is not lost.  All lanes of the warp.
template <typename IN, int N>
__device__ __forceinline__ float largest_of_row(const Pack<IN, N>& x, int group) {
  if constexpr (sizeof(IN) == 2) {
    const uint32_t* two = reinterpret_cast<const uint32_t*>(x.v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) top = __vmaxu2(top, two[i] & 0x7fff7fffu);
    for (int o = group >> 1; o >= 1; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(kFull, top, o));
    const uint16_t one = static_cast<uint16_t>(max(top & 0xffffu, top >> 16));
    return to_float(*reinterpret_cast<const IN*>(&one));
  } else {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(x.v[i]) & 0x7fffffffu);
    for (int o = group >> 1; o >= 1; o >>= 1) top = max(top, __shfl_xor_sync(kFull, top, o));
    return __uint_as_float(top);
  }
}

// Codes and scale of a row whose largest magnitude is `top`.
template <typename IN, typename CACHE, int N>
__device__ __forceinline__ float quantise(const Pack<IN, N>& x, float top, Pack<CACHE, N>& c) {
  constexpr float most = largest_code(CACHE{});
  float v[N];
  to_floats(x, v);
  float s;
  if (top > 0x1p-80f && top < 0x1p90f) {
    constexpr float share = 1.f / most;  // correctly rounded, so that the same theorem gives the scale
    s = top * share;
    s = fmaf(fmaf(-s, most, top), share, s);
    const float inv = __frcp_rn(s);
    if constexpr (sizeof(IN) == 2) {
      const float off = fmaf(-s, most, top);  // exact; its sign is that of e
      if (off != 0.f) {
        const float w = inv * (off > 0.f ? 1.f + 0x1p-21f : 1.f - 0x1p-21f);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= w;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float q0 = v[i] * inv;
          v[i] = fmaf(fmaf(-q0, s, v[i]), inv, q0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = quotient_to_odd(v[i], s, inv);
    }
  } else {
    s = top / most;
    if (s == 0.f) {  // nothing but zeros, or values that no scale above 0 reaches
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 0.f;
    } else {
#pragma unroll 1
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j)  // (registers cannot be indexed)
          if (j == i) v[j] = quotient_by_double(v[j], s, most);
      }
    }
  }
  static_assert(N % 4 == 0, "codes are packed four at a time");
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    reinterpret_cast<uint32_t*>(c.v)[i] = nearest_codes(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], CACHE{});
  return s;
}

template <typename IN, typename CACHE, int P, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 4) write_kernel(const CacheArgs a, int group) {
  constexpr int N = lane_features(P);
  const int lane = threadIdx.x & (group - 1);
  const long long n_rows = a.n_tokens * a.n_heads;
  const int groups = kThreads / group;
  const long long stride = static_cast<long long>(gridDim.x) * groups;
  // all groups of a block go round together (the largest of a row is found by the whole warp)
  for (long long base = static_cast<long long>(blockIdx.x) * groups; base < n_rows; base += stride) {
    const long long r = base + threadIdx.x / group;
    const RowPlace at(a, r < n_rows ? r : n_rows - 1, TypeOf<CACHE>::coded);
    const bool ok = r < n_rows && at.held;
    Pack<IN, N> x[2];
#pragma unroll
    for (int w = 0; w < 2; ++w)
      // (a skipped token's row is loaded too: the loads need not wait for its slot)
      load_row<P, SPLIT>(x[w], static_cast<const IN*>(a.rows[w].data) + at.token_at[w], lane, r < n_rows ? a.dim : 0);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      CACHE* to = static_cast<CACHE*>(a.pools[w].data) + at.page_at[w];
      if constexpr (!TypeOf<CACHE>::coded) {
        store_row<P, SPLIT>(x[w], to, lane, ok ? a.dim : 0);
      } else {
        const float top = largest_of_row(x[w], group);
        Pack<CACHE, N> c;
        const float s = quantise(x[w], ok ? top : 0.f, c);
        store_row<P, SPLIT>(c, to, lane, ok ? a.dim : 0);
        if (ok && lane == 0) a.pools[w].scales[at.scale_at[w]] = s;
      }
    }
  }
}

template <typename CACHE, typename OUT, int P, bool SPLIT>
__global__ void __launch_bounds__(kThreads) read_kernel(const CacheArgs a, int group) {
  constexpr int N = lane_features(P);
  const int lane = threadIdx.x & (group - 1);
  const long long n_rows = a.n_tokens * a.n_heads;
  const int groups = kThreads / group;
  const long long stride = static_cast<long long>(gridDim.x) * groups;
  for (long long r = static_cast<long long>(blockIdx.x) * groups + threadIdx.x / group; r < n_rows; r += stride) {
    const RowPlace at(a, r, TypeOf<CACHE>::coded);
    Pack<CACHE, N> c[2];
    float s[2] = {1.f, 1.f};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      load_row<P, SPLIT>(c[w], static_cast<const CACHE*>(a.pools[w].data) + at.page_at[w], lane, at.held ? a.dim : 0);
      if (TypeOf<CACHE>::coded && at.held) s[w] = a.pools[w].scales[at.scale_at[w]];
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float v[N];
      to_floats(c[w], v);
      Pack<OUT, N> x;
#pragma unroll
      for (int i = 0; i < N; ++i) x.v[i] = from_float<OUT>(TypeOf<CACHE>::coded ? v[i] * s[w] : v[i]);
      store_row<P, SPLIT>(x, static_cast<OUT*>(a.rows[w].data) + at.token_at[w], lane, a.dim);
    }
  }
}

// Rows made of whole 32-byte packs of the wide type that start on 32 bytes are moved in those, rows of whole 16-byte packs
// in pairs of these; anything else takes a warp a row, one feature in 32 a lane.
enum class Form { whole, split, single };
struct Shape {
  Form form;
  int group;  // lanes per row
  unsigned blocks;
};

static Shape shape_of(const CacheArgs& a, int wide_type, int cache_type) {
  const int wide = type_bytes(wide_type), item = type_bytes(cache_type), p = 32 / wide;
  auto fits = [&](int bytes) {  // vectors of that many bytes of the wide type
    const int n = bytes / wide, packed = n * item < 32 ? n * item : 32;
    bool ok = a.dim % n == 0;
    for (int w = 0; w < 2; ++w) ok = ok && rows_aligned(a.rows[w], wide, bytes) && rows_aligned(a.pools[w], item, packed);
    return ok;
  };
  Shape s;
  s.form = fits(32) ? Form::whole : fits(16) ? Form::split : Form::single;
  s.group = 32;
  while (s.form != Form::single && s.group > 1 && s.group / 2 * p >= a.dim) s.group /= 2;
  const long long rows_per_block = kThreads / s.group;
  const long long blocks = (a.n_tokens * a.n_heads + rows_per_block - 1) / rows_per_block;
  s.blocks = static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20));
  return s;
}

template <typename IN, typename CACHE>
static int launch_write(const CacheArgs& a, cudaStream_t stream) {
  constexpr int p = 32 / static_cast<int>(sizeof(IN));
  const Shape s = shape_of(a, TypeOf<IN>::id, TypeOf<CACHE>::id);
  if (s.form == Form::whole) write_kernel<IN, CACHE, p, false><<<s.blocks, kThreads, 0, stream>>>(a, s.group);
  else if (s.form == Form::split) write_kernel<IN, CACHE, p, true><<<s.blocks, kThreads, 0, stream>>>(a, s.group);
  else write_kernel<IN, CACHE, 0, false><<<s.blocks, kThreads, 0, stream>>>(a, s.group);
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
  constexpr int p = 32 / static_cast<int>(sizeof(OUT));
  const Shape s = shape_of(a, TypeOf<OUT>::id, TypeOf<CACHE>::id);
  if (s.form == Form::whole) read_kernel<CACHE, OUT, p, false><<<s.blocks, kThreads, 0, stream>>>(a, s.group);
  else if (s.form == Form::split) read_kernel<CACHE, OUT, p, true><<<s.blocks, kThreads, 0, stream>>>(a, s.group);
  else read_kernel<CACHE, OUT, 0, false><<<s.blocks, kThreads, 0, stream>>>(a, s.group);
  ASG_CUDA(cudaGetLastError());
  return ASG_OK;
}
template <typename CACHE>
static int launch_read(const CacheArgs& a, int out_type, cudaStream_t stream) {
  if (out_type == ASG_TYPE_F32) return launch_read<CACHE, F32>(a, stream);
  if (out_type == ASG_TYPE_BF16) return launch_read<CACHE, BF16>(a, stream);
  return launch_read<CACHE, F16>(a, stream);
}

static int fill_args(CacheArgs& a, const asg_paged_cache_args* args) {
  ASG_REQUIRE(args != nullptr, ASG_EINVAL, "args must not be null");
  const asg_page_pool &key = args->key_pool, &value = args->value_pool;
  if (int rc = check_pools(key, value, args->n_pages, args->page_size, args->n_heads, args->head_dim, args->token_type,
                           args->cache_type)) return rc;
  ASG_REQUIRE(args->n_tokens >= 0, ASG_EINVAL, "n_tokens must be non-negative");
  ASG_REQUIRE(args->n_tokens <= (1ll << 40), ASG_ERANGE, "n_tokens exceeds the kernel index range");
  ASG_REQUIRE(args->n_tokens == 0 || (args->slots != nullptr && args->key.data != nullptr && args->value.data != nullptr),
              ASG_EINVAL, "slots, key and value must not be null");
  a.slots = args->slots;
  a.n_tokens = args->n_tokens;
  a.n_slots = args->n_pages * args->page_size;
  a.rows[0] = args->key;
  a.rows[1] = args->value;
  a.pools[0] = key;
  a.pools[1] = value;
  a.page_size = static_cast<int>(args->page_size);
  a.n_heads = static_cast<int>(args->n_heads);
  a.dim = static_cast<int>(args->head_dim);
  a.by_heads = divisor_of(static_cast<unsigned>(a.n_heads));
  a.by_page = divisor_of(static_cast<unsigned>(a.page_size));
  a.small = a.n_tokens * a.n_heads < (1ll << 31) && a.n_slots < (1ll << 31);
  a.same_rows = a.rows[0].token_stride == a.rows[1].token_stride && a.rows[0].head_stride == a.rows[1].head_stride;
  a.same_pools = key.page_stride == value.page_stride && key.token_stride == value.token_stride &&
                 key.head_stride == value.head_stride && key.scale_page_stride == value.scale_page_stride &&
                 key.scale_head_stride == value.scale_head_stride && key.scale_token_stride == value.scale_token_stride;
  return ASG_OK;
}

}  // namespace paged
}  // namespace asg

extern "C" {

int asg_paged_cache_write(const asg_paged_cache_args* args) {
  using namespace asg;
  using namespace asg::paged;
  CacheArgs a;
  if (int rc = fill_args(a, args)) return rc;
  ASG_REQUIRE(is_coded(args->cache_type) || args->cache_type == args->token_type, ASG_EINVAL,
              "the pages must have the type of the tokens or an 8-bit type");
  if (a.n_tokens == 0 || a.n_slots == 0) return ASG_OK;
  // one tensor for keys and values is written twice alike
  const bool same_tokens = a.same_rows && a.rows[0].data == a.rows[1].data;
  ASG_REQUIRE(same_tokens || (a.pools[0].data != a.pools[1].data &&
                              (!is_coded(args->cache_type) || a.pools[0].scales != a.pools[1].scales)), ASG_EINVAL,
              "different keys and values cannot be written to the same pages or scales");
  DeviceGuard guard(a.pools[0].data);
  ASG_CUDA(guard.status);
  cudaStream_t stream = static_cast<cudaStream_t>(args->stream);
  const int cache_type = static_cast<int>(args->cache_type);
  if (args->token_type == ASG_TYPE_F32) return launch_write<F32>(a, cache_type, stream);
  if (args->token_type == ASG_TYPE_BF16) return launch_write<BF16>(a, cache_type, stream);
  return launch_write<F16>(a, cache_type, stream);
}

int asg_paged_cache_read(const asg_paged_cache_args* args) {
  using namespace asg;
  using namespace asg::paged;
  CacheArgs a;
  if (int rc = fill_args(a, args)) return rc;
  if (a.n_tokens == 0) return ASG_OK;
  DeviceGuard guard(a.rows[0].data);
  ASG_CUDA(guard.status);
  cudaStream_t stream = static_cast<cudaStream_t>(args->stream);
  const int token_type = static_cast<int>(args->token_type);
  switch (args->cache_type) {
    case ASG_TYPE_F32: return launch_read<F32>(a, token_type, stream);
    case ASG_TYPE_BF16: return launch_read<BF16>(a, token_type, stream);
    case ASG_TYPE_F16: return launch_read<F16>(a, token_type, stream);
    case ASG_TYPE_E4M3: return launch_read<E4M3>(a, token_type, stream);
    default: return launch_read<INT8>(a, token_type, stream);
  }
}

}  // extern "C"
