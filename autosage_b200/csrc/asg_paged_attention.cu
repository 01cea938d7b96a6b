// Paged attention: C entry points and the kernel that joins the pieces of items shared by several CTAs.
#include <mutex>

#include "asg_paged_attention.cuh"

namespace asg {
namespace paged {

size_t workspace_bytes_for(int ctas, int gt, int dim) {
  const size_t records = static_cast<size_t>(ctas) * 2 * gt;
  return align256(static_cast<size_t>(ctas) * sizeof(int4)) + align256(records * sizeof(float2)) + align256(records * ((dim + 3) / 4 * 4) * sizeof(float));
}

constexpr int kJoinThreads = 256;

// Block (c, y): if CTA c's last piece starts an item that it does not finish, puts that item together from CTA c's
// piece and the first pieces of the CTAs after it.  A thread owns four features of a head and walks through the
// pieces with a running maximum, like the warps through the tokens.  Usually an item has a few pieces, and a
// thread takes them all; where items are so few that each has many (`sliced`), block y is a head of its own, groups of
// threads take every slices-th piece, and their parts are added in a fixed order.
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttentionArgs a, int ctas, int gt, bool sliced) {
  __shared__ float4 s_acc[kJoinThreads];
  __shared__ float2 s_stat[kJoinThreads];
  const int c = blockIdx.x, tid = threadIdx.x;
  if (blockIdx.y == 0) clear_empty_rows(a, c, ctas);
  pdl_wait_for_primary();
  const int4 piece = a.pieces[c];
  const int n = min(piece.z, ctas - c);  // of its pieces; 0: none starts here
  // (the workspace is the caller's: should anything else have written to it, no row is addressed that is not there)
  if (n <= 0 || static_cast<unsigned>(piece.x) >= static_cast<unsigned>(a.n_rows) ||
      static_cast<unsigned>(piece.y) >= static_cast<unsigned>(a.n_kv_heads * a.subgroups)) return;
  const int kv_head = piece.y / a.subgroups, sub = piece.y - kv_head * a.subgroups;
  const int heads = min(gt, a.group - sub * gt);
  const int fours = (a.dim + 3) / 4;
  int slices = 1;  // a power of two
  while (sliced && slices * 2 * fours <= kJoinThreads) slices *= 2;
  const int columns = sliced ? fours : heads * fours;
  const int slice = sliced ? tid / fours : 0;
  const int column = sliced ? tid - slice * fours : static_cast<int>(blockIdx.y) * kJoinThreads + tid;
  const int g = sliced ? static_cast<int>(blockIdx.y) : column / fours;
  const int d = (column - (sliced ? 0 : g * fours)) * 4;
  const bool active = slice < slices && column < columns && g < heads;
  float top = -CUDART_INF_F, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float2 s, float4 x) {
    const float m = fmaxf(top, s.x);
    const float keep = part_factor(top, sum, m), f = part_factor(s.x, s.y, m);
    top = m;
    sum = sum * keep + s.y * f;
    acc.x = acc.x * keep + x.x * f;
    acc.y = acc.y * keep + x.y * f;
    acc.z = acc.z * keep + x.z * f;
    acc.w = acc.w * keep + x.w * f;
  };
  if (active) {
#pragma unroll 4
    for (int i = slice; i < n; i += slices) {
      const long long record = (static_cast<long long>(c + i) * 2 + (i == 0 ? 1 : 0)) * gt + g;
      add(a.stats[record], *reinterpret_cast<const float4*>(a.partial + record * a.partial_pitch + d));
    }
  }
  if (sliced) {  // uniform
    s_stat[tid] = make_float2(top, sum);
    s_acc[tid] = acc;
    __syncthreads();
    if (active && slice == 0)
      for (int i = 1; i < slices; ++i) add(s_stat[i * fours + column], s_acc[i * fours + column]);
  }
  if (active && slice == 0) {
    const long long row = static_cast<long long>(piece.x) * a.n_heads + kv_head * a.group + sub * gt + g;
    const float scale = sum == 0.f ? 0.f : 1.f / sum;
    store_four(a, row, d, make_float4(acc.x * scale, acc.y * scale, acc.z * scale, acc.w * scale));
    if (a.lse != nullptr && d == 0) a.lse[row] = log_sum(top, sum);
  }
}

static int launch_join(const AttentionArgs& args, int ctas, int gt, int64_t items, cudaStream_t stream) {
  const int heads = args.group < gt ? args.group : gt;
  const bool sliced = items * 8 < ctas;
  const int blocks = sliced ? heads : (heads * ((args.dim + 3) / 4) + kJoinThreads - 1) / kJoinThreads;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(blocks));
  config.blockDim = dim3(kJoinThreads);
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  ASG_CUDA(cudaLaunchKernelEx(&config, join_kernel, args, ctas, gt, sliced));
  return ASG_OK;
}

}  // namespace paged
}  // namespace asg

extern "C" {

size_t asg_paged_attention_workspace_bytes(int n_heads, int n_kv_heads, int head_dim) {
  using namespace asg::paged;
  if (n_heads < 1 || n_kv_heads < 1 || head_dim < 1 || head_dim > kMaxDim || n_heads % n_kv_heads != 0) return 0;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) cudaGetLastError();
  return workspace_bytes_for(asg::sm_count(device) * kMaxCtasPerSm, n_heads / n_kv_heads > 8 ? 16 : 8, head_dim);
}

int asg_paged_attention(const asg_paged_attention_args* args) {
  using namespace asg;
  using namespace asg::paged;
  ASG_REQUIRE(args != nullptr, ASG_EINVAL, "args must not be null");
  const int64_t n_rows = args->n_rows, n_cols = args->n_cols, n_heads = args->n_heads, n_kv_heads = args->n_kv_heads;
  const int64_t page_size = args->page_size, head_dim = args->head_dim, type = args->type, cache_type = args->cache_type;
  if (int rc = check_pools(args->key_pool, args->value_pool, args->n_pages, page_size, n_kv_heads, head_dim, type, cache_type))
    return rc;
  ASG_REQUIRE(is_coded(cache_type) || cache_type == type, ASG_EINVAL,
              "the pages must have the type of the query or an 8-bit type");
  ASG_REQUIRE(n_heads >= 1 && n_heads <= 65535 && n_heads % n_kv_heads == 0, ASG_EINVAL,
              "n_heads must be a positive multiple of n_kv_heads");
  ASG_REQUIRE(n_rows >= 0 && n_cols >= 0, ASG_EINVAL, "sizes must be non-negative");
  ASG_REQUIRE(n_rows < 2147483647ll - 2048 && n_cols < (1ll << 31), ASG_ERANGE, "n_rows or n_cols exceeds the kernel index range");
  ASG_REQUIRE(args->window >= 0, ASG_EINVAL, "window must not be negative");
  if (n_rows == 0) return ASG_OK;
  ASG_REQUIRE(args->crow != nullptr && args->lengths != nullptr && args->q.data != nullptr && args->out != nullptr, ASG_EINVAL,
              "crow, lengths, query and out must not be null");
  ASG_REQUIRE(n_cols == 0 || args->col != nullptr, ASG_EINVAL, "col must not be null");
  ASG_REQUIRE(args->workspace != nullptr, ASG_EWORKSPACE, "workspace pointer is null");
  ASG_REQUIRE((reinterpret_cast<uintptr_t>(args->workspace) & 255u) == 0, ASG_EWORKSPACE, "workspace must be 256-byte aligned");
  DeviceGuard guard(args->out);
  ASG_CUDA(guard.status);
  cudaStream_t stream = static_cast<cudaStream_t>(args->stream);
  AttentionArgs a = {};
  a.crow = args->crow;
  a.col = args->col;
  a.lengths = args->lengths;
  a.q = args->q.data;
  a.out = args->out;
  a.lse = args->lse;
  a.key = args->key_pool;
  a.value = args->value_pool;
  a.q_token_stride = args->q.token_stride;
  a.q_head_stride = args->q.head_stride;
  a.n_cols = n_cols;
  a.n_pages = args->n_pages;
  a.window = args->window;
  a.n_rows = static_cast<int>(n_rows);
  a.page_size = static_cast<int>(page_size);
  a.n_heads = static_cast<int>(n_heads);
  a.n_kv_heads = static_cast<int>(n_kv_heads);
  a.dim = static_cast<int>(head_dim);
  a.group = static_cast<int>(n_heads / n_kv_heads);
  a.type = static_cast<int>(type);
  a.scale_log2 = static_cast<float>(args->scale * 1.4426950408889634);
  a.q_fours = rows_aligned(args->q, type_bytes(type), 4 * type_bytes(type));
  a.same_strides = a.key.page_stride == a.value.page_stride && a.key.token_stride == a.value.token_stride;
  a.out_vector = head_dim % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0;
  a.partial_pitch = static_cast<int>((head_dim + 3) / 4 * 4);
  // Tensor cores wherever 16-byte copies can fetch the rows, save for float32 pages, whose products have to keep 24 bits
  // on both sides; everything else on the FMA pipe
  const int pages_type = static_cast<int>(cache_type);
  Choice choice = is_coded(cache_type) ? choose_tensor8(a, pages_type) : choose_tensor16(a, pages_type);
  if (choice.launch == nullptr) choice = choose_general(a, pages_type);
  a.subgroups = (a.group + choice.gt - 1) / choice.gt;
  // no more CTAs than units there can be (every row may end in a partly filled one)
  const int64_t items = n_kv_heads * a.subgroups;
  const double most = (static_cast<double>(n_cols) * page_size / kUnit + n_rows) * items;
  ASG_REQUIRE(most + static_cast<double>(n_rows) * kStart * items < 2e9, ASG_ERANGE,
              "the page table lists more than 2^37 tokens and heads");
  int ctas = sm_count(guard.target) * choice.ctas_per_sm;
  if (most < ctas) ctas = most < 1 ? 1 : static_cast<int>(most);
  const size_t records = static_cast<size_t>(ctas) * 2 * choice.gt;
  ASG_REQUIRE(args->workspace_bytes >= workspace_bytes_for(ctas, choice.gt, a.dim), ASG_EWORKSPACE,
              "workspace is smaller than asg_paged_attention_workspace_bytes");
  char* at = static_cast<char*>(args->workspace);
  a.pieces = reinterpret_cast<int4*>(at);
  at += align256(static_cast<size_t>(ctas) * sizeof(int4));
  a.stats = reinterpret_cast<float2*>(at);
  at += align256(records * sizeof(float2));
  a.partial = reinterpret_cast<float*>(at);
  // an item of at most one unit is never cut, and no row has more tokens than all pages of the table
  a.join = ctas > 1 && n_cols * page_size > kUnit;
  // the two launches of a call follow one another on the stream also when another host thread calls with the same
  // stream and workspace
  static std::mutex launching;
  std::lock_guard<std::mutex> hold(launching);
  if (int rc = choice.launch(a, ctas, stream)) return rc;
  return !a.join ? ASG_OK : launch_join(a, ctas, choice.gt, items * n_rows, stream);
}

}  // extern "C"
