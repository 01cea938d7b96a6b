// Paged attention: C entry points and the kernel that joins the pieces of items shared by several CTAs.
#include "asg_paged_attention.cuh"

namespace asg {
namespace paged {

size_t workspace_bytes_for(int ctas, int gt, int dim) {
  const size_t records = static_cast<size_t>(ctas) * 2 * gt;
  return align256(static_cast<size_t>(ctas) * sizeof(int4)) + align256(records * sizeof(float2)) + align256(records * ((dim + 3) / 4 * 4) * sizeof(float));
}

constexpr int kJoinThreads = 256;

// Block (c, y): if CTA c's last piece starts an item that it does not finish, puts the heads y, y + gridDim.y, ... of
// that item together from CTA c's piece and the first pieces of the CTAs after it.  The threads of a block share
// a head's features, four a thread, and where some are left over the pieces too; their sums are added in a fixed order.
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttentionArgs a, int ctas, int gt) {
  extern __shared__ float factor[];  // [ctas]
  __shared__ float s_part[kJoinThreads / 32];
  __shared__ float4 s_sum[kJoinThreads];
  __shared__ int s_last;
  const int c = blockIdx.x, tid = threadIdx.x;
  if (blockIdx.y == 0) clear_empty_rows(a, c, ctas);
  pdl_wait_for_primary();
  const int4 piece = a.pieces[c];
  if (piece.z == 0) return;
  const int kv_head = piece.y / a.subgroups, sub = piece.y - kv_head * a.subgroups;
  const int heads = min(gt, a.group - sub * gt);
  // the CTA that ends the item: the first after c whose first piece does not go on
  if (tid == 0) s_last = ctas - 1;
  __syncthreads();
  for (int base = c + 1; base < ctas; base += kJoinThreads) {
    const bool ends = base + tid < ctas && a.pieces[base + tid].w != 2;
    if (ends) atomicMin(&s_last, base + tid);
    if (__syncthreads_or(ends)) break;
  }
  const int n = s_last - c + 1;
  const int fours = (a.dim + 3) / 4;
  int slices = 1;  // threads that share four features, a power of two
  while (slices * 2 * fours <= kJoinThreads) slices *= 2;
  const int slice = tid / fours, column = tid - slice * fours;
  for (int g = blockIdx.y; g < heads; g += gridDim.y) {
    auto record = [&](int i) { return (static_cast<long long>(c + i) * 2 + (i == 0 ? 1 : 0)) * gt + g; };
    __syncthreads();  // factor, s_part and s_sum of the head before have been read
    float top = -CUDART_INF_F;
    for (int i = tid; i < n; i += kJoinThreads) top = fmaxf(top, a.stats[record(i)].x);
    top = warp_max(top);
    if ((tid & 31) == 0) s_part[tid >> 5] = top;
    __syncthreads();
    top = s_part[0];
#pragma unroll
    for (int w = 1; w < kJoinThreads / 32; ++w) top = fmaxf(top, s_part[w]);
    __syncthreads();
    float sum = 0.f;
    for (int i = tid; i < n; i += kJoinThreads) {
      const float2 s = a.stats[record(i)];
      factor[i] = part_factor(s.x, s.y, top);
      sum += factor[i] * s.y;
    }
    sum = warp_sum(sum);
    if ((tid & 31) == 0) s_part[tid >> 5] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) sum += s_part[w];
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (slice < slices) {
#pragma unroll 8
      for (int i = slice; i < n; i += slices) {
        const float4 x = *reinterpret_cast<const float4*>(a.partial + record(i) * a.partial_pitch + column * 4);
        const float f = factor[i];
        acc.x += f * x.x;
        acc.y += f * x.y;
        acc.z += f * x.z;
        acc.w += f * x.w;
      }
      s_sum[tid] = acc;
    }
    __syncthreads();
    const long long row = static_cast<long long>(piece.x) * a.n_heads + kv_head * a.group + sub * gt + g;
    if (slice == 0) {
      for (int i = 1; i < slices; ++i) {
        const float4 x = s_sum[i * fours + column];
        acc.x += x.x;
        acc.y += x.y;
        acc.z += x.z;
        acc.w += x.w;
      }
      const float scale = sum == 0.f ? 0.f : 1.f / sum;
      store_four(a, row, column * 4, make_float4(acc.x * scale, acc.y * scale, acc.z * scale, acc.w * scale));
    }
    if (a.lse != nullptr && tid == 0) a.lse[row] = log_sum(top, sum);
  }
}

static int launch_join(const AttentionArgs& args, int ctas, int gt, int64_t items, cudaStream_t stream) {
  // an item cut into many pieces is worth a block per head (there are few such items, so few blocks find work);
  // where items are cut once, one block goes through the heads
  const int heads = args.group < gt ? args.group : gt;
  const bool many = items * 4 < ctas;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(ctas), many ? static_cast<unsigned>(heads) : 1u);
  config.blockDim = dim3(kJoinThreads);
  config.dynamicSmemBytes = sizeof(float) * static_cast<size_t>(ctas);
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  ASG_CUDA(cudaLaunchKernelEx(&config, join_kernel, args, ctas, gt));
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
  return workspace_bytes_for(asg::sm_count(device) * kMaxCtasPerSm, 16, head_dim);
}

int asg_paged_attention(const int64_t* crow, const int64_t* col, const int64_t* lengths, int64_t n_rows, int64_t n_cols,
                        const asg_token_rows* q, void* out, float* lse, const asg_page_pool* key_pool,
                        const asg_page_pool* value_pool, int64_t n_pages, int64_t page_size, int n_heads,
                        int n_kv_heads, int head_dim, float scale, int64_t window, int type, int cache_type,
                        void* workspace, size_t workspace_bytes, void* stream_ptr) {
  using namespace asg;
  using namespace asg::paged;
  if (int rc = check_pools(key_pool, value_pool, n_pages, page_size, n_kv_heads, head_dim, type, cache_type)) return rc;
  ASG_REQUIRE(is_coded(cache_type) || cache_type == type, ASG_EINVAL,
              "the pages must have the type of the query or an 8-bit type");
  ASG_REQUIRE(n_heads >= 1 && n_heads <= 65535 && n_heads % n_kv_heads == 0, ASG_EINVAL,
              "n_heads must be a positive multiple of n_kv_heads");
  ASG_REQUIRE(n_rows >= 0 && n_cols >= 0, ASG_EINVAL, "sizes must be non-negative");
  ASG_REQUIRE(n_rows < 2147483647ll - 2048 && n_cols < (1ll << 31), ASG_ERANGE, "n_rows or n_cols exceeds the kernel index range");
  ASG_REQUIRE(window >= 0, ASG_EINVAL, "window must not be negative");
  if (n_rows == 0) return ASG_OK;
  ASG_REQUIRE(crow != nullptr && lengths != nullptr && q != nullptr && q->data != nullptr && out != nullptr, ASG_EINVAL,
              "crow, lengths, query and out must not be null");
  ASG_REQUIRE(n_cols == 0 || col != nullptr, ASG_EINVAL, "col must not be null");
  ASG_REQUIRE(workspace != nullptr, ASG_EWORKSPACE, "workspace pointer is null");
  ASG_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, ASG_EWORKSPACE, "workspace must be 256-byte aligned");
  DeviceGuard guard(out);
  ASG_CUDA(guard.status);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  AttentionArgs a = {};
  a.crow = crow;
  a.col = col;
  a.lengths = lengths;
  a.q = q->data;
  a.out = out;
  a.lse = lse;
  a.key = *key_pool;
  a.value = *value_pool;
  a.q_token_stride = q->token_stride;
  a.q_head_stride = q->head_stride;
  a.n_cols = n_cols;
  a.n_pages = n_pages;
  a.window = window;
  a.n_rows = static_cast<int>(n_rows);
  a.page_size = static_cast<int>(page_size);
  a.n_heads = n_heads;
  a.n_kv_heads = n_kv_heads;
  a.dim = head_dim;
  a.group = n_heads / n_kv_heads;
  a.type = type;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.q_pairs = rows_aligned(*q, type_bytes(type), 8);
  a.out_vector = head_dim % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  a.partial_pitch = (head_dim + 3) / 4 * 4;
  // 16-bit queries run on the tensor cores wherever 16-byte copies can fetch the rows; float32 queries, whose
  // products have to keep 24 bits, and everything else on the FMA pipe
  Choice choice = is_coded(cache_type) ? choose_tensor8(a, cache_type) : choose_tensor16(a, cache_type);
  if (choice.launch == nullptr) choice = choose_general(a, cache_type);
  a.subgroups = (a.group + choice.gt - 1) / choice.gt;
  // no more CTAs than units there can be (every row may end in a partly filled one)
  const int64_t items = static_cast<int64_t>(n_kv_heads) * a.subgroups;
  const double most = (static_cast<double>(n_cols) * page_size / kUnit + n_rows) * items;
  int ctas = sm_count(guard.target) * choice.ctas_per_sm;
  if (most < ctas) ctas = most < 1 ? 1 : static_cast<int>(most);
  const size_t records = static_cast<size_t>(ctas) * 2 * choice.gt;
  ASG_REQUIRE(workspace_bytes >= workspace_bytes_for(ctas, choice.gt, head_dim), ASG_EWORKSPACE,
              "workspace is smaller than asg_paged_attention_workspace_bytes");
  char* at = static_cast<char*>(workspace);
  a.pieces = reinterpret_cast<int4*>(at);
  at += align256(static_cast<size_t>(ctas) * sizeof(int4));
  a.stats = reinterpret_cast<float2*>(at);
  at += align256(records * sizeof(float2));
  a.partial = reinterpret_cast<float*>(at);
  if (int rc = choice.launch(a, ctas, stream)) return rc;
  if (ctas == 1) return ASG_OK;  // nothing is shared
  return launch_join(a, ctas, choice.gt, items * n_rows, stream);
}

}  // extern "C"
