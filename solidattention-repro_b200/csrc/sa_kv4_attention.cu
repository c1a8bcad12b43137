// sa_kv4_attention.cu -- GQA attention of a batch's newest tokens over the
// 4-bit paged cache.
//
//   x_t = scale * sum_d q_d (s_t,g c_t,d + m_t,g)      softmax over the tokens seen
//   o_d = sum_t p_t (s'_t,g c'_t,d + m'_t,g) / sum_t p_t
//
// One CTA per (request, new token, query head): each warp walks its share of
// the row's blocks, a lane scoring one token and owning D / 32 output elements,
// with a running maximum and sum; the warps are merged at the end.
#include "sa_kv4.cuh"

namespace sa {
namespace {

constexpr int kMaxLists = 8192;

struct Kv4AttnParams {
  const void* query;
  int64_t stride_request, stride_token, stride_head;
  int query_type, out_type;
  const uint8_t* pool;
  const int32_t* table;
  const int32_t* seq_lens;
  const int32_t* selected;
  const int32_t* selected_count;
  void* out;
  float* lse;
  uint32_t* status;
  int pool_blocks, table_blocks, lists_per_request, budget;
  int requests, new_tokens, query_heads, kv_heads, head_dim;
  float scale;
};

__device__ __forceinline__ float load_as_float(const void* base, int64_t i, int type) {
  if (type == SA_TYPE_F32) return static_cast<const float*>(base)[i];
  if (type == SA_TYPE_F16) return __half2float(static_cast<const __half*>(base)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
}

__device__ __forceinline__ void store_from_float(void* base, int64_t i, int type, float x) {
  if (type == SA_TYPE_F32)
    static_cast<float*>(base)[i] = x;
  else if (type == SA_TYPE_F16)
    static_cast<__half*>(base)[i] = __float2half_rn(x);
  else
    static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
}

// A request's length, 0 (and a status bit) when it is out of range.
__device__ __forceinline__ int checked_length(int length, int table_blocks, uint32_t* status) {
  if (length >= 0 && length <= static_cast<int64_t>(table_blocks) * kBlockTokens) return length;
  raise_status(status, SA_DEV_BAD_BLOCK);
  return 0;
}

constexpr int kWarps = 4;

__global__ void __launch_bounds__(kWarps * 32) attention_simple(const Kv4AttnParams p) {
  __shared__ float q[256];
  __shared__ float part[kWarps][2 + 256];
  const int d = p.head_dim, per_lane = d / 32, groups = d / kKv4Group;
  const int row = blockIdx.x;
  const int head = row % p.query_heads, i = row / p.query_heads % p.new_tokens;
  const int b = row / p.query_heads / p.new_tokens;
  const int kv_head = head / (p.query_heads / p.kv_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < d; e += blockDim.x)
    q[e] = load_as_float(p.query, b * p.stride_request + i * p.stride_token +
                                      head * p.stride_head + e, p.query_type);
  __syncthreads();
  const int length = checked_length(p.seq_lens[b], p.table_blocks, p.status);
  const int seen = length - p.new_tokens + i + 1;  // tokens this row sees
  const int blocks = (length + kBlockTokens - 1) / kBlockTokens;
  const int list = b * p.lists_per_request + kv_head / (p.kv_heads / p.lists_per_request);
  const int32_t* ids = p.selected ? p.selected + static_cast<int64_t>(list) * p.budget : nullptr;
  int entries = blocks;
  if (ids && blocks > 0) entries = min(max(p.selected_count[list], 0), p.budget) + 1;
  float top = -INFINITY, sum = 0.0f, o[8] = {};
  for (int e = warp; e < entries; e += kWarps) {
    int logical = e;
    if (ids) {
      logical = blocks - 1;
      if (e < entries - 1) {
        logical = ids[e];
        if (logical < 0 || logical >= blocks - 1 || (e > 0 && logical <= ids[e - 1])) {
          raise_status(p.status, SA_DEV_BAD_BLOCK);
          continue;
        }
      }
    }
    const int block = p.table[static_cast<int64_t>(b) * p.table_blocks + logical];
    if (block < 0 || block >= p.pool_blocks) {
      raise_status(p.status, SA_DEV_BAD_BLOCK);
      continue;
    }
    const uint8_t* entry = p.pool + (static_cast<int64_t>(block) * p.kv_heads + kv_head) *
                                        kv4_entry_bytes(d);
    const bool sees = logical * kBlockTokens + lane < seen;
    float x = -INFINITY;
    if (sees) {
      x = 0.0f;
      for (int g = 0; g < groups; ++g) {
        float dot = 0.0f, all = 0.0f;
        for (int t = 0; t < 4; ++t) {
          const uint2 w = *reinterpret_cast<const uint2*>(entry + kv4_key_at(d, lane, g, t));
          for (int j = 0; j < 16; ++j) {
            const float qj = q[g * kKv4Group + 16 * t + j];
            dot += qj * static_cast<float>(((j < 8 ? w.x : w.y) >> (4 * (j & 7))) & 15u);
            all += qj;
          }
        }
        const __half2 sm =
            *reinterpret_cast<const __half2*>(entry + kv4_key_scale_at(d, lane, g));
        x += __low2float(sm) * dot + __high2float(sm) * all;
      }
      x *= p.scale;
    }
    float new_top = fmaxf(top, x);
    for (int s = 16; s > 0; s >>= 1)
      new_top = fmaxf(new_top, __shfl_xor_sync(0xffffffffu, new_top, s));
    if (new_top == -INFINITY) continue;
    const float keep = expf(top - new_top), pr = sees ? expf(x - new_top) : 0.0f;
    top = new_top;
    float block_sum = pr;
    for (int s = 16; s > 0; s >>= 1) block_sum += __shfl_xor_sync(0xffffffffu, block_sum, s);
    sum = sum * keep + block_sum;
    for (int j = 0; j < per_lane; ++j) o[j] *= keep;
    for (int r = 0; r < kBlockTokens; ++r) {
      if (logical * kBlockTokens + r >= seen) break;
      const float pt = __shfl_sync(0xffffffffu, pr, r);
      for (int j = 0; j < per_lane; ++j) {
        const int el = lane * per_lane + j, g = el / kKv4Group, in = el % kKv4Group;
        const uint32_t byte =
            entry[kv4_value_at(d, r, g, in / 8, in % 8 / 4, in % 4 / 2)];
        const __half* at = reinterpret_cast<const __half*>(entry + kv4_value_scale_at(d, r, g));
        o[j] += pt * (__half2float(at[0]) * static_cast<float>((byte >> (4 * (in & 1))) & 15u) +
                      __half2float(at[d / 2]));
      }
    }
  }
  if (lane == 0) {
    part[warp][0] = top;
    part[warp][1] = sum;
  }
  for (int j = 0; j < per_lane; ++j) part[warp][2 + lane * per_lane + j] = o[j];
  __syncthreads();
  float all_top = -INFINITY, all_sum = 0.0f;
  for (int w = 0; w < kWarps; ++w) all_top = fmaxf(all_top, part[w][0]);
  for (int w = 0; w < kWarps; ++w)
    if (part[w][1] != 0.0f) all_sum += part[w][1] * expf(part[w][0] - all_top);
  for (int e = threadIdx.x; e < d; e += blockDim.x) {
    float value = 0.0f;
    for (int w = 0; w < kWarps; ++w)
      if (part[w][1] != 0.0f) value += part[w][2 + e] * expf(part[w][0] - all_top);
    store_from_float(p.out, static_cast<int64_t>(row) * d + e, p.out_type,
                     all_sum != 0.0f ? value / all_sum : 0.0f);
  }
  if (p.lse && threadIdx.x == 0)
    p.lse[row] = all_sum != 0.0f ? all_top + logf(all_sum) : -INFINITY;
}

bool known_type(int type) {
  return type == SA_TYPE_F32 || type == SA_TYPE_F16 || type == SA_TYPE_BF16;
}

}  // namespace
}  // namespace sa

using namespace sa;

extern "C" SA_API size_t sa_attention_kv4_workspace_size(size_t requests, size_t new_tokens,
                                                         size_t query_heads, size_t kv_heads,
                                                         size_t head_dim) {
  if (requests == 0 || new_tokens == 0 || kv_heads == 0 || query_heads == 0 ||
      query_heads % kv_heads != 0 || sa_kv4_entry_bytes(head_dim) == 0)
    return 0;
  return 256;
}

extern "C" SA_API sa_status sa_attention_kv4(
    const void* query, int query_type, int64_t stride_request, int64_t stride_token,
    int64_t stride_head, const void* pool, size_t pool_blocks, const int32_t* block_table,
    size_t table_blocks, const int32_t* seq_lens, const int32_t* selected,
    const int32_t* selected_count, size_t select_groups, size_t budget, size_t requests,
    size_t new_tokens, size_t query_heads, size_t kv_heads, size_t head_dim, float scale, void* out,
    int out_type, float* lse_out, void* workspace, size_t workspace_bytes, uint32_t* status,
    void* stream) {
  if (!query || !pool || !block_table || !seq_lens || !out)
    return fail(SA_ERR_INVALID_ARG, "attention_kv4: null pointer");
  if (kv_heads == 0 || query_heads == 0 || query_heads % kv_heads != 0 || requests == 0 ||
      new_tokens == 0 || pool_blocks == 0 || table_blocks == 0)
    return fail(SA_ERR_INVALID_ARG, "invalid GQA attention dimensions");
  if (!known_type(query_type) || !known_type(out_type))
    return fail(SA_ERR_INVALID_ARG, "attention_kv4: unknown element type");
  if (query_type != SA_TYPE_F32 && out_type != query_type)
    return fail(SA_ERR_UNSUPPORTED, "attention_kv4: a 16-bit query gives an output of its own type");
  if (sa_kv4_entry_bytes(head_dim) == 0)
    return fail(SA_ERR_UNSUPPORTED, "attention_kv4: head_dim must be 64, 128 or 256");
  if ((reinterpret_cast<uintptr_t>(pool) & 15u) != 0)
    return fail(SA_ERR_INVALID_ARG, "attention_kv4: the pool must be 16-byte aligned");
  size_t lists = 1;
  if (selected) {
    if (!selected_count || budget == 0 || select_groups == 0 || kv_heads % select_groups != 0)
      return fail(SA_ERR_INVALID_ARG, "attention_kv4: invalid selection");
    if (new_tokens != 1)
      return fail(SA_ERR_UNSUPPORTED, "attention_kv4: a selection serves one new token a request");
    lists = select_groups;
  }
  if (requests * lists > (size_t)kMaxLists || requests > (size_t)kMaxLists)
    return fail(SA_ERR_UNSUPPORTED, "attention_kv4: more than 8192 requests or lists");
  if (pool_blocks > 0x7fffffffu / kBlockTokens || table_blocks > 0x7fffffffu / kBlockTokens)
    return fail(SA_ERR_UNSUPPORTED, "attention_kv4: more than 2^31 slots");
  const size_t need =
      sa_attention_kv4_workspace_size(requests, new_tokens, query_heads, kv_heads, head_dim);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
    return fail(SA_ERR_CAPACITY,
                "attention_kv4: workspace unaligned or smaller than sa_attention_kv4_workspace_size()");
  if (requests * new_tokens * query_heads > 0x7fffffffu)
    return fail(SA_ERR_UNSUPPORTED, "attention_kv4: too many query rows");
  Kv4AttnParams p{};
  p.query = query;
  p.stride_request = stride_request;
  p.stride_token = stride_token;
  p.stride_head = stride_head;
  p.query_type = query_type;
  p.out_type = out_type;
  p.pool = static_cast<const uint8_t*>(pool);
  p.table = block_table;
  p.seq_lens = seq_lens;
  p.selected = selected;
  p.selected_count = selected_count;
  p.out = out;
  p.lse = lse_out;
  p.status = status;
  p.pool_blocks = (int)pool_blocks;
  p.table_blocks = (int)table_blocks;
  p.lists_per_request = (int)lists;
  p.budget = (int)budget;
  p.requests = (int)requests;
  p.new_tokens = (int)new_tokens;
  p.query_heads = (int)query_heads;
  p.kv_heads = (int)kv_heads;
  p.head_dim = (int)head_dim;
  p.scale = scale;
  attention_simple<<<(unsigned)(requests * new_tokens * query_heads), kWarps * 32, 0,
                     static_cast<cudaStream_t>(stream)>>>(p);
  return cuda_status(cudaGetLastError(), "attention_kv4 launch");
}
