// sa_kv4.cu -- rows into and out of the 4-bit cache.
//
// A thread owns 16 consecutive elements of one (token, KV head, key or value,
// group of 64): four neighbouring lanes make a group.
#include "sa_kv4.cuh"

namespace sa {
namespace {

struct PackParams {
  uint8_t* pool;
  const void* rows[2];  // keys, values
  int64_t token_stride[2], head_stride[2];
  const int32_t* slots;
  uint32_t* status;
  int64_t slot_limit;
  int64_t work;  // threads with work: tokens * 2 * kv_heads * groups * 4
  int kv_heads, head_dim;
};

struct UnpackParams {
  const uint8_t* pool;
  void* rows[2];
  const int32_t* slots;
  uint32_t* status;
  int64_t slot_limit;
  int64_t work;
  int kv_heads, head_dim;
};

// The largest FP16 value that is not above x, the smallest that is not below.
__device__ __forceinline__ __half half_below(float x) { return __float2half_rd(x); }
__device__ __forceinline__ __half half_above(float x) { return __float2half_ru(x); }

// What a thread works on.
struct Piece {
  int64_t token;
  int which, head, group, t;
};
__device__ __forceinline__ Piece piece_of(int64_t index, int kv_heads, int groups) {
  Piece c;
  c.t = static_cast<int>(index & 3);
  int64_t rest = index >> 2;
  c.group = static_cast<int>(rest % groups);
  rest /= groups;
  c.head = static_cast<int>(rest % kv_heads);
  rest /= kv_heads;
  c.which = static_cast<int>(rest & 1);
  c.token = rest >> 1;
  return c;
}

template <int TYPE>
__global__ void __launch_bounds__(256) pack_kernel(const PackParams p) {
  using Element = Kv4Type<TYPE>;
  const int64_t index = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const bool live = index < p.work;
  const int groups = p.head_dim / kKv4Group;
  const Piece c = piece_of(live ? index : 0, p.kv_heads, groups);
  const int64_t slot = live ? p.slots[c.token] : -1;
  const bool writes = slot >= 0 && slot < p.slot_limit;
  if (slot >= p.slot_limit && c.t == 0) raise_status(p.status, SA_DEV_BAD_BLOCK);
  float x[16];
  float low = INFINITY, high = -INFINITY;
  bool finite = true;
  const auto* row = static_cast<const typename Element::T*>(p.rows[c.which]) +
                    c.token * p.token_stride[c.which] + c.head * p.head_stride[c.which] +
                    c.group * kKv4Group + c.t * 16;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = writes ? Element::load(row[i]) : 0.0f;
    finite &= isfinite(x[i]);
    x[i] = fminf(fmaxf(x[i], -65504.0f), 65504.0f);
    low = fminf(low, x[i]);
    high = fmaxf(high, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    finite &= static_cast<bool>(__shfl_xor_sync(0xffffffffu, static_cast<int>(finite), o));
  }
  if (!writes) return;
  // Rounding up at each of the three operations gives the smallest FP16 step
  // whose fifteenth multiple reaches the maximum: 15 * step has 15 bits, so no
  // rounding in between can pass it.
  __half minimum = half_below(low);
  __half step = half_above(__fdiv_ru(__fsub_ru(high, __half2float(minimum)), 15.0f));
  const float m = __half2float(minimum), s = __half2float(step);
  uint32_t code[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    code[i] = finite && s > 0.0f ? static_cast<uint32_t>(rintf(__fdiv_rn(x[i] - m, s))) : 0u;
  if (!finite) minimum = step = __ushort_as_half(0x7fffu);
  const int block = static_cast<int>(slot / kBlockTokens), r = static_cast<int>(slot % kBlockTokens);
  uint8_t* entry = p.pool + (static_cast<int64_t>(block) * p.kv_heads + c.head) *
                                kv4_entry_bytes(p.head_dim);
  if (c.which == 0) {
    uint32_t word[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 16; ++i) word[i >> 3] |= code[i] << (4 * (i & 7));
    *reinterpret_cast<uint2*>(entry + kv4_key_at(p.head_dim, r, c.group, c.t)) =
        make_uint2(word[0], word[1]);
    if (c.t == 0)
      *reinterpret_cast<__half2*>(entry + kv4_key_scale_at(p.head_dim, r, c.group)) =
          __halves2half2(step, minimum);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t piece = code[4 * i] | code[4 * i + 1] << 4 | code[4 * i + 2] << 8 |
                             code[4 * i + 3] << 12;
      // the piece's two bytes are elements 4w .. 4w+3 of owner g = 2t + i/2
      *reinterpret_cast<uint16_t*>(
          entry + kv4_value_at(p.head_dim, r, c.group, 2 * c.t + (i >> 1), i & 1, 0)) =
          static_cast<uint16_t>(piece);
    }
    if (c.t == 0) {
      __half* at =
          reinterpret_cast<__half*>(entry + kv4_value_scale_at(p.head_dim, r, c.group));
      at[0] = step;
      at[p.head_dim / 2] = minimum;
    }
  }
}

template <int TYPE>
__global__ void __launch_bounds__(256) unpack_kernel(const UnpackParams p) {
  using Element = Kv4Type<TYPE>;
  const int64_t index = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (index >= p.work) return;
  const int groups = p.head_dim / kKv4Group;
  const Piece c = piece_of(index, p.kv_heads, groups);
  const int64_t slot = p.slots[c.token];
  if (slot >= p.slot_limit && c.t == 0) raise_status(p.status, SA_DEV_BAD_BLOCK);
  auto* row = static_cast<typename Element::T*>(p.rows[c.which]) +
              (c.token * p.kv_heads + c.head) * p.head_dim + c.group * kKv4Group + c.t * 16;
  if (slot < 0 || slot >= p.slot_limit) {
#pragma unroll
    for (int i = 0; i < 16; ++i) row[i] = Element::store(0.0f);
    return;
  }
  const int block = static_cast<int>(slot / kBlockTokens), r = static_cast<int>(slot % kBlockTokens);
  const uint8_t* entry = p.pool + (static_cast<int64_t>(block) * p.kv_heads + c.head) *
                                      kv4_entry_bytes(p.head_dim);
  uint32_t word[2];
  float s, m;
  if (c.which == 0) {
    const uint2 w =
        *reinterpret_cast<const uint2*>(entry + kv4_key_at(p.head_dim, r, c.group, c.t));
    word[0] = w.x;
    word[1] = w.y;
    const __half2 sm =
        *reinterpret_cast<const __half2*>(entry + kv4_key_scale_at(p.head_dim, r, c.group));
    s = __low2float(sm);
    m = __high2float(sm);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint16_t* at = reinterpret_cast<const uint16_t*>(
          entry + kv4_value_at(p.head_dim, r, c.group, 2 * c.t + i, 0, 0));
      word[i] = at[0] | static_cast<uint32_t>(at[2]) << 16;
    }
    const __half* at =
        reinterpret_cast<const __half*>(entry + kv4_value_scale_at(p.head_dim, r, c.group));
    s = __half2float(at[0]);
    m = __half2float(at[p.head_dim / 2]);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float code = static_cast<float>((word[i >> 3] >> (4 * (i & 7))) & 15u);
    row[i] = Element::store(__fadd_rn(__fmul_rn(s, code), m));  // the product is exact
  }
}

bool known_dim(size_t head_dim) { return head_dim == 64 || head_dim == 128 || head_dim == 256; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The checks that pack and unpack share.
sa_status check_rows(const char* what, const void* pool, size_t pool_blocks, const int32_t* slots,
                     size_t tokens, size_t kv_heads, size_t head_dim, int type) {
  if (!pool || (!slots && tokens)) return fail(SA_ERR_INVALID_ARG, std::string(what) + ": null pointer");
  if (kv_heads == 0 || pool_blocks == 0)
    return fail(SA_ERR_INVALID_ARG, std::string(what) + ": no KV heads or no blocks");
  if (type != SA_TYPE_F32 && type != SA_TYPE_F16 && type != SA_TYPE_BF16)
    return fail(SA_ERR_INVALID_ARG, std::string(what) + ": unknown element type");
  if (!known_dim(head_dim))
    return fail(SA_ERR_UNSUPPORTED, std::string(what) + ": head_dim must be 64, 128 or 256");
  if (!aligned16(pool))
    return fail(SA_ERR_INVALID_ARG, std::string(what) + ": the pool must be 16-byte aligned");
  if (pool_blocks > 0x7fffffffu / kBlockTokens || kv_heads > 65536 || tokens > 0x7fffffffu)
    return fail(SA_ERR_UNSUPPORTED, std::string(what) + ": more than 2^31 slots or tokens");
  if (tokens * kv_heads > (size_t(1) << 33))
    return fail(SA_ERR_UNSUPPORTED, std::string(what) + ": too many rows for one call");
  return SA_OK;
}

}  // namespace
}  // namespace sa

using namespace sa;

extern "C" SA_API size_t sa_kv4_entry_bytes(size_t head_dim) {
  return known_dim(head_dim) ? (size_t)kv4_entry_bytes((int)head_dim) : 0;
}

extern "C" SA_API sa_status sa_pack_kv4(void* pool, size_t pool_blocks, const void* key,
                                        const void* value, int type, int64_t key_token_stride,
                                        int64_t key_head_stride, int64_t value_token_stride,
                                        int64_t value_head_stride, const int32_t* slots,
                                        size_t tokens, size_t kv_heads, size_t head_dim,
                                        uint32_t* status, void* stream) {
  const sa_status st = check_rows("pack_kv4", pool, pool_blocks, slots, tokens, kv_heads, head_dim, type);
  if (st != SA_OK) return st;
  if (tokens == 0) return SA_OK;
  if (!key || !value) return fail(SA_ERR_INVALID_ARG, "pack_kv4: null pointer");
  PackParams p{};
  p.pool = static_cast<uint8_t*>(pool);
  p.rows[0] = key;
  p.rows[1] = value;
  p.token_stride[0] = key_token_stride;
  p.token_stride[1] = value_token_stride;
  p.head_stride[0] = key_head_stride;
  p.head_stride[1] = value_head_stride;
  p.slots = slots;
  p.status = status;
  p.slot_limit = (int64_t)pool_blocks * kBlockTokens;
  p.work = (int64_t)tokens * 2 * (int64_t)kv_heads * (int64_t)(head_dim / kKv4Group) * 4;
  p.kv_heads = (int)kv_heads;
  p.head_dim = (int)head_dim;
  const dim3 grid((unsigned)((p.work + 255) / 256));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (type == SA_TYPE_F32)
    pack_kernel<SA_TYPE_F32><<<grid, 256, 0, s>>>(p);
  else if (type == SA_TYPE_F16)
    pack_kernel<SA_TYPE_F16><<<grid, 256, 0, s>>>(p);
  else
    pack_kernel<SA_TYPE_BF16><<<grid, 256, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "pack_kv4 launch");
}

extern "C" SA_API sa_status sa_unpack_kv4(const void* pool, size_t pool_blocks,
                                          const int32_t* slots, size_t tokens, size_t kv_heads,
                                          size_t head_dim, void* key_out, void* value_out,
                                          int type, uint32_t* status, void* stream) {
  const sa_status st =
      check_rows("unpack_kv4", pool, pool_blocks, slots, tokens, kv_heads, head_dim, type);
  if (st != SA_OK) return st;
  if (tokens == 0) return SA_OK;
  if (!key_out || !value_out) return fail(SA_ERR_INVALID_ARG, "unpack_kv4: null pointer");
  if (!aligned16(key_out) || !aligned16(value_out))
    return fail(SA_ERR_INVALID_ARG, "unpack_kv4: outputs must be 16-byte aligned");
  UnpackParams p{};
  p.pool = static_cast<const uint8_t*>(pool);
  p.rows[0] = key_out;
  p.rows[1] = value_out;
  p.slots = slots;
  p.status = status;
  p.slot_limit = (int64_t)pool_blocks * kBlockTokens;
  p.work = (int64_t)tokens * 2 * (int64_t)kv_heads * (int64_t)(head_dim / kKv4Group) * 4;
  p.kv_heads = (int)kv_heads;
  p.head_dim = (int)head_dim;
  const dim3 grid((unsigned)((p.work + 255) / 256));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (type == SA_TYPE_F32)
    unpack_kernel<SA_TYPE_F32><<<grid, 256, 0, s>>>(p);
  else if (type == SA_TYPE_F16)
    unpack_kernel<SA_TYPE_F16><<<grid, 256, 0, s>>>(p);
  else
    unpack_kernel<SA_TYPE_BF16><<<grid, 256, 0, s>>>(p);
  return cuda_status(cudaGetLastError(), "unpack_kv4 launch");
}
