// sa_kv4.cu -- rows into and out of the 4-bit cache.
//
// Both kernels move a row once and are bound by that traffic. A thread owns
// eight consecutive elements (a column) of kTokens consecutive tokens: the
// index arithmetic is done once, the tokens' loads are in flight together, and
// the lanes of a warp read and write whole rows. Eight neighbouring lanes hold
// a group of 64, so its minimum and maximum take three shuffles each.
//
// Rounding. The step is the smallest FP16 number s with 15 s >= max - minimum
// (the difference rounded up; 15 s is exact in FP32, so the comparison decides
// as it would in exact arithmetic). A code is guessed as rint(x * (1 / s)) with
// an approximate reciprocal and settled by its remainder x - code * s, which
// is exact in FP32: only remainders of half a step or more, ties among them,
// need a second look.
#include <cfloat>

#include "sa_kv4.cuh"

namespace sa {
namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 4;  // consecutive tokens of a thread

struct PackParams {
  uint8_t* pool;
  const void* keys;
  const void* values;
  int64_t key_token_stride, key_head_stride, value_token_stride, value_head_stride;
  const int32_t* slots;
  uint32_t* status;
  int64_t slot_limit;
  int tokens, kv_heads;
  int columns;      // of 8 elements in a token's keys and values
  int token_lanes;  // groups of kTokens tokens of a CTA
  int vectors;      // every row is 16-byte aligned
};

struct UnpackParams {
  const uint8_t* pool;
  void* keys;
  void* values;
  const int32_t* slots;
  uint32_t* status;
  int64_t slot_limit;
  int tokens, kv_heads, columns, token_lanes;
};

// Eight elements of a row: `o`-th piece of group `group` of a head.
struct Column {
  int which, head, group, o;
  int64_t first;  // first token
  bool live;
};
template <int NG, class Params>
__device__ __forceinline__ Column column_of(const Params& p) {
  Column c;
  int lane = threadIdx.x, at = blockIdx.y * kThreads;
  if (p.token_lanes > 1) {
    lane = threadIdx.x / p.columns;
    at = threadIdx.x % p.columns;
  } else {
    lane = 0;
    at += threadIdx.x;
  }
  c.live = lane < p.token_lanes && at < p.columns;
  c.first = (static_cast<int64_t>(blockIdx.x) * p.token_lanes + lane) * kTokens;
  c.o = at & 7;
  c.group = (at >> 3) % NG;
  const int rest = (at >> 3) / NG;
  c.which = rest >= p.kv_heads ? 1 : 0;
  c.head = rest - (c.which ? p.kv_heads : 0);
  return c;
}

template <int NG>
__device__ __forceinline__ int64_t entry_of(int slot, int kv_heads, int head) {
  return (static_cast<int64_t>(slot / kBlockTokens) * kv_heads + head) * kv4_entry_bytes(64 * NG);
}

// Eight elements as FP32.
template <int TYPE>
__device__ __forceinline__ void load8(const void* base, int64_t at, bool vectors, float (&x)[8]) {
  using Element = Kv4Type<TYPE>;
  const auto* from = static_cast<const typename Element::T*>(base) + at;
  if (vectors) {
    if constexpr (TYPE == SA_TYPE_F32) {
      const float4 a = reinterpret_cast<const float4*>(from)[0], b = reinterpret_cast<const float4*>(from)[1];
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
      x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(from);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (TYPE == SA_TYPE_BF16) {
          x[2 * i] = __uint_as_float(w[i] << 16);
          x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
          const float2 f = h2x2f(w[i]);
          x[2 * i] = f.x;
          x[2 * i + 1] = f.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Element::load(from[i]);
  }
}

template <int TYPE, int NG>
__global__ void __launch_bounds__(kThreads) pack_kernel(const PackParams p) {
  constexpr int kDim = 64 * NG;
  const Column c = column_of<NG>(p);
  float x[kTokens][8];
  int slot[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    slot[i] = c.live && c.first + i < p.tokens ? p.slots[c.first + i] : -1;
    if (slot[i] >= p.slot_limit) {
      if (c.o == 0) raise_status(p.status, SA_DEV_BAD_BLOCK);
      slot[i] = -1;
    }
  }
  const void* rows = c.which ? p.values : p.keys;
  const int64_t stride = c.which ? p.value_token_stride : p.key_token_stride;
  const int64_t at = c.first * stride +
                     c.head * (c.which ? p.value_head_stride : p.key_head_stride) +
                     c.group * kKv4Group + c.o * 8;
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    if (slot[i] >= 0) {
      load8<TYPE>(rows, at + i * stride, p.vectors, x[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
    }
  }
  uint32_t word[kTokens];
  __half step[kTokens], minimum[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    float low = x[i][0], high = x[i][0];
    bool nan = isnan(x[i][0]);
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      low = fminf(low, x[i][e]);
      high = fmaxf(high, x[i][e]);
      nan |= isnan(x[i][e]);
    }
    // NaN as an infinity, which no finite element gives
    if (nan) high = INFINITY;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
      high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    const bool finite = low >= -FLT_MAX && high <= FLT_MAX;
    if constexpr (TYPE != SA_TYPE_F16) {
      low = fmaxf(low, -65504.0f);
      high = fminf(high, 65504.0f);
      low = fminf(low, 65504.0f);
      high = fmaxf(high, -65504.0f);
    }
    minimum[i] = __float2half_rd(low);
    const float m = __half2float(minimum[i]), range = __fsub_ru(high, m);
    // from just below range / 15 upwards
    uint16_t bits = __half_as_ushort(__float2half_rd(range * 0.066666655f));
#pragma unroll
    for (int k = 0; k < 2; ++k)  // at most one FP16 number lies between them
      if (15.0f * h2f(bits) < range) ++bits;
    step[i] = __ushort_as_half(bits);
    const float s = h2f(bits), inverse = s > 0.0f ? __fdividef(1.0f, s) : 0.0f;
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
    uint32_t sum = 0;
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float y = x[i][e];
      if constexpr (TYPE != SA_TYPE_F16) y = fminf(fmaxf(y, -65504.0f), 65504.0f);
      x[i][e] = y - m;
      const float rounded = fmaf(x[i][e], inverse, kMagic);
      sum += __float_as_uint(rounded) << (4 * e);
      most = fmaxf(most, fabsf(fmaf(-(rounded - kMagic), s, x[i][e])));
    }
    sum -= 0x11111111u * 0x4b400000u;  // kMagic's bits, eight times
    if (2.0f * most >= s) {
      sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float code = fmaf(x[i][e], inverse, kMagic) - kMagic;
        const float twice = 2.0f * fmaf(-code, s, x[i][e]);
        const bool odd = static_cast<int>(code) & 1;
        if (twice > s || (twice == s && odd)) code += 1.0f;
        if (twice < -s || (twice == -s && odd)) code -= 1.0f;
        sum |= static_cast<uint32_t>(s > 0.0f ? code : 0.0f) << (4 * e);
      }
    }
    word[i] = sum;
    if (!finite) {
      word[i] = 0;
      step[i] = minimum[i] = __ushort_as_half(0x7fffu);
    }
  }
  if (c.which == 0) {
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      if (slot[i] < 0) continue;
      const int r = slot[i] % kBlockTokens;
      uint8_t* entry = p.pool + entry_of<NG>(slot[i], p.kv_heads, c.head);
      *reinterpret_cast<uint32_t*>(entry + kv4_key_at(kDim, r, c.group, c.o >> 1) +
                                   4 * (c.o & 1)) = word[i];
      if (c.o == 0)
        *reinterpret_cast<__half2*>(entry + kv4_key_scale_at(kDim, r, c.group)) =
            __halves2half2(step[i], minimum[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      if (slot[i] < 0) continue;
      const int r = slot[i] % kBlockTokens;
      uint8_t* entry = p.pool + entry_of<NG>(slot[i], p.kv_heads, c.head);
      if (c.o == 0) {
        __half* at = reinterpret_cast<__half*>(entry + kv4_value_scale_at(kDim, r, c.group));
        at[0] = step[i];
        at[kDim / 2] = minimum[i];
      }
      uint8_t* to = entry + kv4_value_at(kDim, r, c.group, c.o, 0, 0);
      // two tokens of a pair row at once, or the 16-bit pieces of one
      if (i + 1 < kTokens && (r & 1) == 0 && slot[i + 1 < kTokens ? i + 1 : i] == slot[i] + 1) {
        *reinterpret_cast<uint2*>(to) = make_uint2(__byte_perm(word[i], word[i + 1 < kTokens ? i + 1 : i], 0x5410),
                                                   __byte_perm(word[i], word[i + 1 < kTokens ? i + 1 : i], 0x7632));
      } else if (!(i > 0 && (r & 1) == 1 && slot[i > 0 ? i - 1 : i] == slot[i] - 1)) {
        *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(word[i]);
        *reinterpret_cast<uint16_t*>(to + 4) = static_cast<uint16_t>(word[i] >> 16);
      }
    }
  }
}

template <int TYPE, int NG>
__global__ void __launch_bounds__(kThreads) unpack_kernel(const UnpackParams p) {
  using Element = Kv4Type<TYPE>;
  constexpr int kDim = 64 * NG;
  const Column c = column_of<NG>(p);
  if (!c.live) return;
  int slot[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    slot[i] = c.first + i < p.tokens ? p.slots[c.first + i] : -1;
    if (slot[i] >= p.slot_limit) {
      if (c.o == 0) raise_status(p.status, SA_DEV_BAD_BLOCK);
      slot[i] = -1;
    }
  }
  uint32_t word[kTokens];
  __half step[kTokens], minimum[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    word[i] = 0;
    step[i] = minimum[i] = __ushort_as_half(0);
    if (slot[i] < 0) continue;
    const int r = slot[i] % kBlockTokens;
    const uint8_t* entry = p.pool + entry_of<NG>(slot[i], p.kv_heads, c.head);
    if (c.which == 0) {
      word[i] = *reinterpret_cast<const uint32_t*>(
          entry + kv4_key_at(kDim, r, c.group, c.o >> 1) + 4 * (c.o & 1));
      const __half2 sm =
          *reinterpret_cast<const __half2*>(entry + kv4_key_scale_at(kDim, r, c.group));
      step[i] = __low2half(sm);
      minimum[i] = __high2half(sm);
    } else {
      const uint2 pair =
          *reinterpret_cast<const uint2*>(entry + kv4_value_at(kDim, r & ~1, c.group, c.o, 0, 0));
      word[i] = __byte_perm(pair.x, pair.y, r & 1 ? 0x7632 : 0x5410);
      const __half* at =
          reinterpret_cast<const __half*>(entry + kv4_value_scale_at(kDim, r, c.group));
      step[i] = at[0];
      minimum[i] = at[kDim / 2];
    }
  }
  auto* row = static_cast<typename Element::T*>(c.which ? p.values : p.keys) +
              (c.first * p.kv_heads + c.head) * kDim + c.group * kKv4Group + c.o * 8;
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    if (c.first + i >= p.tokens) break;
    const float s = __half2float(step[i]), m = __half2float(minimum[i]);
    alignas(16) typename Element::T y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)  // the product is exact, so this rounds once
      y[e] = Element::store(fmaf(s, static_cast<float>((word[i] >> (4 * e)) & 15u), m));
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(y) / 16); ++k)
      reinterpret_cast<uint4*>(row + static_cast<int64_t>(i) * p.kv_heads * kDim)[k] =
          reinterpret_cast<const uint4*>(y)[k];
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
  if (pool_blocks > 0x7fffffffu / kBlockTokens || tokens > 0x7fffffffu)
    return fail(SA_ERR_UNSUPPORTED, std::string(what) + ": more than 2^31 slots or tokens");
  if (kv_heads > 65536)
    return fail(SA_ERR_UNSUPPORTED, std::string(what) + ": more than 65536 KV heads");
  return SA_OK;
}

// The grid over (tokens, columns) that column_of() reads; narrow rows put
// several groups of tokens into a CTA.
template <class Params>
dim3 row_grid(Params& p, size_t tokens, size_t kv_heads, size_t head_dim) {
  p.tokens = (int)tokens;
  p.kv_heads = (int)kv_heads;
  p.columns = (int)(2 * kv_heads * (head_dim / 8));
  p.token_lanes = p.columns < kThreads ? kThreads / p.columns : 1;
  const size_t each = (size_t)p.token_lanes * kTokens;
  return dim3((unsigned)((tokens + each - 1) / each), (unsigned)((p.columns + kThreads - 1) / kThreads));
}

template <int NG>
void launch_pack(const PackParams& p, dim3 grid, int type, cudaStream_t s) {
  if (type == SA_TYPE_F32)
    pack_kernel<SA_TYPE_F32, NG><<<grid, kThreads, 0, s>>>(p);
  else if (type == SA_TYPE_F16)
    pack_kernel<SA_TYPE_F16, NG><<<grid, kThreads, 0, s>>>(p);
  else
    pack_kernel<SA_TYPE_BF16, NG><<<grid, kThreads, 0, s>>>(p);
}

template <int NG>
void launch_unpack(const UnpackParams& p, dim3 grid, int type, cudaStream_t s) {
  if (type == SA_TYPE_F32)
    unpack_kernel<SA_TYPE_F32, NG><<<grid, kThreads, 0, s>>>(p);
  else if (type == SA_TYPE_F16)
    unpack_kernel<SA_TYPE_F16, NG><<<grid, kThreads, 0, s>>>(p);
  else
    unpack_kernel<SA_TYPE_BF16, NG><<<grid, kThreads, 0, s>>>(p);
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
  p.keys = key;
  p.values = value;
  p.key_token_stride = key_token_stride;
  p.key_head_stride = key_head_stride;
  p.value_token_stride = value_token_stride;
  p.value_head_stride = value_head_stride;
  p.slots = slots;
  p.status = status;
  p.slot_limit = (int64_t)pool_blocks * kBlockTokens;
  const size_t element = type == SA_TYPE_F32 ? 4 : 2;
  p.vectors = ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value) |
                (size_t)(key_token_stride | key_head_stride | value_token_stride |
                         value_head_stride) * element) & 15u) == 0;
  const dim3 grid = row_grid(p, tokens, kv_heads, head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (head_dim == 64)
    launch_pack<1>(p, grid, type, s);
  else if (head_dim == 128)
    launch_pack<2>(p, grid, type, s);
  else
    launch_pack<4>(p, grid, type, s);
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
  p.keys = key_out;
  p.values = value_out;
  p.slots = slots;
  p.status = status;
  p.slot_limit = (int64_t)pool_blocks * kBlockTokens;
  const dim3 grid = row_grid(p, tokens, kv_heads, head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (head_dim == 64)
    launch_unpack<1>(p, grid, type, s);
  else if (head_dim == 128)
    launch_unpack<2>(p, grid, type, s);
  else
    launch_unpack<4>(p, grid, type, s);
  return cuda_status(cudaGetLastError(), "unpack_kv4 launch");
}
