// sa_kv4.cu -- rows into and out of the 4-bit cache.
//
// Both kernels move a row once and are bound by that traffic. A thread owns 16
// consecutive elements (a column) of kTokens consecutive tokens: the index
// arithmetic is done once, the tokens' loads are in flight together, and the
// lanes of a warp read and write whole rows. Four neighbouring lanes hold a
// group of 64, so its minimum and maximum take two shuffles each. (Eight
// elements of four tokens a thread spent 2.5 times the instructions: prompts of
// 99,991 tokens, 5 heads of 64, packed and read back in 145 us, now 86 us.)
// Measured on the device: 32,768 tokens, 8 heads of 128, packed in 40 us in BF16,
// 38 in FP16 and 52 in FP32, read back in 35, 35 and 71 us, against floors of 26,
// 26 and 47; a chunk of 8,192 tokens in FP16 packed and read back in 21.4 us.
// Packing is bound by instructions (81 % of the issue slots, 17 an element, two
// thirds of them for rows and scales rather than codes), unpacking by the latency
// of its loads and nearly by instructions (72 % of the slots, 12 an element).
//
// Rounding. The step is the smallest FP16 number s with 15 s >= max - minimum
// (the difference rounded up; 15 s is exact in FP32, so the comparison decides
// as it would in exact arithmetic). A code is rint(d / s) with d = x - minimum
// in FP32: the reciprocal is held as the sum of two FP32 numbers, its error of
// 2^-44 vanishes in the rounding of d * (r0 + r1) to FP32, so exact halves come
// out exact and go to the even code; and no other quotient rounds to a half,
// since d (24 bits) and a half times s (16 bits) that differ do so by more than
// half a unit in the quotient's last place.
#include <cfloat>
#include <type_traits>

#include "sa_kv4.cuh"

namespace sa {
namespace {

constexpr int kThreads = 128;
constexpr int kTokens = 2;  // consecutive tokens of a thread

struct PackParams {
  uint8_t* pool;
  const void* keys;
  const void* values;
  int64_t key_token_stride, key_head_stride, value_token_stride, value_head_stride;
  const int32_t* slots;
  uint32_t* status;
  int64_t slot_limit;
  int tokens, kv_heads;
  int columns;      // of 16 elements in a token's keys and values
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

// Sixteen elements of a row: the t-th part of group `group` of a head.
struct Column {
  int which, head, group, t;
  int64_t first;  // first token
  bool live;
};
template <int NG, class Params>
__device__ __forceinline__ Column column_of(const Params& p) {
  Column c;
  int lane = 0, at = blockIdx.y * kThreads + threadIdx.x;
  if (p.token_lanes > 1) {
    lane = threadIdx.x / p.columns;
    at = threadIdx.x % p.columns;
  }
  c.live = lane < p.token_lanes && at < p.columns;
  c.first = (static_cast<int64_t>(blockIdx.x) * p.token_lanes + lane) * kTokens;
  c.t = at & 3;
  c.group = (at >> 2) % NG;
  const int rest = (at >> 2) / NG;
  c.which = rest >= p.kv_heads ? 1 : 0;
  c.head = rest - (c.which ? p.kv_heads : 0);
  return c;
}

// The slots of a column's tokens, -1 where there is nothing to do.
template <class Params>
__device__ __forceinline__ void slots_of(const Params& p, const Column& c, int (&slot)[kTokens]) {
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    slot[i] = c.live && c.first + i < p.tokens ? p.slots[c.first + i] : -1;
    if (slot[i] >= p.slot_limit) {
      if (c.t == 0) raise_status(p.status, SA_DEV_BAD_BLOCK);
      slot[i] = -1;
    }
  }
}

template <int NG>
__device__ __forceinline__ int64_t entry_of(int slot, int kv_heads, int head) {
  return (static_cast<int64_t>(slot / kBlockTokens) * kv_heads + head) * kv4_entry_bytes(64 * NG);
}

// Sixteen elements as they are loaded: 16-bit types stay packed until their
// minimum and maximum are known.
template <int TYPE>
struct Row16 {
  using Pair = std::conditional_t<TYPE == SA_TYPE_BF16, __nv_bfloat162, __half2>;
  uint32_t word[8];
  __device__ __forceinline__ void load(const void* base, int64_t at, bool vectors) {
    const auto* from = static_cast<const uint16_t*>(base) + at;
    if (vectors) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint4 v = reinterpret_cast<const uint4*>(from)[k];
        word[4 * k] = v.x, word[4 * k + 1] = v.y, word[4 * k + 2] = v.z, word[4 * k + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) word[i] = from[2 * i] | static_cast<uint32_t>(from[2 * i + 1]) << 16;
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) word[i] = 0u;
  }
  __device__ __forceinline__ void values(float (&x)[16]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (TYPE == SA_TYPE_BF16) {
        x[2 * i] = __uint_as_float(word[i] << 16);
        x[2 * i + 1] = __uint_as_float(word[i] & 0xffff0000u);
      } else {
        const float2 f = h2x2f(word[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void limits(float& low, float& high) const {
    Pair a = pair(0), b = a;
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      a = __hmin2_nan(a, pair(i));
      b = __hmax2_nan(b, pair(i));
    }
    low = min_nan(first(a), second(a));
    high = max_nan(first(b), second(b));
  }

 private:
  __device__ __forceinline__ Pair pair(int i) const { return *reinterpret_cast<const Pair*>(&word[i]); }
  static __device__ __forceinline__ float first(Pair a) { return Kv4Type<TYPE>::load(a.x); }
  static __device__ __forceinline__ float second(Pair a) { return Kv4Type<TYPE>::load(a.y); }
};
template <>
struct Row16<SA_TYPE_F32> {
  float x[16];
  __device__ __forceinline__ void load(const void* base, int64_t at, bool vectors) {
    const auto* from = static_cast<const float*>(base) + at;
    if (vectors) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 v = reinterpret_cast<const float4*>(from)[k];
        x[4 * k] = v.x, x[4 * k + 1] = v.y, x[4 * k + 2] = v.z, x[4 * k + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = from[i];
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.0f;
  }
  __device__ __forceinline__ void values(float (&y)[16]) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = x[i];
  }
  __device__ __forceinline__ void limits(float& low, float& high) const {
    low = high = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) {
      low = min_nan(low, x[i]);
      high = max_nan(high, x[i]);
    }
  }
};

template <int TYPE, int NG>
__global__ void __launch_bounds__(kThreads) pack_kernel(const PackParams p) {
  constexpr int kDim = 64 * NG;
  const Column c = column_of<NG>(p);
  int slot[kTokens];
  slots_of(p, c, slot);
  const void* rows = c.which ? p.values : p.keys;
  const int64_t stride = c.which ? p.value_token_stride : p.key_token_stride;
  const int64_t at = c.first * stride +
                     c.head * (c.which ? p.value_head_stride : p.key_head_stride) +
                     c.group * kKv4Group + c.t * 16;
  Row16<TYPE> row[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    if (slot[i] >= 0)
      row[i].load(rows, at + i * stride, p.vectors);
    else
      row[i].clear();
  }
  uint32_t word[kTokens][2];
  __half step[kTokens], minimum[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    float low, high;
    row[i].limits(low, high);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
      high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    const bool finite = low >= -FLT_MAX && high <= FLT_MAX;
    float x[16];
    row[i].values(x);
    if (TYPE != SA_TYPE_F16 && (low < -65504.0f || high > 65504.0f)) {
      low = fminf(fmaxf(low, -65504.0f), 65504.0f);
      high = fminf(fmaxf(high, -65504.0f), 65504.0f);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = fminf(fmaxf(x[e], -65504.0f), 65504.0f);
    }
    minimum[i] = __float2half_rd(low);
    const float m = __half2float(minimum[i]), range = __fsub_ru(high, m);
    // from just below range / 15 upwards
    uint16_t bits = __half_as_ushort(__float2half_rd(range * 0.066666655f));
#pragma unroll
    for (int k = 0; k < 2; ++k)  // at most one FP16 number lies between them
      if (15.0f * h2f(bits) < range) ++bits;
    step[i] = __ushort_as_half(bits);
    const float s = h2f(bits), r0 = s > 0.0f ? __fdividef(1.0f, s) : 0.0f;
    const float r1 = fmaf(-s, r0, 1.0f) * r0;
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = x[8 * k + e] - m;
        sum += __float_as_uint(fmaf(d, r0, d * r1) + kMagic) << (4 * e);
      }
      word[i][k] = finite ? sum - 0x11111111u * 0x4b400000u : 0u;  // without kMagic's bits
    }
    if (!finite) step[i] = minimum[i] = __ushort_as_half(0x7fffu);
  }
  if (c.which == 0) {
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      if (slot[i] < 0) continue;
      const int r = slot[i] % kBlockTokens;
      uint8_t* entry = p.pool + entry_of<NG>(slot[i], p.kv_heads, c.head);
      *reinterpret_cast<uint2*>(entry + kv4_key_at(kDim, r, c.group, c.t)) =
          make_uint2(word[i][0], word[i][1]);
      if (c.t == 0)
        *reinterpret_cast<__half2*>(entry + kv4_key_scale_at(kDim, r, c.group)) =
            __halves2half2(step[i], minimum[i]);
    }
  } else {
    // the two tokens of a pair row at once where the slots allow it
    const bool pair = slot[0] >= 0 && (slot[0] & 1) == 0 && slot[1] == slot[0] + 1;
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      if (slot[i] < 0) continue;
      const int r = slot[i] % kBlockTokens;
      uint8_t* entry = p.pool + entry_of<NG>(slot[i], p.kv_heads, c.head);
      if (c.t == 0) {
        __half* to = reinterpret_cast<__half*>(entry + kv4_value_scale_at(kDim, r, c.group));
        to[0] = step[i];
        to[kDim / 2] = minimum[i];
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint8_t* to = entry + kv4_value_at(kDim, r, c.group, 2 * c.t + k, 0, 0);
        if (pair) {
          if (i == 0)
            *reinterpret_cast<uint2*>(to) = make_uint2(__byte_perm(word[0][k], word[1][k], 0x5410),
                                                       __byte_perm(word[0][k], word[1][k], 0x7632));
        } else {
          *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(word[i][k]);
          *reinterpret_cast<uint16_t*>(to + 4) = static_cast<uint16_t>(word[i][k] >> 16);
        }
      }
    }
  }
}

template <int TYPE, int NG>
__global__ void __launch_bounds__(kThreads) unpack_kernel(const UnpackParams p) {
  using Element = Kv4Type<TYPE>;
  constexpr int kDim = 64 * NG;
  const Column c = column_of<NG>(p);
  int slot[kTokens];
  slots_of(p, c, slot);
  uint32_t word[kTokens][2];
  __half step[kTokens], minimum[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    word[i][0] = word[i][1] = 0;
    step[i] = minimum[i] = __ushort_as_half(0);
    if (slot[i] < 0) continue;
    const int r = slot[i] % kBlockTokens;
    const uint8_t* entry = p.pool + entry_of<NG>(slot[i], p.kv_heads, c.head);
    if (c.which == 0) {
      const uint2 w = *reinterpret_cast<const uint2*>(entry + kv4_key_at(kDim, r, c.group, c.t));
      word[i][0] = w.x;
      word[i][1] = w.y;
      const __half2 sm =
          *reinterpret_cast<const __half2*>(entry + kv4_key_scale_at(kDim, r, c.group));
      step[i] = __low2half(sm);
      minimum[i] = __high2half(sm);
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint2 w = *reinterpret_cast<const uint2*>(
            entry + kv4_value_at(kDim, r & ~1, c.group, 2 * c.t + k, 0, 0));
        word[i][k] = __byte_perm(w.x, w.y, r & 1 ? 0x7632 : 0x5410);
      }
      const __half* at =
          reinterpret_cast<const __half*>(entry + kv4_value_scale_at(kDim, r, c.group));
      step[i] = at[0];
      minimum[i] = at[kDim / 2];
    }
  }
  auto* row = static_cast<typename Element::T*>(c.which ? p.values : p.keys) +
              (c.first * p.kv_heads + c.head) * kDim + c.group * kKv4Group + c.t * 16;
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    const float s = __half2float(step[i]), m = __half2float(minimum[i]);
    alignas(16) typename Element::T y[16];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // codes e and e + 4 as 1024 + c, then c, in FP16
        const uint32_t both = (word[i][k] >> (4 * e) & 0x000f000fu) | 0x64006400u;
        const float2 code = __half22float2(
            __hsub2(*reinterpret_cast<const __half2*>(&both), __half2half2(__ushort_as_half(0x6400u))));
        y[8 * k + e] = Element::store(fmaf(s, code.x, m));  // the product is exact: one rounding
        y[8 * k + e + 4] = Element::store(fmaf(s, code.y, m));
      }
    if constexpr (TYPE == SA_TYPE_F16) {
      __half2* pairs = reinterpret_cast<__half2*>(y);
#pragma unroll
      for (int k = 0; k < 8; ++k) pairs[k] = __hmin2_nan(pairs[k], __float2half2_rn(kHalfMost));
    }
    // Two lanes exchange quads, so that each store of the warp writes whole
    // 32-byte sectors.
    uint4* to = reinterpret_cast<uint4*>(row + static_cast<int64_t>(i) * p.kv_heads * kDim);
    const uint4* from = reinterpret_cast<const uint4*>(y);
    constexpr int kQuads = static_cast<int>(sizeof(y) / 16);
    const bool odd = threadIdx.x & 1, writes = c.live && c.first + i < p.tokens;
#pragma unroll
    for (int k = 0; k < kQuads; k += 2) {
      const uint4 keep = odd ? from[k + 1] : from[k], give = odd ? from[k] : from[k + 1];
      uint4 got;
      got.x = __shfl_xor_sync(0xffffffffu, give.x, 1);
      got.y = __shfl_xor_sync(0xffffffffu, give.y, 1);
      got.z = __shfl_xor_sync(0xffffffffu, give.z, 1);
      got.w = __shfl_xor_sync(0xffffffffu, give.w, 1);
      if (writes) {
        to[odd ? k + 1 - kQuads : k] = odd ? got : keep;  // the even lane's quads
        to[odd ? k + 1 : k + kQuads] = odd ? keep : got;  // the odd lane's
      }
    }
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
  p.columns = (int)(2 * kv_heads * (head_dim / 16));
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
