// sa_kv4_attention.cu -- GQA attention of a batch's newest tokens over the
// 4-bit paged cache.
//
//   x_t = scale * sum_d q_d (s_t,g c_t,d + m_t,g)      softmax over the tokens seen
//   o_d = sum_t p_t (s'_t,g c'_t,d + m'_t,g) / sum_t p_t
//
// The codes are never dequantised. A nibble in the low bits of a 16-bit lane is
// an FP16 subnormal, c * 2^-24 (c * 2^-20 for the next nibble, whose factor 16
// goes into the query for keys and into the output row for values), so one AND
// turns eight codes into a matrix operand register pair, and the tensor cores
// multiply codes exactly:
//
//   x_t = F sum_g s_t,g (sum_d q'_d c_t,d) + sum_g m_t,g Q_g,   Q_g = sum_d q_d
//   o_d = sum_t (p_t s'_t,g) c'_t,d + sum_t p_t m'_t,g
//
// with q' = q scaled by a power of two per row to [2^14, 2^15), the key scales
// applied to the FP32 products, and the value steps folded into the FP16
// weights (one extra matrix row a group gives the second sum). Tokens are the
// matrix rows of the first product and query rows its columns, so that up to 8
// query rows (heads of a KV head times new tokens) cost one m16n8k16 column
// tile; the weights become the second product's operand by an 8x8 transpose of
// registers (movmatrix).
//
// Rounding. FP32 queries are split into two FP16 parts. Where the output is
// BF16, weights are rounded to FP16, and again when the step is multiplied in
// (2^-11 each against the output's own 2^-8): the error against float64 is
// 1.73e-3 where FP32 weights leave 1.66e-3 (8,192 tokens; 1.67e-3 and 1.65e-3
// over 997). Weights in two parts would close that at 136 us for the 115 of 64
// requests of 8K, 166 with centred codes. Other outputs have them in two parts.
// There the value codes are also centred, c - 8 with minimum + 8 step (in two
// FP16 parts): over a long context the output is a small difference of large
// sums otherwise, and the matrix unit's truncating sums lost 1e-4 of it at
// 4,128 tokens (9e-7 for plain FP32). FP32 queries centre the key codes too,
// and add the products of their small parts apart. Logits, maxima, sums and
// partial results are FP32.
//
// The value steps of each group of 64 elements are scaled by a power of two
// 2^-E that follows the group's largest finite one, so that weight * step
// stays inside FP16. Groups are separate output elements: a huge or NaN step
// of one leaves the others as they are. Inside a group, steps more than 2^-14
// below the largest one that a warp has seen lose bits (they are FP16
// subnormals then, off by 2^-25 of 2^E), an error of 2^-24 of the group's
// largest value.
//
// Work split. All (list, KV head, row tile) units' entries form one flat list;
// every CTA takes an equal contiguous range of it, whatever the lengths, and
// its warps equal contiguous parts of that, each streaming its entries through
// a ring of its own. A unit that a warp covers alone is written at once. Parts
// of units go to the workspace as (maximum, sum, weighted values), joined by
// the CTA first where its whole range lies in one unit, and merge_kernel joins
// them in the order of the list.
//
// Measured (device time, both launches, bursts of ten calls; 32 query heads of
// 128 over 8): 64 requests of 8,192 tokens in BF16 115 us, 5.3 TB/s of cache,
// 0.80 of the copy rate (136 us, 0.68, in a loop of seconds, where the power
// cap lowers the clock); FP16 164 us and FP32 193 us, bound by instructions
// (weights and, for FP32, queries in two parts). One request of 997 tokens: 10.4
// to 11 us, launches, the chain of dependent reads and code that runs once.
#include <algorithm>
#include <type_traits>

#include "sa_kv4.cuh"

namespace sa {
namespace {

constexpr int kMaxLists = 8192;
// Warps of an attention CTA, one CTA an SM: 16 of 128 registers, 12 of 168, or 8
// of 255 for the larger tiles. Medians over eight places of the cache in memory,
// between which one binary differs by 1 to 8 %: 32 requests of 8K, 8 rows a tile,
// 67.2 us with 12 warps (66.9 to 68.6, once 72.9), 73.6 with 8 (73.2 to 73.8), 64
// requests 115 and 130; FP32 queries 105 and 108; head_dim 64 77.7 with 16 warps,
// 81.3 with 12, 97 with 8. 16 rows a tile, 16 query heads a KV head: 63.6 us with
// 8 warps, 71.6 with 12 (400 to 560 bytes of spills a thread); four drafts of
// two sets of ragged requests 149 and 153, 182 and 175.
__host__ __device__ constexpr int attention_warps(int head_dim, int tile) {
  return tile > 8 || head_dim > 128 ? 8 : head_dim == 64 ? 16 : 12;
}
constexpr float kHeadroom = 4.0f;  // log2 by which a weight may exceed its row's running maximum
constexpr float kWeightLog2 = 11.0f;  // weights are held as 2^11 p: at most 2^15 in FP16

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
  int requests, new_tokens, query_heads, kv_heads;
  int group;           // query heads per KV head
  int rows;            // query rows of a KV head: group * new_tokens
  int row_tiles;       // tiles of 8 * NT rows
  int units_per_list;  // KV heads of a list * row_tiles
  float scale_log2;    // softmax scale * log2(e)
  int ctas, warps;     // of the attention grid, of its CTAs
  int vector_rows;     // query rows are 16-byte aligned
  int* starts;         // workspace: [lists + 1] entries of the lists before each
  float* part_ml;      // workspace: [warps][2][rows of a tile][max, sum]
  float* part_o;       // workspace: [warps][2][rows of a tile][head_dim]
};

// ---- elements of the calls' types ------------------------------------------------

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t pack_bf162(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Outputs in FP16: finite ones stay so.
__device__ __forceinline__ uint32_t pack_output(float a, float b) {
  return pack_half2(min_nan(a, kHalfMost), min_nan(b, kHalfMost));
}

// Eight consecutive elements from element `i` on (a multiple of 8).
__device__ __forceinline__ void store8(void* base, int64_t i, int type, const float (&x)[8]) {
  if (type == SA_TYPE_F32) {
    float4* at = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
    at[0] = make_float4(x[0], x[1], x[2], x[3]);
    at[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else if (type == SA_TYPE_F16) {
    *reinterpret_cast<uint4*>(static_cast<__half*>(base) + i) =
        make_uint4(pack_output(x[0], x[1]), pack_output(x[2], x[3]), pack_output(x[4], x[5]),
                   pack_output(x[6], x[7]));
  } else {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + i) =
        make_uint4(pack_bf162(x[0], x[1]), pack_bf162(x[2], x[3]), pack_bf162(x[4], x[5]),
                   pack_bf162(x[6], x[7]));
  }
}

// Four of them (a multiple of 4).
__device__ __forceinline__ void store4(void* base, int64_t i, int type, float a, float b, float c,
                                       float d) {
  if (type == SA_TYPE_F32)
    *reinterpret_cast<float4*>(static_cast<float*>(base) + i) = make_float4(a, b, c, d);
  else if (type == SA_TYPE_F16)
    *reinterpret_cast<uint2*>(static_cast<__half*>(base) + i) =
        make_uint2(pack_output(a, b), pack_output(c, d));
  else
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(base) + i) =
        make_uint2(pack_bf162(a, b), pack_bf162(c, d));
}

__device__ __forceinline__ void cp_async16_at(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to),
               "l"(reinterpret_cast<uint64_t>(from))
               : "memory");
}

// ---- matrix fragments -------------------------------------------------------------

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8x8 matrix of 16-bit elements held one row per four lanes.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^k, -126 <= k <= 127.
__device__ __forceinline__ float power_of_2(int k) { return __int_as_float((k + 127) << 23); }

// E for a group's largest step, given as FP16 bits: 2^E is above it. Steps stay as they are
// while the largest is in [2^-8, 1).
__device__ __forceinline__ int step_exponent(uint32_t largest) {
  const int exponent = static_cast<int>(largest >> 10) - 14;
  return exponent > -8 && exponent <= 0 ? 0 : exponent;
}

// k of a power of two 2^k held as FP16 bits in the low half (k up to 16, one above FP16's largest exponent).
__device__ __forceinline__ int step_log2(uint32_t bits) { return static_cast<int>(bits >> 10 & 31u) - 15; }

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hadd2(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2_rn(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  return hadd2(a, b ^ 0x80008000u);
}
__device__ __forceinline__ float2 half2_floats(uint32_t a) {
  return __half22float2(*reinterpret_cast<const __half2*>(&a));
}

constexpr uint32_t kNibble0 = 0x000f000fu;  // c * 2^-24 in both halves
constexpr uint32_t kNibble1 = 0x00f000f0u;  // c * 2^-20

// Codes as an operand register: c * 2^-24, or centred c - 8 (1024 + c,
// then minus 1032); the odd ones are 16 times that.
template <bool CENTRED>
__device__ __forceinline__ uint32_t even_codes(uint32_t word) {
  return CENTRED ? hadd2((word & kNibble0) | 0x64006400u, 0xe408e408u) : word & kNibble0;
}
template <bool CENTRED>
__device__ __forceinline__ uint32_t odd_codes(uint32_t word) {
  return CENTRED ? hadd2((word & kNibble1) | 0x64006400u, 0xe480e480u) : word & kNibble1;
}

// ln(sum * 2^base); -inf for an empty row.
__device__ __forceinline__ float log_of_sum(float base, float sum) {
  return sum != 0.0f ? (base + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

// ---- lists and units ----------------------------------------------------------------

// Row of the output of query row `row` of a KV head.
__device__ __forceinline__ int64_t output_row(const Kv4AttnParams& p, int b, int kv_head, int row) {
  return (static_cast<int64_t>(b) * p.new_tokens + row / p.group) * p.query_heads +
         static_cast<int64_t>(kv_head) * p.group + row % p.group;
}

// A request's length, 0 when it is out of range.
__device__ __forceinline__ int checked_length(int length, int table_blocks) {
  return length >= 0 && length <= static_cast<int64_t>(table_blocks) * kBlockTokens ? length : 0;
}

// Entries of a list: its request's blocks, or the selected ones and the newest.
__device__ __forceinline__ int list_entries(const Kv4AttnParams& p, int list, bool* bad) {
  const int raw = p.seq_lens[list / p.lists_per_request];
  const int length = checked_length(raw, p.table_blocks);
  *bad = length != raw;
  if (length == 0) return 0;
  if (!p.selected) return (length + kBlockTokens - 1) / kBlockTokens;
  return min(max(p.selected_count[list], 0), p.budget) + 1;
}

// The last list whose first entry is not behind `at`.
__device__ __forceinline__ int list_of(const int* starts, int lists, int at) {
  int low = 0, high = lists;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (starts[mid] <= at)
      low = mid;
    else
      high = mid;
  }
  return low;
}

// The ranges of the flat list: `cta` entries for each CTA, `warp` of them for
// each of its warps.
struct Quota {
  int entries, cta, warp;
};
__device__ __forceinline__ Quota quota_of(int entries, int ctas, int warps) {
  Quota q;
  q.entries = entries;
  q.cta = max((entries + ctas - 1) / ctas, 1);
  q.warp = (q.cta + warps - 1) / warps;
  return q;
}

// 16 elements as FP32.
template <int TYPE>
__device__ __forceinline__ void load16(const void* base, int64_t at, bool vectors, float (&x)[16]) {
  using Element = Kv4Type<TYPE>;
  const auto* from = static_cast<const typename Element::T*>(base) + at;
  if (vectors) {
    constexpr int kEach = 16 / sizeof(typename Element::T);
#pragma unroll
    for (int k = 0; k < 16 / kEach; ++k) {
      const uint4 v = reinterpret_cast<const uint4*>(from)[k];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (TYPE == SA_TYPE_F32) {
          x[4 * k + i] = __uint_as_float(w[i]);
        } else if constexpr (TYPE == SA_TYPE_BF16) {
          x[8 * k + 2 * i] = __uint_as_float(w[i] << 16);
          x[8 * k + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          x[8 * k + 2 * i] = f.x;
          x[8 * k + 2 * i + 1] = f.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = Element::load(from[i]);
  }
}

// ---- attention -------------------------------------------------------------------------

template <int NG, int NT>
struct Ring {
  static constexpr int kWarps = attention_warps(64 * NG, 8 * NT);
  static constexpr int kEntry = 36 * 64 * NG;
  static constexpr int kStages = NG == 4 ? 2 : 3;
  static constexpr int kStage = kEntry + 16;  // 16 zero bytes: the minima of lanes without a group
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kBytes = kWarps * kWarpBytes;
};

// Stages are read with the lanes' fragment pattern, so 16-byte pieces are
// permuted inside their rows on the way in: piece x of key row r, or of value
// pair row r, goes to place x ^ swizzle. Eight consecutive lanes then read all
// 32 banks (value reads took four passes without it, 50 shared-memory wavefronts
// more a block; 0.03 now).
template <int NG>
__device__ __forceinline__ int key_swizzle(int r) {
  return NG == 4 ? r & 1 : 0;
}
template <int NG>
__device__ __forceinline__ int value_swizzle(int r) {
  return NG == 1 ? r & 2 : NG == 2 ? 2 * (r & 3) : (r & 1) | 2 * (r & 2);
}

// MODE 0: 16-bit queries, BF16 output. 1: 16-bit queries, FP16 output (weights
// in two parts). 2: FP32 queries (queries and weights in two parts).
template <int NG, int NT, int MODE>
__global__ void __launch_bounds__(Ring<NG, NT>::kWarps * 32, 1)
    attention_kernel(const Kv4AttnParams p) {
  constexpr int kWarps = Ring<NG, NT>::kWarps;
  constexpr int kDim = 64 * NG, kEntry = Ring<NG, NT>::kEntry, kStages = Ring<NG, NT>::kStages;
  constexpr int kTile = 8 * NT;               // query rows of a unit
  constexpr int kParts = MODE == 2 ? 2 : 1;   // FP16 parts of a query
  constexpr int kWeights = MODE == 0 ? 1 : 2;  // FP16 parts of a weight
  constexpr bool kCentred = kWeights == 2;    // value codes as c - 8
  constexpr bool kCentredKeys = kParts == 2;  // key codes too
  constexpr int kPieces = kEntry / 16;        // 16-byte pieces of an entry
  constexpr int kStage = Ring<NG, NT>::kStage;
  constexpr int kQuery = MODE == 0 ? SA_TYPE_BF16 : MODE == 1 ? SA_TYPE_F16 : SA_TYPE_F32;
  extern __shared__ __align__(128) uint8_t kv4_smem[];
  __shared__ int scan_scratch[33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = kv4_smem + warp * Ring<NG, NT>::kWarpBytes;
  int* starts = reinterpret_cast<int*>(kv4_smem + Ring<NG, NT>::kBytes);
  const int lists = p.requests * p.lists_per_request;
  // Where a lane's 16-byte pieces of an entry go: piece 32 k + lane of the keys
  // and of the values (k even, odd), less 512 k bytes.
  const uint32_t ring_at = smem_addr(ring);
  const uint32_t key_place = 16 * (lane ^ key_swizzle<NG>(lane / (2 * NG)));
  const uint32_t value_place[2] = {16u * (lane ^ value_swizzle<NG>(lane / (4 * NG))),
                                   16u * (lane ^ value_swizzle<NG>((32 + lane) / (4 * NG)))};

  if (lane < kStages)
    *reinterpret_cast<uint4*>(ring + lane * kStage + kEntry) = make_uint4(0u, 0u, 0u, 0u);
  // Entries before each list. Up to 32 lists each warp sums by itself (all
  // write the same values) and needs no barrier.
  int base = 0;
  if (lists <= 32) {
    bool bad = false;
    const int n = lane < lists ? list_entries(p, lane, &bad) : 0;
    if (bad && blockIdx.x == 0 && warp == 0) raise_status(p.status, SA_DEV_BAD_BLOCK);
    int inclusive = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int before = __shfl_up_sync(0xffffffffu, inclusive, o);
      if (lane >= o) inclusive += before;
    }
    base = __shfl_sync(0xffffffffu, inclusive, 31);
    if (lane < lists) starts[lane + 1] = inclusive;
    if (lane == 0) starts[0] = 0;
    if (blockIdx.x == 0 && warp == 0) {
      if (lane < lists) p.starts[lane + 1] = inclusive;
      if (lane == 0) p.starts[0] = 0;
    }
    __syncwarp();
  } else {
    for (int first = 0; first < lists; first += blockDim.x) {
      const int list = first + threadIdx.x;
      bool bad = false;
      const int n = list < lists ? list_entries(p, list, &bad) : 0;
      if (bad && blockIdx.x == 0) raise_status(p.status, SA_DEV_BAD_BLOCK);
      int total;
      const int before = base + block_exclusive_scan(n, scan_scratch, &total);
      if (list < lists) starts[list] = before;
      base += total;
    }
    if (threadIdx.x == 0) starts[lists] = base;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i <= lists; i += blockDim.x) p.starts[i] = starts[i];
  }

  const Quota quota = quota_of(base * p.units_per_list, p.ctas, kWarps);
  const int cta_begin = min(static_cast<int>(blockIdx.x) * quota.cta, quota.entries);
  const int cta_end = min(cta_begin + quota.cta, quota.entries);
  const int warp_begin = min(cta_begin + warp * quota.warp, cta_end);
  const int end = min(warp_begin + quota.warp, cta_end);

  for (int at = warp_begin; at < end;) {
    // The unit of flat entry `at`, and the part of it in this warp's range.
    const int list = list_of(starts, lists, at / p.units_per_list);
    const int n = starts[list + 1] - starts[list];
    const int in_list = at - starts[list] * p.units_per_list;
    const int unit = in_list / n, first = in_list % n;
    const int count = min(n - first, end - at);
    // the CTA's whole range lies in this unit: its warps join their parts
    const int unit_begin = at - first;
    const bool joined = unit_begin <= cta_begin && unit_begin + n >= cta_end;
    const int b = list / p.lists_per_request;
    const int kv_head = list % p.lists_per_request * (p.kv_heads / p.lists_per_request) +
                        unit / p.row_tiles;
    const int row0 = unit % p.row_tiles * kTile;
    const int length = checked_length(p.seq_lens[b], p.table_blocks);
    const int newest = (length - 1) / kBlockTokens;
    const int32_t* table = p.table + static_cast<int64_t>(b) * p.table_blocks;
    const int32_t* ids =
        p.selected ? p.selected + static_cast<int64_t>(list) * p.budget : nullptr;
    const uint8_t* lane_pool = p.pool + static_cast<int64_t>(kv_head) * kEntry + 16 * lane;
    const int64_t block_stride = static_cast<int64_t>(p.kv_heads) * kEntry;

    // Physical blocks of 32 entries from `from` on, one per lane; -1 where
    // there is none to read.
    auto blocks_from = [&](int from) {
      const int e = from + lane;
      int block = -1;
      if (e < first + count) {
        int logical = e;
        bool good = true;
        if (ids) {
          logical = newest;
          if (e < n - 1) {
            logical = ids[e];
            good = logical >= 0 && logical < newest && (e == 0 || logical > ids[e - 1]);
          }
        }
        if (good) block = table[logical];
        if (block < 0 || block >= p.pool_blocks) {
          block = -1;
          raise_status(p.status, SA_DEV_BAD_BLOCK);
        }
      }
      return block;
    };
    int blocks = blocks_from(first);
    uint32_t unread = 0;  // bit s: stage s holds no entry
    auto fetch = [&](int i, int stage) {  // entry first + i into a stage
      if (i < count) {
        if (i > 0 && (i & 31) == 0) blocks = blocks_from(first + i);
        const int block = __shfl_sync(0xffffffffu, blocks, i & 31);
        unread &= ~(1u << stage);
        if (block < 0) {
          unread |= 1u << stage;
        } else {
          // 32 NG pieces of keys, 32 NG of values in rows of 2 NG and 4 NG
          // pieces, then the scales
          const uint8_t* from = lane_pool + block * block_stride;
          const uint32_t to = ring_at + stage * kStage;
#pragma unroll
          for (int k = 0; k < (kPieces + 31) / 32; ++k) {
            const uint32_t place = k < 2 * NG ? key_place : k < 4 * NG ? value_place[k & 1] : 16 * lane;
            if (kPieces % 32 == 0 || k * 32 + lane < kPieces)
              cp_async16_at(to + place + 512 * k, from + 512 * k);
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kStages; ++s) fetch(s, s);

    // Query fragments: lane (g, t) holds elements 64 gr + 16 t .. + 15 of row g.
    uint32_t q[NT][kParts][NG][8];
    float row_factor[NT][2];   // F of columns 2t, 2t + 1
    float row_sum[NT][NG][2];  // Q_g of columns 2t, 2t + 1
    int limit[NT][2];          // tokens that columns 2t, 2t + 1 see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + nt * 8 + g;
      const bool live = row < p.rows;
      const int i = live ? row / p.group : 0, h = live ? row % p.group : 0;
      const int64_t from = b * p.stride_request + i * p.stride_token +
                           (static_cast<int64_t>(kv_head) * p.group + h) * p.stride_head + 16 * t;
      float x[NG][16], sums[NG];
      float top = 0.0f;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        if (live) {
          load16<kQuery>(p.query, from + 64 * gr, p.vector_rows, x[gr]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) x[gr][e] = 0.0f;
        }
        sums[gr] = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          top = fmaxf(top, fabsf(x[gr][e]));
          sums[gr] += x[gr][e];
        }
        sums[gr] += __shfl_xor_sync(0xffffffffu, sums[gr], 1);
        sums[gr] += __shfl_xor_sync(0xffffffffu, sums[gr], 2);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^(14 - floor(log2 top)), kept inside FP32 for the smallest rows
      const int exponent = max((__float_as_int(top) >> 23) - 127, -100);
      const float up = __int_as_float((14 - exponent + 127) << 23);
      const float down = __int_as_float((exponent - 14 + 127) << 23);
#pragma unroll
      for (int gr = 0; gr < NG; ++gr)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int e = 8 * w + 2 * s;
            const float even0 = x[gr][e] * up, even1 = x[gr][e + 4] * up;
            const float odd0 = x[gr][e + 1] * up * 0.0625f, odd1 = x[gr][e + 5] * up * 0.0625f;
            const int k = (w * 2 + s) * 2;
            q[nt][0][gr][k] = pack_half2(even0, even1);
            q[nt][0][gr][k + 1] = pack_half2(odd0, odd1);
            if constexpr (kParts == 2) {
              const float2 he = half2_floats(q[nt][0][gr][k]), ho = half2_floats(q[nt][0][gr][k + 1]);
              q[nt][1][gr][k] = pack_half2(even0 - he.x, even1 - he.y);
              q[nt][1][gr][k + 1] = pack_half2(odd0 - ho.x, odd1 - ho.y);
            }
          }
      const float factor = p.scale_log2 * down * (kCentredKeys ? 1.0f : 16777216.0f);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int source = (2 * t + c) * 4;
        row_factor[nt][c] = __shfl_sync(0xffffffffu, factor, source);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
          row_sum[nt][gr][c] = p.scale_log2 * __shfl_sync(0xffffffffu, sums[gr], source);
        const int r = row0 + nt * 8 + 2 * t + c;
        limit[nt][c] = length - p.new_tokens + 1 + (r < p.rows ? r / p.group : 0);
      }
    }
    const int least = length - p.new_tokens + 1 + row0 / p.group;  // what every row sees
    // what the last row sees
    const int longest = length - p.new_tokens + 1 + (min(row0 + kTile, p.rows) - 1) / p.group;

    float o[NT][NG][2][2][4];  // codes' sums of element 64 gr + 8 g + 4 w + 2 s (+ 1, times 16)
    float low[NT][2];          // minima's sums: lane group g holds value group g's
    float base[NT][2], sum[NT][2];  // running maximum - 11; sum of 2^(x - base)
    uint32_t step_bits[NG];         // 2^E of each group as FP16 bits in both halves, 0 before the first block
    uint32_t step_unit[NG];         // 2^-E in both halves: value steps are held as s * 2^-E
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) step_bits[gr] = step_unit[gr] = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        base[nt][c] = -3.0e38f;
        sum[nt][c] = 0.0f;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) low[nt][c] = 0.0f;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr)
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nt][gr][m >> 1][m & 1][c] = 0.0f;
    }

    // One entry. Blocks that every row sees whole take the copy without masks.
    // Of the block whose first token is token0, the other one takes the rows
    // that see at least `from` and at most `to` of its tokens.
    auto process = [&](const uint8_t* entry, int token0, int from, int to, auto masks) {
      constexpr bool kMasked = decltype(masks)::value;
      bool sees[NT][2];  // columns 2t, 2t + 1 take part
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int held = min(limit[nt][c] - token0, kBlockTokens);
          sees[nt][c] = !kMasked || (held >= from && held <= to);
        }
      // ---- logits
      float x[NT][2][4];
      uint4 scales[NG];  // (step, minimum) of rows g, g + 8, g + 16, g + 24
#pragma unroll
      for (int gr = 0; gr < NG; ++gr)
        scales[gr] = *reinterpret_cast<const uint4*>(entry + kv4_key_scales(kDim) + gr * 128 + g * 16);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t word[2][2 * NG];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* from = entry + (16 * j + 8 * h + g) * (kDim / 2);
          if constexpr (NG == 1) {
            const uint2 w = *reinterpret_cast<const uint2*>(from + 8 * t);
            word[h][0] = w.x;
            word[h][1] = w.y;
          } else {
#pragma unroll
            for (int k = 0; k < NG / 2; ++k) {
              const uint4 w = *reinterpret_cast<const uint4*>(
                  from + 16 * ((NG / 2 * t + k) ^ key_swizzle<NG>(g)));
              word[h][4 * k] = w.x;
              word[h][4 * k + 1] = w.y;
              word[h][4 * k + 2] = w.z;
              word[h][4 * k + 3] = w.w;
            }
          }
        }
        float lowest[NT][4];
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          float acc[NT][kParts][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
              for (int c = 0; c < 4; ++c) acc[nt][part][c] = 0.0f;
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const uint32_t r0 = word[0][2 * gr + w] >> (8 * s), r1 = word[1][2 * gr + w] >> (8 * s);
              const uint32_t a0 = even_codes<kCentredKeys>(r0), a1 = even_codes<kCentredKeys>(r1),
                             a2 = odd_codes<kCentredKeys>(r0), a3 = odd_codes<kCentredKeys>(r1);
              const int k = (w * 2 + s) * 2;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int part = 0; part < kParts; ++part)
                  mma16816(acc[nt][part], a0, a1, a2, a3, q[nt][part][gr][k], q[nt][part][gr][k + 1]);
            }
          const uint32_t sm0 = j == 0 ? scales[gr].x : scales[gr].z;
          const uint32_t sm1 = j == 0 ? scales[gr].y : scales[gr].w;
          float2 f0 = half2_floats(sm0), f1 = half2_floats(sm1);
          if constexpr (kCentredKeys) {
            f0.y = fmaf(8.0f, f0.x, f0.y);
            f1.y = fmaf(8.0f, f1.x, f1.y);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float step = c < 2 ? f0.x : f1.x, minimum = c < 2 ? f0.y : f1.y;
              const float dot =
                  kParts == 2 ? acc[nt][0][c] + acc[nt][kParts - 1][c] : acc[nt][0][c];
              x[nt][j][c] = gr == 0 ? step * dot : fmaf(step, dot, x[nt][j][c]);
              lowest[nt][c] = gr == 0 ? minimum * row_sum[nt][gr][c & 1]
                                      : fmaf(minimum, row_sum[nt][gr][c & 1], lowest[nt][c]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            x[nt][j][c] = fmaf(x[nt][j][c], row_factor[nt][c & 1], lowest[nt][c]);
      }
      if constexpr (kMasked) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (!sees[nt][c & 1] || token0 + 16 * j + 8 * (c >> 1) + g >= limit[nt][c & 1])
                x[nt][j][c] = -INFINITY;
      }

      // ---- value scales: pairs of tokens (16 j + 8 h + 2 t, + 1)
      uint32_t step[NG][2][2], minimum[2][2];
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        const uint4 w =
            *reinterpret_cast<const uint4*>(entry + kv4_value_scales(kDim) + gr * 64 + t * 16);
        step[gr][0][0] = w.x;
        step[gr][0][1] = w.y;
        step[gr][1][0] = w.z;
        step[gr][1][1] = w.w;
      }
      {
        const uint4 w = *reinterpret_cast<const uint4*>(
            entry + (g < NG ? kv4_value_scales(kDim) + kDim + g * 64 + t * 16 : kEntry));
        minimum[0][0] = w.x;
        minimum[0][1] = w.y;
        minimum[1][0] = w.z;
        minimum[1][1] = w.w;
      }
      if constexpr (kMasked) {  // tokens that no row sees: nothing of them may enter a product
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = 16 * j + 8 * h + 2 * t;
            const uint32_t keep = (r < to ? 0xffffu : 0u) | (r + 1 < to ? 0xffff0000u : 0u);
            minimum[j][h] &= keep;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) step[gr][j][h] &= keep;
          }
      }
      // ---- running maxima of the logits and of the value steps, raised only
      // when a logit passes its row's by the headroom or a step passes 2^E
      uint32_t above = 0;  // bits 15 and 31: a step is not below its 2^E
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        const uint32_t most = __vmaxu2(__vimax3_u16x2(step[gr][0][0], step[gr][0][1], step[gr][1][0]),
                                       step[gr][1][1]);
        above |= (most | 0x80008000u) - step_bits[gr];  // 15-bit values: the halves do not borrow
      }
      bool passes = (above & 0x80008000u) != 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          passes |= fmaxf(fmaxf(x[nt][0][c], x[nt][0][c + 2]), fmaxf(x[nt][1][c], x[nt][1][c + 2])) >
                    base[nt][c] + (kHeadroom + kWeightLog2);
      if (__any_sync(0xffffffffu, passes)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m = fmaxf(fmaxf(x[nt][0][c], x[nt][0][c + 2]), fmaxf(x[nt][1][c], x[nt][1][c + 2]));
            m -= kWeightLog2;
            m = fmaxf(m, base[nt][c]);
#pragma unroll
            for (int s = 4; s < 32; s <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
            const float keep = exp2_approx(base[nt][c] - m);
            base[nt][c] = m;
            sum[nt][c] *= keep;
            low[nt][c] *= keep;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                o[nt][gr][k >> 1][k & 1][c] *= keep;
                o[nt][gr][k >> 1][k & 1][c + 2] *= keep;
              }
          }
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          // NaN and infinite steps (from 0x7c00 on) carry themselves through the products
          uint32_t most = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t w = step[gr][k >> 1][k & 1];
            most = __vmaxu2(most, w & __vcmpltu2(w, 0x7c007c00u));
          }
          uint32_t largest = max(most & 0xffffu, most >> 16);
          largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
          largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
          const uint32_t bits = step_bits[gr] & 0xffffu;
          if (largest < bits) continue;  // the same in every lane
          const int exponent = step_exponent(largest);
          const float keep = bits == 0 ? 0.0f : power_of_2(step_log2(bits) - exponent);
          step_bits[gr] = static_cast<uint32_t>(exponent + 15) * 0x04000400u;
          const __half2 unit = __half2half2(__float2half_rn(power_of_2(-exponent)));
          step_unit[gr] = *reinterpret_cast<const uint32_t*>(&unit);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int c = 0; c < 4; ++c) o[nt][gr][k >> 1][k & 1][c] *= keep;
        }
      }
      // ---- weights, as columns of the second product
      uint32_t weight[NT][kWeights][2][2];  // part, matrix step j, half h
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float a = exp2_approx(x[nt][j][2 * h] - base[nt][0]);
            const float c = exp2_approx(x[nt][j][2 * h + 1] - base[nt][1]);
            sum[nt][0] += a;
            sum[nt][1] += c;
            const uint32_t high = pack_half2(a, c);
            weight[nt][0][j][h] = transpose8(high);
            if constexpr (kWeights == 2) {
              const float2 f = half2_floats(high);
              weight[nt][1][j][h] = transpose8(pack_half2(a - f.x, c - f.y));
            }
          }

      // ---- weighted minima: row g of the operand, what rounding the centred
      // ones to FP16 lost in row g + 8
      uint32_t rest[2][2] = {{0u, 0u}, {0u, 0u}};
      float low_unit = 1.0f;
      if constexpr (kCentred) {
        // minimum + 8 step as an unevaluated sum of two FP16 numbers (Knuth's
        // two-sum), halved where 8 step could pass FP16's largest
        uint32_t bits = step_bits[0];
#pragma unroll
        for (int gr = 1; gr < NG; ++gr) bits = g == gr ? step_bits[gr] : bits;
        const bool large = step_log2(bits) > 12;
        low_unit = large ? 2.0f : 1.0f;
        const uint32_t eight = large ? 0x44004400u : 0x48004800u, one = large ? 0x38003800u : 0x3c003c00u;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t mine = step[0][j][h];
#pragma unroll
            for (int gr = 1; gr < NG; ++gr) mine = g == gr ? step[gr][j][h] : mine;
            const uint32_t a = hmul2(g < NG ? mine : 0u, eight), c = hmul2(minimum[j][h], one);
            const uint32_t all = hadd2(a, c), back = hsub2(all, a);
            rest[j][h] = hadd2(hsub2(a, hsub2(all, back)), hsub2(c, back));
            minimum[j][h] = all;
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int part = 0; part < kWeights; ++part)
            mma16816(acc, minimum[j][0], rest[j][0], minimum[j][1], rest[j][1],
                     weight[nt][part][j][0], weight[nt][part][j][1]);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (sees[nt][c])
            low[nt][c] = kCentred ? fmaf(acc[c] + acc[c + 2], low_unit, low[nt][c]) : low[nt][c] + acc[c];
      }
      // ---- weighted codes
      uint32_t word[2][2][2 * NG];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* from = entry + kv4_value_codes(kDim) + (8 * j + 4 * h + t) * kDim;
          if constexpr (NG == 1) {
            const uint2 w = *reinterpret_cast<const uint2*>(
                from + 16 * ((g >> 1) ^ value_swizzle<NG>(t)) + 8 * (g & 1));
            word[j][h][0] = w.x;
            word[j][h][1] = w.y;
          } else {
#pragma unroll
            for (int k = 0; k < NG / 2; ++k) {
              const uint4 w = *reinterpret_cast<const uint4*>(
                  from + 16 * ((NG / 2 * g + k) ^ value_swizzle<NG>(t)));
              word[j][h][4 * k] = w.x;
              word[j][h][4 * k + 1] = w.y;
              word[j][h][4 * k + 2] = w.z;
              word[j][h][4 * k + 3] = w.w;
            }
          }
        }
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        uint32_t scaled[NT][kWeights][2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t s = hmul2(step[gr][j][h], step_unit[gr]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              scaled[nt][0][j][h] = hmul2(weight[nt][0][j][h], s);
              if constexpr (kWeights == 2)  // what the first part's rounding lost, and the rest
                scaled[nt][1][j][h] =
                    hfma2(weight[nt][1][j][h], s,
                          hfma2(weight[nt][0][j][h], s, scaled[nt][0][j][h] ^ 0x80008000u));
            }
          }
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const uint32_t r0 = word[j][0][2 * gr + w] >> (8 * s);
                const uint32_t r1 = word[j][1][2 * gr + w] >> (8 * s);
#pragma unroll
                for (int part = 0; part < kWeights; ++part)
                  mma16816(acc, even_codes<kCentred>(r0), odd_codes<kCentred>(r0),
                           even_codes<kCentred>(r1), odd_codes<kCentred>(r1),
                           scaled[nt][part][j][0], scaled[nt][part][j][1]);
              }
#pragma unroll
              for (int c = 0; c < 4; ++c)
                if (sees[nt][c & 1]) o[nt][gr][w][s][c] += acc[c];
            }
      }
    };

    // A token that some rows see and others do not has a weight of zero for
    // these, which leaves them as they are unless its values are not finite (zero
    // times that is NaN) or its steps raise their group's exponent. Does one of
    // an entry's tokens from .. to - 1 forbid to take such rows together? (Always
    // apart, 16 requests with 4 drafts each took 171 us instead of 150.)
    auto parts_rows = [&](const uint8_t* entry, int from, int to) {
      bool parts = false;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        const auto* at = reinterpret_cast<const uint16_t*>(entry + kv4_value_scale_at(kDim, lane, gr));
        const uint32_t step = at[0];
        uint32_t bound = step_bits[gr] & 0xffffu;
        if (bound == 0)  // none yet: the one that the tokens seen by all rows will set
          bound = (step_exponent(__reduce_max_sync(0xffffffffu, lane < from && step < 0x7c00u ? step : 0u)) + 15) << 10;
        parts |= step >= bound || (at[kDim / 2] & 0x7c00u) == 0x7c00u;
      }
      return __any_sync(0xffffffffu, parts && lane >= from && lane < to);
    };

    int stage = 0, seen = 0;  // seen: tokens of a masked block that its last turn's rows saw
    for (int i = 0; i < count;) {
      if (seen == 0) {
        cp_async_wait<kStages - 1>();
        __syncwarp();
      }
      if (!(unread >> stage & 1)) {
        const uint8_t* entry = ring + stage * kStage;
        const int logical = ids ? newest : first + i;  // with ids, used for the newest block only
        const int token0 = logical * kBlockTokens;
        if ((!ids || first + i == n - 1) && token0 + kBlockTokens > least) {
          const int from = max(least - token0, seen + 1), most = min(longest - token0, kBlockTokens);
          seen = most;
          if (from <= most) {
            if (from < most && parts_rows(entry, from, most)) seen = from;
            process(entry, token0, from, seen, std::true_type{});
          }
          if (seen < most) continue;
        } else {
          process(entry, token0, 0, kBlockTokens, std::false_type{});
        }
      }
      seen = 0;
      __syncwarp();  // every lane has read the stage
      fetch(i + kStages, stage);
      stage = stage + 1 == kStages ? 0 : stage + 1;
      ++i;
    }
    cp_async_wait<0>();

    // ---- the segment's result
    const bool whole = count == n;
    const int part = ((static_cast<int>(blockIdx.x) * kWarps + warp) * 2 + (at == warp_begin ? 0 : 1)) * kTile;
    const bool shared = joined && !whole;  // joined through shared memory
    float* mine = reinterpret_cast<float*>(ring);  // [kTile][kDim], then [kTile][2]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s = sum[nt][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const int r = nt * 8 + 2 * t + c, row = row0 + r;
        const float scale = whole ? (s != 0.0f ? 1.0f / s : 0.0f) : 1.0f;
        const int64_t out_row = output_row(p, b, kv_head, row);
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          const float minima = __shfl_sync(0xffffffffu, low[nt][c], gr * 4 + t);
          const float code_unit = power_of_2((kCentred ? 0 : 24) + step_log2(step_bits[gr]));
          float y[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float* acc = o[nt][gr][k >> 1][k & 1];
            y[2 * k] = fmaf(acc[c], code_unit, minima) * scale;
            y[2 * k + 1] = fmaf(acc[c + 2], code_unit * 0.0625f, minima) * scale;
          }
          if (row < p.rows) {
            const int e = 64 * gr + 8 * g;
            if (whole)
              store8(p.out, out_row * kDim + e, MODE == 2 ? p.out_type : kQuery, y);
            else if (shared)
              store8(mine, r * kDim + e, SA_TYPE_F32, y);
            else
              store8(p.part_o, static_cast<int64_t>(part + r) * kDim + e, SA_TYPE_F32, y);
          }
        }
        if (g == 0 && row < p.rows) {
          if (whole) {
            if (p.lse) p.lse[out_row] = log_of_sum(base[nt][c], s);
          } else {
            float* ml = shared ? mine + kTile * kDim + r * 2 : p.part_ml + (part + r) * 2;
            ml[0] = base[nt][c];
            ml[1] = s;
          }
        }
      }
    if (shared) {
      // Every active warp of the CTA has this one segment.
      const int active = (cta_end - cta_begin + quota.warp - 1) / quota.warp;
      if (active > 1)
        asm volatile("bar.sync 1, %0;" ::"r"(active * 32) : "memory");
      else
        __syncwarp();
      const bool complete = unit_begin == cta_begin && unit_begin + n == cta_end;
      const int cta_part = static_cast<int>(blockIdx.x) * kWarps * 2 * kTile;
      constexpr int kVectors = kDim / 4;
      for (int i = threadIdx.x; i < kTile * kVectors; i += active * 32) {
        const int r = i / kVectors, e = i % kVectors * 4, row = row0 + r;
        if (row >= p.rows) break;
        float top = -INFINITY, s = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < active; ++w) {
          const float* from = reinterpret_cast<const float*>(kv4_smem + w * Ring<NG, NT>::kWarpBytes);
          top = fmaxf(top, from[kTile * kDim + r * 2]);
        }
        for (int w = 0; w < active; ++w) {
          const float* from = reinterpret_cast<const float*>(kv4_smem + w * Ring<NG, NT>::kWarpBytes);
          const float weight = exp2_approx(from[kTile * kDim + r * 2] - top);
          s = fmaf(weight, from[kTile * kDim + r * 2 + 1], s);
          const float4 v = *reinterpret_cast<const float4*>(from + r * kDim + e);
          y[0] = fmaf(weight, v.x, y[0]);
          y[1] = fmaf(weight, v.y, y[1]);
          y[2] = fmaf(weight, v.z, y[2]);
          y[3] = fmaf(weight, v.w, y[3]);
        }
        if (complete) {
          const int64_t out_row = output_row(p, b, kv_head, row);
          const float scale = s != 0.0f ? 1.0f / s : 0.0f;
          store4(p.out, out_row * kDim + e, MODE == 2 ? p.out_type : kQuery, y[0] * scale,
                 y[1] * scale, y[2] * scale, y[3] * scale);
          if (p.lse && e == 0) p.lse[out_row] = log_of_sum(top, s);
        } else {
          store4(p.part_o, static_cast<int64_t>(cta_part + r) * kDim + e, SA_TYPE_F32, y[0], y[1],
                 y[2], y[3]);
          if (e == 0) {
            p.part_ml[(cta_part + r) * 2] = top;
            p.part_ml[(cta_part + r) * 2 + 1] = s;
          }
        }
      }
    }
    at += count;
  }
}

// Where the parts of a unit [begin, end) of the flat list are: those of the
// first CTA's warps, one of each CTA between, those of the last CTA's; a CTA
// whose whole range lies in the unit has one, its warp 0's.
struct Parts {
  int begin, first, first_warp, first_parts, ctas, count;
};
__device__ __forceinline__ Parts parts_of(const Quota& q, int begin, int end) {
  Parts u{};
  u.begin = begin;
  if (begin == end) return u;
  u.first = begin / q.cta;
  const int last = (end - 1) / q.cta;
  u.ctas = last - u.first + 1;
  const auto covers = [&](int cta) {
    return begin <= cta * q.cta && end >= min((cta + 1) * q.cta, q.entries);
  };
  u.first_warp = (begin - u.first * q.cta) / q.warp;
  u.first_parts = covers(u.first)
                      ? 1
                      : (min(end - u.first * q.cta, q.cta) - 1) / q.warp - u.first_warp + 1;
  u.count = u.first_parts;
  if (u.ctas > 1) u.count += u.ctas - 1 + (covers(last) ? 0 : (end - 1 - last * q.cta) / q.warp);
  return u;
}
// Slot of a unit's i-th part.
__device__ __forceinline__ int part_slot(const Parts& u, const Quota& q, int warps, int i) {
  int cta = u.first, w = u.first_warp + i;
  if (i >= u.first_parts) {
    i -= u.first_parts;
    cta = u.first + 1 + min(i, u.ctas - 2);
    w = max(i - (u.ctas - 2), 0);
  }
  const bool inside = cta * q.cta + w * q.warp < u.begin;  // begins inside the warp's range
  return (cta * warps + w) * 2 + (inside ? 1 : 0);
}

// Joins parts first, first + stride, ... of row r of a unit in one warp: lane l
// gets elements l, l + 32, ...; UNROLL parts' loads are in flight together.
template <int NG, int UNROLL>
__device__ __forceinline__ void join_parts(const Kv4AttnParams& p, const Quota& q, const Parts& u,
                                           int tile, int r, int first, int stride, float& top,
                                           float& sum, float (&o)[2 * NG]) {
  constexpr int kDim = 64 * NG, kPerLane = 2 * NG;
  const int lane = threadIdx.x & 31;
  for (int i = first; i < u.count; i += stride * UNROLL) {
    float ml[UNROLL][2], v[UNROLL][kPerLane];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int64_t at =
          static_cast<int64_t>(part_slot(u, q, p.warps, min(i + k * stride, u.count - 1))) * tile + r;
      const float2 pair = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
      ml[k][0] = pair.x;
      ml[k][1] = pair.y;
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) v[k][j] = p.part_o[at * kDim + j * 32 + lane];
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      if (i + k * stride >= u.count) break;
      const float now = fmaxf(top, ml[k][0]);
      const float keep = exp2_approx(top - now), weight = exp2_approx(ml[k][0] - now);
      top = now;
      sum = fmaf(sum, keep, weight * ml[k][1]);
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) o[j] = fmaf(o[j], keep, weight * v[k][j]);
    }
  }
}

__device__ __forceinline__ void store1(void* base, int64_t i, int type, float x) {
  if (type == SA_TYPE_F32)
    static_cast<float*>(base)[i] = x;
  else if (type == SA_TYPE_F16)
    static_cast<__half*>(base)[i] = __float2half_rn(min_nan(x, kHalfMost));
  else
    static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
}

// Joins the parts of split units and writes the rows of empty ones. SHARED: one
// CTA a query row, its warps sharing the row's parts, of which few units can have
// hundreds. Otherwise one CTA a unit and a warp a row: most of the cost is then
// finding the parts, and many units have none left to join (512 requests of 100
// tokens: 62 us with a CTA a row, 47 us so).
template <int NG, int WARPS, bool SHARED>
__global__ void __launch_bounds__(WARPS * 32) merge_kernel(const Kv4AttnParams p, int tile) {
  constexpr int kDim = 64 * NG, kPerLane = kDim / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = min(tile, p.rows);
  const int u = SHARED ? blockIdx.x / rows : blockIdx.x;
  const int list = u / p.units_per_list, unit = u % p.units_per_list;
  const int start = p.starts[list], n = p.starts[list + 1] - start;
  const Quota quota =
      quota_of(p.starts[p.requests * p.lists_per_request] * p.units_per_list, p.ctas, p.warps);
  const int begin = start * p.units_per_list + unit * n;
  const Parts parts = parts_of(quota, begin, begin + n);
  if (parts.count == 1) return;  // written by the attention
  const int b = list / p.lists_per_request;
  const int kv_head =
      list % p.lists_per_request * (p.kv_heads / p.lists_per_request) + unit / p.row_tiles;
  const int row0 = unit % p.row_tiles * tile;
  if constexpr (!SHARED) {
    for (int r = warp; r < rows && row0 + r < p.rows; r += WARPS) {
      float top = -INFINITY, sum = 0.0f, o[kPerLane] = {};
      join_parts<NG, 8>(p, quota, parts, tile, r, 0, 1, top, sum, o);
      const int64_t out_row = output_row(p, b, kv_head, row0 + r);
      const float scale = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
      for (int j = 0; j < kPerLane; ++j)
        store1(p.out, out_row * kDim + j * 32 + lane, p.out_type, o[j] * scale);
      if (p.lse && lane == 0) p.lse[out_row] = log_of_sum(top, sum);
    }
  } else {
    __shared__ float shared_o[WARPS][kDim];
    __shared__ float shared_ml[WARPS][2];
    const int r = blockIdx.x % rows;
    if (row0 + r >= p.rows) return;
    float top = -INFINITY, sum = 0.0f, o[kPerLane] = {};
    join_parts<NG, 4>(p, quota, parts, tile, r, warp, WARPS, top, sum, o);
    if (lane == 0) {
      shared_ml[warp][0] = top;
      shared_ml[warp][1] = sum;
    }
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) shared_o[warp][j * 32 + lane] = o[j];
    __syncthreads();
    top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, shared_ml[w][0]);
    const int64_t out_row = output_row(p, b, kv_head, row0 + r);
    for (int e = threadIdx.x; e < kDim; e += WARPS * 32) {
      float y = 0.0f;
      sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w >= parts.count) break;
        const float weight = exp2_approx(shared_ml[w][0] - top);
        sum = fmaf(weight, shared_ml[w][1], sum);
        y = fmaf(weight, shared_o[w][e], y);
      }
      store1(p.out, out_row * kDim + e, p.out_type, sum != 0.0f ? y / sum : 0.0f);
      if (p.lse && e == 0) p.lse[out_row] = log_of_sum(top, sum);
    }
  }
}

// ---- host ---------------------------------------------------------------------------------

// Query rows of a unit: 16 where a KV head has more than 8 and registers allow
// (BF16 and FP16 at head_dim up to 128), else 8.
int tile_rows(size_t rows, size_t head_dim, int query_type) {
  return rows > 8 && head_dim <= 128 && query_type != SA_TYPE_F32 ? 16 : 8;
}

// Rows of the parts that a grid of one CTA an SM may write: two units a warp.
size_t part_rows(size_t head_dim, int tile) {
  return (size_t)device_sm_count() * attention_warps((int)head_dim, tile) * 2 * tile;
}

size_t round256(size_t x) { return (x + 255) & ~size_t(255); }

template <int NG, int NT, int MODE>
sa_status launch(const Kv4AttnParams& p, int lists, cudaStream_t stream) {
  static int configured[kMaxDevices];
  const auto kernel = attention_kernel<NG, NT, MODE>;
  constexpr int kMost = Ring<NG, NT>::kBytes + (kMaxLists + 1) * (int)sizeof(int);
  const sa_status st = ensure_smem_limit(reinterpret_cast<const void*>(kernel), kMost, configured);
  if (st != SA_OK) return st;
  const size_t smem = Ring<NG, NT>::kBytes + (size_t)(lists + 1) * sizeof(int);
  SA_CUDA_TRY(launch_kernel(kernel, dim3(p.ctas), dim3(Ring<NG, NT>::kWarps * 32), smem, stream, false, p));
  // A warp a row where units have some four parts (all warps' ranges over the
  // units), else a CTA a row: 16, 32 and 64 requests of 8K (14, 7 and 3.5 parts)
  // took 43.1, 67.3 and 117.4 us with a CTA a row, 48.4, 69.0 and 115.2 us with a
  // warp (medians over eight places of the cache; 0.5, 1.9 and 1.8 us between the
  // ends of either).
  const int units = lists * p.units_per_list, rows = std::min(p.rows, 8 * NT);
  const auto merge = [&](auto kernel_, int grid, int warps) {
    return launch_kernel(kernel_, dim3(grid), dim3(warps * 32), 0, stream, false, p, 8 * NT);
  };
  const cudaError_t err = units < p.ctas * p.warps / 4 ? merge(merge_kernel<NG, 4, true>, units * rows, 4)
                          : rows <= 4                   ? merge(merge_kernel<NG, 4, false>, units, 4)
                          : rows <= 8                   ? merge(merge_kernel<NG, 8, false>, units, 8)
                                                        : merge(merge_kernel<NG, 16, false>, units, 16);
  return cuda_status(err, "attention_kv4 merge launch");
}

template <int NG>
sa_status launch_dim(const Kv4AttnParams& p, int lists, int tile, cudaStream_t stream) {
  const int mode = p.query_type == SA_TYPE_F32 ? 2 : p.out_type == SA_TYPE_F16 ? 1 : 0;
  if constexpr (NG <= 2) {
    if (tile == 16)
      return mode == 0 ? launch<NG, 2, 0>(p, lists, stream) : launch<NG, 2, 1>(p, lists, stream);
  }
  return mode == 0   ? launch<NG, 1, 0>(p, lists, stream)
         : mode == 1 ? launch<NG, 1, 1>(p, lists, stream)
                     : launch<NG, 1, 2>(p, lists, stream);
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
  const size_t rows = std::max(part_rows(head_dim, 8), part_rows(head_dim, 16));
  return round256((kMaxLists + 1) * sizeof(int)) + rows * (2 + head_dim) * sizeof(float);
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
  if ((reinterpret_cast<uintptr_t>(pool) & 15u) != 0 || (reinterpret_cast<uintptr_t>(out) & 15u) != 0)
    return fail(SA_ERR_INVALID_ARG, "attention_kv4: the pool and out must be 16-byte aligned");
  size_t lists = 1, list_blocks = table_blocks;
  if (selected) {
    if (!selected_count || budget == 0 || select_groups == 0 || kv_heads % select_groups != 0)
      return fail(SA_ERR_INVALID_ARG, "attention_kv4: invalid selection");
    if (new_tokens != 1)
      return fail(SA_ERR_UNSUPPORTED, "attention_kv4: a selection serves one new token a request");
    lists = select_groups;
    list_blocks = budget + 1;
  }
  if (requests > (size_t)kMaxLists || lists > (size_t)kMaxLists || requests * lists > (size_t)kMaxLists)
    return fail(SA_ERR_UNSUPPORTED, "attention_kv4: more than 8192 requests or lists");
  constexpr size_t kMost = 0x7fffffffu;
  if (pool_blocks > kMost / kBlockTokens || table_blocks > kMost / kBlockTokens || budget >= kMost ||
      requests * lists * list_blocks > kMost)
    return fail(SA_ERR_UNSUPPORTED, "attention_kv4: more than 2^31 slots or listed blocks");
  // every row of every tile, and every entry of every unit, has a 31-bit index
  if (query_heads > 65536 || new_tokens > 65536 || requests * (query_heads + 16 * kv_heads) > kMost / new_tokens)
    return fail(SA_ERR_UNSUPPORTED, "attention_kv4: too many query rows");
  const size_t need =
      sa_attention_kv4_workspace_size(requests, new_tokens, query_heads, kv_heads, head_dim);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
    return fail(SA_ERR_CAPACITY,
                "attention_kv4: workspace unaligned or smaller than sa_attention_kv4_workspace_size()");
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
  p.group = (int)(query_heads / kv_heads);
  p.rows = p.group * p.new_tokens;
  const int tile = tile_rows((size_t)p.rows, head_dim, query_type);
  p.row_tiles = (p.rows + tile - 1) / tile;
  p.units_per_list = (int)(kv_heads / lists) * p.row_tiles;
  if (requests * lists * list_blocks > (kMost >> 1) / (size_t)p.units_per_list)
    return fail(SA_ERR_UNSUPPORTED, "attention_kv4: more than 2^30 (block, KV head, row tile) entries");
  p.scale_log2 = scale * 1.4426950408889634f;
  const size_t element = query_type == SA_TYPE_F32 ? 4 : 2;
  p.vector_rows = ((reinterpret_cast<uintptr_t>(query) | (size_t)stride_request * element |
                    (size_t)stride_token * element | (size_t)stride_head * element) & 15u) == 0;
  p.ctas = device_sm_count();
  p.warps = attention_warps((int)head_dim, tile);
  char* ws = static_cast<char*>(workspace);
  p.starts = reinterpret_cast<int*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + round256((kMaxLists + 1) * sizeof(int)));
  p.part_o = p.part_ml + part_rows(head_dim, tile) * 2;
  const int all = (int)(requests * lists);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return head_dim == 64    ? launch_dim<1>(p, all, tile, s)
         : head_dim == 128 ? launch_dim<2>(p, all, tile, s)
                           : launch_dim<4>(p, all, tile, s);
}
