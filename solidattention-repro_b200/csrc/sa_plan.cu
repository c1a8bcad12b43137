// sa_plan.cu -- block tables and slot maps on the device from request lengths.
//
// One launch brings a batch's block tables, lengths and free list from one
// step to the next and writes the slot of every new token. Everything follows
// from prefix sums over the requests:
//
//   grow = max(add, 0)            token i of request b is row cu[b] + i
//   want = ceil(new length / 32)  need = max(want - held, 0) blocks are taken
//                                 gone = max(held - want, 0) are given back
//   a-th block taken  (request order, then logical) = free_list[top - 1 - a]
//   r-th block given back goes to free_list[top - A + R - 1 - r]
//
// (A, R: all taken, all given back.) Taking from the top down and giving back
// in reverse makes a step and its inverse restore the list. Every output has a
// place of its own, so nothing depends on the order of threads.
//
// The work is a few bytes a request and 8 a token, and its time is the chain
// of dependent reads (lengths, scan, list, table), so it is one launch: a
// single CTA for small steps, one cluster for large ones (the scans are
// repeated in each CTA, the writes are split; a cluster barrier stands between
// the last read of the old state and the first write over it).
//
// Measured on the device: 8 requests stepping by a token 3.1 us, 256 requests
// with 40 prompts 8.4 us, 2,000 requests with 600 prompts (156,200 rows of slots)
// 14.2 us a plan: launch, three passes over the lengths, two scans, one read of a
// block, the barrier.
#include "sa_device.cuh"

namespace sa {
namespace {

constexpr int kPlanMaxRequests = 8192;
constexpr int kPlanArrays = 5;  // of one int a request in shared memory
constexpr int kFew = 4;         // new tokens that a request's own thread writes
constexpr int kChunk = 128;     // new tokens that a warp writes at a time otherwise
// The largest cluster. 2,000 requests, 156,200 rows of slots: 14.2 us a plan with 16 CTAs, 18.9 with 8, 42 with
// 2, 71 with one.
constexpr int kPlanCluster = 16;

struct PlanParams {
  const int32_t* add;
  int32_t* seq_lens;
  int32_t* table;
  int32_t* free_list;
  int32_t* free_top;
  int32_t* slots;
  int32_t* positions;  // nullable
  int32_t* cu_tokens;  // nullable
  uint32_t* status;
  int requests, table_blocks, pool_blocks, max_tokens;
};

__device__ __forceinline__ int cluster_ctas() {
  int n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}

// Execution and memory barrier of the cluster (the grid is one cluster).
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Sums are capped at 2^31 - 1 (a cap commutes with sums of what is not
// negative), so that 32 bits hold them whatever the lengths.
constexpr uint32_t kCap = 0x7fffffffu;
__device__ __forceinline__ uint32_t add_capped(uint32_t a, uint32_t b) { return min(a + b, kCap); }

// Exclusive capped sums of N values over the block's threads; totals get the
// block's. narrow: over each warp's lanes alone (the warps hold the same values).
template <int N>
__device__ __forceinline__ void scan(const uint32_t (&value)[N], uint32_t (&before)[N],
                                     uint32_t (&totals)[N], uint32_t (*scratch)[32], bool narrow) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t sum = value[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t n = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum = add_capped(sum, n);
    }
    before[i] = __shfl_up_sync(0xffffffffu, sum, 1);
    if (lane == 0) before[i] = 0;
    totals[i] = __shfl_sync(0xffffffffu, sum, 31);
  }
  if (narrow) return;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane == 0) scratch[i][warp] = totals[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {  // every warp sums the warps' totals for itself
    uint32_t sum = lane < warps ? scratch[i][lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t n = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum = add_capped(sum, n);
    }
    totals[i] = __shfl_sync(0xffffffffu, sum, 31);
    const uint32_t mine = __shfl_sync(0xffffffffu, sum, max(warp - 1, 0));
    if (warp > 0) before[i] = add_capped(before[i], mine);
  }
}

// The last index in [0, n) whose start is not above `at` (starts[0] is 0).
__device__ __forceinline__ int owner_of(const int32_t* starts, int n, int at) {
  int low = 0, high = n;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (starts[mid] <= at)
      low = mid;
    else
      high = mid;
  }
  return low;
}

__device__ __forceinline__ int blocks_of(int tokens) {
  return static_cast<int>((static_cast<long long>(tokens) + kBlockTokens - 1) / kBlockTokens);
}

// Slot and position of a request's k-th new token, row i: its block is in the
// table if the request held it, else in the list. `len`: the length before, bit
// 31 set when the request is refused; `take`: its first block in taking order.
__device__ __forceinline__ void write_token(const PlanParams& p, int i, int k, int len, int take,
                                            int b, int top) {
  const int before = len & 0x7fffffff;
  const int position =
      static_cast<int>(min(static_cast<long long>(before) + k, 0x7fffffffll));  // far only when refused
  int slot = -1;
  if (len >= 0) {
    const int at = position / kBlockTokens, held = blocks_of(before);
    const int block = at < held ? p.table[static_cast<int64_t>(b) * p.table_blocks + at]
                                : p.free_list[top - 1 - (take + at - held)];
    if (block >= 0 && block < p.pool_blocks)
      slot = block * kBlockTokens + position % kBlockTokens;
    else
      raise_status(p.status, SA_DEV_BAD_BLOCK);
  }
  p.slots[i] = slot;
  if (p.positions) p.positions[i] = position;
}

// What a step wants of a request whose new tokens start at row tok_at.
struct Request {
  int before, grow, held, want;  // length before, new tokens, blocks before and after
  int rows;                      // new tokens inside the slot map
  bool broken, full, over;
  __device__ __forceinline__ bool refused() const { return broken || full || over; }
  __device__ __forceinline__ bool few() const { return grow <= kFew; }
};
__device__ __forceinline__ Request request_of(const PlanParams& p, int b, uint32_t tok_at) {
  const long long limit = static_cast<long long>(p.table_blocks) * kBlockTokens;
  const int before = p.seq_lens[b], add = p.add[b];
  Request r;
  r.broken = before < 0 || before > limit;
  r.before = r.broken ? 0 : before;
  const long long after = max(0ll, static_cast<long long>(r.before) + add);
  r.grow = max(add, 0);
  r.full = !r.broken && after > limit;
  const uint32_t room = max(p.max_tokens - static_cast<int>(tok_at), 0);
  // only what grows needs rows: requests that end or shrink behind a prompt too
  // long for the slot map give their blocks back all the same
  r.over = r.grow > 0 && add_capped(tok_at, r.grow) > static_cast<uint32_t>(p.max_tokens);
  r.rows = static_cast<int>(min(static_cast<uint32_t>(r.grow), room));
  r.held = blocks_of(r.before);
  r.want = r.refused() ? r.held : blocks_of(static_cast<int>(after));
  return r;
}

__global__ void __launch_bounds__(1024) plan_kernel(const PlanParams p) {
  extern __shared__ int32_t plan_smem[];
  __shared__ uint32_t scratch[4][32];
  __shared__ int taken_shared;
  const int n = p.requests, rank = blockIdx.x, ctas = cluster_ctas();
  int32_t* tok = plan_smem;       // [n] first row of a request's new tokens
  int32_t* take = tok + n;        // [n] first of its blocks in taking order
  int32_t* give = take + n;       // [n] first of its blocks in giving order
  int32_t* len = give + n;        // [n] its length before, bit 31 set when refused
  int32_t* chunk = len + n;       // [n] first of its chunks of kChunk tokens
  if (threadIdx.x == 0) taken_shared = 0;
  if (n <= 32) __syncthreads();  // before any warp's maximum; for more requests the scans have barriers

  int top = *p.free_top;
  if (top < 0 || top > p.pool_blocks) {
    if (rank == 0 && threadIdx.x == 0) raise_status(p.status, SA_DEV_BAD_BLOCK);
    top = min(max(top, 0), p.pool_blocks);
  }
  // A thread has `each` consecutive requests; up to 32 requests each warp has
  // all of them and scans by itself. Lengths are read again in each pass.
  const bool narrow = n <= 32;
  const int each = narrow ? 1 : (n + blockDim.x - 1) / blockDim.x;
  const int mine = narrow ? threadIdx.x & 31 : threadIdx.x * each;
  const int mine_end = min(mine + each, n);
  const bool speaks = !narrow || threadIdx.x < 32;  // for its requests, in this CTA
  uint32_t grown[1] = {0}, grown_before[1], grown_total[1];
  for (int b = mine; b < mine_end; ++b) grown[0] = add_capped(grown[0], max(p.add[b], 0));
  scan(grown, grown_before, grown_total, scratch, narrow);

  uint32_t moved[3] = {0, 0, 0}, moved_before[3], moved_total[3];  // taken, given back, chunks
  uint32_t tok_at = grown_before[0];
  for (int b = mine; b < mine_end; ++b) {
    const Request r = request_of(p, b, tok_at);
    moved[0] = add_capped(moved[0], max(r.want - r.held, 0));
    moved[1] = add_capped(moved[1], max(r.held - r.want, 0));
    moved[2] += r.few() ? 0 : (r.rows + kChunk - 1) / kChunk;
    tok_at = add_capped(tok_at, r.grow);
  }
  scan(moved, moved_before, moved_total, scratch + 1, narrow);

  tok_at = grown_before[0];
  uint32_t take_at = moved_before[0], give_at = moved_before[1], chunk_at = moved_before[2];
  for (int b = mine; b < mine_end; ++b) {
    const Request r = request_of(p, b, tok_at);
    const uint32_t need = max(r.want - r.held, 0), behind = add_capped(take_at, need);
    const bool short_of = need > 0 && behind > static_cast<uint32_t>(top);
    const bool refused = r.refused() || short_of;
    if (need > 0 && !short_of) atomicMax(&taken_shared, static_cast<int>(behind));
    tok[b] = static_cast<int>(tok_at);
    take[b] = static_cast<int>(take_at);
    give[b] = static_cast<int>(give_at);
    len[b] = r.before | (refused ? static_cast<int>(0x80000000u) : 0);
    chunk[b] = static_cast<int>(chunk_at);
    // requests that grow by a few tokens write them at once, those of 32 in one CTA
    if (r.few() && (b >> 5) % ctas == rank && speaks)
      for (int k = 0; k < r.rows; ++k) write_token(p, tok[b] + k, k, len[b], take[b], b, top);
    if (rank == 0 && speaks) {
      if (r.broken) raise_status(p.status, SA_DEV_BAD_BLOCK);
      if (r.full) raise_status(p.status, SA_DEV_TABLE_FULL);
      if (r.over && !r.broken && !r.full) raise_status(p.status, SA_DEV_SLOTS_FULL);
      if (short_of) raise_status(p.status, SA_DEV_POOL_EMPTY);
    }
    tok_at = add_capped(tok_at, r.grow);
    take_at = behind;
    give_at = add_capped(give_at, max(r.held - r.want, 0));
    chunk_at += r.few() ? 0 : (r.rows + kChunk - 1) / kChunk;
  }
  __syncthreads();
  const int taken = taken_shared;
  const int given = static_cast<int>(moved_total[1]);
  const int tokens = min(static_cast<int>(grown_total[0]), p.max_tokens);
  const int chunks = static_cast<int>(moved_total[2]);
  const int me = rank * blockDim.x + threadIdx.x, all = ctas * blockDim.x;

  for (int a = me; a < taken; a += all) {
    const int b = owner_of(take, n, a);
    const int id = p.free_list[top - 1 - a];
    if (id < 0 || id >= p.pool_blocks) raise_status(p.status, SA_DEV_BAD_BLOCK);
    p.table[static_cast<int64_t>(b) * p.table_blocks + blocks_of(len[b]) + a - take[b]] = id;
  }
  // Tokens of the requests that grow by more than kFew, a warp for each chunk of one.
  const int lane = threadIdx.x & 31;
  for (int c = me >> 5; c < chunks; c += all >> 5) {
    const int b = owner_of(chunk, n, c);
    const int end = min(b + 1 < n ? tok[b + 1] : tokens, tokens);
#pragma unroll
    for (int k = 0; k < kChunk / 32; ++k) {
      const int i = tok[b] + (c - chunk[b]) * kChunk + k * 32 + lane;
      if (i < end) write_token(p, i, i - tok[b], len[b], take[b], b, top);
    }
  }
  for (int i = tokens + me; i < p.max_tokens; i += all) {
    p.slots[i] = -1;
    if (p.positions) p.positions[i] = 0;
  }
  // Every CTA has read the lengths and the list before any of them changes.
  if (ctas > 1)
    cluster_barrier();
  else
    __syncthreads();

  // up to 2^31 - 1 where lengths claim more blocks than the pool has: r + all passes 31 bits
  for (uint32_t r = me; r < static_cast<uint32_t>(given); r += all) {
    const int b = owner_of(give, n, static_cast<int>(r));
    const int before = len[b] & 0x7fffffff;
    const int after = max(before + p.add[b], 0);  // gives back, so add < 0 and not refused
    const int id = p.table[static_cast<int64_t>(b) * p.table_blocks + blocks_of(after) + r - give[b]];
    const long long at = static_cast<long long>(top) - taken + given - 1 - r;
    if (id < 0 || id >= p.pool_blocks || at >= p.pool_blocks)
      raise_status(p.status, SA_DEV_BAD_BLOCK);
    if (at < p.pool_blocks) p.free_list[at] = id;
  }
  if (rank == 0) {
    for (int b = threadIdx.x; b < n; b += blockDim.x) {
      if (len[b] >= 0) p.seq_lens[b] = max(len[b] + p.add[b], 0);
      if (p.cu_tokens) p.cu_tokens[b] = tok[b];
    }
    if (threadIdx.x == 0) {
      if (p.cu_tokens) p.cu_tokens[n] = static_cast<int>(grown_total[0]);
      *p.free_top = static_cast<int>(
          min(static_cast<long long>(top) - taken + given, static_cast<long long>(p.pool_blocks)));
    }
  }
}

int g_plan_smem[kMaxDevices];
// Cluster size for up to kPlanHalf bytes of shared memory a CTA (two may share an SM), and above; 0: not yet asked.
constexpr int kPlanHalf = 100 * 1024, kPlanMost = kPlanMaxRequests * kPlanArrays * (int)sizeof(int32_t);
int g_plan_cluster[kMaxDevices][2];

int plan_device() {
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess && device >= 0 && device < kMaxDevices ? device : 0;
}

cudaLaunchConfig_t plan_config(cudaLaunchAttribute* attr, int ctas, int threads, int bytes) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = ctas;
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  return cfg;
}

// CTAs of a large step: the largest cluster that the current device can place (one on a share of a GPU
// without so many SMs side by side). The kernel takes any size.
sa_status plan_cluster(int bytes, int* ctas) {
  const int wide = bytes > kPlanHalf;
  int& known = g_plan_cluster[plan_device()][wide];
  if (known == 0) {
    SA_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(plan_kernel),
                                     cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    int size = kPlanCluster;
    for (; size > 1; size /= 2) {
      cudaLaunchAttribute attr;
      const cudaLaunchConfig_t cfg = plan_config(&attr, size, 1024, wide ? kPlanMost : kPlanHalf);
      int active = 0;
      if (cudaOccupancyMaxActiveClusters(&active, plan_kernel, &cfg) == cudaSuccess && active > 0) break;
      cudaGetLastError();  // a size that cannot be asked for is one that does not fit
    }
    known = size;
  }
  *ctas = known;
  return SA_OK;
}

}  // namespace
}  // namespace sa

using namespace sa;

extern "C" SA_API sa_status sa_plan_blocks(const int32_t* add, size_t requests, int32_t* seq_lens,
                                           int32_t* block_table, size_t table_blocks,
                                           int32_t* free_list, size_t pool_blocks,
                                           int32_t* free_top, size_t max_tokens,
                                           int32_t* slots_out, int32_t* positions_out,
                                           int32_t* cu_tokens_out, uint32_t* status,
                                           void* stream) {
  if (!add || !seq_lens || !block_table || !free_list || !free_top || (!slots_out && max_tokens))
    return fail(SA_ERR_INVALID_ARG, "plan: null pointer");
  if (requests == 0 || table_blocks == 0 || pool_blocks == 0)
    return fail(SA_ERR_INVALID_ARG, "plan: no requests, table or pool");
  if (requests > (size_t)kPlanMaxRequests)
    return fail(SA_ERR_UNSUPPORTED, "plan: more than 8192 requests");
  // slots are 32-bit, and the sums of a step stay below 2^31
  const size_t most = 0x7fffffffu / kBlockTokens;
  if (pool_blocks > most || table_blocks > most || max_tokens > 0x7fffffffu - (1u << 20) ||
      requests * table_blocks > 0x7fffffffu)
    return fail(SA_ERR_UNSUPPORTED, "plan: pool, table or slot map above 2^31 entries");
  PlanParams p{add,       seq_lens,  block_table,   free_list, free_top,
               slots_out, positions_out, cu_tokens_out, status,    (int)requests,
               (int)table_blocks, (int)pool_blocks, (int)max_tokens};
  // One CTA up to 4096 tokens and 1024 requests, else one cluster.
  const bool small = max_tokens <= 4096 && requests <= 1024;
  const int threads = small && requests <= 256 && max_tokens <= 1024 ? 256 : 1024;
  const int bytes = (int)requests * kPlanArrays * (int)sizeof(int32_t);
  const sa_status st =
      ensure_smem_limit(reinterpret_cast<const void*>(plan_kernel), kPlanMost, g_plan_smem);
  if (st != SA_OK) return st;
  int ctas = 1;
  if (!small) {
    const sa_status placed = plan_cluster(bytes, &ctas);
    if (placed != SA_OK) return placed;
  }
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = plan_config(&attr, ctas, threads, bytes);
  cfg.stream = static_cast<cudaStream_t>(stream);
  return cuda_status(cudaLaunchKernelEx(&cfg, plan_kernel, p), "plan launch");
}
