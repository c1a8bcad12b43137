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
// single CTA for small steps, one cluster of 8 for large ones (the scans are
// repeated in each CTA, the writes are split; a cluster barrier orders the
// blocks taken before the table is read).
#include "sa_device.cuh"

namespace sa {
namespace {

constexpr int kPlanMaxRequests = 8192;
constexpr int kPlanCluster = 8;

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

// Exclusive sum over the block's threads; *total gets the block's sum.
__device__ __forceinline__ long long scan64(long long value, long long* scratch,
                                            long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long inclusive = value;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, inclusive, o);
    if (lane >= o) inclusive += n;
  }
  if (lane == 31) scratch[warp] = inclusive;
  __syncthreads();
  if (warp == 0) {
    long long w = lane < warps ? scratch[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long n = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += n;
    }
    scratch[lane] = w;
  }
  __syncthreads();
  const long long before = (warp > 0 ? scratch[warp - 1] : 0) + inclusive - value;
  *total = scratch[warps - 1];
  __syncthreads();
  return before;
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

__global__ void __launch_bounds__(1024) plan_kernel(const PlanParams p) {
  extern __shared__ int32_t plan_smem[];
  __shared__ long long scratch[32];
  __shared__ int taken_shared;
  const int n = p.requests, rank = blockIdx.x, ctas = cluster_ctas();
  int32_t* tok = plan_smem;       // [n] first row of a request's new tokens
  int32_t* take = tok + n;        // [n] first of its blocks in taking order
  int32_t* give = take + n;       // [n] first of its blocks in giving order
  int32_t* len = give + n;        // [n] its length before, bit 31 set when refused
  if (threadIdx.x == 0) taken_shared = 0;

  int top = *p.free_top;
  if (top < 0 || top > p.pool_blocks) {
    if (rank == 0 && threadIdx.x == 0) raise_status(p.status, SA_DEV_BAD_BLOCK);
    top = min(max(top, 0), p.pool_blocks);
  }
  long long tok_base = 0, take_base = 0, give_base = 0;
  const long long limit = static_cast<long long>(p.table_blocks) * kBlockTokens;
  for (int first = 0; first < n; first += blockDim.x) {
    const int b = first + threadIdx.x;
    const bool live = b < n;
    const int before = live ? p.seq_lens[b] : 0;
    const int add = live ? p.add[b] : 0;
    const bool broken = before < 0 || before > limit;
    const long long after = broken ? 0 : max(0ll, static_cast<long long>(before) + add);
    const long long grow = max(add, 0);
    long long total;
    const long long tok_at = tok_base + scan64(grow, scratch, &total);
    tok_base += total;
    const bool full = !broken && after > limit;
    const bool over = tok_at + grow > p.max_tokens;
    bool refused = broken || full || over;
    const int held = broken ? 0 : blocks_of(before);
    const int want = refused ? held : blocks_of(static_cast<int>(after));
    const int need = max(want - held, 0);
    const long long take_at = take_base + scan64(need, scratch, &total);
    take_base += total;
    const bool short_of = need > 0 && take_at + need > top;
    refused |= short_of;
    if (need > 0 && !short_of) atomicMax(&taken_shared, static_cast<int>(take_at + need));
    const long long give_at = give_base + scan64(max(held - want, 0), scratch, &total);
    give_base += total;
    if (live) {
      tok[b] = static_cast<int>(min(tok_at, 0x7fffffffll));
      take[b] = static_cast<int>(min(take_at, 0x7fffffffll));
      give[b] = static_cast<int>(give_at);
      len[b] = (broken ? 0 : before) | (refused ? static_cast<int>(0x80000000u) : 0);
      if (rank == 0) {
        if (broken) raise_status(p.status, SA_DEV_BAD_BLOCK);
        if (full) raise_status(p.status, SA_DEV_TABLE_FULL);
        if (over && !broken && !full) raise_status(p.status, SA_DEV_SLOTS_FULL);
        if (short_of) raise_status(p.status, SA_DEV_POOL_EMPTY);
      }
    }
  }
  __syncthreads();
  const int taken = taken_shared;
  const int given = static_cast<int>(min(give_base, static_cast<long long>(0x7fffffff)));
  const int tokens = static_cast<int>(min(tok_base, static_cast<long long>(p.max_tokens)));
  const int me = rank * blockDim.x + threadIdx.x, all = ctas * blockDim.x;

  for (int a = me; a < taken; a += all) {
    const int b = owner_of(take, n, a);
    const int id = p.free_list[top - 1 - a];
    if (id < 0 || id >= p.pool_blocks) raise_status(p.status, SA_DEV_BAD_BLOCK);
    p.table[static_cast<int64_t>(b) * p.table_blocks + blocks_of(len[b]) + a - take[b]] = id;
  }
  // Taken blocks are in the table, and every CTA has read the lengths and the
  // list, before any of them changes.
  if (ctas > 1)
    cluster_barrier();
  else
    __syncthreads();

  for (int i = me; i < p.max_tokens; i += all) {
    int slot = -1, position = 0;
    if (i < tokens) {
      const int b = owner_of(tok, n, i);
      const int before = len[b];
      position = static_cast<int>(
          min((before & 0x7fffffffll) + (i - tok[b]), 0x7fffffffll));  // far only when refused
      if (before >= 0) {
        const int id = p.table[static_cast<int64_t>(b) * p.table_blocks + position / kBlockTokens];
        if (id >= 0 && id < p.pool_blocks)
          slot = id * kBlockTokens + position % kBlockTokens;
        else
          raise_status(p.status, SA_DEV_BAD_BLOCK);
      }
    }
    p.slots[i] = slot;
    if (p.positions) p.positions[i] = position;
  }
  for (int r = me; r < given; r += all) {
    const int b = owner_of(give, n, r);
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
      if (p.cu_tokens) p.cu_tokens[n] = static_cast<int>(min(tok_base, 0x7fffffffll));
      *p.free_top = static_cast<int>(
          min(static_cast<long long>(top) - taken + given, static_cast<long long>(p.pool_blocks)));
    }
  }
}

int g_plan_smem[kMaxDevices];

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
  // One CTA up to 4096 tokens and 1024 requests, else a cluster of 8.
  const bool small = max_tokens <= 4096 && requests <= 1024;
  const int threads = small && requests <= 256 && max_tokens <= 1024 ? 256 : 1024;
  const int bytes = (int)requests * 4 * (int)sizeof(int32_t);
  const sa_status st =
      ensure_smem_limit(reinterpret_cast<const void*>(plan_kernel),
                        kPlanMaxRequests * 4 * (int)sizeof(int32_t), g_plan_smem);
  if (st != SA_OK) return st;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(small ? 1 : kPlanCluster);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cfg.gridDim.x;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = small ? 0 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, plan_kernel, p), "plan launch");
}
