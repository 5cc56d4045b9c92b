// What surrounds the attention in a speculative decoding step and would
// otherwise be host work or dozens of small launches: the step's block tables
// and slots (from the requests' lengths, with a free list on the device), the
// accepted path of each drafted tree, and the move of the accepted slots to
// consecutive positions.  Whole numbers and bytes only; all three are bound by
// latency (a few dependent reads) at a decode step's sizes.  Kernel times on one
// MI355X: tables of 64 requests with a tree of 8 nodes, pages taken and given back,
// 8.4 us; of nine prompts with up to 4096 tokens 5.1 and 5.5 us (pages, then tokens);
// a call from Python takes 12-19 us of host time, which covers them.
#include "ftq_device.h"
#include "ftq_internal.h"

#include <algorithm>

namespace ftq {
namespace {

constexpr int STEP_BATCH = 4096;   // requests of a call: their counts are held in LDS
constexpr int STEP_FUSED = 4096;   // tokens that the allocating workgroup maps itself

struct StepArgs {
  const int32_t *qsl, *past, *depths;
  int32_t* bt;
  int64_t bt_row;
  int B, max_blocks, bs;
  int64_t tokens;
  int32_t *have, *free, *count;      // null without a free list
  int pool;                          // entries of the free list
  int64_t *slots, *pos;
  int32_t *req, *lens, *missing;
};

// largest i in [lo, hi) with at[i] <= x, given at[lo] <= x; at ascends
template <typename P>
__device__ __forceinline__ int find_below(const P at, int lo, int hi, int x) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// token t's request (qsl: starts, in LDS), slot and position
__device__ __forceinline__ void step_token(const StepArgs& a, const int* qsl, int64_t t) {
  int64_t slot = -1, pos = 0;
  int b = -1;
  if (t >= qsl[0] && t < qsl[a.B]) {
    b = find_below(qsl, 0, a.B, (int)t);
    const int i = (int)t - qsl[b], past = max(a.past[b], 0);
    const int64_t at = (int64_t)past + i, page = at / a.bs;
    const int limit = a.have != nullptr ? a.have[b] : a.max_blocks;
    const int id = page < limit ? a.bt[b * a.bt_row + page] : -1;
    if (id >= 0) slot = (int64_t)id * a.bs + (at - page * a.bs);
    pos = past + (int64_t)(a.depths != nullptr ? a.depths[t] : i);
  }
  a.slots[t] = slot;
  a.pos[t] = pos;
  a.req[t] = b;
}

// of a request; past 2^31 - 1: that
__device__ __forceinline__ int step_len(const StepArgs& a, int i) {
  const int64_t n = (int64_t)a.qsl[i + 1] - a.qsl[i], len = (int64_t)max(a.past[i], 0) + (n > 0 ? n : 0);
  return (int)(len < 0x7fffffff ? len : 0x7fffffff);
}

// Without a free list: a workgroup per 1024 tokens.
__global__ __launch_bounds__(256) void step_map_kernel(const StepArgs a) {
  extern __shared__ int starts[];
  for (int i = threadIdx.x; i <= a.B; i += 256) starts[i] = a.qsl[i];
  if (a.have == nullptr && blockIdx.x == 0) {
    for (int i = threadIdx.x; i < a.B; i += 256) a.lens[i] = step_len(a, i);
    if (threadIdx.x == 0) *a.missing = 0;
  }
  __syncthreads();
  for (int k = 0; k < 4; ++k) {
    const int64_t t = (int64_t)blockIdx.x * 1024 + 256 * k + threadIdx.x;
    if (t < a.tokens) step_token(a, starts, t);
  }
}

// Block tables brought to the requests' lengths.  With have and want the pages a
// request holds and needs, released pages (want <= page < have) go on top of the
// free list in the order of the requests and pages, and the new ones (have <= page
// < want) come from its top in that order: new page k is entry avail - 1 - k of
// the old list followed by the released pages.  Both orders are prefix sums over
// the requests, so every page is found by two binary searches and no order of
// execution matters.  One workgroup: nothing that it overwrites is read by another.
// map: also the tokens.
__global__ __launch_bounds__(1024) void step_alloc_kernel(const StepArgs a, int map) {
  extern __shared__ int lds[];
  int *relp = lds, *newp = relp + a.B + 1, *want = newp + a.B + 1, *starts = want + a.B;
  __shared__ int wsum[3][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int PER = STEP_BATCH / 1024;
  int rel[PER], fresh[PER], have[PER];
  int sr = 0, sn = 0, sx = 0;  // released, new, pages past the table's width
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = tid * PER + k;
    rel[k] = fresh[k] = have[k] = 0;
    if (i < a.B) {
      const int len = step_len(a, i), need = (int)(((int64_t)len + a.bs - 1) / a.bs), w = min(need, a.max_blocks);
      have[k] = min(max(a.have[i], 0), a.max_blocks);
      rel[k] = max(have[k] - w, 0);
      fresh[k] = max(w - have[k], 0);
      want[i] = w;
      a.lens[i] = len;
      sx += need - w;
    }
    sr += rel[k];
    sn += fresh[k];
  }
  const int count = min(max(*a.count, 0), a.pool);
  // inclusive sums over the lanes, then the waves
  int ir = sr, in = sn;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int pr = __shfl_up(ir, m), pn = __shfl_up(in, m);
    if (lane >= m) {
      ir += pr;
      in += pn;
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sx += __shfl_xor(sx, m);
  if (lane == 63) {
    wsum[0][wave] = ir;
    wsum[1][wave] = in;
    wsum[2][wave] = sx;
  }
  if (map)
    for (int i = tid; i <= a.B; i += 1024) starts[i] = a.qsl[i];
  __syncthreads();
  int br = ir - sr, bn = in - sn, R = 0, N = 0, X = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    if (w < wave) {
      br += wsum[0][w];
      bn += wsum[1][w];
    }
    R += wsum[0][w];
    N += wsum[1][w];
    X += wsum[2][w];
  }
  const int avail = count + R, given = min(N, avail);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = tid * PER + k;
    if (i <= a.B) {
      relp[i] = br;
      newp[i] = bn;
    }
    if (i < a.B) a.have[i] = have[k] - rel[k] + min(max(given - bn, 0), fresh[k]);
    br += rel[k];
    bn += fresh[k];
  }
  if (tid * PER + PER == a.B) {  // the last thread's requests end the batch
    relp[a.B] = br;
    newp[a.B] = bn;
  }
  __syncthreads();
  // released page r: of request j, page want[j] + (r - relp[j])
  auto released = [&](int r) {
    const int j = find_below(relp, 0, a.B, r);
    return a.bt[j * a.bt_row + want[j] + (r - relp[j])];
  };
  for (int k = tid; k < given; k += 1024) {
    const int i = find_below(newp, 0, a.B, k), s = avail - 1 - k;
    const int id = s < count ? a.free[s] : released(s - count);
    a.bt[i * a.bt_row + want[i] - (newp[i + 1] - newp[i]) + (k - newp[i])] = id;
  }
  // rows that release take nothing, so no released entry is overwritten above;
  // the free list is read below `count` and written from there on
  for (int r = tid; r < avail - given - count; r += 1024)
    if (count + r < a.pool) a.free[count + r] = released(r);
  __syncthreads();  // the tables and counts are complete, and every free entry is read
  if (tid == 0) {
    *a.count = min(avail - given, a.pool);
    *a.missing = X + N - given;
  }
  if (map)
    for (int64_t t = tid; t < a.tokens; t += 1024) step_token(a, starts, t);
}

// One wave per tree: its nodes in LDS, then from the root the lowest child whose
// token is the answer at the current node, 64 nodes at a time.  Latency of the loads
// and of a step per accepted node: 2.3 us for three trees of 8 nodes, 4.7 for 64
// of 61.
__global__ __launch_bounds__(64) void tree_accept_kernel(const int64_t* __restrict__ tokens, const int32_t* __restrict__ parents,
                                                         const int64_t* __restrict__ targets, const int32_t* __restrict__ qsl,
                                                         int64_t num_tokens, int width, int32_t* __restrict__ path,
                                                         int32_t* __restrict__ counts, int64_t* __restrict__ out) {
  extern __shared__ __attribute__((aligned(8))) int64_t nodes[];  // tokens, targets, parents
  const int b = blockIdx.x, lane = threadIdx.x;
  const int64_t q0 = qsl[b];
  const int64_t room = q0 >= 0 ? num_tokens - q0 : 0;
  const int n = (int)max(min(min((int64_t)qsl[b + 1] - q0, room), (int64_t)width), (int64_t)0);
  int64_t *tok = nodes, *ans = nodes + width;
  int32_t* par = reinterpret_cast<int32_t*>(nodes + 2 * (int64_t)width);
  for (int i = lane; i < n; i += 64) {
    tok[i] = tokens[q0 + i];
    ans[i] = targets[q0 + i];
    par[i] = parents[q0 + i];
  }
  __syncthreads();
  int64_t* o = out + (int64_t)b * width;
  int32_t* p = path + (int64_t)b * width;
  int cur = 0, count = 0;
  while (cur < n) {  // cur ascends
    const int64_t want = ans[cur];
    if (lane == 0) {
      p[count] = cur;
      o[count] = want;
    }
    ++count;
    int next = n;
    for (int j0 = cur + 1; j0 < n; j0 += 64) {
      const int j = j0 + lane;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(j < n && par[j] == cur && tok[j] == want);
      if (hit != 0) {
        next = j0 + __builtin_ctzll(hit);
        break;
      }
    }
    cur = next;
  }
  for (int i = count + lane; i < width; i += 64) {
    p[i] = -1;
    o[i] = -1;
  }
  if (lane == 0) counts[b] = count;
}

constexpr int COMMIT_LAYERS = 64;  // caches of a launch

struct CommitArgs {
  uint8_t* cache[COMMIT_LAYERS];
  int64_t nb, sblk, spos, shead;
  int bs, hkv, units;       // units: T-sized pieces of a slot
  const int32_t* bt;
  int64_t bt_row;
  int max_blocks, width;
  const int32_t *past, *path, *counts;
};

// Position past + path[j] to past + j, j = 0, 1, ...: a workgroup takes 256 pieces
// of a sequence's slots in one layer.  The path ascends, so path[j] >= j and no
// piece is overwritten before it is read: a thread moves the same piece of every
// position, and reads a group of four before it writes them (what it writes lies
// at or below what it reads).  All layers in one launch: 3.1 MB moved in 32 layers in
// 7.3 us, most of it the latency of path, table and slot in turn.
template <typename T>
__global__ __launch_bounds__(256) void commit_slots_kernel(const CommitArgs a) {
  constexpr int NP = 256;  // path entries at a time
  __shared__ int64_t src[NP], dst[NP];
  __shared__ int end;
  const int b = blockIdx.y, tid = threadIdx.x, u = blockIdx.x * 256 + tid;
  const int past = max(a.past[b], 0), count = min(max(a.counts[b], 0), a.width);
  const int32_t* path = a.path + (int64_t)b * a.width;
  const bool on = u < a.hkv * a.units;
  const int h = on ? u / a.units : 0;
  T* base = reinterpret_cast<T*>(a.cache[blockIdx.z] + (int64_t)h * a.shead) + (on ? u - h * a.units : 0);
  auto slot = [&](int64_t at) -> int64_t {  // byte offset of a position, or -1
    const int64_t page = at / a.bs;
    const int id = page < a.max_blocks ? a.bt[b * a.bt_row + page] : -1;
    return id >= 0 && id < a.nb ? id * a.sblk + (at - page * a.bs) * a.spos : -1;
  };
  for (int j0 = 0; j0 < count; j0 += NP) {
    __syncthreads();
    if (tid == 0) end = min(count - j0, NP);
    __syncthreads();
    const int j = j0 + tid;
    if (j < count) {
      const int at = path[j];
      // an entry that does not ascend ends the path
      if (at < 0 || (j > 0 && at <= path[j - 1])) atomicMin(&end, tid);
      const int64_t s = at > j ? slot((int64_t)past + at) : -1, d = at > j ? slot((int64_t)past + j) : -1;
      src[tid] = d >= 0 ? s : -1;
      dst[tid] = d;
    }
    __syncthreads();
    const int n = end;
    if (on) {
      for (int k = 0; k < n; k += 4) {
        T x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (k + i < n && src[k + i] >= 0) x[i] = *reinterpret_cast<const T*>(reinterpret_cast<const uint8_t*>(base) + src[k + i]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (k + i < n && src[k + i] >= 0) *reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(base) + dst[k + i]) = x[i];
      }
    }
    if (n < min(count - j0, NP)) break;  // uniform
  }
}

}  // namespace
}  // namespace ftq

using namespace ftq;

extern "C" int ftq_step_tables(const int32_t* query_start_loc, const int32_t* past_lens, const int32_t* depths, int batch,
                               int64_t num_tokens, int32_t* block_table, int64_t table_stride, int max_blocks, int block_size,
                               int32_t* num_blocks_held, int32_t* free_blocks, int32_t* free_count, int pool_size,
                               int64_t* slot_mapping, int64_t* positions, int32_t* token_request, int32_t* seq_lens,
                               int32_t* missing, void* stream) {
  FTQ_REQUIRE(batch >= 0 && batch <= STEP_BATCH, "step tables: at most 4096 requests");
  FTQ_REQUIRE(num_tokens >= 0 && num_tokens <= INT32_MAX - 1024, "step tables: bad token count");
  FTQ_REQUIRE(block_size >= 1 && max_blocks >= 0 && table_stride >= max_blocks && pool_size >= 0, "step tables: bad sizes");
  const bool alloc = num_blocks_held != nullptr || free_blocks != nullptr || free_count != nullptr;
  FTQ_REQUIRE(!alloc || ((num_blocks_held || batch == 0) && free_count && (free_blocks || pool_size == 0)),
              "step tables: num_blocks, free_blocks and free_count go together");
  FTQ_REQUIRE(!alloc || (int64_t)batch * max_blocks <= INT32_MAX - pool_size, "step tables: too many table entries");
  FTQ_REQUIRE(missing && query_start_loc, "null pointer argument");
  FTQ_REQUIRE(batch == 0 || (past_lens && seq_lens && (block_table || max_blocks == 0)), "null pointer argument");
  FTQ_REQUIRE(num_tokens == 0 || (slot_mapping && positions && token_request), "null pointer argument");
  StepArgs a{query_start_loc, past_lens, depths, block_table, table_stride, batch, max_blocks, block_size, num_tokens,
             num_blocks_held, free_blocks, free_count, pool_size, slot_mapping, positions, token_request, seq_lens, missing};
  hipStream_t st = (hipStream_t)stream;
  if (alloc) {
    const bool map = num_tokens <= STEP_FUSED;
    const size_t lds = ((size_t)3 * batch + 2 + (map ? batch + 1 : 0)) * 4;
    step_alloc_kernel<<<dim3(1), dim3(1024), lds, st>>>(a, map);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || map) return hip_status(e);
  }
  step_map_kernel<<<dim3((unsigned)std::max<int64_t>((num_tokens + 1023) / 1024, 1)), dim3(256), ((size_t)batch + 1) * 4, st>>>(a);
  return hip_status(hipGetLastError());
}

extern "C" int ftq_tree_accept(const int64_t* tokens, const int32_t* parents, const int64_t* targets,
                               const int32_t* query_start_loc, int batch, int64_t num_tokens, int max_nodes, int32_t* path,
                               int32_t* counts, int64_t* accepted, void* stream) {
  FTQ_REQUIRE(batch >= 0 && num_tokens >= 0, "tree accept: bad counts");
  FTQ_REQUIRE(max_nodes >= 1 && max_nodes <= 2048, "tree accept: max_nodes must be in [1, 2048]");
  if (batch == 0) return FTQ_OK;
  FTQ_REQUIRE(query_start_loc && path && counts && accepted && (num_tokens == 0 || (tokens && parents && targets)),
              "null pointer argument");
  tree_accept_kernel<<<dim3((unsigned)batch), dim3(64), (size_t)max_nodes * 20, (hipStream_t)stream>>>(
      tokens, parents, targets, query_start_loc, num_tokens, max_nodes, path, counts, accepted);
  return hip_status(hipGetLastError());
}

extern "C" int ftq_commit_slots(uint8_t* const* kv_caches, int num_caches, int64_t num_blocks, int block_size,
                                int64_t stride_block, int64_t stride_pos, int64_t stride_head, int num_kv_heads,
                                int slot_bytes, const int32_t* block_table, int64_t table_stride, int max_blocks,
                                const int32_t* past_lens, const int32_t* path, const int32_t* counts, int max_nodes,
                                int batch, void* stream) {
  FTQ_REQUIRE(num_caches >= 0 && batch >= 0 && batch <= 65535 && max_nodes >= 0 && block_size >= 1 && max_blocks >= 0 &&
                  table_stride >= max_blocks && slot_bytes > 0 && num_kv_heads > 0,
              "commit slots: bad counts (at most 65535 sequences)");
  FTQ_REQUIRE(stride_head >= slot_bytes && cache_strides_ok(num_blocks, stride_block, stride_pos, stride_head, num_kv_heads, block_size),
              "kv_cache strides must describe [num_blocks][block_size][num_kv_heads][slot]");
  FTQ_REQUIRE(((stride_block | stride_pos | stride_head | slot_bytes) & 3) == 0, "kv_cache strides must be multiples of 4 bytes");
  if (num_caches == 0 || batch == 0 || max_nodes == 0 || num_blocks == 0 || max_blocks == 0) return FTQ_OK;
  FTQ_REQUIRE(kv_caches && block_table && past_lens && path && counts, "null pointer argument");
  bool wide = ((stride_block | stride_pos | stride_head | slot_bytes) & 15) == 0;
  for (int i = 0; i < num_caches; ++i) {
    FTQ_REQUIRE(kv_caches[i] != nullptr && aligned4(kv_caches[i]), "kv_cache must be 4-byte aligned");
    wide = wide && aligned16(kv_caches[i]);
  }
  const int64_t units = slot_bytes / (wide ? 16 : 4);
  FTQ_REQUIRE(units * num_kv_heads <= INT32_MAX - 256, "commit slots: slot too large");
  for (int at = 0; at < num_caches; at += COMMIT_LAYERS) {
    CommitArgs a{};
    const int n = std::min(num_caches - at, COMMIT_LAYERS);
    for (int i = 0; i < n; ++i) a.cache[i] = kv_caches[at + i];
    a.nb = num_blocks; a.sblk = stride_block; a.spos = stride_pos; a.shead = stride_head;
    a.bs = block_size; a.hkv = num_kv_heads; a.units = (int)units;
    a.bt = block_table; a.bt_row = table_stride; a.max_blocks = max_blocks; a.width = max_nodes;
    a.past = past_lens; a.path = path; a.counts = counts;
    const dim3 grid((unsigned)((units * num_kv_heads + 255) / 256), (unsigned)batch, (unsigned)n);
    if (wide) commit_slots_kernel<uint4><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a);
    else commit_slots_kernel<uint32_t><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_status(e);
  }
  return FTQ_OK;
}
