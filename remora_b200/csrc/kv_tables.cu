// kv_tables.cu -- block tables and slot maps of a paged key-value cache, built
// on the GPU from the requests' lengths (no counterpart in the reference,
// which has no cache; it serves the attention beside it).
//
// One step of a serving loop appends n_r tokens to each request r (or releases
// it).  With bs tokens per block, request r owns ceil(len_r / bs) blocks and
// needs ceil((len_r + n_r) / bs) - ceil(len_r / bs) more.  The free blocks are
// a stack; released blocks are pushed on it in (request, page) order, then the
// needed ones are popped in the same order: the j-th block of the step is
// entry have - 1 - j of the stack, so every token finds its own block from
// three prefix sums (tokens, blocks needed, blocks released) and no block is
// handed out by an atomic whose order could change the result.
//
// The call is latency bound (a few KB per thousand tokens): 4.9 us on the
// device for 8 requests, 9.0 for 256, 14.8 for 128544 tokens.  It is therefore
// one launch of one cluster: every CTA scans the requests by itself (at most
// 8192 lengths), the CTAs meet at a cluster barrier before anything is written,
// and tokens are then spread over all threads, four to each, which find their
// request by binary search in the shared-memory prefix sums.
#include <algorithm>

#include "runtime.cuh"

namespace rb {
namespace kv {

constexpr int kMaxRequests = 8192;

struct TableArgs {
  const int32_t *lens, *fresh;
  int32_t* table;
  int64_t ld_table;
  int32_t *free_blocks, *lens_out, *free_out, *cu, *slots, *positions, *requests, *status;
  const int32_t* free_count;
  int32_t R, max_blocks, num_blocks, bs, max_tokens;
  Divisor by_bs;
  int32_t vectors;  // slots, positions and requests are 16-byte aligned
};

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}

__device__ __forceinline__ int32_t sat32(int64_t v) {
  return v > 0x7fffffffll ? 0x7fffffff : (int32_t)v;
}

// What one request asks for: tokens, blocks needed, blocks released.
struct Ask {
  int64_t tokens, need, back;
  bool bad, append;
  // Refused where the tokens up to its own end are t?  A release has no tokens that could lie past
  // the room for them, and its blocks are pushed whatever the requests in front of it ask for.
  __device__ __forceinline__ bool refused(int64_t t, int32_t max_tokens) const {
    return bad || (append && t > max_tokens);
  }
};

// A block id as it may enter the table or the stack: one outside the cache becomes -1 (`bad`: it
// is to be reported).
__device__ __forceinline__ int32_t checked_id(const TableArgs& a, int32_t id, bool& bad) {
  const bool in = (uint32_t)id < (uint32_t)a.num_blocks;
  bad |= !in;
  return in ? id : -1;
}

// Blocks of n tokens, n in [0, 2^31).
__device__ __forceinline__ int32_t blocks_of(const TableArgs& a, int32_t n) {
  return n > 0 ? a.by_bs.div(n - 1) + 1 : 0;
}

__device__ __forceinline__ Ask ask_of(const TableArgs& a, int32_t len, int32_t n) {
  Ask q{0, 0, 0, false, n >= 0};
  const int64_t room = (int64_t)a.max_blocks * a.bs;  // below 2^31
  const bool held = len >= 0 && len <= room;
  const int32_t own = held ? blocks_of(a, len) : 0;
  if (n >= 0) {
    q.tokens = n;
    q.bad = !held || (int64_t)len + n > room;
    if (!q.bad) q.need = blocks_of(a, len + n) - own;
  } else {
    q.bad = n != REMORA_B200_KV_RELEASE || !held;
    if (!q.bad) q.back = own;
  }
  return q;
}

// Inclusive sum over the lanes of a warp.
__device__ __forceinline__ int64_t warp_scan(int64_t x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// Largest i with prefix[i] <= v, over prefix[0..n] (prefix[0] = 0, v >= 0).
__device__ __forceinline__ int find_le(const int32_t* prefix, int n, int32_t v) {
  int lo = 0, hi = n + 1;  // prefix[lo] <= v < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(1024) k_block_table(const TableArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* cu = sm;                    // [R + 1] tokens before request r
  int32_t* need = cu + a.R + 1;        // [R + 1] blocks needed before request r
  int32_t* back = need + a.R + 1;      // [R + 1] blocks released before request r
  int32_t* len0 = back + a.R + 1;      // [R] length before the step; bit 31: refused
  __shared__ int64_t part[3][32];
  __shared__ int32_t taken;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int nw = nt >> 5;
  if (tid == 0) taken = 0;
  const int32_t count_in = *a.free_count;

  // prefix sums: each thread sums a run of requests, then warps, then the block.  A request
  // whose tokens pass max_tokens is refused and its blocks are not counted, so the tokens are
  // summed first.
  const int c = (a.R + nt - 1) / nt;
  const int r0 = min(tid * c, a.R), r1 = min(r0 + c, a.R);
  const int32_t len_r0 = r0 < r1 ? a.lens[r0] : 0, n_r0 = r0 < r1 ? a.fresh[r0] : 0;
  const Ask ask_r0 = ask_of(a, len_r0, n_r0);
  auto ask = [&](int r) { return r == r0 ? ask_r0 : ask_of(a, a.lens[r], a.fresh[r]); };
  int64_t s0 = 0, s1 = 0, s2 = 0;
  for (int r = r0; r < r1; ++r) s0 += ask(r).tokens;
  const int64_t x0 = warp_scan(s0, lane);
  if (lane == 31) part[0][warp] = x0;
  __syncthreads();
  const int64_t w0 = lane < nw ? part[0][lane] : 0, i0 = warp_scan(w0, lane);
  const int64_t before = __shfl_sync(~0u, i0 - w0, warp) + x0 - s0;
  {
    int64_t t = before;
    for (int r = r0; r < r1; ++r) {
      const Ask q = ask(r);
      t += q.tokens;
      if (t <= a.max_tokens) s1 += q.need;
      s2 += q.back;
    }
  }
  const int64_t x1 = warp_scan(s1, lane), x2 = warp_scan(s2, lane);
  if (lane == 31) { part[1][warp] = x1; part[2][warp] = x2; }
  __syncthreads();
  const int64_t w1 = lane < nw ? part[1][lane] : 0, w2 = lane < nw ? part[2][lane] : 0;
  const int64_t i1 = warp_scan(w1, lane), i2 = warp_scan(w2, lane);
  const int64_t b1 = __shfl_sync(~0u, i1 - w1, warp), b2 = __shfl_sync(~0u, i2 - w2, warp);
  const int64_t all2 = __shfl_sync(~0u, i2, 31);
  const int32_t count0 = min(max(count_in, 0), a.num_blocks);
  const int32_t have = (int32_t)min((int64_t)count0 + all2, (int64_t)a.num_blocks);
  {
    int64_t t = before, p1 = b1 + x1 - s1, p2 = b2 + x2 - s2;
    int32_t top = 0;
    for (int r = r0; r < r1; ++r) {
      const int32_t len = r == r0 ? len_r0 : a.lens[r];
      const Ask q = ask(r);
      cu[r] = sat32(t);
      need[r] = sat32(p1);
      back[r] = sat32(p2);
      t += q.tokens;
      const bool bad = q.refused(t, a.max_tokens);
      if (t <= a.max_tokens) p1 += q.need;
      p2 += q.back;
      const bool dry = !bad && q.need > 0 && p1 > have;
      if (!bad && !dry && q.need > 0) top = (int32_t)p1;
      len0[r] = (len & 0x7fffffff) | (bad || dry ? 0x80000000 : 0);
    }
    if (r1 == a.R) {  // several threads when R is short of the block: the same values
      cu[a.R] = sat32(t);
      need[a.R] = sat32(p1);
      back[a.R] = sat32(p2);
    }
    if (top > 0) atomicMax(&taken, top);
  }
  const uint32_t rank = cluster_rank(), ctas = cluster_size();
  const int me = rank * nt + tid, step = ctas * nt;
  cluster_barrier();  // every CTA has read the lengths and the count: they may be overwritten

  bool bad = count_in != count0 || (int64_t)count0 + all2 > a.num_blocks;

  // push the released blocks
  const int32_t n_back = back[a.R];
  if (n_back > 0) {  // the same in every CTA of the cluster
    const int room = min(n_back, a.num_blocks - count0);
    for (int64_t i = me; i < room; i += step) {
      const int j = (int)i, r = find_le(back, a.R, j);
      a.free_blocks[count0 + j] = checked_id(a, a.table[(int64_t)r * a.ld_table + (j - back[r])], bad);
    }
    cluster_barrier();
  }

  // each token's slot, four neighbours to a thread (mostly of one request and one block); the
  // token that opens a block enters it into the table
  const int32_t total = cu[a.R];
  const int64_t quads = ((int64_t)a.max_tokens + 3) / 4;
  for (int64_t i = me; i < quads; i += step) {
    const int32_t t4 = (int32_t)(4 * i);
    int32_t slot[4], pos[4], req[4];
    int32_t r = t4 < total ? find_le(cu, a.R, t4) : a.R, seen_r = -1, seen_page = -1, id = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t t = (int64_t)t4 + e;
      slot[e] = -1;
      pos[e] = 0;
      req[e] = -1;
      if (t >= min(total, a.max_tokens)) continue;
      while (t >= cu[r + 1]) ++r;
      req[e] = r;
      const int32_t l = len0[r];
      if (l < 0) continue;
      pos[e] = l + (int32_t)(t - cu[r]);
      const int32_t page = a.by_bs.div(pos[e]), off = pos[e] - page * a.bs;
      if (r != seen_r || page != seen_page) {
        const int32_t own = blocks_of(a, l);
        if (page < own) {
          id = checked_id(a, a.table[(int64_t)r * a.ld_table + page], bad);
        } else {
          id = checked_id(a, __ldcg(a.free_blocks + (have - 1 - (need[r] + page - own))), bad);
          if (off == 0) a.table[(int64_t)r * a.ld_table + page] = id;
        }
        seen_r = r;
        seen_page = page;
      }
      if (id >= 0) slot[e] = id * a.bs + off;
    }
    if (a.vectors && t4 + 3 < a.max_tokens) {
      *reinterpret_cast<int4*>(a.slots + t4) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.positions + t4) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(a.requests + t4) = make_int4(req[0], req[1], req[2], req[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((int64_t)t4 + e < a.max_tokens) {
          a.slots[t4 + e] = slot[e];
          a.positions[t4 + e] = pos[e];
          a.requests[t4 + e] = req[e];
        }
    }
  }

  if (bad) atomicExch(&g_device_error, 3);

  for (int r = me; r < a.R; r += step) {
    const int32_t n = a.fresh[r], l = len0[r];
    const bool no = l < 0;
    // a refused request keeps its length, whatever it is
    if (!no) a.lens_out[r] = n >= 0 ? l + n : 0;
    else if (a.lens_out != a.lens) a.lens_out[r] = a.lens[r];
    const bool dry = no && n >= 0 && cu[r + 1] <= a.max_tokens &&
                     !ask_of(a, a.lens[r], n).bad;
    a.status[r] = !no ? 0 : dry ? 1 : 2;
    a.cu[r] = cu[r];
  }
  if (me == 0) {
    a.cu[a.R] = total;
    *a.free_out = have - taken;
  }
}

struct Launch {
  int ctas, threads;
  size_t smem;
};

// A thread for each request or four tokens, in one CTA while 1024 are enough.  (16 CTAs, which
// no cluster is sure to get, took 10.6 us for 128544 tokens where 8 take 14.5 and 4 take 22.)
inline Launch launch_of(int64_t R, int64_t max_tokens) {
  const int64_t wide = std::max<int64_t>(R, (max_tokens + 3) / 4);
  return Launch{wide > 1024 ? 8 : 1,
                (int)std::min<int64_t>(1024, std::max<int64_t>(128, (wide + 31) / 32 * 32)),
                (4 * (size_t)R + 3) * sizeof(int32_t)};
}

}  // namespace kv
}  // namespace rb

extern "C" int remora_b200_kv_block_table(const remora_b200_kv_block_table_args* args,
                                          void* stream) {
  using namespace rb;
  using namespace rb::kv;
  clear_error();
  RB_CHECK_ARG(args, "kv_block_table: args is null");
  const remora_b200_kv_block_table_args& x = *args;
  RB_CHECK_ARG(x.R >= 0 && x.R <= kMaxRequests, "kv_block_table: R must be in [0, %d], got %lld",
               kMaxRequests, (long long)x.R);
  RB_CHECK_ARG(x.max_tokens >= 0 && x.max_tokens < 0x7fffffff,
               "kv_block_table: max_tokens must be in [0, 2^31 - 1)");
  RB_CHECK_ARG(x.block_size >= 1 && x.num_blocks >= 1 && x.num_blocks < 0x7fffffff &&
                   x.block_size <= 0x7fffffff && x.num_blocks <= 0x7fffffff / x.block_size,
               "kv_block_table: num_blocks * block_size must be in [1, 2^31)");
  RB_CHECK_ARG(x.max_blocks >= 1 && x.max_blocks <= 0x7fffffff / x.block_size,
               "kv_block_table: max_blocks * block_size must be in [1, 2^31)");
  RB_CHECK_ARG(x.ld_table >= x.max_blocks, "kv_block_table: ld_table must be at least max_blocks");
  RB_CHECK_ARG(x.free_blocks && x.free_count && x.free_count_out && x.cu_tokens,
               "kv_block_table: null pointer");
  RB_CHECK_ARG(x.R == 0 || (x.lens && x.new_tokens && x.block_table && x.lens_out && x.status),
               "kv_block_table: null pointer");
  RB_CHECK_ARG(x.max_tokens == 0 || (x.slots && x.positions && x.requests),
               "kv_block_table: null pointer");
  RB_CHECK_ARG(aligned4(x.lens, x.new_tokens, x.block_table, x.free_blocks, x.free_count,
                        x.lens_out, x.free_count_out, x.cu_tokens, x.slots, x.positions,
                        x.requests, x.status),
               "kv_block_table: a pointer is not aligned to its elements");
  TableArgs a{x.lens, x.new_tokens, x.block_table, x.ld_table, x.free_blocks, x.lens_out,
              x.free_count_out, x.cu_tokens, x.slots, x.positions, x.requests, x.status,
              x.free_count, (int32_t)x.R, (int32_t)x.max_blocks, (int32_t)x.num_blocks,
              (int32_t)x.block_size, (int32_t)x.max_tokens, Divisor((uint32_t)x.block_size),
              aligned16(x.slots) && aligned16(x.positions) && aligned16(x.requests)};
  const Launch l = launch_of(x.R, x.max_tokens);
  if (l.smem > 48 * 1024)
    RB_CUDA(cudaFuncSetAttribute(k_block_table, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (4 * kMaxRequests + 3) * (int)sizeof(int32_t)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(l.ctas);
  cfg.blockDim = dim3(l.threads);
  cfg.dynamicSmemBytes = l.smem;
  cfg.stream = as_stream(stream);
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)l.ctas, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  RB_CUDA(cudaLaunchKernelEx(&cfg, k_block_table, a));
  return REMORA_B200_OK;
}
