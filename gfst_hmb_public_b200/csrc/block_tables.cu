// Block tables of the paged memory, and the write of new tokens to their slots.
//
// Requests of ragged lengths share one pool of n_blocks blocks of L tokens.
// Request b holds ceil(len_b / L) blocks, listed in its table row; the free
// blocks are a ring (free_ring, with head and count in free_state): a step
// takes blocks at the head in request order and puts the blocks of ended
// requests behind the tail, so nothing the step reads from the ring is
// overwritten by it (head + count + returned <= head + n_blocks).
//
//   held_b = min(ceil(len_b / L), W)      need_b = min(ceil((len_b + new_b) / L), W)
//   rank of request b's j-th new block = sum_{a < b} (need_a - held_a) + j
//   new token i of request b (packed position cu_b + i) has position
//   p = len_b + i and slot  block(p / L) * L + p % L
//
// Every output is a function of three exclusive prefix sums over the requests
// (new tokens, blocks taken, blocks returned).  One launch: every CTA computes
// the sums itself (the lengths stay in L2 and a scan of 4096 requests is four
// loads and one block scan), then fills its share of the table entries and of
// the slots, each found by its own arithmetic -- no CTA waits for another.
// What bounds it: launch and scan latency for a decode batch; for thousands
// of requests the table rows written, 4 B per entry.
#include "gfst_common.cuh"

namespace gfst {
namespace {

constexpr int kMaxRequests = 16384;  // three prefix sums of the step in one CTA's shared memory
constexpr int kTablesMaxThreads = 1024;

struct TablesArgs {
  const int32_t* lens;
  const int32_t* new_lens;
  const int32_t* tables;  // may be tables_out
  int32_t* free_ring;
  const int32_t* free_state;
  int32_t* tables_out;
  int32_t* lens_out;
  int32_t* cu_new;
  int32_t* slot_map;
  int32_t* free_state_out;
  int32_t* n_short;
  int B, W, L, F;
  int64_t n_tokens;
};

struct Need {
  int64_t add;   // new tokens
  int held, need, back;
  int64_t want;  // blocks asked for, beyond the table's width too
};

__device__ __forceinline__ Need need_of(const TablesArgs& a, int b) {
  Need r;
  const int64_t len = max(a.lens[b], 0);
  const int nw = a.new_lens[b];
  r.add = nw > 0 ? nw : 0;
  const int64_t held = (len + a.L - 1) / a.L;
  r.held = (int)min(held, (int64_t)a.W);
  r.want = nw < 0 ? r.held : (len + r.add + a.L - 1) / a.L;
  r.need = nw < 0 ? r.held : (int)min(r.want, (int64_t)a.W);
  r.back = nw < 0 ? r.held : 0;
  return r;
}

template <typename T>
__device__ __forceinline__ T warp_inclusive(T v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

__global__ void __launch_bounds__(kTablesMaxThreads) block_tables_kernel(const TablesArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* s_cu = sm;               // [B + 1] first packed position of each request
  int32_t* s_first = sm + a.B + 1;  // [B] rank of its first new block
  int32_t* s_back = s_first + a.B;  // [B] rank of its first returned block
  __shared__ int64_t w_add[32], w_want[32];
  __shared__ int w_grow[32], w_back[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_warps = blockDim.x >> 5;

  // thread t owns requests [t * per, (t + 1) * per)
  const int per = (a.B + blockDim.x - 1) / blockDim.x;
  const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  int64_t add = 0, want = 0;
  int grow = 0, back = 0;
  for (int b = b0; b < b1; ++b) {
    const Need n = need_of(a, b);
    add += n.add;
    grow += n.need - n.held;
    back += n.back;
    want += n.want - n.need;
  }
  const int64_t i_add = warp_inclusive(add), i_want = warp_inclusive(want);
  const int i_grow = warp_inclusive(grow), i_back = warp_inclusive(back);
  if (lane == 31) {
    w_add[warp] = i_add;
    w_want[warp] = i_want;
    w_grow[warp] = i_grow;
    w_back[warp] = i_back;
  }
  __syncthreads();
  int64_t x_add = i_add - add, t_add = 0, t_want = 0;
  int x_grow = i_grow - grow, x_back = i_back - back, t_grow = 0, t_back = 0;
  for (int w = 0; w < n_warps; ++w) {
    if (w < warp) {
      x_add += w_add[w];
      x_grow += w_grow[w];
      x_back += w_back[w];
    }
    t_add += w_add[w];
    t_want += w_want[w];
    t_grow += w_grow[w];
    t_back += w_back[w];
  }
  // packed positions past the int32 range are past every slot map as well
  auto clamp32 = [](int64_t v) { return (int32_t)min(v, (int64_t)0x7fffffff); };
  for (int b = b0; b < b1; ++b) {
    const Need n = need_of(a, b);
    s_cu[b] = clamp32(x_add);
    s_first[b] = x_grow;
    s_back[b] = x_back;
    x_add += n.add;
    x_grow += n.need - n.held;
    x_back += n.back;
  }
  if (tid == 0) s_cu[a.B] = clamp32(t_add);
  __syncthreads();

  const int head = min(max(a.free_state[0], 0), a.F - 1);
  const int count = min(max(a.free_state[1], 0), a.F);
  const int taken = min(t_grow, count);
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  const int64_t first = (int64_t)blockIdx.x * blockDim.x + tid;

  if (blockIdx.x == 0) {
    for (int b = tid; b <= a.B; b += blockDim.x) a.cu_new[b] = s_cu[b];
    for (int b = tid; b < a.B; b += blockDim.x) {
      const int nw = a.new_lens[b];
      a.lens_out[b] = nw < 0 ? 0 : clamp32((int64_t)max(a.lens[b], 0) + nw);
    }
    if (tid == 0) {
      a.free_state_out[0] = (int)(((int64_t)head + taken) % a.F);
      // a table that lists more blocks than the ring has room for overflows no count
      a.free_state_out[1] = (int)min((int64_t)a.F, (int64_t)count - taken + t_back);
      a.n_short[0] = clamp32((int64_t)(t_grow - taken) + t_want);
    }
  }

  // the entry of block j >= held of request b
  auto fresh = [&](int b, int j, int held) -> int32_t {
    const int64_t rank = (int64_t)s_first[b] + j - held;
    return rank < count ? a.free_ring[(head + rank) % a.F] : -1;
  };

  const int64_t entries = (int64_t)a.B * a.W;
  for (int64_t i = first; i < entries; i += stride) {
    const int b = (int)(i / a.W), j = (int)(i - (int64_t)b * a.W);
    const Need n = need_of(a, b);
    int32_t v = -1;
    if (j < n.held) {
      v = a.tables[i];
      if (n.back > 0) {
        const int64_t rank = (int64_t)count + s_back[b] + j;
        // returned entries past the ring's room (a block listed twice) are dropped
        if (rank < a.F) a.free_ring[(head + rank) % a.F] = v;
        v = -1;
      }
    } else if (j < n.need) {
      v = fresh(b, j, n.held);
    }
    a.tables_out[i] = v;
  }

  const int total = s_cu[a.B];
  for (int64_t i = first; i < a.n_tokens; i += stride) {
    int32_t slot = -1;
    if (i < total) {
      // the last request whose first packed position is <= i (idle requests share it with the next one)
      int lo = 0, hi = a.B;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= i) lo = mid;
        else hi = mid;
      }
      const Need n = need_of(a, lo);
      const int64_t p = (int64_t)max(a.lens[lo], 0) + (i - s_cu[lo]);
      const int64_t j = p / a.L;
      if (j < a.W) {
        const int32_t blk = j < n.held ? a.tables[(int64_t)lo * a.W + j] : fresh(lo, (int)j, n.held);
        if (blk >= 0 && blk < a.F) slot = (int32_t)((int64_t)blk * a.L + (p - j * a.L));
      }
    }
    a.slot_map[i] = slot;
  }
}

// 16-byte vectors of one row group: token t, head h, vector v of the row.  A
// thread moves kAppendIlp vectors with their loads in flight together.
constexpr int kAppendIlp = 4;
constexpr int kAppendThreads = 256;

__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(
    const uint4* __restrict__ K, int64_t k_st, int64_t k_sh, const uint4* __restrict__ V, int64_t v_st, int64_t v_sh,
    uint4* __restrict__ pool_K, uint4* __restrict__ pool_V, const int32_t* __restrict__ slot_map, int64_t n_tokens,
    int64_t n_slots, int L, int H, int kv, int vv, int64_t k_items, int64_t items) {
  const int64_t base = (int64_t)blockIdx.x * (kAppendThreads * kAppendIlp) + threadIdx.x;
  uint4 x[kAppendIlp];
  uint4* dst[kAppendIlp];
#pragma unroll
  for (int u = 0; u < kAppendIlp; ++u) {
    const int64_t i = base + u * kAppendThreads;
    dst[u] = nullptr;
    if (i >= items) continue;
    const bool is_v = i >= k_items;
    const int64_t r = is_v ? i - k_items : i;
    const int vpr = is_v ? vv : kv;
    const int64_t row = r / vpr;
    const int v = (int)(r - row * vpr);
    const int64_t t = row / H;
    const int h = (int)(row - t * H);
    const int64_t slot = slot_map[t];
    if (slot < 0 || slot >= n_slots) continue;
    const int64_t blk = slot / L;
    const int off = (int)(slot - blk * L);
    const uint4* src = is_v ? V + t * v_st + h * v_sh + v : K + t * k_st + h * k_sh + v;
    x[u] = __ldg(src);
    dst[u] = (is_v ? pool_V : pool_K) + ((blk * H + h) * L + off) * vpr + v;
  }
#pragma unroll
  for (int u = 0; u < kAppendIlp; ++u)
    if (dst[u] != nullptr) *dst[u] = x[u];
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return n;
}

}  // namespace
}  // namespace gfst

using namespace gfst;

extern "C" int gfst_block_tables(const int32_t* lens, const int32_t* new_lens, const int32_t* tables,
                                 int32_t* free_ring, const int32_t* free_state, int n_requests, int width, int L,
                                 int64_t n_blocks, int64_t n_tokens, int32_t* tables_out, int32_t* lens_out,
                                 int32_t* cu_new, int32_t* slot_map, int32_t* free_state_out, int32_t* n_short,
                                 cudaStream_t stream) {
  GFST_REQUIRE(n_requests >= 1 && n_requests <= kMaxRequests, GFST_ERR_SHAPE, "n_requests %d outside [1, %d]",
               n_requests, kMaxRequests);
  GFST_REQUIRE(width >= 1 && L >= 1, GFST_ERR_SHAPE, "table width %d and block length %d must be positive", width, L);
  GFST_REQUIRE((int64_t)width * L < (1LL << 31) && (int64_t)n_requests * width < (1LL << 31), GFST_ERR_SHAPE,
               "width %d x L %d or x n_requests %d exceeds the int32 range", width, L, n_requests);
  GFST_REQUIRE(n_blocks >= 1 && n_blocks * L < (1LL << 31), GFST_ERR_SHAPE,
               "pool of %lld blocks of %d tokens exceeds the int32 slot range", (long long)n_blocks, L);
  GFST_REQUIRE(n_tokens >= 0 && n_tokens < (1LL << 31), GFST_ERR_SHAPE, "n_tokens %lld outside [0, 2^31)",
               (long long)n_tokens);
  GFST_REQUIRE(lens && new_lens && tables && free_ring && free_state && tables_out && lens_out && cu_new &&
                   (slot_map || n_tokens == 0) && free_state_out && n_short,
               GFST_ERR_ARG, "null pointer");
  GFST_REQUIRE(lens_out != lens && lens_out != new_lens && free_state_out != free_state, GFST_ERR_ARG,
               "lens_out and free_state_out must not alias the inputs");
  const int sms = sm_count();
  GFST_REQUIRE(sms > 0, GFST_ERR_DEVICE, "no CUDA device");
  const TablesArgs a{lens,     new_lens, tables,         free_ring, free_state, tables_out, lens_out, cu_new,
                     slot_map, free_state_out, n_short, n_requests, width, L, (int)n_blocks, n_tokens};
  const int threads = n_requests <= 1024 ? 256 : kTablesMaxThreads;
  const int64_t work = (int64_t)n_requests * width + n_tokens;
  // four elements per thread before a CTA more; every CTA repeats the scan
  const int64_t want = (work + 4 * threads - 1) / (4 * threads);
  const int grid = (int)(want < 2 * sms ? want : 2 * sms);
  const size_t smem = ((size_t)3 * n_requests + 1) * 4;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(block_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (kMaxRequests * 3 + 1) * 4);
    GFST_REQUIRE(e == cudaSuccess, GFST_ERR_DEVICE, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  }
  block_tables_kernel<<<grid, threads, smem, stream>>>(a);
  return check_launch("block_tables_kernel");
}

extern "C" int gfst_paged_append(const void* K, int64_t k_stride_t, int64_t k_stride_h, const void* V,
                                 int64_t v_stride_t, int64_t v_stride_h, void* pool_K, void* pool_V,
                                 const int32_t* slot_map, int64_t n_tokens, int64_t n_blocks, int L, int n_heads, int d,
                                 int dv, int dtype, cudaStream_t stream) {
  GFST_REQUIRE(dtype == GFST_F32 || dtype == GFST_BF16 || dtype == GFST_F16, GFST_ERR_DTYPE, "dtype %d", dtype);
  const int es = dtype == GFST_F32 ? 4 : 2, pv = 16 / es;
  GFST_REQUIRE(n_tokens >= 0 && n_blocks >= 1 && L >= 1 && n_heads >= 1 && d >= 1 && dv >= 1, GFST_ERR_SHAPE,
               "n_tokens %lld n_blocks %lld L %d heads %d d %d dv %d", (long long)n_tokens, (long long)n_blocks, L,
               n_heads, d, dv);
  GFST_REQUIRE(n_blocks * L < (1LL << 31) && n_tokens < (1LL << 31), GFST_ERR_SHAPE,
               "slots or tokens exceed the int32 range");
  if (n_tokens == 0) return GFST_OK;
  GFST_REQUIRE(K && V && pool_K && pool_V && slot_map, GFST_ERR_ARG, "null pointer");
  GFST_REQUIRE(d % pv == 0 && dv % pv == 0, GFST_ERR_ALIGN, "rows of %d and %d elements are no multiple of 16 bytes", d,
               dv);
  GFST_REQUIRE(aligned16(K) && aligned16(V) && aligned16(pool_K) && aligned16(pool_V) && k_stride_t % pv == 0 &&
                   k_stride_h % pv == 0 && v_stride_t % pv == 0 && v_stride_h % pv == 0,
               GFST_ERR_ALIGN, "K, V and the pools need 16-byte aligned rows");
  const int kv = d / pv, vv = dv / pv;
  const int64_t k_items = n_tokens * n_heads * kv, items = k_items + n_tokens * n_heads * vv;
  const int64_t grid = (items + kAppendThreads * kAppendIlp - 1) / (kAppendThreads * kAppendIlp);
  GFST_REQUIRE(grid < (1LL << 31), GFST_ERR_SHAPE, "too many rows for one launch");
  paged_append_kernel<<<(unsigned)grid, kAppendThreads, 0, stream>>>(
      static_cast<const uint4*>(K), k_stride_t / pv, k_stride_h / pv, static_cast<const uint4*>(V), v_stride_t / pv,
      v_stride_h / pv, static_cast<uint4*>(pool_K), static_cast<uint4*>(pool_V), slot_map, n_tokens, n_blocks * L, L,
      n_heads, kv, vv, k_items, items);
  return check_launch("paged_append_kernel");
}
