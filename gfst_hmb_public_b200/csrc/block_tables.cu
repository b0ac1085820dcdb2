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
// the slots, each found by its own arithmetic -- no CTA waits for another.  A
// step in place that wants more blocks than there are, or has more tokens than
// slots to fill, leaves everything as it was (every CTA knows it from the sums), so
// that it can be taken again.
// What bounds it: launch and scan latency for a decode batch (256 requests of up
// to 512 blocks: 5 us); for thousands of requests the table rows written, 4 B per
// entry (4096 x 1024 entries and 0.8 M tokens: 16 us for 25 MB).
#include "gfst_common.cuh"

namespace gfst {
namespace {

constexpr int kMaxRequests = 16384;  // three prefix sums of the step in one CTA's shared memory
constexpr int kTablesMaxThreads = 1024;
constexpr int kTablesStatic = 1024;  // at least the kernel's own shared memory (its warps' sums)

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
  int lane_bits;  // lanes of a table row, as a power of two
  int shift;      // L == 1 << shift, or shift < 0
};

// v / L for v below 2^32
__device__ __forceinline__ uint32_t over_L(const TablesArgs& a, uint32_t v) {
  return a.shift >= 0 ? v >> a.shift : v / (uint32_t)a.L;
}

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
  const int held = (int)over_L(a, (uint32_t)len + (uint32_t)a.L - 1u);  // both below 2^31
  r.held = min(held, a.W);
  const int64_t end = len + r.add + a.L - 1;
  r.want = nw < 0 ? r.held : (end >> 32) == 0 ? (int64_t)over_L(a, (uint32_t)end) : end / a.L;
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
  __shared__ int64_t w_add[33], w_want[33];  // by warp, then exclusive sums and the total
  __shared__ int w_grow[33], w_back[33];
  static_assert(sizeof(w_add) + sizeof(w_want) + sizeof(w_grow) + sizeof(w_back) <= kTablesStatic, "shared memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_warps = blockDim.x >> 5;

  const int head = min(max(a.free_state[0], 0), a.F - 1);
  const int count = min(max(a.free_state[1], 0), a.F);
  // each request's numbers, a request a thread at a time (coalesced) ...
  int64_t want = 0;
#pragma unroll 4
  for (int b = tid; b < a.B; b += blockDim.x) {
    const Need n = need_of(a, b);
    s_cu[b] = (int)n.add;
    s_first[b] = n.need - n.held;
    s_back[b] = n.back;
    want += n.want - n.need;
  }
  __syncthreads();
  // ... and their prefix sums, thread t over requests [t * per, (t + 1) * per)
  // (an odd run: the threads' reads then fall on different banks)
  const int per = ((a.B + blockDim.x - 1) / blockDim.x) | 1;
  const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  int64_t add = 0;
  int grow = 0, back = 0;
  for (int b = b0; b < b1; ++b) {
    add += s_cu[b];
    grow += s_first[b];
    back += s_back[b];
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
  if (warp == 0) {
    const bool in = lane < n_warps;
    const int64_t a0 = in ? w_add[lane] : 0, a1 = in ? w_want[lane] : 0;
    const int a2 = in ? w_grow[lane] : 0, a3 = in ? w_back[lane] : 0;
    const int64_t s0 = warp_inclusive(a0), s1 = warp_inclusive(a1);
    const int s2 = warp_inclusive(a2), s3 = warp_inclusive(a3);
    w_add[lane] = s0 - a0, w_grow[lane] = s2 - a2, w_back[lane] = s3 - a3;
    if (lane == 31) w_add[32] = s0, w_want[32] = s1, w_grow[32] = s2, w_back[32] = s3;
  }
  __syncthreads();
  int64_t x_add = w_add[warp] + i_add - add;
  int x_grow = w_grow[warp] + i_grow - grow, x_back = w_back[warp] + i_back - back;
  const int64_t t_add = w_add[32], t_want = w_want[32];
  const int t_grow = w_grow[32], t_back = w_back[32];
  // packed positions past the int32 range are past every slot map as well
  auto clamp32 = [](int64_t v) { return (int32_t)min(v, (int64_t)0x7fffffff); };
  for (int b = b0; b < b1; ++b) {
    const int na = s_cu[b], ng = s_first[b], nb = s_back[b];
    s_cu[b] = clamp32(x_add);
    s_first[b] = x_grow;
    s_back[b] = x_back;
    x_add += na;
    x_grow += ng;
    x_back += nb;
  }
  if (tid == 0) s_cu[a.B] = clamp32(t_add);
  __syncthreads();

  const int taken = min(t_grow, count);
  const bool in_place = a.tables == a.tables_out;
  // in place, tokens that the slot map has no room for are lacking as well: they
  // would count as held and never be written
  const int64_t unheld = in_place ? max(t_add - a.n_tokens, (int64_t)0) : 0;
  const int32_t lacking = clamp32((int64_t)(t_grow - taken) + t_want + unheld);
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  const int64_t first = (int64_t)blockIdx.x * blockDim.x + tid;

  if (lacking > 0 && in_place) {
    // a step in place that cannot be had: lengths, tables and ring stay, no token has a slot
    if (blockIdx.x == 0) {
      for (int b = tid; b <= a.B; b += blockDim.x) a.cu_new[b] = 0;
      for (int b = tid; b < a.B; b += blockDim.x) a.lens_out[b] = a.lens[b];
      if (tid == 0) {
        a.free_state_out[0] = a.free_state[0];
        a.free_state_out[1] = a.free_state[1];
        a.n_short[0] = lacking;
      }
    }
    for (int64_t i = first; i < a.n_tokens; i += stride) a.slot_map[i] = -1;
    return;
  }

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
      a.n_short[0] = lacking;
    }
  }

  // ring position of `head + offset`, offset below F (and F below 2^31)
  auto ring_at = [&](int offset) -> uint32_t {
    const uint32_t at = (uint32_t)head + (uint32_t)offset;
    return at >= (uint32_t)a.F ? at - (uint32_t)a.F : at;
  };
  // the entry of block j >= held of request b, j < W
  auto fresh = [&](int b, int j, int held) -> int32_t {
    const int rank = s_first[b] + j - held;
    return rank < count ? a.free_ring[ring_at(rank)] : -1;
  };
  // slot of position p of request b (held blocks); positions lie below 2^32
  auto slot_of = [&](int b, int held, uint32_t p) -> int32_t {
    const uint32_t j = over_L(a, p);
    if (j >= (uint32_t)a.W) return -1;
    const int32_t blk = (int)j < held ? a.tables[(int64_t)b * a.W + j] : fresh(b, (int)j, held);
    return blk >= 0 && blk < a.F ? (int32_t)((uint32_t)blk * (uint32_t)a.L + (p - j * (uint32_t)a.L)) : -1;
  };

  // Table rows: a group of lanes a row (a power of two near the width, so that
  // short rows leave few lanes idle), four entries a lane in flight.
  const int lanes = 1 << a.lane_bits;
  const int64_t groups = ((int64_t)gridDim.x * blockDim.x) >> a.lane_bits;
  const int gl = tid & (lanes - 1);
  for (int64_t b = ((int64_t)blockIdx.x * blockDim.x + tid) >> a.lane_bits; b < a.B; b += groups) {
    const Need n = need_of(a, (int)b);
    const int32_t* row = a.tables + b * a.W;
    int32_t* out = a.tables_out + b * a.W;
    for (int j0 = gl; j0 < a.W; j0 += 4 * lanes) {
      int32_t v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u * lanes;
        v[u] = -1;
        if (j >= a.W) continue;
        if (j < n.held) v[u] = row[j];
        else if (j < n.need) v[u] = fresh((int)b, j, n.held);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u * lanes;
        if (j >= a.W) continue;
        if (n.back > 0) {
          if (j < n.held) {
            const int64_t rank = (int64_t)count + s_back[b] + j;
            // returned entries past the ring's room (a block listed twice) are dropped
            if (rank < a.F) a.free_ring[ring_at((int)rank)] = v[u];
          }
          v[u] = -1;
        }
        out[j] = v[u];
      }
    }
  }

  // Slots: four tokens in a row a thread (one while there are threads enough), the
  // last CTAs first, which have the fewest rows.  The first token's request, the
  // last whose first packed position is not behind it (idle requests share theirs
  // with the next), is found by bisection in shared memory; the others follow it.
  const int total = (int)min((int64_t)s_cu[a.B], a.n_tokens);
  int step0 = 1;
  while (step0 * 2 < a.B) step0 *= 2;
  const int run = a.n_tokens > stride ? 4 : 1;
  const bool vec = run == 4 && (reinterpret_cast<uintptr_t>(a.slot_map) & 15) == 0;
#pragma unroll 1
  for (int64_t i0 = (stride - 1 - first) * run; i0 < a.n_tokens; i0 += stride * run) {
    int32_t slot[4] = {-1, -1, -1, -1};
    int b = 0, held = 0, end = -1;  // request, its blocks, where its tokens end
    uint32_t p = 0;
    if (i0 < total) {
#pragma unroll 1
      for (int step = step0; step > 0; step >>= 1) {
        const int x = b + step;
        if (x < a.B && s_cu[x] <= (int)i0) b = x;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = (int)i0 + u;
        if (i >= total || u >= run) break;
        if (u == 0 || i >= end) {
          if (u > 0) {
            do ++b;
            while (s_cu[b + 1] <= i);
          }
          end = s_cu[b + 1];
          held = need_of(a, b).held;
          p = (uint32_t)max(a.lens[b], 0) + (uint32_t)(i - s_cu[b]);
          slot[u] = slot_of(b, held, p);
        } else {
          ++p;
          const bool same = a.shift >= 0 ? (p & (uint32_t)(a.L - 1)) != 0 : p % (uint32_t)a.L != 0;
          slot[u] = same ? (slot[u - 1] < 0 ? -1 : slot[u - 1] + 1) : slot_of(b, held, p);
        }
      }
    }
    if (vec && i0 + 4 <= a.n_tokens) {
      *reinterpret_cast<int4*>(a.slot_map + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (u < run && i0 + u < a.n_tokens) a.slot_map[i0 + u] = slot[u];
    }
  }
}

// A token's keys and values are H (kv + vv) 16-byte vectors.  A thread keeps its
// vector (head and piece) and walks tokens, so the only division left is the
// slot's block (a shift where L is a power of two); kAppendIlp tokens are in
// flight at once.  A copy: the bytes of K and V read and written bound it (65,000
// tokens of 8 heads of 128, 533 MB: 87.5 us, 6.1 TB/s).
constexpr int kAppendIlp = 4;
constexpr int kAppendThreads = 256;

struct AppendArgs {
  const uint4* K;
  const uint4* V;
  int64_t k_st, k_sh, v_st, v_sh;  // strides in vectors
  uint4* pool_K;
  uint4* pool_V;
  const int32_t* slot_map;
  int64_t n_tokens, n_slots;
  int L, shift;       // L == 1 << shift, or shift < 0
  int H, kv, vv;      // vectors of a key and of a value row
  int per, abreast;   // vectors of a token; tokens side by side in a CTA
};

__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs a) {
  const int side = a.abreast > 1 ? (int)threadIdx.x / a.per : 0;
  const int64_t t0 = (int64_t)blockIdx.x * (a.abreast * kAppendIlp) + side;
  for (int x = a.abreast > 1 ? (int)threadIdx.x - side * a.per : (int)threadIdx.x; x < a.per && side < a.abreast;
       x += a.abreast > 1 ? a.per : kAppendThreads) {
    const bool is_v = x >= a.H * a.kv;
    const int y = is_v ? x - a.H * a.kv : x, row = is_v ? a.vv : a.kv;
    const int h = y / row, v = y - h * row;
    const uint4* src = is_v ? a.V + h * a.v_sh + v : a.K + h * a.k_sh + v;
    const int64_t st = is_v ? a.v_st : a.k_st;
    uint4* pool = (is_v ? a.pool_V : a.pool_K) + (int64_t)h * a.L * row + v;
    const int64_t block = (int64_t)a.H * a.L * row;
    int slot[kAppendIlp];
    uint4 d[kAppendIlp];
#pragma unroll
    for (int u = 0; u < kAppendIlp; ++u) {
      const int64_t t = t0 + u * a.abreast;
      slot[u] = t < a.n_tokens ? a.slot_map[t] : -1;
    }
#pragma unroll
    for (int u = 0; u < kAppendIlp; ++u) {
      if (slot[u] >= a.n_slots) slot[u] = -1;
      if (slot[u] >= 0) d[u] = __ldg(src + (t0 + u * a.abreast) * st);
    }
#pragma unroll
    for (int u = 0; u < kAppendIlp; ++u) {
      if (slot[u] < 0) continue;
      const int blk = a.shift >= 0 ? slot[u] >> a.shift : (int)((uint32_t)slot[u] / (uint32_t)a.L);
      pool[blk * block + (int64_t)(slot[u] - blk * a.L) * row] = d[u];
    }
  }
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
  int lane_bits = 0;
  while (lane_bits < 5 && (4 << lane_bits) < width) ++lane_bits;
  const TablesArgs a{lens,     new_lens, tables,         free_ring, free_state, tables_out, lens_out, cu_new,
                     slot_map, free_state_out, n_short, n_requests, width, L, (int)n_blocks, n_tokens, lane_bits,
                     (L & (L - 1)) == 0 ? ilog2(L) : -1};
  const int threads = n_requests <= 1024 ? 256 : kTablesMaxThreads;
  const int64_t work = (int64_t)n_requests * width + n_tokens;
  // four elements per thread before a CTA more; every CTA repeats the scan, so one wave
  const int64_t want = (work + 4 * threads - 1) / (4 * threads);
  const int64_t wave = (int64_t)sms * (threads < kTablesMaxThreads ? 2 : 1);
  const int grid = (int)(want < wave ? want : wave);
  const size_t smem = ((size_t)3 * n_requests + 1) * 4;
  if (smem + kTablesStatic > 48 * 1024) {  // without leave, a launch has 48 KB of both together
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
  GFST_REQUIRE((int64_t)n_heads * (d + dv) < (1LL << 30), GFST_ERR_SHAPE, "rows of %d heads are too long", n_heads);
  AppendArgs a;
  a.K = static_cast<const uint4*>(K), a.V = static_cast<const uint4*>(V);
  a.k_st = k_stride_t / pv, a.k_sh = k_stride_h / pv, a.v_st = v_stride_t / pv, a.v_sh = v_stride_h / pv;
  a.pool_K = static_cast<uint4*>(pool_K), a.pool_V = static_cast<uint4*>(pool_V);
  a.slot_map = slot_map, a.n_tokens = n_tokens, a.n_slots = n_blocks * L;
  a.L = L, a.shift = (L & (L - 1)) == 0 ? ilog2(L) : -1;
  a.H = n_heads, a.kv = d / pv, a.vv = dv / pv;
  a.per = n_heads * (a.kv + a.vv);
  a.abreast = a.per < kAppendThreads ? kAppendThreads / a.per : 1;
  const int64_t grid = (n_tokens + a.abreast * kAppendIlp - 1) / (a.abreast * kAppendIlp);
  paged_append_kernel<<<(unsigned)grid, kAppendThreads, 0, stream>>>(a);
  return check_launch("paged_append_kernel");
}
