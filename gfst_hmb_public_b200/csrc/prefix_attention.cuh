// Attention of a batch that shares a prefix: the work list, its cut into equal
// shares, and the partial results, shared by the tensor-core kernel, the FP32
// kernel and the merge.
//
// Per new token (query) i of request b, KV head h and query head hq = h G + g:
//     o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j)
// over the prefix_len positions of the shared prefix and the positions
// j <= len_b - n_b + i of the request's own blocks (n_b new tokens, the last of
// its len_b).  Softmax splits over disjoint key sets (the online softmax of Milakov
// and Gimelshein, 2018): with m the running maximum of a set (in units of log2), l = sum 2^(s - m) and o unnormalised,
// sets join as m* = max m, l* = sum l 2^(m - m*), o* = sum o 2^(m - m*).
//
// Items.  A prefix item is MR rows of ALL queries of one KV head (row = token
// * G + g over the whole batch) against the whole prefix, so a prefix key is
// read once for MR queries and not once per request.  An own item is MR rows
// of one request and KV head (row = (token - first) * G + g) against that
// request's positions, up to the last one its rows see.  An item's cost is
// c0 + w * (number of KT-key tiles), w by its rows.
//
// Shares.  All items of a cut, in a fixed order, make one line of cost; a
// worker (a CTA, or one of its two streams) takes an interval of it and computes
// the tiles that begin there: any mixture of lengths loads all SMs alike, and a
// long request is split over many workers without a plan made on the host.  The
// part of an item that holds its first tile writes to the row's own place
// (prefix or own); a later part is the first work of its worker, so one
// continuation buffer per worker is enough.  The row records where its
// continuations lie: those of the next workers in order.
//
// Pieces.  A worker hands out its tiles of an item in pieces of at most
// kAttnMostKeys keys; a piece behind the first is joined to what the worker wrote
// before.  The tensor cores cut what they add to a sum off to the sum's last bits:
// with values of one sign, a piece of 65,536 keys comes out 3.1e-4 too small (half
// a step of fp16 is 4.9e-4, of bf16 3.9e-3), one of 1,048,576 keys 5.2e-3 and one
// of 8,388,608 keys 4.0e-2.  It also bounds how long any role waits for another.
#pragma once

#include <atomic>

#include "gfst_common.cuh"

namespace gfst {

struct AttnArgs {
  const void* Q;
  int64_t q_st, q_sh;      // strides of Q in elements (token, head)
  const void* pool_K;
  const void* pool_V;
  int64_t n_blocks;
  int L, H, G, d, dv;
  const int32_t* tables;   // [B, width], rows table_st apart
  int64_t table_st;
  int width;
  const int32_t* lens;     // [B] own positions, the new ones included
  const int32_t* cu;       // [B + 1] first token of each request
  int B;
  int n_tokens;            // rows of Q
  const int32_t* prefix_table;
  int prefix_width;
  const int32_t* prefix_len;  // [1]
  float scale_log2;        // scale * log2(e)
  void* out;
  float* lse;              // or null
  int fill_tail;           // out of tokens behind the last request: 1 = write 0, 0 = leave (lse: -inf)
  // partial results
  float* part_o[2];        // [n_tokens * H * G, dv]: prefix, own
  float2* part_ml[2];      // (m, l)
  int2* part_next[2];      // attn_next()
  float* cont_o;           // [continuation rows, dv]
  float2* cont_ml;         // [continuation rows]
};

__device__ __forceinline__ int attn_tokens(const AttnArgs& a) { return min(max(a.cu[a.B], 0), a.n_tokens); }
__device__ __forceinline__ int attn_prefix_len(const AttnArgs& a) {
  const int64_t most = (int64_t)a.prefix_width * a.L;
  return (int)min((int64_t)max(a.prefix_len ? a.prefix_len[0] : 0, 0), most);
}

struct AttnRequest {
  int tok0, n;   // first token, tokens (those that Q has rows for)
  int len;       // own positions that they see between them: token i sees those < len - n + i + 1
};
__device__ __forceinline__ AttnRequest attn_request(const AttnArgs& a, int b) {
  AttnRequest r;
  r.tok0 = min(max(a.cu[b], 0), a.n_tokens);
  const int end = max(a.cu[b + 1], r.tok0);
  r.n = min(end, a.n_tokens) - r.tok0;
  // Q may have fewer rows than there are new tokens: the positions of those behind
  // them are seen by none
  r.len = max((int)min((int64_t)max(a.lens[b], 0), (int64_t)a.width * a.L) - (end - r.tok0 - r.n), 0);
  return r;
}

// One worker's part of an item.
struct AttnPart {
  uint8_t own;    // 0: prefix, 1: a request's own positions
  uint8_t first;  // holds the item's first tile: writes the row's own place
  uint8_t again;  // a piece behind the first: joined to what is there
  int b, h;
  int tok0;       // first token of the item's row group
  int row0, rows; // rows [row0, row0 + rows) of the group
  int len;        // keys: positions [0, len)
  int see0;       // row r sees positions < min(len, see0 + r / G + 1) (own items)
  int t0, t1;     // tiles of this part (of one piece of it)
  int n_cont;     // continuations of the item (first part only), by workers worker + 1 ..
};

constexpr int kAttnMostKeys = 65536;

// Sets a (written before) and b (computed now) of a row joined: the reference and
// sum of both, and the factors of their values.  Equal references need no
// exponential, and no inf - inf.
struct AttnJoin {
  float2 ml;
  float fa, fb;
  __device__ __forceinline__ AttnJoin(float2 a, float2 b) {
    ml.x = fmaxf(a.x, b.x);
    fa = a.x == ml.x ? 1.f : exp2f(a.x - ml.x);
    fb = b.x == ml.x ? 1.f : exp2f(b.x - ml.x);
    ml.y = fmaf(a.y, fa, b.y * fb);
  }
};

// x / n for x >= 0, n > 0: costs hardly ever leave 32 bits, where a division is a
// fifth as long.
__device__ __forceinline__ int64_t attn_div(int64_t x, int64_t n) {
  return ((x | n) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)n) : x / n;
}

// How a group of R rows is cut into items, and what an item costs: C0 + weight()
// per tile, which is at most W.  MR is the most rows of an item.  (Here items of
// up to four rows weigh 1 where `few` rows have a way of their own, and others
// the more the more rows they have.)
template <int MR_, int KT_, int C0_, int W_>
struct AttnCutAll {
  static constexpr int MR = MR_, KT = KT_, C0 = C0_, W = W_;
  __device__ static __forceinline__ int weight(int rows, int few) {
    return few && rows <= 4 ? 1 : min(W, 2 + rows * W / MR * 3 / 4);
  }
  __device__ static __forceinline__ int count(int R) { return (R + MR - 1) / MR; }
  __device__ static __forceinline__ int row0(int, int m) { return m * MR; }
  __device__ static __forceinline__ int rows(int R, int m) { return min(MR, R - m * MR); }
};
// Items of more than HALF rows, up to two HALF-row tiles that share their keys ...
template <int HALF, int KT_, int C0_, int W_>
struct AttnCutPairs {
  static constexpr int MR = 2 * HALF, KT = KT_, C0 = C0_, W = W_;
  __device__ static __forceinline__ int weight(int, int) { return W; }
  __device__ static __forceinline__ int count(int R) { return R > HALF ? (R - HALF + MR - 1) / MR : 0; }
  __device__ static __forceinline__ int row0(int, int m) { return m * MR; }
  __device__ static __forceinline__ int rows(int R, int m) { return min(MR, R - m * MR); }
};
// ... and what they leave: at most one item of up to HALF rows.
template <int HALF, int KT_, int C0_, int W_>
struct AttnCutRest {
  using Pairs = AttnCutPairs<HALF, KT_, C0_, W_>;
  static constexpr int MR = HALF, KT = KT_, C0 = C0_, W = W_;
  __device__ static __forceinline__ int weight(int, int) { return W; }
  __device__ static __forceinline__ int row0(int R, int) { return Pairs::count(R) * 2 * HALF; }
  __device__ static __forceinline__ int rows(int R, int) { return R - row0(R, 0); }
  __device__ static __forceinline__ int count(int R) { return rows(R, 0) > 0 ? 1 : 0; }
};

// The line of all items of one cut.
template <class C>
struct AttnLine {
  int64_t U, prefix_all, prefix_cost;
  int prefix_len, prefix_rows, prefix_mt, prefix_nt, few;
  // this thread's requests [b0, b1): their cost and the cost before them
  int b0, b1;
  int64_t before, sum;
  // the last of them, and the cost of one of its heads
  AttnRequest last;
  int64_t last_cost;

  __device__ __forceinline__ int prefix_w_rows() const { return min(C::MR, prefix_rows); }
  __device__ static __forceinline__ int tiles(int len) { return max(1, (len + C::KT - 1) / C::KT); }
  // positions that the rows up to `last_row` of a request see between them
  __device__ static __forceinline__ int see(const AttnRequest& r, int last_row, int G) {
    return min(r.len, max(0, r.len - r.n + last_row / G + 1));
  }
  __device__ static __forceinline__ int own_tiles(const AttnRequest& r, int m, int G) {
    const int R = r.n * G;
    return tiles(see(r, C::row0(R, m) + C::rows(R, m) - 1, G));
  }
  // cost of an item of nt tiles and of `rows` rows (the prefix's items all count as their first)
  __device__ __forceinline__ int64_t item_cost(int nt, int rows) const {
    return C::C0 + (int64_t)C::weight(rows, few) * nt;
  }
  __device__ __forceinline__ int64_t own_cost(const AttnRequest& r, int m, int G) const {
    return item_cost(own_tiles(r, m, G), C::rows(r.n * G, m));
  }
  __device__ __forceinline__ int64_t head_cost(const AttnRequest& r, int G) const {
    int64_t c = 0;
    const int mt = C::count(r.n * G);
#pragma unroll 1
    for (int m = 0; m < mt; ++m) c += own_cost(r, m, G);
    return c;
  }
  // attn_lines() in pieces: the prefix's part; one request; the scan over threads
  __device__ __forceinline__ void begin(const AttnArgs& a, int prefix, int tokens) {
    few = a.d <= 128 && a.dv <= 128;
    prefix_len = prefix;
    prefix_rows = prefix > 0 ? tokens * a.G : 0;
    prefix_mt = C::count(prefix_rows);
    prefix_nt = tiles(prefix_len);
    prefix_cost = item_cost(prefix_nt, prefix_w_rows());
    prefix_all = prefix_cost * prefix_mt * a.H;
    sum = 0;
  }
  __device__ __forceinline__ void add(const AttnArgs& a, const AttnRequest& r) {
    last = r;
    last_cost = head_cost(r, a.G);
    sum += last_cost * a.H;
  }
  __device__ __forceinline__ void scan_warp(int64_t* s_sum) {
    const int lane = threadIdx.x & 31;
    int64_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) s_sum[threadIdx.x >> 5] = inc;
    before = prefix_all + inc - sum;
  }
  template <int WARPS>
  __device__ __forceinline__ void scan_block(const int64_t* s_sum) {
    const int warp = threadIdx.x >> 5;
    U = prefix_all;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int64_t v = s_sum[w];
      before += w < warp ? v : 0;
      U += v;
    }
  }
};

// Sums up one or more lines; called by every thread of the CTA (WARPS warps) with
// its own line objects.  One barrier; s_sum (one row a line) may be used again
// after the caller's next one.
template <int WARPS, class... C>
__device__ __forceinline__ void attn_lines(const AttnArgs& a, int64_t (*s_sum)[32], AttnLine<C>&... line) {
  const int prefix = attn_prefix_len(a), tokens = attn_tokens(a);
  (line.begin(a, prefix, tokens), ...);
  const int per = (a.B + WARPS * 32 - 1) / (WARPS * 32);
  const int b0 = min(a.B, (int)threadIdx.x * per), b1 = min(a.B, b0 + per);
  ((line.b0 = b0, line.b1 = b1), ...);
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    const AttnRequest r = attn_request(a, b);
    (line.add(a, r), ...);
  }
  int k = 0;
  (line.scan_warp(s_sum[k++]), ...);
  __syncthreads();
  k = 0;
  (line.template scan_block<WARPS>(s_sum[k++]), ...);
}

// Equal shares of a line over n workers, rounded up: the last ones may be short
// or empty.
struct AttnEven {
  int64_t U, step;
  int n;
  __device__ __forceinline__ void init(int64_t u, int workers) {
    U = u, n = workers;
    step = max(attn_div(u + n - 1, max(n, 1)), (int64_t)1);
  }
  __device__ __forceinline__ int64_t bound(int i) const { return min(U, step * i); }
  __device__ __forceinline__ int worker_of(int64_t u) const { return (int)attn_div(u, step); }
};

// How the two lines are shared: CTAs [0, pairs.n) take pairs and the others of n
// the rest, in the ratio of their costs, so that a pair's rows are split over no
// more CTAs than its cost needs and compute-bound and memory-bound work run side
// by side.  A CTA of the rest is one worker, or two (its streams) if there is
// enough.  There are workers for shares of `least`, an item's fixed cost and one
// tile; the split by cost rounds them down by half at most, which still is more
// than a tile, so every worker between the first and the last of an item holds
// one of its tiles.
struct AttnShares {
  AttnEven pairs, rest;
  int two;

  __device__ __forceinline__ void init(int64_t P, int64_t S, int grid, int least_p, int least_s) {
    const int64_t T = P + S;
    const int least = P > 0 ? max(least_p, least_s) : least_s;
    const int n = T >= (int64_t)grid * least ? grid : max(1, (int)T / least);
    // a CTA more than the ratio's whole part once that would leave the pairs' 15 % behind
    int np = (int)ceilf((float)P * n / (float)max(T, (int64_t)1) - 0.15f);
    np = P == 0 ? 0 : S == 0 ? n : min(max(np, 1), max(n - 1, 1));
    const int ns = S == 0 ? 0 : max(n - np, 1);
    two = S >= (int64_t)ns * (2 * least_s);
    pairs.init(P, np);
    rest.init(S, two ? 2 * ns : ns);
  }
  // worker number of stream j of CTA c among the rest, or -1
  __device__ __forceinline__ int rest_worker(int c, int j) const {
    const int w = two ? 2 * (c - pairs.n) + j : j == 0 ? c - pairs.n : -1;
    return c < pairs.n || w >= rest.n ? -1 : w;
  }
};

// Walks a share [u0, u1) of a line; the state is the calling thread's.
template <class C>
struct AttnWalk {
  static constexpr int kMost = kAttnMostKeys / C::KT;  // tiles of a piece
  int64_t u0, u1, at;
  int64_t cost;  // of the item at `at`, once it has been handed out
  int go_on;     // its tile at which the next piece begins, or -1: it was the last
  int own, b, h, m;
  AttnRequest req;

  // The walk of the share [from, to) into *s (to be read behind a barrier); called
  // by every thread with its line: the one whose requests hold `from`, or thread 0
  // for the prefix and an empty share, knows where it begins.
  __device__ static __forceinline__ void find(const AttnArgs& a, const AttnLine<C>& ln, int64_t from, int64_t to,
                                              AttnWalk* s) {
    const bool none = from >= to, prefix = from < ln.prefix_all;
    if (none || prefix ? threadIdx.x != 0 : from < ln.before || from >= ln.before + ln.sum) return;
    AttnWalk w;
    w.u0 = from;
    w.u1 = to;
    w.own = !prefix;
    w.m = w.h = w.b = 0;
    w.at = 0;
    if (none) {
      w.own = 1;
      w.b = a.B;
      w.at = to;
    } else if (prefix) {
      const int64_t k = attn_div(from, ln.prefix_cost);
      w.h = (int)attn_div(k, ln.prefix_mt);
      w.m = (int)(k - (int64_t)w.h * ln.prefix_mt);
      w.at = k * ln.prefix_cost;
    } else {
      w.at = ln.before;
      w.b = ln.b1 - 1;
      w.req = ln.last;
      int64_t hc = ln.last_cost;
      if (ln.b0 < w.b) {
#pragma unroll 1
        for (w.b = ln.b0;; ++w.b) {
          w.req = attn_request(a, w.b);
          hc = ln.head_cost(w.req, a.G);
          if (from < w.at + hc * a.H) break;
          w.at += hc * a.H;
        }
      }
      w.h = (int)attn_div(from - w.at, hc);
      w.at += hc * w.h;
      const int items = C::count(w.req.n * a.G);
#pragma unroll 1
      for (; w.m + 1 < items; ++w.m) {
        const int64_t c = ln.own_cost(w.req, w.m, a.G);
        if (from < w.at + c) break;
        w.at += c;
      }
    }
    w.cost = -1;
    w.go_on = -1;
    *s = w;
  }

  // to the next item of the line
  __device__ __forceinline__ void step(const AttnArgs& a, const AttnLine<C>& ln) {
    at += cost;
    if (++m < C::count(own ? req.n * a.G : ln.prefix_rows)) return;
    m = 0;
    if (++h < a.H) return;
    h = 0;
    if (!own) {
      own = 1;
      b = -1;
    }
    do {
      if (++b >= a.B) break;
      req = attn_request(a, b);
    } while (C::count(req.n * a.G) == 0);
  }

  // The next part (or piece of one) with at least one tile; false at the end of the share.
  // share_of(p): number of the worker whose share holds position p.
  template <class F>
  __device__ __forceinline__ bool next(const AttnArgs& a, const AttnLine<C>& ln, F&& share_of, AttnPart& it) {
#pragma unroll 1
    for (;;) {
      if (cost >= 0 && go_on < 0) step(a, ln);  // only now: the next request's lengths are not waited for before
      if (at >= u1 || (own && b >= a.B)) return false;
      const int R = own ? req.n * a.G : ln.prefix_rows;
      int nt;
      it.own = (uint8_t)own;
      it.h = h;
      it.row0 = C::row0(R, m);
      it.rows = C::rows(R, m);
      if (!own) {
        nt = ln.prefix_nt;
        it.b = -1;
        it.tok0 = 0;
        it.len = ln.prefix_len;
        it.see0 = 0;
      } else {
        it.b = b;
        it.tok0 = req.tok0;
        it.len = ln.see(req, it.row0 + it.rows - 1, a.G);
        it.see0 = req.len - req.n;
        nt = ln.tiles(it.len);
      }
      // tile j begins at cost position base + j * w
      const int w_rows = own ? it.rows : ln.prefix_w_rows();
      const int w = C::weight(w_rows, ln.few);
      const int64_t base = at + C::C0;
      auto tile_from = [&](int64_t u) -> int {
        return u <= base ? 0 : (int)min((int64_t)nt, (u - base + w - 1) / w);
      };
      it.t0 = tile_from(u0);
      it.t1 = tile_from(u1);
      it.first = it.t0 == 0;
      it.n_cont = 0;
      if (it.first && it.t1 < nt) it.n_cont = share_of(base + (int64_t)(nt - 1) * w) - share_of(base);
      cost = ln.item_cost(nt, w_rows);
      it.again = go_on >= 0;
      if (it.again) it.t0 = go_on;
      go_on = it.t1 - it.t0 > kMost ? it.t0 + kMost : -1;
      if (go_on >= 0) it.t1 = go_on;
      if (it.t1 > it.t0) return true;
    }
  }
};

// part_next of a row: where its continuations begin and how far they lie apart
__device__ __forceinline__ int2 attn_next(int cont_row, int n_cont, int stride) {
  return make_int2(cont_row, n_cont * 512 + stride);
}

// Block holding position p (or -1 where the table names none of the pool's).
__device__ __forceinline__ int attn_block(const AttnArgs& a, const AttnPart& it, int index) {
  const int32_t* t = it.own ? a.tables + (int64_t)it.b * a.table_st : a.prefix_table;
  const int blk = t[index];
  return blk >= 0 && blk < a.n_blocks ? blk : -1;
}

// Query row r of a part: token and head
__device__ __forceinline__ void attn_row(const AttnArgs& a, const AttnPart& it, int r, int& tok, int& hq) {
  const int rg = it.row0 + r;
  const int t = rg / a.G;
  tok = it.tok0 + t;
  hq = it.h * a.G + rg - t * a.G;
}

// Largest dynamic shared memory of a kernel, set once per device.
template <typename K>
int attn_allow_smem(K kern, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return GFST_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  GFST_REQUIRE(e == cudaSuccess, GFST_ERR_DEVICE, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return GFST_OK;
}

// A launch that may begin while the one before it on the stream ends: the
// kernels wait (griddepcontrol.wait) before they touch memory.
template <typename... P, typename... A>
int attn_launch(const char* what, void (*kern)(P...), int64_t grid, int threads, int smem, cudaStream_t stream,
                const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, P(args)...);
  if (e == cudaSuccess) return GFST_OK;
  cudaGetLastError();  // reported here
  set_last_error("%s: %s", what, cudaGetErrorString(e));
  return GFST_ERR_LAUNCH;
}

// the kernels' launchers (each returns a status)
constexpr int kAttnMaxGrid = 160;      // CTAs of a launch (two per SM of the FP32 kernel count as one here)
constexpr int kAttnFmaRows = 64;       // rows of an item of the FP32 kernel
constexpr int kAttnTcHalf = 128;       // rows of a tile of the tensor-core kernel
// continuation rows: 64 for each of 320 CTAs of the FP32 kernel; 256 for a CTA's
// pairs and 128 for each of its two streams of the tensor-core kernel
constexpr int kAttnFmaContRows = 2 * kAttnMaxGrid * kAttnFmaRows;
constexpr int kAttnTcContRows = kAttnMaxGrid * 4 * kAttnTcHalf;
int launch_prefix_attention_fma(const AttnArgs& a, int dtype, int sms, cudaStream_t stream);
bool prefix_attention_tc_takes(const AttnArgs& a, int dtype);
int launch_prefix_attention_tc(const AttnArgs& a, int dtype, int sms, cudaStream_t stream);

}  // namespace gfst
