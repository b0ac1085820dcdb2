// Attention of a batch that shares a prefix: the work list, its cut into equal
// shares, and the partial results, shared by the tensor-core kernel, the FP32
// kernel and the merge.
//
// Per new token (query) i of request b, KV head h and query head hq = h G + g:
//     o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j)
// over the prefix_len positions of the shared prefix and the positions
// j <= len_b - n_b + i of the request's own blocks (n_b new tokens, the last of
// its len_b).  Softmax splits over disjoint key sets: with m the running
// maximum of a set (in units of log2), l = sum 2^(s - m) and o unnormalised,
// sets join as m* = max m, l* = sum l 2^(m - m*), o* = sum o 2^(m - m*).
//
// Items.  A prefix item is MR rows of ALL queries of one KV head (row = token
// * G + g over the whole batch) against the whole prefix, so a prefix key is
// read once for MR queries and not once per request.  An own item is MR rows
// of one request and KV head (row = (token - first) * G + g) against that
// request's positions, up to the last one its rows see.  An item's cost is
// c0 + w * (number of KT-key tiles).
//
// Shares.  All items in a fixed order make one line of cost U; CTA c of n
// takes [U c / n, U (c + 1) / n) and computes the tiles that begin there: any
// mixture of lengths loads all SMs alike, and a long request is split over
// many CTAs without a plan made on the host.  The part of an item that holds
// its first tile writes to the row's own place (prefix or own); a later part
// is the first work of its CTA, so one continuation buffer per CTA is enough.
// The row records where its continuations lie: CTAs first + 1 .. first + n.
#pragma once

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
  int fill_tail;           // tokens behind the last request: 1 = write 0 / -inf, 0 = leave
  // partial results
  float* part_o[2];        // [n_tokens * H * G, dv]: prefix, own
  float2* part_ml[2];      // (m, l)
  int2* part_next[2];      // (row in the continuation buffer, continuations)
  float* cont_o;           // [grid, MR, dv]
  float2* cont_ml;         // [grid, MR]
};

__device__ __forceinline__ int attn_tokens(const AttnArgs& a) { return min(max(a.cu[a.B], 0), a.n_tokens); }
__device__ __forceinline__ int attn_prefix_len(const AttnArgs& a) {
  const int64_t most = (int64_t)a.prefix_width * a.L;
  return (int)min((int64_t)max(a.prefix_len ? a.prefix_len[0] : 0, 0), most);
}

struct AttnRequest {
  int tok0, n;   // first token, tokens
  int len;       // own positions
};
__device__ __forceinline__ AttnRequest attn_request(const AttnArgs& a, int b) {
  AttnRequest r;
  r.tok0 = min(max(a.cu[b], 0), a.n_tokens);
  r.n = min(max(a.cu[b + 1], r.tok0), a.n_tokens) - r.tok0;
  r.len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.width * a.L);
  return r;
}

// One CTA's part of an item.
struct AttnPart {
  int own;        // 0: prefix, 1: a request's own positions
  int b, h;
  int tok0;       // first token of the item's row group
  int row0, rows; // rows [row0, row0 + rows) of the group
  int len;        // keys: positions [0, len)
  int see0;       // row r sees positions < min(len, see0 + r / G + 1) (own items)
  int t0, t1;     // tiles of this part
  int first;      // holds the item's first tile: writes the row's own place
  int n_cont;     // continuations of the item (first part only), in CTAs cta + 1 ..
};

template <int MR_, int KT_, int C0_, int W1_, int W2_, int ROWS1_>
struct AttnCost {
  static constexpr int MR = MR_, KT = KT_;
  // an item's fixed cost, and a tile's for items of up to ROWS1 rows and of more
  static constexpr int C0 = C0_, W1 = W1_, W2 = W2_, ROWS1 = ROWS1_;
  static constexpr int WMAX = W1 > W2 ? W1 : W2;
  __device__ static __forceinline__ int weight(int rows) { return rows <= ROWS1 ? W1 : W2; }
};

// Walks a CTA's share.  init() is called by every thread of the CTA; next() by
// any set of threads, each for itself (the state is per thread).
template <class C>
struct AttnWalk {
  int64_t U, u0, u1;           // whole cost, this CTA's share
  int n_cta;
  int prefix_len, prefix_rows, prefix_mt, prefix_nt;
  int64_t prefix_cost;         // one prefix item
  // current item
  int own, b, h, m;
  int64_t at;                  // cost position where the current item begins
  AttnRequest req;

  __device__ static __forceinline__ int tiles(int len) { return max(1, (len + C::KT - 1) / C::KT); }
  __device__ static __forceinline__ int row_tiles(int rows) { return (rows + C::MR - 1) / C::MR; }
  // positions that rows [row0, row0 + rows) of a request see between them
  __device__ static __forceinline__ int see(const AttnRequest& r, int last_row, int G) {
    return min(r.len, max(0, r.len - r.n + last_row / G + 1));
  }
  __device__ static __forceinline__ int64_t own_item_cost(const AttnRequest& r, int m, int G) {
    const int all = r.n * G, rows = min(C::MR, all - m * C::MR);
    return C::C0 + (int64_t)C::weight(rows) * tiles(see(r, m * C::MR + rows - 1, G));
  }
  __device__ static __forceinline__ int64_t head_cost(const AttnRequest& r, int G) {
    int64_t c = 0;
    const int mt = row_tiles(r.n * G);
    for (int m = 0; m < mt; ++m) c += own_item_cost(r, m, G);
    return c;
  }

  // Shares over at most `grid` CTAs, none smaller than the costliest tile plus
  // an item's fixed cost.
  __device__ void init(const AttnArgs& a, int grid, int cta) {
    __shared__ int64_t s_sum[32];
    __shared__ int s_b;
    __shared__ int64_t s_at;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_warps = (blockDim.x + 31) >> 5;
    prefix_len = attn_prefix_len(a);
    prefix_rows = prefix_len > 0 ? attn_tokens(a) * a.G : 0;
    prefix_mt = row_tiles(prefix_rows);
    prefix_nt = tiles(prefix_len);
    prefix_cost = C::C0 + (int64_t)C::weight(prefix_rows) * prefix_nt;
    const int64_t prefix_all = prefix_cost * prefix_mt * a.H;
    // thread t owns requests [t * per, (t + 1) * per)
    const int per = (a.B + blockDim.x - 1) / blockDim.x;
    const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    int64_t sum = 0;
    for (int i = b0; i < b1; ++i) sum += head_cost(attn_request(a, i), a.G) * a.H;
    int64_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) s_sum[warp] = inc;
    if (tid == 0) s_b = a.B;
    __syncthreads();
    int64_t before = prefix_all + inc - sum;
    U = prefix_all;
    for (int w = 0; w < n_warps; ++w) {
      if (w < warp) before += s_sum[w];
      U += s_sum[w];
    }
    const int64_t most = U / (C::C0 + C::WMAX);
    n_cta = (int)max((int64_t)1, min((int64_t)grid, most));
    u0 = cta < n_cta ? U * cta / n_cta : U;
    u1 = cta < n_cta ? U * (cta + 1) / n_cta : U;
    if (u0 >= prefix_all && before <= u0 && u0 < before + sum) {
      int64_t p = before;
      int i = b0;
      for (; i < b1; ++i) {
        const int64_t c = head_cost(attn_request(a, i), a.G) * a.H;
        if (u0 < p + c) break;
        p += c;
      }
      s_b = i;
      s_at = p;
    }
    __syncthreads();
    own = u0 >= prefix_all;
    m = h = b = 0;
    at = 0;
    if (u0 >= U) {  // nothing for this CTA
      own = 1;
      b = a.B;
      at = U;
    } else if (!own) {
      const int64_t i = u0 / prefix_cost;
      h = (int)(i / prefix_mt);
      m = (int)(i - (int64_t)h * prefix_mt);
      at = i * prefix_cost;
    } else {
      b = s_b;
      at = s_at;
      req = attn_request(a, b);
      const int64_t hc = head_cost(req, a.G);
      h = (int)((u0 - at) / hc);
      at += hc * h;
      for (;;) {
        const int64_t c = own_item_cost(req, m, a.G);
        if (u0 < at + c) break;
        at += c;
        ++m;
      }
    }
  }

  // CTA whose share holds cost position p
  __device__ __forceinline__ int cta_of(int64_t p) const { return (int)(((p + 1) * n_cta - 1) / U); }

  // The next part with at least one tile; false at the end of the share.
  __device__ bool next(const AttnArgs& a, AttnPart& it) {
    for (;;) {
      if (at >= u1 || (own && b >= a.B)) return false;
      int rows, nt;
      int64_t cost;
      it.own = own;
      it.h = h;
      if (!own) {
        rows = min(C::MR, prefix_rows - m * C::MR);
        nt = prefix_nt;
        cost = prefix_cost;
        it.b = -1;
        it.tok0 = 0;
        it.len = prefix_len;
        it.see0 = 0;
      } else {
        rows = min(C::MR, req.n * a.G - m * C::MR);
        const int last = see(req, m * C::MR + rows - 1, a.G);
        nt = tiles(last);
        cost = C::C0 + (int64_t)C::weight(rows) * nt;
        it.b = b;
        it.tok0 = req.tok0;
        it.len = last;
        it.see0 = req.len - req.n;
      }
      it.row0 = m * C::MR;
      it.rows = rows;
      // tile j begins at cost position at + C0 + j * w
      const int w = C::weight(own ? rows : prefix_rows);
      const int64_t base = at + C::C0;
      auto tile_from = [&](int64_t u) -> int {
        return u <= base ? 0 : (int)min((int64_t)nt, (u - base + w - 1) / w);
      };
      it.t0 = tile_from(u0);
      it.t1 = tile_from(u1);
      it.first = it.t0 == 0;
      it.n_cont = 0;
      if (it.first && it.t1 < nt) it.n_cont = cta_of(base + (int64_t)(nt - 1) * w) - cta_of(base);
      // step to the next item
      at += cost;
      ++m;
      if (!own) {
        if (m == prefix_mt) {
          m = 0;
          if (++h == a.H) {
            h = 0;
            own = 1;
            b = -1;
            advance_request(a);
          }
        }
      } else if (m * C::MR >= req.n * a.G) {
        m = 0;
        if (++h == a.H) {
          h = 0;
          advance_request(a);
        }
      }
      if (it.t1 > it.t0) return true;
    }
  }

  __device__ __forceinline__ void advance_request(const AttnArgs& a) {
    do {
      if (++b >= a.B) return;
      req = attn_request(a, b);
    } while (req.n == 0);
  }
};

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

// device kernels' launchers (each returns a status)
constexpr int kAttnMaxGrid = 320;      // continuation buffers
constexpr int kAttnFmaRows = 32;       // MR of the FP32 kernel
constexpr int kAttnTcRows = 256;       // MR of the tensor-core kernel
int launch_prefix_attention_fma(const AttnArgs& a, int dtype, int sms, cudaStream_t stream);

}  // namespace gfst
