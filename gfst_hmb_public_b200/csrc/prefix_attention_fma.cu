// Shared-prefix attention on the FP32 units: every element type, block length
// and head size (rows a multiple of 16 bytes, up to 256 elements).  It serves
// the 32-bit memory, whose products the tensor cores would round, and the
// shapes the tensor-core kernel does not tile.
//
// One CTA walks its share of the items (prefix_attention.cuh), up to 64 query rows
// against 32-key tiles.  Keys and values arrive by cp.async in the pools' own
// type, the next tile under this one's arithmetic.  Warp w has rows w, w + 8, ..
// to itself: a lane scores up to two of them against four keys (items of up to
// eight rows: one row against one key), eight lanes reduce a row's maximum and sum
// by shuffles, the weights go to the warp's own corner of shared memory, and then
// value rows are added, four of every 32 columns a lane -- no barrier but the
// tile's two.  What bounds it: the latency of shared-memory reads with 16 warps on
// an SM (registers allow no more), 3.4 wavefronts each for 16 or 32 products.
//
// Items of up to four rows (a decode step's) would leave warps idle and wait for
// each tile: they go key by key instead.  Eight lanes have a key, 16 bytes of
// every 128 each; a warp four keys of the 32-key tile.  A lane copies the pieces
// that it reads itself, two tiles ahead, so that it waits for its own copies alone.
// Every group of eight lanes keeps its own maximum, sum and values over its keys
// and all are joined when the part ends, so the loop has no barrier at all.
//
// Measured (device time with the merge), 32-bit, d = 128: 16 one-token requests of
// up to 8000 tokens (8 heads x 4) 113 us, 2.9 TB/s; prompt pieces of 200 to 600
// tokens (4 heads x 2) 497 us, 17 TFLOP/s; d = 64, 64 requests behind 4000 tokens (4
// x 4) 91 us, 12 TFLOP/s.  (The compiler's choice of registers at the cap of 128
// moves these by up to 3 %.)
// Keys read straight into registers: 144 us for the first, 1.3 us less for the
// smallest call.  Without the way of few rows: 216 us for the first; without one
// row a warp, 32 requests of 500 to 3000 tokens with eight query heads a key head:
// 228 us for 110; with two rows a lane where one does, 20 rows over 20,000 keys: 142
// us for 120.
#include <cuda_fp16.h>

#include "prefix_attention.cuh"

namespace gfst {

GFST_DEFINE_ERROR_WORD(g_attn_fma_error, take_attn_fma_error, "attention")

namespace {

// a status recorded as the kernel records it
__global__ void attn_fma_error_kernel(int status) { atomicMax(&g_attn_fma_error, (unsigned)status); }

constexpr int kRows = kAttnFmaRows;   // 64
constexpr int kKeys = 32;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPer = kRows / kWarps;  // rows of a warp
constexpr int kWeightPitch = kKeys + 4;  // floats of a row of weights
// A 32-key tile of 64 rows counts eight of one of up to four rows, an item four
// (queries in, partials out).  12 or 16 for a tile of 64 rows, and costs of 2 to 10
// for an item, were slower over the range (decode 115-135 us for 110, prompt pieces
// 484-514 for 499).
using Cut = AttnCutAll<kRows, kKeys, 4, 8>;

template <typename T>
struct Vec;  // 16 bytes of T as floats
template <>
struct Vec<float> {
  static constexpr int N = 4;
  __device__ static __forceinline__ void get(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static __forceinline__ void get(const uint4& v, float* f) {
    f[0] = bf16_lo(v.x), f[1] = bf16_hi(v.x), f[2] = bf16_lo(v.y), f[3] = bf16_hi(v.y);
    f[4] = bf16_lo(v.z), f[5] = bf16_hi(v.z), f[6] = bf16_lo(v.w), f[7] = bf16_hi(v.w);
  }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  __device__ static __forceinline__ void get(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
};
// Where a row's partial result goes: its own place, or this CTA's continuation
// buffer.  Called by a warp's lanes that hold the row, `write` for one of them,
// which writes (m, l).  A later piece is joined to what is there: the lanes read
// the (m, l) of before, which `write` changes only when all have, and their
// columns' values, which they wrote themselves.
struct FmaPut {
  float* o;
  float keep, f;  // factors of the values there and of the new ones
  __device__ __forceinline__ FmaPut(const AttnArgs& a, const AttnPart& it, int r, float2 ml, bool live, bool write) {
    int tok, hq;
    attn_row(a, it, live ? r : 0, tok, hq);
    const int64_t row = (int64_t)tok * (a.H * a.G) + hq;
    const int64_t crow = (int64_t)blockIdx.x * kRows + r;
    float2* at = it.first ? a.part_ml[it.own] + row : a.cont_ml + crow;
    o = it.first ? a.part_o[it.own] + row * a.dv : a.cont_o + crow * a.dv;
    keep = 0.f, f = 1.f;
    if (it.again) {
      if (live) {
        const AttnJoin j(*at, ml);
        ml = j.ml, keep = j.fa, f = j.fb;
      }
      __syncwarp();
    }
    if (live && write) {
      *at = ml;
      if (it.first) a.part_next[it.own][row] = attn_next((blockIdx.x + 1) * kRows + r, it.n_cont, kRows);
    }
  }
  // four columns
  __device__ __forceinline__ void store(const AttnPart& it, int c, float4 v) const {
    float4* to = reinterpret_cast<float4*>(o + c);
    if (it.again) {
      const float4 u = *to;
      v = make_float4(fmaf(u.x, keep, v.x * f), fmaf(u.y, keep, v.y * f), fmaf(u.z, keep, v.z * f),
                      fmaf(u.w, keep, v.w * f));
    }
    *to = v;
  }
};
// Row r of an item lies in slot r / 8 of warp r % 8's eight: neighbours for the
// lanes of a warp, and few rows are spread over all warps.
__device__ __forceinline__ int slot_of(int r) { return (r & (kWarps - 1)) * kPer + (r >> 3); }

// four elements of a row in shared memory
template <typename T>
__device__ __forceinline__ float4 four(const uint8_t* row, int c) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(row + c * 4);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(row + c * 2);
    float f[8];
    Vec<T>::get(make_uint4(v.x, v.y, 0, 0), f);
    return make_float4(f[0], f[1], f[2], f[3]);
  }
}

// Shared memory, in bytes.  Key and value rows are padded by 16 bytes, so that a
// quarter-warp's 16-byte reads of eight rows cover all banks.
struct FmaLayout {
  int kp, vp, qp;              // row pitches: keys, values (bytes), queries (floats)
  int kv, stage, q, w, rows, bytes;
  __host__ __device__ FmaLayout(int d, int dv, int es) {
    kp = d * es + 16;
    vp = dv * es + 16;
    qp = d + 4;
    stage = kKeys * (kp + vp);  // keys, then values
    kv = 0;
    q = 2 * stage;
    w = q + kRows * qp * 4;
    rows = w + kRows * kWeightPitch * 4;
    bytes = rows + 2 * kKeys * 8;
  }
};

// Up to NR rows, key by key (see above); d and dv up to 128; qp: from one row's
// queries to the next.  smem: two stages, and when the part is done the warps'
// sets, NR rows of dv + 4 floats each.  Returns whether a table entry outside the
// pool was met.
template <typename T, int NR>
__device__ __forceinline__ bool few_rows(const AttnArgs& a, const AttnPart& it, const float* sq, int qp,
                                         const FmaLayout& ly, uint8_t* smem) {
  constexpr int N = Vec<T>::N, S = 16 / N;            // elements and 16-byte pieces of a lane
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, grp = lane >> 3, piece = lane & 7;
  const int kvr = a.d / N, vvr = a.dv / N;
  bool bad = false;
  // pool row of this group's key in tile t (-1: zeros, -2: none)
  auto row_of = [&](int t) -> int64_t {
    const int p = t * kKeys + warp * 4 + grp;
    if (t >= it.t1 || p >= it.len) return -2;
    const int j = p / a.L;
    const int blk = attn_block(a, it, j);
    bad |= blk < 0;
    return blk >= 0 ? ((int64_t)blk * a.H + it.h) * a.L + (p - j * a.L) : -1;
  };
  float m[NR], l[NR], acc[NR][16];
  int see[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    m[i] = -INFINITY, l[i] = 0.f;
    see[i] = i >= it.rows ? 0 : it.own ? min(it.len, it.see0 + (it.row0 + i) / a.G + 1) : it.len;
#pragma unroll
    for (int c = 0; c < 16; ++c) acc[i][c] = 0.f;
  }
  // two tiles ahead: a lane copies what it will read itself, so it only waits for
  // its own copies
  uint8_t* sk = smem + (warp * 4 + grp) * ly.kp + piece * 16;
  uint8_t* sv = smem + kKeys * ly.kp + (warp * 4 + grp) * ly.vp + piece * 16;
  auto fetch = [&](int t) {
    const int64_t row = row_of(t);
    if (row != -2) {
      const int64_t at = max(row, (int64_t)0);
      const int bytes = row >= 0 ? 16 : 0;  // a table entry outside the pool: zeros
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint8_t* src = kv ? reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.pool_V) + at * a.dv)
                                : reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.pool_K) + at * a.d);
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared((kv ? sv : sk) + (t & 1) * ly.stage);
#pragma unroll
        for (int s = 0; s < S; ++s)
          if (s * 8 + piece < (kv ? vvr : kvr))
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + s * 128),
                         "l"(src + (s * 8 + piece) * 16), "r"(bytes)
                         : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(it.t0);
  fetch(it.t0 + 1);
#pragma unroll 1
  for (int t = it.t0; t < it.t1; ++t) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    const int p0 = t * kKeys + warp * 4 + grp;
    const bool key = p0 < it.len;
    const uint8_t* ks = sk + (t & 1) * ly.stage;
    const uint8_t* vs = sv + (t & 1) * ly.stage;
    float x[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) x[i] = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s * 8 + piece < kvr) {
        float f[N];
        Vec<T>::get(*reinterpret_cast<const uint4*>(ks + s * 128), f);
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int c = 0; c < N; c += 4) {
            const float4 u = *reinterpret_cast<const float4*>(sq + i * qp + (s * 8 + piece) * N + c);
            x[i] = fmaf(f[c], u.x, x[i]), x[i] = fmaf(f[c + 1], u.y, x[i]);
            x[i] = fmaf(f[c + 2], u.z, x[i]), x[i] = fmaf(f[c + 3], u.w, x[i]);
          }
      }
    }
    float w[NR];
    bool any = false;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
#pragma unroll
      for (int o = 4; o >= 1; o >>= 1) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
      // a key that the row does not see is left out (its values may be inf or NaN)
      const bool seen = key && p0 < see[i];
      const float s = x[i] * a.scale_log2;
      w[i] = -1.f;
      if (seen) {
        if (s > m[i]) {
          const float al = exp2f(m[i] - s);
          m[i] = s;
          l[i] *= al;
#pragma unroll
          for (int c = 0; c < 16; ++c) acc[i][c] *= al;
        }
        // only scores of -inf seen: weight 0
        w[i] = exp2f(s - (m[i] == -INFINITY ? 0.f : m[i]));
        l[i] += w[i];
        any = true;
      }
    }
    if (any) {
#pragma unroll
      for (int q = 0; q < S; ++q) {
        if (q * 8 + piece >= vvr) continue;
        float f[N];
        Vec<T>::get(*reinterpret_cast<const uint4*>(vs + q * 128), f);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          if (w[i] < 0.f) continue;
#pragma unroll
          for (int c = 0; c < N; ++c) acc[i][q * N + c] = fmaf(w[i], f[c], acc[i][q * N + c]);
        }
      }
    }
    fetch(t + 2);  // into the stage just read
  }
  __syncthreads();  // all warps are done with the stages
  float* sj = reinterpret_cast<float*>(smem);
  // the warp's four groups, then the warps through shared memory
#pragma unroll
  for (int i = 0; i < NR; ++i) {
#pragma unroll
    for (int o = 8; o <= 16; o <<= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m[i], o), ol = __shfl_xor_sync(0xffffffffu, l[i], o);
      const float now = fmaxf(m[i], om);
      const float fa = m[i] == now ? 1.f : exp2f(m[i] - now), fb = om == now ? 1.f : exp2f(om - now);
      m[i] = now;
      l[i] = l[i] * fa + ol * fb;
#pragma unroll
      for (int c = 0; c < 16; ++c) acc[i][c] = acc[i][c] * fa + __shfl_xor_sync(0xffffffffu, acc[i][c], o) * fb;
    }
    float* set = sj + (warp * NR + i) * (a.dv + 4);
    if (grp == 0) {
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (s * 8 + piece < vvr) {
#pragma unroll
          for (int c = 0; c < N; c += 4)
            *reinterpret_cast<float4*>(set + 4 + (s * 8 + piece) * N + c) =
                make_float4(acc[i][s * N + c], acc[i][s * N + c + 1], acc[i][s * N + c + 2], acc[i][s * N + c + 3]);
        }
      if (piece == 0) set[0] = m[i], set[1] = l[i];
    }
  }
  __syncthreads();
  // row `warp` of the item: its eight sets, four columns a lane
  if (warp < it.rows) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sj[(w * NR + warp) * (a.dv + 4)]);
    float sum = 0.f;
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* set = sj + (w * NR + warp) * (a.dv + 4);
      const float f = set[0] == top ? 1.f : exp2f(set[0] - top);
      sum += set[1] * f;
      if (lane * 4 < a.dv) {
        const float4 u = *reinterpret_cast<const float4*>(set + 4 + lane * 4);
        o.x += u.x * f, o.y += u.y * f, o.z += u.z * f, o.w += u.w * f;
      }
    }
    const FmaPut put(a, it, warp, make_float2(top, sum), true, lane == 0);
    if (lane * 4 < a.dv) put.store(it, lane * 4, o);
  }
  return bad;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) prefix_attention_fma_kernel(const __grid_constant__ AttnArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  const FmaLayout ly(a.d, a.dv, (int)sizeof(T));
  float* sq = reinterpret_cast<float*>(smem + ly.q);
  int64_t* s_row = reinterpret_cast<int64_t*>(smem + ly.rows);  // [2][kKeys] pool row of a key, -1: zeros, -2: none
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float* sw = reinterpret_cast<float*>(smem + ly.w) + warp * (kPer * kWeightPitch);  // the warp's weights
  const T* Q = static_cast<const T*>(a.Q);
  const int kvr = a.d / Vec<T>::N, vvr = a.dv / Vec<T>::N, vpr = kvr + vvr;

  // the walk is one thread's, its state in shared memory: 40 registers less a thread
  __shared__ int64_t s_sum[1][32];
  __shared__ int s_more;
  __shared__ AttnLine<Cut> s_line;
  __shared__ AttnEven s_shares;
  __shared__ AttnWalk<Cut> s_walk;
  __shared__ AttnPart s_it;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  {
    AttnLine<Cut> line;
    attn_lines<kWarps>(a, s_sum, line);
    AttnEven shares;
    constexpr int least = Cut::C0 + Cut::W;
    shares.init(line.U, line.U >= (int64_t)gridDim.x * least ? (int)gridDim.x : max(1, (int)line.U / least));
    AttnWalk<Cut>::find(a, line, shares.bound(blockIdx.x), shares.bound(blockIdx.x + 1), &s_walk);
    if (tid == 32) s_line = line;
    if (tid == 64) s_shares = shares;
  }
  bool bad = false;
#pragma unroll 1
  for (;;) {
    __syncthreads();  // the last part's reads of the stages, the queries and s_it are done
    if (tid == 0) s_more = s_walk.next(a, s_line, [&](int64_t p) { return s_shares.worker_of(p); }, s_it);
    __syncthreads();
    if (!s_more) break;
    const AttnPart it = s_it;
    // where a tile's keys lie (32 threads)
    auto find_rows = [&](int t) {
      if (tid >= kKeys || t >= it.t1) return;
      const int p = t * kKeys + tid;
      int64_t row = -2;
      if (p < it.len) {
        const int j = p / a.L;
        const int blk = attn_block(a, it, j);
        row = blk >= 0 ? ((int64_t)blk * a.H + it.h) * a.L + (p - j * a.L) : -1;
        bad |= blk < 0;
      }
      s_row[(t & 1) * kKeys + tid] = row;
    };
    // a tile's keys and values on their way into stage t & 1
    auto fetch = [&](int t) {
      uint8_t* st = smem + (t & 1) * ly.stage;
      for (int i = tid; i < kKeys * vpr; i += kThreads) {
        const int key = i / vpr, v = i - key * vpr;
        const int64_t row = s_row[(t & 1) * kKeys + key];
        if (row == -2) continue;
        const bool is_v = v >= kvr;
        const int64_t at = max(row, (int64_t)0);
        const T* src = is_v ? static_cast<const T*>(a.pool_V) + at * a.dv + (v - kvr) * Vec<T>::N
                            : static_cast<const T*>(a.pool_K) + at * a.d + v * Vec<T>::N;
        uint8_t* dst = is_v ? st + kKeys * ly.kp + key * ly.vp + (v - kvr) * 16 : st + key * ly.kp + v * 16;
        // a table entry outside the pool: zeros
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)),
                     "l"(src), "r"(row >= 0 ? 16 : 0)
                     : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    for (int i = tid; i < it.rows * kvr; i += kThreads) {
      const int r = i / kvr, v = i - r * kvr;
      int tok, hq;
      attn_row(a, it, r, tok, hq);
      float f[Vec<T>::N];
      Vec<T>::get(__ldg(reinterpret_cast<const uint4*>(Q + tok * a.q_st + hq * a.q_sh) + v), f);
#pragma unroll
      for (int x = 0; x < Vec<T>::N; x += 4)
        *reinterpret_cast<float4*>(sq + slot_of(r) * ly.qp + v * Vec<T>::N + x) = make_float4(f[x], f[x + 1], f[x + 2], f[x + 3]);
    }
    if (it.rows <= 4 && s_line.few) {
      __syncthreads();
      const int qp = slot_of(1) * ly.qp;
      bad |= it.rows == 1   ? few_rows<T, 1>(a, it, sq, qp, ly, smem)
             : it.rows == 2 ? few_rows<T, 2>(a, it, sq, qp, ly, smem)
                            : few_rows<T, 4>(a, it, sq, qp, ly, smem);
      continue;
    }
    find_rows(it.t0);
    find_rows(it.t0 + 1);
    __syncthreads();
    fetch(it.t0);
    // NR: rows of a lane (0: one row a warp, whose keys its lanes share out); Q: runs
    // of 32 columns of a lane's values
    auto run = [&](auto nr, auto nq) {
      constexpr bool ONE = decltype(nr)::value == 0;
      constexpr int NR = ONE ? 1 : decltype(nr)::value, Q32 = decltype(nq)::value, NK = ONE ? 1 : 4;
      // scores: rows ry, ry + 4 of the warp's, keys kx, kx + 8 .. (ONE: key `lane`)
      const int ry = lane >> 3, kx = lane & 7, key = ONE ? lane : kx;
      constexpr int kOver = ONE ? 16 : 4;  // a row's lanes: 32 or 8
      float m[NR], l[NR];
      float4 acc[NR][Q32];
      const float* q[NR];
      int row[NR];
#pragma unroll
      for (int u = 0; u < NR; ++u) {
        m[u] = -INFINITY, l[u] = 0.f;
        // (rows behind the item's last repeat it)
        row[u] = ONE ? warp : warp + kWarps * (ry + 4 * u);
        q[u] = sq + slot_of(min(row[u], it.rows - 1)) * ly.qp;
#pragma unroll
        for (int c = 0; c < Q32; ++c) acc[u][c] = make_float4(0, 0, 0, 0);
      }
#pragma unroll 1
      for (int t = it.t0; t < it.t1; ++t) {
        if (t + 1 < it.t1) {
          fetch(t + 1);
          asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        find_rows(t + 2);
        const uint8_t* sk = smem + (t & 1) * ly.stage;
        const uint8_t* sv = sk + kKeys * ly.kp;
        const int key0 = t * kKeys, n = min(kKeys, it.len - key0);
        if (warp < it.rows) {
          float x[NR][NK];
#pragma unroll
          for (int u = 0; u < NR; ++u)
#pragma unroll
            for (int k = 0; k < NK; ++k) x[u][k] = 0.f;
          const uint8_t* kr = sk + key * ly.kp;
#pragma unroll 2
          for (int v = 0; v < kvr; ++v) {
            float f[NK][Vec<T>::N];
#pragma unroll
            for (int k = 0; k < NK; ++k) Vec<T>::get(*reinterpret_cast<const uint4*>(kr + k * 8 * ly.kp + v * 16), f[k]);
#pragma unroll
            for (int c = 0; c < Vec<T>::N; c += 4)
#pragma unroll
              for (int u = 0; u < NR; ++u) {
                const float4 y = *reinterpret_cast<const float4*>(q[u] + v * Vec<T>::N + c);
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                  x[u][k] = fmaf(f[k][c], y.x, x[u][k]), x[u][k] = fmaf(f[k][c + 1], y.y, x[u][k]);
                  x[u][k] = fmaf(f[k][c + 2], y.z, x[u][k]), x[u][k] = fmaf(f[k][c + 3], y.w, x[u][k]);
                }
              }
          }
          // keys that a row sees, running maximum and sum over its lanes
          int see[NR];
#pragma unroll
          for (int u = 0; u < NR; ++u) {
            see[u] = it.own ? min(n, it.see0 + (it.row0 + min(row[u], it.rows - 1)) / a.G + 1 - key0) : n;
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < NK; ++k) {
              x[u][k] = key + 8 * k < see[u] ? x[u][k] * a.scale_log2 : -INFINITY;
              top = fmaxf(top, x[u][k]);
            }
#pragma unroll
            for (int o = kOver; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float now = fmaxf(m[u], top);
            const float base = now == -INFINITY ? 0.f : now;  // nothing seen yet: weights 0, and no inf - inf
            const float al = exp2f(m[u] - base);
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < NK; ++k) {
              const float p = exp2f(x[u][k] - base);
              sum += p;
              sw[(ONE ? 0 : (ry + 4 * u) * kWeightPitch) + key + 8 * k] = p;
            }
#pragma unroll
            for (int o = kOver; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            m[u] = now;
            l[u] = l[u] * al + sum;
#pragma unroll
            for (int c = 0; c < Q32; ++c)
              acc[u][c].x *= al, acc[u][c].y *= al, acc[u][c].z *= al, acc[u][c].w *= al;
          }
          __syncwarp();
          // values, four of every 32 columns a lane; a key beyond a row's own has
          // weight 0, but 0 * (inf or NaN) is NaN, so it is left out
          const bool ragged = it.own && key0 + n > it.see0 + it.row0 / a.G + 1;
          auto add = [&](auto guard) {
#pragma unroll 1
            for (int j0 = 0; j0 < n; j0 += 4) {
              if constexpr (ONE) {
                // a key every eight lanes
                const int j = j0 + ry;
                if (j >= (decltype(guard)::value ? see[0] : n)) continue;
                const float w = sw[j];
#pragma unroll
                for (int c = 0; c < Q32; ++c) {
                  if (c * 32 >= a.dv) break;
                  const float4 v = four<T>(sv + j * ly.vp, c * 32 + kx * 4);
                  acc[0][c].x = fmaf(w, v.x, acc[0][c].x), acc[0][c].y = fmaf(w, v.y, acc[0][c].y);
                  acc[0][c].z = fmaf(w, v.z, acc[0][c].z), acc[0][c].w = fmaf(w, v.w, acc[0][c].w);
                }
                continue;
              }
              float4 p[NR];
#pragma unroll
              for (int u = 0; u < NR; ++u)
                p[u] = *reinterpret_cast<const float4*>(sw + (ry + 4 * u) * kWeightPitch + j0);
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                if (j0 + y >= n) break;
#pragma unroll
                for (int c = 0; c < Q32; ++c) {
                  if (c * 32 >= a.dv) break;  // (a lane's columns behind the last are not kept)
                  const float4 v = four<T>(sv + (j0 + y) * ly.vp, c * 32 + kx * 4);
#pragma unroll
                  for (int u = 0; u < NR; ++u) {
                    if (decltype(guard)::value && j0 + y >= see[u]) continue;
                    const float w = y == 0 ? p[u].x : y == 1 ? p[u].y : y == 2 ? p[u].z : p[u].w;
                    acc[u][c].x = fmaf(w, v.x, acc[u][c].x), acc[u][c].y = fmaf(w, v.y, acc[u][c].y);
                    acc[u][c].z = fmaf(w, v.z, acc[u][c].z), acc[u][c].w = fmaf(w, v.w, acc[u][c].w);
                  }
                }
              }
            }
          };
          if (ragged) add(IC<1>{});
          else add(IC<0>{});
          __syncwarp();  // the weights may be written again
        }
        __syncthreads();  // the stage may be filled again, and the next rows are known
      }
      if constexpr (ONE) {
#pragma unroll
        for (int c = 0; c < Q32; ++c)
#pragma unroll
          for (int o = 8; o <= 16; o <<= 1) {
            acc[0][c].x += __shfl_xor_sync(0xffffffffu, acc[0][c].x, o);
            acc[0][c].y += __shfl_xor_sync(0xffffffffu, acc[0][c].y, o);
            acc[0][c].z += __shfl_xor_sync(0xffffffffu, acc[0][c].z, o);
            acc[0][c].w += __shfl_xor_sync(0xffffffffu, acc[0][c].w, o);
          }
      }
      // partial results: the row's own place, or this CTA's continuation buffer
#pragma unroll
      for (int u = 0; u < NR; ++u) {
        const bool mine = row[u] < it.rows && !(ONE && ry > 0);
        const FmaPut put(a, s_it, row[u], make_float2(m[u], l[u]), mine, kx == 0);  // (s_it: no registers in the loop)
#pragma unroll
        for (int c = 0; c < Q32; ++c)
          if (mine && c * 32 + kx * 4 < a.dv) put.store(s_it, c * 32 + kx * 4, acc[u][c]);
      }
    };
    auto rows = [&](auto nq) {
      if (it.rows <= kWarps) run(IC<0>{}, nq);
      else if (it.rows <= 4 * kWarps) run(IC<1>{}, nq);
      else run(IC<2>{}, nq);
    };
    if (a.dv <= 128) rows(IC<4>{});
    else rows(IC<8>{});
  }
  if (bad) atomicMax(&g_attn_fma_error, (unsigned)GFST_ERR_ARG);
}

template <typename T>
int launch(const AttnArgs& a, int sms, cudaStream_t stream) {
  const FmaLayout ly(a.d, a.dv, (int)sizeof(T));
  auto kern = prefix_attention_fma_kernel<T>;
  static std::atomic<uint64_t> allowed{0};
  const int st = attn_allow_smem(kern, FmaLayout(256, 256, (int)sizeof(T)).bytes, allowed);
  if (st != GFST_OK) return st;
  const int per_sm = ly.bytes <= 110 * 1024 ? 2 : 1;
  const int grid = (sms < kAttnMaxGrid ? sms : kAttnMaxGrid) * per_sm;
  return attn_launch("prefix_attention_fma_kernel", kern, grid, kThreads, ly.bytes, stream, a);
}

}  // namespace

int launch_attn_fma_error(int status, cudaStream_t stream) {
  attn_fma_error_kernel<<<1, 1, 0, stream>>>(status);
  return check_launch("attn_fma_error_kernel");
}

int launch_prefix_attention_fma(const AttnArgs& a, int dtype, int sms, cudaStream_t stream) {
  if (dtype == GFST_F32) return launch<float>(a, sms, stream);
  if (dtype == GFST_BF16) return launch<__nv_bfloat16>(a, sms, stream);
  return launch<__half>(a, sms, stream);
}

}  // namespace gfst
