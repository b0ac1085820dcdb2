// Shared-prefix attention on the FP32 units: every element type, block length
// and head size (rows a multiple of 16 bytes, up to 256 elements).  It serves
// the 32-bit memory, whose products the tensor cores would round, and the
// shapes the tensor-core kernel does not tile.
//
// One CTA walks its share of the items (prefix_attention.cuh): 32 query rows
// and a 64-key tile in shared memory as fp32, scores one key per thread and
// four rows a pass, running maximum and sum per row in shared memory, values
// accumulated in registers (four columns per thread).  Row groups without
// valid rows are skipped, so a decode step of a few rows reads each key from
// shared memory once.
#include <cuda_fp16.h>

#include "prefix_attention.cuh"

namespace gfst {

GFST_DEFINE_ERROR_WORD(g_attn_fma_error, read_attn_fma_error, "attention")

namespace {

constexpr int kRows = kAttnFmaRows;   // 32
constexpr int kKeys = 64;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
// An item's fixed cost is about two 64-key tiles (queries in, partials out).
using Cut = AttnCutAll<kRows, kKeys, 2, 1>;

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

// shared memory: rows padded by 4 floats, so that the float4 reads of eight
// consecutive rows cover all banks once
struct FmaLayout {
  int qp, vp, q, k, v, s, stat, rows, bytes;
  __host__ __device__ FmaLayout(int d, int dv) {
    qp = d + 4;
    vp = dv + 4;
    q = 0;
    k = q + kRows * qp;
    v = k + kKeys * qp;
    s = v + kKeys * vp;
    stat = s + kRows * (kKeys + 1);
    rows = stat + 3 * kRows;      // int64 row offsets, 8-byte aligned below
    rows = (rows + 1) & ~1;
    bytes = (rows + 2 * kKeys) * 4;
  }
};

template <typename T>
__device__ __forceinline__ void stage_row(float* dst, const T* src, int v) {
  float f[Vec<T>::N];
  const uint4 x = src != nullptr ? __ldg(reinterpret_cast<const uint4*>(src) + v) : make_uint4(0, 0, 0, 0);
  Vec<T>::get(x, f);
#pragma unroll
  for (int i = 0; i < Vec<T>::N; i += 4)
    *reinterpret_cast<float4*>(dst + v * Vec<T>::N + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) prefix_attention_fma_kernel(const AttnArgs a) {
  extern __shared__ float4 smem4[];
  float* sm = reinterpret_cast<float*>(smem4);
  const FmaLayout ly(a.d, a.dv);
  float* sq = sm + ly.q;
  float* sk = sm + ly.k;
  float* sv = sm + ly.v;
  float* ss = sm + ly.s;                 // [kRows][kKeys + 1]
  float* s_m = sm + ly.stat;             // running maximum (log2 units)
  float* s_l = s_m + kRows;              // running sum
  float* s_a = s_l + kRows;              // this tile's rescale
  int64_t* s_row = reinterpret_cast<int64_t*>(sm + ly.rows);  // pool row of each key, -1 = none
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* Q = static_cast<const T*>(a.Q);
  const T* pK = static_cast<const T*>(a.pool_K);
  const T* pV = static_cast<const T*>(a.pool_V);
  const int kvr = a.d / Vec<T>::N, vvr = a.dv / Vec<T>::N;

  // value columns: thread owns columns [4 col, 4 col + 4) of rows grp, grp + n_grp, ...
  const int n_col = a.dv / 4, n_grp = kThreads / n_col;
  const int grp = tid / n_col, col = (tid - grp * n_col) * 4;
  constexpr int kAcc = 8;                // rows per thread at dv = 256; fewer below

  __shared__ int64_t s_sum[1][32], s_at;
  __shared__ int s_b;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  AttnLine<Cut> line;
  attn_lines(a, s_sum, line);
  AttnEven shares;
  constexpr int least = Cut::C0 + Cut::W;
  shares.init(line.U, line.U >= (int64_t)gridDim.x * least ? (int)gridDim.x : max(1, (int)line.U / least));
  const int64_t u0 = shares.bound(blockIdx.x), u1 = shares.bound(blockIdx.x + 1);
  line.find(a, u0, &s_b, &s_at);
  __syncthreads();
  AttnWalk<Cut> walk;
  walk.begin(a, line, u0, u1, s_b, s_at);
  auto share_of = [&](int64_t p) { return shares.worker_of(p); };
  AttnPart it;
  bool bad = false;
  while (walk.next(a, line, share_of, it)) {
    __syncthreads();
    for (int i = tid; i < it.rows * kvr; i += kThreads) {
      const int r = i / kvr;
      int tok, hq;
      attn_row(a, it, r, tok, hq);
      stage_row<T>(sq + r * ly.qp, Q + tok * a.q_st + hq * a.q_sh, i - r * kvr);
    }
    if (tid < kRows) {
      s_m[tid] = -INFINITY;
      s_l[tid] = 0.f;
    }
    float acc[kAcc][4];
#pragma unroll
    for (int i = 0; i < kAcc; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;

    for (int t = it.t0; t < it.t1; ++t) {
      const int key0 = t * kKeys;
      __syncthreads();
      if (tid < kKeys) {
        const int p = key0 + tid;
        int64_t row = -1;
        if (p < it.len) {
          const int j = p / a.L;
          const int blk = attn_block(a, it, j);
          if (blk >= 0) row = ((int64_t)blk * a.H + it.h) * a.L + (p - j * a.L);
          else bad = true;
        }
        s_row[tid] = row;
      }
      __syncthreads();
      for (int i = tid; i < kKeys * kvr; i += kThreads) {
        const int r = i / kvr;
        const int64_t row = s_row[r];
        stage_row<T>(sk + r * ly.qp, row >= 0 ? pK + row * a.d : nullptr, i - r * kvr);
      }
      for (int i = tid; i < kKeys * vvr; i += kThreads) {
        const int r = i / vvr;
        const int64_t row = s_row[r];
        stage_row<T>(sv + r * ly.vp, row >= 0 ? pV + row * a.dv : nullptr, i - r * vvr);
      }
      __syncthreads();
      {  // scores: key tid % 64, rows tid / 64 + 4 i
        const int key = tid & (kKeys - 1);
        const float4* kr = reinterpret_cast<const float4*>(sk + key * ly.qp);
        for (int r0 = 0; r0 < it.rows; r0 += 8) {
          const int ra = min(r0 + (tid >> 6), it.rows - 1), rb = min(r0 + 4 + (tid >> 6), it.rows - 1);
          const float4* qa = reinterpret_cast<const float4*>(sq + ra * ly.qp);
          const float4* qb = reinterpret_cast<const float4*>(sq + rb * ly.qp);
          float x = 0.f, y = 0.f;
          for (int c = 0; c < a.d / 4; ++c) {
            const float4 k = kr[c], u = qa[c], w = qb[c];
            x = fmaf(k.x, u.x, x), x = fmaf(k.y, u.y, x), x = fmaf(k.z, u.z, x), x = fmaf(k.w, u.w, x);
            y = fmaf(k.x, w.x, y), y = fmaf(k.y, w.y, y), y = fmaf(k.z, w.z, y), y = fmaf(k.w, w.w, y);
          }
          const int p = key0 + key;
          auto put = [&](int r, float s) {
            const int lim = it.own ? min(it.len, it.see0 + (it.row0 + r) / a.G + 1) : it.len;
            ss[r * (kKeys + 1) + key] = p < lim ? s * a.scale_log2 : -INFINITY;
          };
          put(ra, x);
          if (rb != ra) put(rb, y);
        }
      }
      __syncthreads();
      // running maximum and sum: warp w takes rows w, w + 8, ...
      for (int r = warp; r < it.rows; r += kWarps) {
        float* sr = ss + r * (kKeys + 1);
        const float x = sr[lane], y = sr[lane + 32];
        float m = fmaxf(x, y);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float old = s_m[r];
        const float now = fmaxf(old, m);
        // a row that has seen nothing keeps weight 0 (and no inf - inf)
        const float base = now == -INFINITY ? 0.f : now;
        const float px = exp2f(x - base), py = exp2f(y - base);
        sr[lane] = px;
        sr[lane + 32] = py;
        float l = px + py;
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (lane == 0) {
          const float al = exp2f(old - base);
          s_a[r] = al;
          s_m[r] = now;
          s_l[r] = s_l[r] * al + l;
        }
      }
      __syncthreads();
      if (grp < n_grp) {
        // keys beyond a row's own limit carry weight 0, but 0 * (inf or NaN) is NaN: they are left out
        const bool ragged = it.own && key0 + kKeys > it.see0 + it.row0 / a.G + 1;
#pragma unroll
        for (int i = 0; i < kAcc; ++i) {
          const int r = grp + i * n_grp;
          if (r < it.rows) {
            const float al = s_a[r];
            float o0 = acc[i][0] * al, o1 = acc[i][1] * al, o2 = acc[i][2] * al, o3 = acc[i][3] * al;
            const float* pr = ss + r * (kKeys + 1);
            int n = min(kKeys, it.len - key0);
            if (ragged) n = min(n, it.see0 + (it.row0 + r) / a.G + 1 - key0);
            for (int j = 0; j < n; ++j) {
              const float p = pr[j];
              const float4 v = *reinterpret_cast<const float4*>(sv + j * ly.vp + col);
              o0 = fmaf(p, v.x, o0), o1 = fmaf(p, v.y, o1), o2 = fmaf(p, v.z, o2), o3 = fmaf(p, v.w, o3);
            }
            acc[i][0] = o0, acc[i][1] = o1, acc[i][2] = o2, acc[i][3] = o3;
          }
        }
      }
    }
    __syncthreads();
    // partial results: the row's own place, or this CTA's continuation buffer
    if (grp < n_grp) {
#pragma unroll
      for (int i = 0; i < kAcc; ++i) {
        const int r = grp + i * n_grp;
        if (r < it.rows) {
          int tok, hq;
          attn_row(a, it, r, tok, hq);
          const int64_t row = (int64_t)tok * (a.H * a.G) + hq;
          const int64_t crow = (int64_t)blockIdx.x * kRows + r;
          float* o = it.first ? a.part_o[it.own] + row * a.dv : a.cont_o + crow * a.dv;
          *reinterpret_cast<float4*>(o + col) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
          if (col == 0) {
            const float2 ml = make_float2(s_m[r], s_l[r]);
            if (it.first) {
              a.part_ml[it.own][row] = ml;
              a.part_next[it.own][row] = attn_next((blockIdx.x + 1) * kRows + r, it.n_cont, kRows);
            } else {
              a.cont_ml[crow] = ml;
            }
          }
        }
      }
    }
  }
  if (bad) atomicExch(&g_attn_fma_error, (unsigned)GFST_ERR_ARG);
}

template <typename T>
int launch(const AttnArgs& a, int sms, cudaStream_t stream) {
  const FmaLayout ly(a.d, a.dv);
  auto kern = prefix_attention_fma_kernel<T>;
  static std::atomic<uint64_t> allowed{0};
  const int st = attn_allow_smem(kern, FmaLayout(256, 256).bytes, allowed);
  if (st != GFST_OK) return st;
  const int per_sm = ly.bytes <= 110 * 1024 ? 2 : 1;
  const int grid = (sms < kAttnMaxGrid ? sms : kAttnMaxGrid) * per_sm;
  return attn_launch("prefix_attention_fma_kernel", kern, grid, kThreads, ly.bytes, stream, a);
}

}  // namespace

int launch_prefix_attention_fma(const AttnArgs& a, int dtype, int sms, cudaStream_t stream) {
  if (dtype == GFST_F32) return launch<float>(a, sms, stream);
  if (dtype == GFST_BF16) return launch<__nv_bfloat16>(a, sms, stream);
  return launch<__half>(a, sms, stream);
}

}  // namespace gfst
