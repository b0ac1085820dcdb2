// Shared-prefix attention: argument checks, workspace, kernel choice and the
// merge of the partial results (prefix_attention.cuh).
//
// The merge is one warp per (token, query head): the prefix part, the own part
// and their continuations, at most a few, weighted by 2^(m_i - max m), divided
// by the joined sum and rounded once to the output type.  It reads each partial
// once; what bounds it is their 4 B per value: for 300,768 rows of two parts of
// 128 columns, 385 MB, it takes 95 us (4.1 TB/s).  A row's two parts and their (m, l)
// are loaded at once, before it is known which of them are needed: one memory
// latency a warp instead of four in a chain (which took 217 us).  One row a warp:
// two or four, with their loads together, were slower from 16 rows (11.7 and 13.0
// us for attention and merge together, 11.2 with one) to those (934 and 979 us, 931
// with one, before later steps that are not the merge's).
#include <cuda_fp16.h>

#include <cmath>

#include "prefix_attention.cuh"

namespace gfst {

namespace {

constexpr int kMergeThreads = 128;

template <typename T>
__device__ __forceinline__ void store4(T* dst, float4 v);
template <>
__device__ __forceinline__ void store4<float>(float* dst, float4 v) { *reinterpret_cast<float4*>(dst) = v; }
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* dst, float4 v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
template <>
__device__ __forceinline__ void store4<__half>(__half* dst, float4 v) {
  const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// What a row's sets have given so far: o is relative to 2^m.
template <int V>
struct MergeRow {
  float m = -INFINITY, l = 0.f;
  float4 o[V] = {};
  // weight of a set of reference x under the reference `now` (equal ones need no
  // exponential, and no inf - inf)
  __device__ static __forceinline__ float weight(float x, float now) { return x == now ? 1.f : exp2f(x - now); }
  __device__ __forceinline__ void add(int i, const float4& v, float w) {
    o[i].x = fmaf(v.x, w, o[i].x), o[i].y = fmaf(v.y, w, o[i].y);
    o[i].z = fmaf(v.z, w, o[i].z), o[i].w = fmaf(v.w, w, o[i].w);
  }
};
// an empty set (a NaN sum is kept)
__device__ __forceinline__ bool merge_empty(float2 ml) { return !(ml.y > 0.f) && ml.y == ml.y; }

// V: runs of 128 columns.
template <typename T, int V>
__global__ void __launch_bounds__(kMergeThreads) prefix_attention_merge_kernel(const AttnArgs a, int cont_rows) {
  const int lane = threadIdx.x & 31;
  const int heads = a.H * a.G;
  const int64_t row = (int64_t)blockIdx.x * (kMergeThreads / 32) + (threadIdx.x >> 5);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (row >= (int64_t)a.n_tokens * heads) return;
  // everything that lies at the row's own place in one go, whether it is needed or
  // not (a set that was not written is not looked at)
  int2 next[2] = {};
  float2 ml[2];
  float4 o[2][V];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k == 0 && a.prefix_len == nullptr) continue;
    next[k] = a.part_next[k][row];
    ml[k] = a.part_ml[k][row];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * 32 + lane) * 4;
      if (c < a.dv) o[k][i] = *reinterpret_cast<const float4*>(a.part_o[k] + row * a.dv + c);
    }
  }
  const int tok = (int)row / heads;
  const bool live = tok < attn_tokens(a) && tok >= a.cu[0], prefix = live && attn_prefix_len(a) > 0;
  if (!live && !a.fill_tail) {  // the caller's rows of out stay, the log-sum-exp is of nothing
    if (a.lse != nullptr && lane == 0) a.lse[row] = -INFINITY;
    return;
  }
  const bool has[2] = {prefix && !merge_empty(ml[0]), live && !merge_empty(ml[1])};
  MergeRow<V> x;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (has[k]) x.m = fmaxf(x.m, ml[k].x);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (!has[k]) continue;
    const float w = MergeRow<V>::weight(ml[k].x, x.m);
    x.l = fmaf(ml[k].y, w, x.l);
#pragma unroll
    for (int i = 0; i < V; ++i) x.add(i, o[k][i], w);
  }
  // Continuations, 32 sets at a time, one per lane: weights first, then the
  // values with their loads in flight together.  (Offsets that cover no item leave
  // `next` unset: sets outside the buffer are left out.)
  const int n0 = prefix ? min(max(next[0].y >> 9, 0), cont_rows) : 0;
  const int n1 = live ? min(max(next[1].y >> 9, 0), cont_rows) : 0;
  for (int s0 = 0; s0 < n0 + n1; s0 += 32) {
    const int s = s0 + lane;
    const float* src = nullptr;
    float2 y = make_float2(-INFINITY, 0.f);
    if (s < n0 + n1) {
      const int own = s >= n0;
      const int2 nx = own ? next[1] : next[0];
      const int64_t c = nx.x + (int64_t)(own ? s - n0 : s) * (nx.y & 511);
      if (c >= 0 && c < cont_rows) {
        y = a.cont_ml[c];
        src = a.cont_o + c * a.dv;
      }
    }
    if (merge_empty(y)) src = nullptr;
    if (src == nullptr) y = make_float2(-INFINITY, 0.f);
    float now = fmaxf(x.m, y.x);
#pragma unroll
    for (int i = 16; i >= 1; i >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, i));
    const float w = src == nullptr ? 0.f : MergeRow<V>::weight(y.x, now);
    float sum = y.y * w;
#pragma unroll
    for (int i = 16; i >= 1; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    const float keep = MergeRow<V>::weight(x.m, now);
    x.m = now;
    x.l = x.l * keep + sum;
#pragma unroll
    for (int i = 0; i < V; ++i) x.o[i].x *= keep, x.o[i].y *= keep, x.o[i].z *= keep, x.o[i].w *= keep;
    const int n = min(32, n0 + n1 - s0);
    for (int g = 0; g < n; g += 4) {
      float wt[4];
      float4 v[4][V];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = g + q;
        const float* p = reinterpret_cast<const float*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), k & 31));
        wt[q] = __shfl_sync(0xffffffffu, w, k & 31);
        if (k >= n) p = nullptr;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = (i * 32 + lane) * 4;
          v[q][i] = p != nullptr && c < a.dv ? *reinterpret_cast<const float4*>(p + c) : make_float4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (g + q >= n) break;
#pragma unroll
        for (int i = 0; i < V; ++i) x.add(i, v[q][i], wt[q]);
      }
    }
  }
  // a row that sees nothing: zeros and -inf
  const float inv = x.l == 0.f ? 0.f : 1.f / x.l;
  T* out = static_cast<T*>(a.out) + row * a.dv;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * 32 + lane) * 4;
    if (c < a.dv) store4<T>(out + c, make_float4(x.o[i].x * inv, x.o[i].y * inv, x.o[i].z * inv, x.o[i].w * inv));
  }
  if (a.lse != nullptr && lane == 0) a.lse[row] = x.l == 0.f ? -INFINITY : (x.m + log2f(x.l)) * 0.69314718055994531f;
}

template <typename T, int V>
int launch_merge_of(const AttnArgs& a, int cont_rows, cudaStream_t stream) {
  constexpr int per = kMergeThreads / 32;
  const int64_t rows = (int64_t)a.n_tokens * a.H * a.G;
  return attn_launch("prefix_attention_merge_kernel", prefix_attention_merge_kernel<T, V>, (rows + per - 1) / per,
                     kMergeThreads, 0, stream, a, cont_rows);
}

template <typename T>
int launch_merge(const AttnArgs& a, cudaStream_t stream) {
  return a.dv > 128 ? launch_merge_of<T, 2>(a, kAttnFmaContRows, stream)
                    : launch_merge_of<T, 1>(a, kAttnTcContRows, stream);
}

struct Workspace {
  size_t o, ml, next, cont_o, cont_ml, bytes;  // o, ml, next: two of each (prefix, own)
  int64_t rows;
  Workspace(int64_t n_tokens, int heads, int dv) {
    rows = n_tokens * heads;
    auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
    size_t at = 0;
    o = at, at += 2 * up((size_t)rows * dv * 4);
    ml = at, at += 2 * up((size_t)rows * 8);
    next = at, at += 2 * up((size_t)rows * 8);
    // the tensor-core kernel takes dv <= 128
    const size_t cont = dv <= 128 ? (size_t)kAttnTcContRows : (size_t)kAttnFmaContRows;
    cont_o = at, at += up(cont * dv * 4);
    cont_ml = at, at += up(cont * 8);
    bytes = at;
  }
};

int check_dims(int64_t n_tokens, int H, int G, int dv) {
  GFST_REQUIRE(n_tokens >= 0 && H >= 1 && G >= 1 && dv >= 1 && dv <= 256, GFST_ERR_SHAPE,
               "n_tokens %lld kv heads %d group %d dv %d", (long long)n_tokens, H, G, dv);
  GFST_REQUIRE(n_tokens * H < (1LL << 31) && n_tokens * H * G < (1LL << 31), GFST_ERR_SHAPE,
               "%lld tokens of %d heads exceed the int32 row range", (long long)n_tokens, H * G);
  return GFST_OK;
}

}  // namespace
}  // namespace gfst

using namespace gfst;

extern "C" int gfst_prefix_attention_workspace_bytes(int64_t n_tokens, int n_kv_heads, int group, int dv,
                                                     size_t* bytes) {
  GFST_REQUIRE(bytes != nullptr, GFST_ERR_ARG, "null pointer");
  const int st = check_dims(n_tokens, n_kv_heads, group, dv);
  if (st != GFST_OK) return st;
  *bytes = Workspace(n_tokens, n_kv_heads * group, dv).bytes;
  return GFST_OK;
}

extern "C" int gfst_prefix_attention(const void* Q, int64_t q_stride_t, int64_t q_stride_h, const void* pool_K,
                                     const void* pool_V, int64_t n_blocks, int L, int n_kv_heads, int group, int d,
                                     int dv, int dtype, const int32_t* tables, int64_t table_stride, int width,
                                     const int32_t* lens, const int32_t* cu_new, int n_requests, int64_t n_tokens,
                                     const int32_t* prefix_table, int prefix_width, const int32_t* prefix_len,
                                     float scale, void* out, float* lse, int fill_tail, void* workspace,
                                     size_t workspace_bytes, cudaStream_t stream) {
  GFST_REQUIRE(dtype == GFST_F32 || dtype == GFST_BF16 || dtype == GFST_F16, GFST_ERR_DTYPE, "dtype %d", dtype);
  int st = check_dims(n_tokens, n_kv_heads, group, dv);
  if (st != GFST_OK) return st;
  const int es = dtype == GFST_F32 ? 4 : 2, pv = 16 / es;
  GFST_REQUIRE(d >= 1 && d <= 256, GFST_ERR_SHAPE, "d=%d outside [1, 256]", d);
  GFST_REQUIRE(d % pv == 0 && dv % pv == 0, GFST_ERR_ALIGN, "rows of %d and %d elements are no multiple of 16 bytes", d,
               dv);
  const float scale_log2 = (float)((double)scale * 1.4426950408889634);
  GFST_REQUIRE(std::isfinite(scale_log2), GFST_ERR_ARG, "scale %g is not finite", (double)scale);
  GFST_REQUIRE(n_requests >= 1 && n_requests <= 65536 && width >= 1 && L >= 1 && n_blocks >= 1 && prefix_width >= 0,
               GFST_ERR_SHAPE, "requests %d width %d L %d blocks %lld prefix width %d", n_requests, width, L,
               (long long)n_blocks, prefix_width);
  constexpr int64_t kMostKeys = (1LL << 31) - 1024;  // a tile's last position stays in range
  GFST_REQUIRE((int64_t)width * L <= kMostKeys && (int64_t)prefix_width * L <= kMostKeys, GFST_ERR_SHAPE,
               "positions exceed the int32 range");
  if (n_tokens == 0) return GFST_OK;
  GFST_REQUIRE(Q && pool_K && pool_V && tables && lens && cu_new && out && workspace, GFST_ERR_ARG, "null pointer");
  GFST_REQUIRE(prefix_width == 0 || (prefix_table && prefix_len), GFST_ERR_ARG, "null prefix table or length");
  GFST_REQUIRE(aligned16(Q) && aligned16(pool_K) && aligned16(pool_V) && aligned16(out) && q_stride_t % pv == 0 &&
                   q_stride_h % pv == 0,
               GFST_ERR_ALIGN, "Q, out and the pools need 16-byte aligned rows");
  GFST_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, GFST_ERR_ALIGN, "workspace must be 256-byte aligned");
  const Workspace ws(n_tokens, n_kv_heads * group, dv);
  GFST_REQUIRE(workspace_bytes >= ws.bytes, GFST_ERR_SHAPE, "workspace of %zu bytes, %zu needed", workspace_bytes,
               ws.bytes);
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  GFST_REQUIRE(e == cudaSuccess, GFST_ERR_DEVICE, "device query: %s", cudaGetErrorString(e));

  uint8_t* w = static_cast<uint8_t*>(workspace);
  auto half = [&](size_t at, size_t next) { return w + at + (next - at) / 2; };
  AttnArgs a;
  a.Q = Q, a.q_st = q_stride_t, a.q_sh = q_stride_h;
  a.pool_K = pool_K, a.pool_V = pool_V, a.n_blocks = n_blocks;
  a.L = L, a.H = n_kv_heads, a.G = group, a.d = d, a.dv = dv;
  a.tables = tables, a.table_st = table_stride, a.width = width, a.lens = lens, a.cu = cu_new, a.B = n_requests;
  a.n_tokens = (int)n_tokens;
  a.prefix_table = prefix_table, a.prefix_width = prefix_width, a.prefix_len = prefix_width > 0 ? prefix_len : nullptr;
  a.scale_log2 = scale_log2;
  a.out = out, a.lse = lse, a.fill_tail = fill_tail;
  a.part_o[0] = reinterpret_cast<float*>(w + ws.o);
  a.part_o[1] = reinterpret_cast<float*>(half(ws.o, ws.ml));
  a.part_ml[0] = reinterpret_cast<float2*>(w + ws.ml);
  a.part_ml[1] = reinterpret_cast<float2*>(half(ws.ml, ws.next));
  a.part_next[0] = reinterpret_cast<int2*>(w + ws.next);
  a.part_next[1] = reinterpret_cast<int2*>(half(ws.next, ws.cont_o));
  a.cont_o = reinterpret_cast<float*>(w + ws.cont_o);
  a.cont_ml = reinterpret_cast<float2*>(w + ws.cont_ml);

  st = prefix_attention_tc_takes(a, dtype) ? launch_prefix_attention_tc(a, dtype, sms, stream)
                                           : launch_prefix_attention_fma(a, dtype, sms, stream);
  if (st != GFST_OK) return st;
  if (dtype == GFST_F32) return launch_merge<float>(a, stream);
  if (dtype == GFST_BF16) return launch_merge<__nv_bfloat16>(a, stream);
  return launch_merge<__half>(a, stream);
}
