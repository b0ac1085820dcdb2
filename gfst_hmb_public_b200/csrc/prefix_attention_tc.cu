// Shared-prefix attention on the 5th-generation tensor cores: bf16 or fp16,
// d = dv = 64 or 128, blocks that tile 128 keys (L a divisor of 128 from 8 up,
// or a multiple of 128).
//
// A CTA (one per SM) runs two streams, each with a 128-row query tile, over units
// of 64 keys (half of a 128-key stage):
//   S = Q K^T     tcgen05.mma, both operands in shared memory, S in one of two TMEM
//                 buffers, so that the next unit's scores are there in time
//   P = 2^(c S - m) by four warps, one row per thread, rounded to the pools'
//                 type and stored back to TMEM over S
//   O += P V      tcgen05.mma, P from TMEM, V from shared memory (keys along
//                 the contraction: V is the MN-major operand), O in TMEM
// While one stream's rows are exponentiated, the other's products run.  For a unit
// of both streams at d = 128 the products take 1230 tensor cycles (S 384: its
// operands come from shared memory at 128 bytes a cycle; O 230) and the 16,384
// exponentials 1024 cycles of the SM's special-function units; a unit takes 1930,
// because a thread's loads, maximum, exponentials, sums and stores follow one
// another and there is room for two such warps on a quarter of the SM.
//
// Measured, bf16, d = 128, device time with the merge (graph replays, SMs near 1.9
// GHz; calls one after another under the power limit in brackets): 512 one-token
// requests behind 32,768 tokens (4 heads x 8) 344 us, 800 TFLOP/s (377 us); prompt
// pieces of 12 requests behind 4096 tokens (8 x 4) 876 us, 837 TFLOP/s (965 us); 16
// requests of 4096 to 32,767 tokens 142 us, 5.8 TB/s (162 us); 64 requests behind
// 8192 tokens 47 us (49 us).  Tried and slower: two threads a
// row, each with half of the keys, that exchange maxima (the same for the document,
// 7 % slower for prompts); a polynomial in place of some exponentials; tiles
// prefetched into L2.
//
// Two kinds of work (prefix_attention.cuh), each cut evenly over the CTAs:
//   pairs   items of more than 128 rows: both streams take the same K and V
//           tiles (one load for 256 rows), through a ring of all stages
//   rest    items of up to 128 rows: every stream walks its own share with its
//           own stages, so two items are in flight on an SM
//
// Warps: 0-3 and 4-7 softmax of stream 0 and 1 (warp w reads TMEM lanes 32 (w %
// 4) ..); 8, 9 the streams' producers (work list, K and V by TMA, one box per block
// and 64 columns, queries by cp.async but for the first part's, which the softmax
// warps fetch); 10, 11 their MMA issuers.
//
// The maximum is followed lazily: m only moves when a row's new maximum exceeds
// it by more than 8 (in log2), so O in TMEM is rescaled a few times per row and
// not once a tile; sums then stay below 2^8 times their keys, exact softmax all
// the same because every term uses the same m.  For fp16 the reference is
// lowered by 7, so that p lies in [2^7, 2^15] at the top and the smallest
// weights keep their bits.
//
// Masked keys get p = 0 by selection.  Since 0 * (inf or NaN) is NaN in the
// product, value rows behind the last key are zeroed in shared memory, and a
// value row that only some of the tile's rows see and that is not finite is
// taken out of the product and added by the threads whose rows see it.
//
// Every wait is bounded; one that gives up sets the CTA's abort flag, every role
// leaves its loop, copies in flight are waited for, TMEM is freed and the sticky
// error word records GFST_ERR_TIMEOUT.
#include <cuda_fp16.h>

#include "prefix_attention.cuh"
#include "umma.cuh"

namespace gfst {

GFST_DEFINE_ERROR_WORD(g_attn_tc_error, take_attn_tc_error, "attention")

namespace {

// a status recorded as the kernel records it
__global__ void attn_tc_error_kernel(int status) { atomicMax(&g_attn_tc_error, (unsigned)status); }

constexpr int kHalf = kAttnTcHalf;  // rows of a stream's tile
constexpr int kKeys = 128;          // keys of a tile (a stage)
constexpr int kUnit = 64;           // keys of a score buffer
constexpr int kThreads = 384;
constexpr int kProducer = 8, kMma = 10;
constexpr int kItems = 4;           // parts announced ahead
constexpr uint32_t kTmemCols = 512; // per stream: S (P over it) 128, O 128
constexpr float kLazy = 8.f;

constexpr int kJoinRows = 16;                         // rows of joining copies staged at a time
constexpr int kStageBytes = 2 * kJoinRows * 128 * 4;  // a stream's rows of joining copies (copies_of)

// Costs in units of about 500 cycles of a CTA, from measured parts: a 256-row
// tile takes about 4200 cycles; of the rest two streams run at once, so a tile of
// 3400 counts 1700 and an item's 8000 (queries in, first scores, partials out)
// count 4000.  A pair's item alone would count 16,000, but 48 units spread the work
// better: with 30, prompt pieces took 929 us for 868; with 60, drafted tokens 45.5
// for 41.6; from 22 to 60 the other cases are within 2 %.
using Pairs = AttnCutPairs<kHalf, kKeys, 48, 8>;
using Rest = AttnCutRest<kHalf, kKeys, 8, 3>;

template <int D>
struct TcAttn {
  static constexpr int NC = D / 64;                // 64-column chunks (128-byte swizzle rows)
  static constexpr int TILE_BYTES = NC * 128 * 128;  // a 128-row tile of Q, K or V
  static constexpr int NS = D == 64 ? 4 : 2;       // stages of a stream
  static constexpr int RING = 2 * NS;              // stages of the pairs' ring
  static constexpr int Q_OFF = 0;
  static constexpr int KV_OFF = 2 * TILE_BYTES;
  static constexpr int STAGE_OFF = KV_OFF + RING * TILE_BYTES;  // rows of joining copies
  static constexpr int CTRL_OFF = STAGE_OFF + 2 * kStageBytes;
};

struct StreamCtrl {
  uint64_t item_full[kItems], item_empty[kItems];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_ready[2], pv_done[2];  // of the two score buffers
  uint64_t care;               // the softmax warps among themselves
  uint64_t full[4], empty[4];  // the stream's own stages
  AttnPart item[kItems];
  int paired[kItems];          // 1: pair, 0: rest, -1: no more work
  uint32_t bad[2][4];          // value rows that are not finite (one bit each), two tiles in turn
  int accumulate;              // the part's first product adds to O
  float2 ml[2][32];            // joining copies' references and sums
};
struct Ctrl {
  StreamCtrl s[2];
  uint64_t full[8], empty[8];  // the pairs' ring
  uint64_t care;                 // both streams' softmax warps
  uint64_t done[2];              // a stream's products are done
  int64_t sum[2][32];
  AttnLine<Pairs> pairs;         // the lines (their common part)
  AttnLine<Rest> rest;
  AttnShares shares;
  AttnWalk<Pairs> walk_pairs;    // where the shares begin
  AttnWalk<Rest> walk_rest[2];
  int gone[2][4];                // softmax warps of pairs that have left
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Weights take the pools' 16-bit type: both operands of a product have one, and V
// is read as it lies in the pool.  Half a step of a weight (bf16 2^-8, fp16 2^-11)
// beside half a step of the output: against 64 bits the outputs are off by 2.3e-3
// (fp16 2.9e-4) where 32-bit weights would leave 1.7e-3 (2.1e-4).  Weights in two
// 16-bit parts would double the second product; 32-bit pools round none.  The sums
// l are of the weights before this rounding.
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
  uint32_t r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
  tmem_st32(taddr, r);
}
__device__ __forceinline__ float tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  return __uint_as_float(r);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// D[tmem] += A[tmem] B[smem]
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 128B-swizzled, MN-major operand: 64-element column chunks `chunk` bytes apart,
// groups of 8 contraction rows 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t chunk) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(chunk >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16 instruction descriptor, 128 x N, A and B of one 16-bit type; b_mn: B is MN-major
__host__ __device__ constexpr uint32_t idesc16(bool f16, int N, bool b_mn) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}

// the lane that issues for its warp (always the same one)
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// One role's waits.  A wait that gives up, or finds that another role has, sets
// the CTA's abort flag and is false.
struct Waiter {
  volatile int* abort;
  __device__ __forceinline__ bool spin(uint64_t* bar, uint32_t parity) const {
    const long long t0 = clock64();
    for (int i = 1; !mbar_try_wait(bar, parity); ++i) {
      if ((i & 15) == 0 && (*abort != 0 || clock64() - t0 > kMbarWaitCycles)) {
        *abort = 1;
        return false;
      }
    }
    return true;
  }
  // the whole warp waits; lanes leave together
  __device__ __forceinline__ bool warp(uint64_t* bar, uint32_t parity) const {
    const bool ok = mbar_try_wait(bar, parity);
    if (__all_sync(0xffffffffu, ok)) return true;
    return __all_sync(0xffffffffu, ok || spin(bar, parity));
  }
};

// An item of few rows would leave most softmax threads idle and one warp with all
// 64 scores of a unit to exponentiate.  Up to 32 rows are laid out twice in the
// query tile (64 rows apart): the products give both copies all scores, copy k
// takes only its 32 keys of each unit (its other weights are 0), and the copies'
// rows, softmaxes over disjoint keys, are joined when the part ends.  (64 requests
// behind 8192 tokens 47.6 us for 50.8 with one copy, 16 long ones 140 for 145; up to
// six drafted tokens 41.7 for 41.0.)
__device__ __forceinline__ int copies_of(int paired, int rows) { return paired || rows > 32 ? 1 : 2; }

// Query rows [r0, r1) of a stream's tile by one warp, swizzled as TMA would: a lane
// finds a row's place, then whole rows are copied, D / 8 lanes a row.
template <int D>
__device__ __forceinline__ void copy_queries(const AttnArgs& a, const AttnPart& it, int paired, int j, uint8_t* sq,
                                             int r0, int r1) {
  const int lane = threadIdx.x & 31;
  const int r_first = paired ? j * kHalf : 0, rows = min(kHalf, it.rows - r_first);
  const int copies = copies_of(paired, it.rows);
  constexpr int PIECES = D / 8, ROWS = 32 / PIECES;  // rows of a step
  const int v = lane % PIECES, sub = lane / PIECES;
  const uint32_t col = smem_u32(sq) + (v >> 3) * (128 * 128);
  r1 = min(r1, rows);
#pragma unroll 1
  for (; r0 < r1; r0 += 32) {
    int tok, hq;
    attn_row(a, it, r_first + min(r0 + lane, rows - 1), tok, hq);
    const int64_t at = tok * a.q_st + hq * a.q_sh;
#pragma unroll 4
    for (int x = 0; x < 32; x += ROWS) {
      const int r = r0 + x + sub;
      const uint16_t* src = static_cast<const uint16_t*>(a.Q) + __shfl_sync(0xffffffffu, at, x + sub) + v * 8;
      const uint32_t dst = col + r * 128 + (((v & 7) ^ (r & 7)) << 4);
      if (r < rows) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
        if (copies > 1)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + (kHalf / 2) * 128), "l"(src) : "memory");
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  fence_async_smem();
  __syncwarp();
}

// One softmax thread: a row of its stream's tile.
template <int D, bool F16>
struct Softmax {
  using TC = TcAttn<D>;
  static constexpr int NS = TC::NS, RING = TC::RING, NC = TC::NC, TILE = TC::TILE_BYTES;
  static constexpr float kBias = F16 ? 7.f : 0.f;
  const AttnArgs& a;
  Ctrl* ctl;
  uint8_t* smem;
  const int j, quad, lane, tid;
  StreamCtrl& c;
  const uint32_t tS, tO;
  const Waiter wait;
  uint32_t n_tile = 0, n_unit = 0, n_own = 0, n_ring = 0, n_care = 0, n_care2 = 0;

  __device__ __forceinline__ Softmax(const AttnArgs& a_, Ctrl* ctl_, uint8_t* smem_, uint32_t tmem, int j_)
      : a(a_), ctl(ctl_), smem(smem_), j(j_), quad((threadIdx.x >> 5) & 3), lane(threadIdx.x & 31),
        tid(threadIdx.x & 127), c(ctl_->s[j_]), tS(tmem + j_ * 256 + ((uint32_t)(quad * 32) << 16)), tO(tS + 128),
        wait{&ctl_->abort} {}

  // a bounded barrier of the stream's softmax warps, for a pair of both streams'
  __device__ __forceinline__ bool meet(int paired) {
    __syncwarp();
    uint64_t* bar = paired ? &ctl->care : &c.care;
    uint32_t& n = paired ? n_care2 : n_care;
    if (lane == 0) mbar_arrive(bar);
    return wait.warp(bar, n++ & 1);
  }
  // A pair's streams tend to reach their exponentials together, share the
  // special-function units and then leave them idle through the rest (the slow
  // CTAs of a launch took 650,000 cycles where the others took 450,000).  Warps w
  // and w + 4, on the same quarter of the SM, take turns instead, stream 0 first:
  // named barriers of the two warps, 1 + quad for stream 0's turn and 5 + quad
  // for stream 1's (through an mbarrier a handover took 200 cycles more).  A warp
  // that gives up sets the abort flag and goes on giving turns until the other
  // one, which looks at the flag before it takes one, has left too (turn_leave).
  __device__ __forceinline__ void turn_give() const {
    asm volatile("barrier.cta.arrive %0, 64;" ::"r"(1 + (j ^ 1) * 4 + quad) : "memory");
  }
  __device__ __forceinline__ bool turn_take() const {
    if (__any_sync(0xffffffffu, *wait.abort != 0)) return false;
    asm volatile("barrier.cta.sync %0, 64;" ::"r"(1 + j * 4 + quad) : "memory");
    return true;
  }
  // After the pairs; ok: this warp did all its work.  Bounded by a few seconds:
  // the other warp's waits are.
  __device__ __forceinline__ void turn_leave(bool ok) const {
    if (ok && j == 0) ok = turn_take();  // the turn that stream 1 gave last
    volatile int* gone = &ctl->gone[0][0];
    if (lane == 0) gone[j * 4 + quad] = 1;
    for (int i = 0; !ok && i < 4000000; ++i) {
      if (__any_sync(0xffffffffu, gone[(j ^ 1) * 4 + quad] != 0)) break;
      turn_give();
      __nanosleep(1000);
    }
  }
  __device__ __forceinline__ void zero_row(uint8_t* vs) const {
#pragma unroll
    for (int i = 0; i < NC * 8; ++i)
      *reinterpret_cast<uint4*>(vs + (i >> 3) * (128 * 128) + tid * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  // O += p v for the value row k, over this thread's row (fresh: O holds nothing yet)
  __device__ __forceinline__ void add_row(const uint8_t* vs, int k, float p, bool add, bool fresh) const {
#pragma unroll 1
    for (int i = 0; i < D; i += 32) {
      float o[32];
      tmem_ld32(tO + i, o);
      tmem_wait_ld();
#pragma unroll
      for (int q = 0; q < 32; q += 8) {
        const int col = i + q;
        const uint4 v = *reinterpret_cast<const uint4*>(vs + (col >> 6) * (128 * 128) + k * 128 +
                                                        ((((col & 63) >> 3) ^ (k & 7)) << 4));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float lo, hi;
          if constexpr (F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[x]));
            lo = f.x, hi = f.y;
          } else {
            lo = bf16_lo(w[x]), hi = bf16_hi(w[x]);
          }
          const float a0 = fresh ? 0.f : o[q + 2 * x], a1 = fresh ? 0.f : o[q + 2 * x + 1];
          o[q + 2 * x] = add ? fmaf(p, lo, a0) : a0;
          o[q + 2 * x + 1] = add ? fmaf(p, hi, a1) : a1;
        }
      }
      tmem_st32(tO + i, o);
      tmem_wait_st();
    }
  }

  // C: copies of the rows
  template <int C>
  __device__ __forceinline__ bool part(const AttnPart& it, int paired) {
    constexpr int copies = C, N = kUnit / C;              // N: keys of a unit that this thread takes
    const int copy = copies > 1 ? tid >> 6 : 0;
    const int r = copies > 1 ? tid & 63 : (paired ? j * kHalf : 0) + tid;  // row of the item
    const bool live = r < it.rows;
    const bool warp_live = __any_sync(0xffffffffu, live);
    const float scale = a.scale_log2;
    const int key_off = copy * N;
    // keys this row sees, and the first row of the item (fewest)
    const int sees = it.own ? min(it.len, it.see0 + (it.row0 + r) / a.G + 1) : it.len;
    const int fewest = it.own ? min(it.len, it.see0 + it.row0 / a.G + 1) : it.len;
    const uint32_t stages = paired ? RING : NS;
    uint64_t* fulls = paired ? ctl->full : c.full;
    float m = -INFINITY, l = 0.f;                        // m: reference, bias included
#pragma unroll 1
    for (int t = it.t0; t < it.t1; ++t) {
      const uint32_t n = (paired ? n_ring : n_own) + 1;  // the value stage (for tiles that need care)
      const uint32_t v_stage = n % stages;
      uint8_t* vs = smem + TC::KV_OFF + ((paired ? 0 : j * NS) + v_stage) * TILE;
      n_ring += paired ? 2 : 0;
      n_own += paired ? 0 : 2;
      const bool care = t * kKeys + kKeys > fewest;
      uint32_t any_bad = 0;
      const int units = it.len - t * kKeys > kUnit ? 2 : 1;
#pragma unroll 1
      for (int u = 0; u < units; ++u, ++n_unit) {
        const uint32_t buf = n_unit & 1;
        const uint32_t tP = tS + buf * kUnit;
        const bool first_unit = t == it.t0 && u == 0;
        const int seen = sees - (t * kKeys + u * kUnit + key_off);  // of this thread's keys, those the row sees
        // O as the products up to the last unit left it (they may still run)
        auto o_stable = [&]() -> bool {
          if (first_unit) return true;
          const bool done = wait.warp(&c.pv_done[buf ^ 1], ((n_unit - 1) >> 1) & 1);
          tc_fence_after();
          return done;
        };
        if (!wait.warp(&c.s_full[buf], (n_unit >> 1) & 1)) return false;
        tc_fence_after();
        float2 x[N / 2];
        if (warp_live) {
          float s[N];
#pragma unroll
          for (int q = 0; q < N; q += 32) tmem_ld32(tP + key_off + q, s + q);
          tmem_wait_ld();
          if (care) {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] = i < seen ? s[i] : -INFINITY;
          }
          float m0 = s[0], m1 = s[1], m2 = s[2], m3 = s[3];
#pragma unroll
          for (int i = 4; i < N; i += 4) {
            m0 = fmaxf(m0, s[i]), m1 = fmaxf(m1, s[i + 1]);
            m2 = fmaxf(m2, s[i + 2]), m3 = fmaxf(m3, s[i + 3]);
          }
#pragma unroll
          for (int i = 0; i < N / 2; ++i) x[i] = make_float2(s[2 * i], s[2 * i + 1]);
          const float top = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * scale - kBias;
          const bool move = live && top > m + kLazy;
          if (__any_sync(0xffffffffu, move)) {
            const float al = move ? ex2(m - top) : 1.f;  // m = -inf: 0
            if (move) m = top;
            l *= al;
            if (!first_unit) {
              if (!o_stable()) return false;
#pragma unroll 1
              for (int i = 0; i < D; i += 32) {
                float o[32];
                tmem_ld32(tO + i, o);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] *= al;
                tmem_st32(tO + i, o);
              }
              tmem_wait_st();
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
        if (care) {
          uint32_t* bad = c.bad[n_tile & 1];
          if (u == 0) {
            // values: rows behind the last key become zero; rows that only some
            // query rows see are looked at
            if (!wait.warp(&fulls[v_stage], (n / stages) & 1)) return false;
            const int valid = min(kKeys, it.len - t * kKeys), from = fewest - t * kKeys;
            if (tid >= valid) zero_row(vs);
            if (from < valid) {
              bool odd = false;
              if (tid >= from && tid < valid) {
                constexpr uint32_t E = F16 ? 0x7c00u : 0x7f80u;
#pragma unroll 1
                for (int i = 0; i < NC * 8; ++i) {
                  const uint4 v = *reinterpret_cast<const uint4*>(vs + (i >> 3) * (128 * 128) + tid * 128 + (i & 7) * 16);
                  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                  for (int q = 0; q < 4; ++q) odd |= (w[q] & E) == E || ((w[q] >> 16) & E) == E;
                }
              }
              const uint32_t mask = __ballot_sync(0xffffffffu, odd);
              if (lane == 0) bad[quad] = mask;
              // both streams of a pair look at the same rows of the same stage
              if (!meet(paired)) return false;
              any_bad = bad[0] | bad[1] | bad[2] | bad[3];
            }
          }
          if (any_bad != 0) {
            if (!o_stable()) return false;
            bool fresh = first_unit;
#pragma unroll 1
            for (int k = u * kUnit; k < u * kUnit + kUnit; ++k) {
              if (!((bad[k >> 5] >> (k & 31)) & 1)) continue;
              if (tid == 0 && first_unit) c.accumulate = 1;
              if (warp_live) {
                const float sk = tmem_ld1(tP + (k - u * kUnit));
                tmem_wait_ld();
                const int mine = k - u * kUnit - key_off;
                const bool add = mine >= 0 && mine < N && mine < seen;
                add_row(vs, k, add ? ex2(fmaf(sk, scale, -base)) : 0.f, add, fresh);
              }
              fresh = false;
            }
            if (!meet(paired)) return false;  // every row has read them
            if ((tid >> 6) == u && ((bad[quad] >> lane) & 1)) zero_row(vs);
          }
          fence_async_smem();
        }
        if (warp_live) {
          const float2 sc = make_float2(scale, scale), nb = make_float2(-base, -base);
          if (paired && !turn_take()) return false;
#pragma unroll
          for (int i = 0; i < N / 2; ++i) x[i] = ffma2(x[i], sc, nb);
#pragma unroll
          for (int i = 0; i < N / 2; ++i) {
            x[i].x = ex2(x[i].x);
            x[i].y = ex2(x[i].y);
          }
          float2 sum0 = x[0], sum1 = x[1];
#pragma unroll
          for (int i = 2; i < N / 2; i += 2) {
            sum0 = __fadd2_rn(sum0, x[i]);
            sum1 = __fadd2_rn(sum1, x[i + 1]);
          }
          if (paired) turn_give();
          // weights go over scores already taken
#pragma unroll
          for (int q = 0; q < N / 2; q += 16) {
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = pack2<F16>(x[q + i].x, x[q + i].y);
            tmem_st16(tP + key_off / 2 + q, p);
          }
          if constexpr (C > 1) {
            const uint32_t zero[16] = {};
            tmem_st16(tP + (copy ^ 1) * 16, zero);
          }
          l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
          tmem_wait_st();
        } else if (paired) {
          if (!turn_take()) return false;
          turn_give();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&c.p_ready[buf]);
      }
      n_tile += care ? 1 : 0;
    }
    // the part's last product, then its rows out.  Continuation rows: the pairs'
    // of all CTAs, then the workers' of the rest
    const int64_t crow0 = paired ? (int64_t)blockIdx.x * (2 * kHalf)
                                 : (int64_t)gridDim.x * (2 * kHalf) +
                                       (int64_t)ctl->shares.rest_worker(blockIdx.x, j) * kHalf;
    const int stride = paired ? 2 * kHalf : kHalf;
    auto put = [&](int r_, float2 ml, bool write) -> float* {  // a row's (m, l) out; where its values go
      int tok, hq;
      attn_row(a, it, r_, tok, hq);
      const int64_t row = (int64_t)tok * (a.H * a.G) + hq;
      if (it.first) {
        if (write) {
          a.part_ml[it.own][row] = ml;
          a.part_next[it.own][row] = attn_next((int)(crow0 + r_ + stride), it.n_cont, stride);
        }
        return a.part_o[it.own] + row * D;
      }
      if (write) a.cont_ml[crow0 + r_] = ml;
      return a.cont_o + (crow0 + r_) * D;
    };
    // A later piece: what is there of a row, all lanes' own writes, joined with the
    // new (m, l); `ml` becomes the joined one.
    auto join = [&](int r_, float2& ml) -> AttnJoin {
      int tok, hq;
      attn_row(a, it, r_, tok, hq);
      const AttnJoin j(it.first ? a.part_ml[it.own][(int64_t)tok * (a.H * a.G) + hq] : a.cont_ml[crow0 + r_], ml);
      ml = j.ml;
      return j;
    };
    auto joined = [](float4 u, float keep, float4 v, float f) {
      return make_float4(fmaf(u.x, keep, v.x * f), fmaf(u.y, keep, v.y * f), fmaf(u.z, keep, v.z * f),
                         fmaf(u.w, keep, v.w * f));
    };
    if (!wait.warp(&c.pv_done[(n_unit - 1) & 1], ((n_unit - 1) >> 1) & 1)) return false;
    tc_fence_after();
    // only here: that product waited for this part's weights of all four warps, which
    // by then were done with the last part's references (read behind the next meeting)
    if (C > 1 && live) c.ml[copy][r] = make_float2(m, l);
    if constexpr (C == 1) {
      if (warp_live) {
        // 32 columns of the warp's 32 rows at a time through shared memory, so that
        // a store writes whole 128-byte lines (four rows) and not 32 sectors
        float4* st = reinterpret_cast<float4*>(smem + TC::STAGE_OFF + j * kStageBytes) + quad * (32 * 8);
        float2 ml = make_float2(m, l);
        float keep = 0.f, f = 1.f;
        if (it.again && live) {
          const AttnJoin jn = join(r, ml);
          keep = jn.fa, f = jn.fb;
        }
        float* dst = live ? put(r, ml, true) : nullptr;
#pragma unroll 1
        for (int i = 0; i < D; i += 32) {
          float o[32];
          tmem_ld32(tO + i, o);
          tmem_wait_ld();
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k)
            st[lane * 8 + (k ^ (lane & 7))] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          __syncwarp();
          auto row_to = [&](int row) {
            float* to = reinterpret_cast<float*>(
                __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), row));
            return to == nullptr ? nullptr : reinterpret_cast<float4*>(to + i + (lane & 7) * 4);
          };
          if (it.again) {  // (apart: drafted tokens took 44.4 us for 42.3 with it in the loop below)
#pragma unroll 1
            for (int k = 0; k < 8; ++k) {
              const int row = k * 4 + (lane >> 3);
              const float k0 = __shfl_sync(0xffffffffu, keep, row), f0 = __shfl_sync(0xffffffffu, f, row);
              float4* to = row_to(row);
              if (to != nullptr) *to = joined(*to, k0, st[row * 8 + ((lane & 7) ^ (row & 7))], f0);
            }
            continue;
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int row = k * 4 + (lane >> 3);
            float4* to = row_to(row);
            const float4 v = st[row * 8 + ((lane & 7) ^ (row & 7))];
            if (to != nullptr) *to = v;
          }
        }
      }
    } else {
      // both copies through shared memory, 16 rows at a time; the four warps join
      // them at the larger reference, a row of D values a warp.  (The next part
      // writes the stage and c.ml behind its last product, which waits for all four
      // warps' weights.)
      constexpr int P = D / 4;                           // 16-byte pieces of a row
      float4* st = reinterpret_cast<float4*>(smem + TC::STAGE_OFF + j * kStageBytes);
#pragma unroll 1
      for (int r0 = 0; r0 < it.rows; r0 += kJoinRows) {
        if (r0 > 0 && !meet(0)) return false;            // the rows before are out
        const bool mine = live && r >= r0 && r < r0 + kJoinRows;
        if (__any_sync(0xffffffffu, mine)) {
#pragma unroll 1
          for (int i = 0; i < D; i += 32) {
            float o[32];
            tmem_ld32(tO + i, o);
            tmem_wait_ld();
            if (mine) {
              float4* dst = st + (copy * kJoinRows + r - r0) * P;
#pragma unroll
              for (int k = 0; k < 32; k += 4)  // pieces in an order that spreads the rows over the banks
                dst[((i + k) / 4) ^ (r & 7)] = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            }
          }
        }
        if (!meet(0)) return false;
        const int rows = min(kJoinRows, it.rows - r0);
#pragma unroll 1
        for (int x = quad; x < rows; x += 4) {
          const float2 v0 = c.ml[0][r0 + x], v1 = c.ml[1][r0 + x];
          const float mx = fmaxf(v0.x, v1.x);
          // equal references (both empty: -inf) need no exponential
          const float f0 = v0.x == mx ? 1.f : ex2(v0.x - mx), f1 = v1.x == mx ? 1.f : ex2(v1.x - mx);
          float2 ml = make_float2(mx, fmaf(v0.y, f0, v1.y * f1));
          if (it.again) {
            const AttnJoin jn = join(r0 + x, ml);
            __syncwarp();  // all lanes have read what lane 0 writes
            float* dst = put(r0 + x, ml, lane == 0);
            if (lane < P) {
              float4* to = reinterpret_cast<float4*>(dst + lane * 4);
              *to = joined(*to, jn.fa,
                           joined(st[x * P + (lane ^ (x & 7))], f0, st[(kJoinRows + x) * P + (lane ^ (x & 7))], f1),
                           jn.fb);
            }
            continue;
          }
          float* dst = put(r0 + x, ml, lane == 0);
          if (lane < P)
            *reinterpret_cast<float4*>(dst + lane * 4) =
                joined(st[x * P + (lane ^ (x & 7))], f0, st[(kJoinRows + x) * P + (lane ^ (x & 7))], f1);
        }
      }
    }
    tc_fence_before();
    return true;
  }
};

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_attention_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                               const __grid_constant__ AttnArgs a, int64_t pool_rows) {
  using TC = TcAttn<D>;
  constexpr int NS = TC::NS, RING = TC::RING, NC = TC::NC, TILE = TC::TILE_BYTES;
  extern __shared__ __align__(1024) uint8_t smem[];  // tiles in 1024-byte swizzle atoms
  Ctrl* ctl = reinterpret_cast<Ctrl*>(smem + TC::CTRL_OFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((smem_u32(smem) & 1023u) != 0) {  // cannot be: no other shared memory
    if (threadIdx.x == 0) atomicMax(&g_attn_tc_error, (unsigned)GFST_ERR_ALIGN);
    return;
  }

  // Everything up to here and the barriers touch no memory of earlier work, so
  // they run while the launch before this one ends.
  if (lane == 0 && warp < 2) {
    StreamCtrl& c = ctl->s[warp];
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&c.item_full[i], 1);
      mbar_init(&c.item_empty[i], 5);  // four softmax warps, the MMA warp
    }
    mbar_init(&c.q_full, 4);
    mbar_init(&c.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c.s_full[i], 1);
      mbar_init(&c.p_ready[i], 4);
      mbar_init(&c.pv_done[i], 1);
    }
    mbar_init(&c.care, 4);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&c.full[i], 1);
      mbar_init(&c.empty[i], 1);
    }
    c.accumulate = 0;
    mbar_init(&ctl->done[warp], 1);
    mbar_init_fence();
  } else if (lane == 0 && warp == 2) {
    for (int i = 0; i < 8; ++i) {
      mbar_init(&ctl->full[i], 1);
      mbar_init(&ctl->empty[i], 2);  // both streams' products
    }
    mbar_init(&ctl->care, 8);
    for (int i = 0; i < 8; ++i) (&ctl->gone[0][0])[i] = 0;
    ctl->abort = 0;
    mbar_init_fence();
  }
  if (warp == kMma) tmem_alloc(&ctl->tmem, kTmemCols);
  if (warp == kProducer && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmK)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmV)) : "memory");
  }
  tc_fence_before();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // the work: this CTA's share of the pairs, and its streams' shares of the rest
  {
    AttnLine<Pairs> pl;
    AttnLine<Rest> rl;
    attn_lines<kThreads / 32>(a, ctl->sum, pl, rl);
    AttnShares sh;
    sh.init(pl.U, rl.U, gridDim.x, Pairs::C0 + Pairs::W, Rest::C0 + Rest::W);
    if (blockIdx.x < sh.pairs.n) {
      AttnWalk<Pairs>::find(a, pl, sh.pairs.bound(blockIdx.x), sh.pairs.bound(blockIdx.x + 1), &ctl->walk_pairs);
    } else {
      for (int j = 0; j < 2; ++j) {
        const int w = sh.rest_worker(blockIdx.x, j);
        if (w >= 0) AttnWalk<Rest>::find(a, rl, sh.rest.bound(w), sh.rest.bound(w + 1), &ctl->walk_rest[j]);
      }
    }
    // (different warps: they run side by side)
    if (threadIdx.x == 32) ctl->pairs = pl;
    if (threadIdx.x == 64) ctl->rest = rl;
    if (threadIdx.x == 96) ctl->shares = sh;
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;

  const Waiter wait{&ctl->abort};
  uint32_t issued_own = 0, issued_ring = 0;  // stages filled by this producer (for the drain)

  // the softmax threads hold 64 scores: they take registers from the other four
  // warps (2 x 128 x 208 + 128 x 88 of the 384 x 168 launched)
  if (warp >= kProducer) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp < kMma) {
    // ------------------------------------------------------------- producer
    const int j = warp - kProducer;
    StreamCtrl& c = ctl->s[j];
    uint8_t* sq = smem + TC::Q_OFF + j * TILE;
    uint32_t n_item = 0;
    bool bad = false, ok = true;

    // one part: announce it, its queries, its keys and values (for pairs the
    // first stream's producer loads them for both)
    auto part = [&](const AttnPart& it, int paired) -> bool {
      const int slot = n_item % kItems;
      if (!wait.warp(&c.item_empty[slot], ((n_item / kItems) & 1) ^ 1)) return false;
      if (lane == 0) {
        c.item[slot] = it;
        c.paired[slot] = paired;
        mbar_arrive(&c.item_full[slot]);
      }
      // queries of this stream; those of its first part come by the softmax warps
      auto queries = [&]() -> bool {
        if (n_item == 0) return true;
        if (!wait.warp(&c.q_empty, (n_item & 1) ^ 1)) return false;
        copy_queries<D>(a, it, paired, j, sq, 0, kHalf);
        if (lane < 4) mbar_arrive(&c.q_full);
        return true;
      };
      if (paired && j == 1) {
        const bool sent = queries();
        ++n_item;
        return sent;
      }
      const int box = min(a.L, kKeys);         // rows of a copy
      const int boxes = kKeys / box;           // copies of a full tile, one per lane
      auto block_row = [&](int t) -> int64_t {  // pool row of this lane's box in tile t
        const int p = t * kKeys + lane * box;
        if (lane >= boxes || p >= it.len) return -1;
        const int idx = p / a.L;
        const int blk = attn_block(a, it, idx);
        // an entry outside the pool: a row behind its end, which TMA fills with zeros
        if (blk < 0) return pool_rows;
        return ((int64_t)blk * a.H + it.h) * a.L + (p - idx * a.L);
      };
      int64_t row = block_row(it.t0);
      for (int t = it.t0; t < it.t1; ++t) {
        const int64_t ahead = t + 1 < it.t1 ? block_row(t + 1) : -1;
        if (row == pool_rows) bad = true;
        const int n = __popc(__ballot_sync(0xffffffffu, row >= 0));
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          uint64_t *full, *empty;
          uint8_t* dst;
          uint32_t parity;
          if (paired) {
            const uint32_t st = issued_ring % RING;
            full = &ctl->full[st], empty = &ctl->empty[st];
            parity = (issued_ring / RING) & 1;
            dst = smem + TC::KV_OFF + st * TILE;
            ++issued_ring;
          } else {
            const uint32_t st = issued_own % NS;
            full = &c.full[st], empty = &c.empty[st];
            parity = (issued_own / NS) & 1;
            dst = smem + TC::KV_OFF + (j * NS + st) * TILE;
            ++issued_own;
          }
          if (!wait.warp(empty, parity ^ 1)) {
            if (paired) --issued_ring;
            else --issued_own;
            return false;
          }
          if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(n * box * NC * 128));
          __syncwarp();
          if (row >= 0) {
#pragma unroll
            for (int ch = 0; ch < NC; ++ch)
              tma_load_2d(dst + ch * (128 * 128) + lane * box * 128, kv ? &tmV : &tmK, full, ch * 64, (int)row);
          }
          if (kv == 0 && t == it.t0 && !queries()) return false;  // while the first keys are on their way
        }
        row = ahead;
      }
      ++n_item;
      return true;
    };

    AttnPart it;
    const AttnShares& sh = ctl->shares;
    if (blockIdx.x < sh.pairs.n) {
      AttnWalk<Pairs> w = ctl->walk_pairs;
#pragma unroll 1
      while (ok && w.next(a, ctl->pairs, [&](int64_t p) { return sh.pairs.worker_of(p); }, it)) ok = part(it, 1);
    } else if (sh.rest_worker(blockIdx.x, j) >= 0) {
      AttnWalk<Rest> w = ctl->walk_rest[j];
#pragma unroll 1
      while (ok && w.next(a, ctl->rest, [&](int64_t p) { return sh.rest.worker_of(p); }, it)) ok = part(it, 0);
    }
    const int slot = n_item % kItems;
    if (ok && wait.warp(&c.item_empty[slot], ((n_item / kItems) & 1) ^ 1) && lane == 0) {
      c.paired[slot] = -1;
      mbar_arrive(&c.item_full[slot]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (bad) atomicMax(&g_attn_tc_error, (unsigned)GFST_ERR_ARG);
  } else {
    // ------------------------------------------------------------------ MMA
    // the whole warp walks the loop on warp-uniform values (descriptors then come
    // from uniform registers); one elected lane issues
    const int j = warp - kMma;
    StreamCtrl& c = ctl->s[j];
    constexpr uint32_t idesc_s = idesc16(F16, kUnit, false), idesc_o = idesc16(F16, D, true);
    const uint32_t tbase = __shfl_sync(0xffffffffu, tmem, 0) + j * 256;
    const uint32_t tS = tbase, tO = tbase + 128;
    const uint32_t base = smem_u32(smem);
    const uint64_t q_desc = sw128_desc(base + TC::Q_OFF + j * TILE);
    const bool issuer = elect_one();
    uint32_t n_item = 0, n_unit = 0, n_own = 0, n_ring = 0;
    bool ok = true;
    while (ok) {
      const int slot = n_item % kItems;
      if (!wait.warp(&c.item_full[slot], (n_item / kItems) & 1)) break;
      const int paired = __shfl_sync(0xffffffffu, c.paired[slot], 0);
      if (paired < 0) break;
      const int t0 = __shfl_sync(0xffffffffu, c.item[slot].t0, 0), t1 = __shfl_sync(0xffffffffu, c.item[slot].t1, 0);
      const int len_of_slot = c.item[slot].len;
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.item_empty[slot]);
      if (!wait.warp(&c.q_full, n_item & 1)) break;
      const int len = __shfl_sync(0xffffffffu, len_of_slot, 0);
      ++n_item;
      const uint32_t stages = paired ? RING : NS;
      uint64_t* fulls = paired ? ctl->full : c.full;
      uint64_t* empties = paired ? ctl->empty : c.empty;
      const uint32_t stage0 = base + TC::KV_OFF + (paired ? 0 : j * NS * TILE);
      const uint32_t n0 = paired ? n_ring : n_own;  // stage number of the part's first tile
      n_ring += paired ? 2 * (t1 - t0) : 0;
      n_own += paired ? 0 : 2 * (t1 - t0);
      // units of 64 keys; the last tile has one if its second half holds no key
      const int units = 2 * (t1 - t0) - (len - (t1 - 1) * kKeys > kUnit ? 0 : 1);
      // scores of unit u, into buffer (n_unit + u) & 1: its weights two units ago
      // lie there, so their product has to be done
      auto scores = [&](int u) -> bool {
        const uint32_t n = n0 + 2 * (u >> 1), ks = n % stages, g = n_unit + u, buf = g & 1;
        if ((u & 1) == 0 && !wait.warp(&fulls[ks], (n / stages) & 1)) return false;
        if (g >= 2 && !wait.warp(&c.pv_done[buf], ((g >> 1) & 1) ^ 1)) return false;
        tc_fence_after();
        if (issuer) {
          const uint64_t k_desc = sw128_desc(stage0 + ks * TILE + (u & 1) * (kUnit * 128));
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
            umma_bf16(tS + buf * kUnit, q_desc + off, k_desc + off, idesc_s, kk > 0 ? 1u : 0u);
          }
          umma_commit(&c.s_full[buf]);
          if ((u & 1) || u == units - 1) umma_commit(&empties[ks]);
          if (u == units - 1) umma_commit(&c.q_empty);
        }
        __syncwarp();
        return true;
      };
      if (!(ok = scores(0))) break;
      for (int u = 0; u < units; ++u) {
        if (u + 1 < units && !(ok = scores(u + 1))) break;
        const uint32_t n = n0 + 2 * (u >> 1) + 1, vs = n % stages, g = n_unit + u, buf = g & 1;
        if ((u & 1) == 0 && !(ok = wait.warp(&fulls[vs], (n / stages) & 1))) break;
        if (!(ok = wait.warp(&c.p_ready[buf], (g >> 1) & 1))) break;
        tc_fence_after();
        uint32_t acc = 1;
        if (u == 0) acc = __shfl_sync(0xffffffffu, c.accumulate, 0);
        if (issuer) {
          const uint64_t v_desc = sw128_mn_desc(stage0 + vs * TILE, 128 * 128) + (u & 1) * (kUnit * 128 >> 4);
#pragma unroll
          for (int kk = 0; kk < kUnit / 16; ++kk)
            umma_ts(tO, tS + buf * kUnit + kk * 8, v_desc + kk * (2048 >> 4), idesc_o, kk > 0 ? 1u : acc);
          umma_commit(&c.pv_done[buf]);
          if ((u & 1) || u == units - 1) umma_commit(&empties[vs]);
          if (u == 0) c.accumulate = 0;
        }
        __syncwarp();
      }
      n_unit += units;
    }
    if (issuer) umma_commit(&ctl->done[j]);
    __syncwarp();
  }
  } else {
    // -------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int j = warp >> 2;
    StreamCtrl& c = ctl->s[j];
    Softmax<D, F16> sm(a, ctl, smem, tmem, j);
    // pairs: the first turn is stream 0's
    const bool turns = blockIdx.x < ctl->shares.pairs.n;
    if (turns && j == 1) sm.turn_give();
    bool ok = false;
    for (uint32_t n_item = 0;; ++n_item) {
      const int slot = n_item % kItems;
      if (!wait.warp(&c.item_full[slot], (n_item / kItems) & 1)) break;
      const int paired = c.paired[slot];
      if ((ok = paired < 0)) break;
      const AttnPart it = c.item[slot];
      __syncwarp();
      if (lane == 0) mbar_arrive(&c.item_empty[slot]);
      if (n_item == 0) {
        // nothing to do yet: these warps fetch the first queries, each its rows (the
        // producer, which is ahead later on, needs 2000 cycles for them)
        copy_queries<D>(a, it, paired, j, smem + TC::Q_OFF + j * TILE, (warp & 3) * 32, (warp & 3) * 32 + 32);
        if (lane == 0) mbar_arrive(&c.q_full);
      }
      if (!(copies_of(paired, it.rows) > 1 ? sm.template part<2>(it, 0) : sm.template part<1>(it, paired))) break;
    }
    if (turns) sm.turn_leave(ok);
  }
  __syncthreads();
  if (ctl->abort) {
    // copies that were issued and may still land
    if (warp >= kProducer && warp < kProducer + 2 && lane == 0) {
      StreamCtrl& c = ctl->s[warp - kProducer];
      for (uint32_t i = issued_own > NS ? issued_own - NS : 0; i < issued_own; ++i)
        mbar_wait(&c.full[i % NS], (i / NS) & 1);
      for (uint32_t i = issued_ring > RING ? issued_ring - RING : 0; i < issued_ring; ++i)
        mbar_wait(&ctl->full[i % RING], (i / RING) & 1);
    }
    __syncthreads();
  }
  if (warp == kMma) {
    for (int j = 0; j < 2; ++j) mbar_wait(&ctl->done[j], 0);
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (threadIdx.x == 0 && ctl->abort) atomicMax(&g_attn_tc_error, (unsigned)GFST_ERR_TIMEOUT);
}

template <int D, bool F16>
int launch(const AttnArgs& a, int sms, cudaStream_t stream) {
  constexpr int smem = TcAttn<D>::CTRL_OFF + (int)sizeof(Ctrl);
  static_assert(smem <= 227 * 1024, "shared memory");
  auto kern = prefix_attention_tc_kernel<D, F16>;
  static std::atomic<uint64_t> allowed{0};
  int st = attn_allow_smem(kern, smem, allowed);
  if (st != GFST_OK) return st;
  const int64_t rows = a.n_blocks * a.H * a.L;
  CUtensorMap mk, mv;
  const int box = a.L < kKeys ? a.L : kKeys;
  st = make_bf16_map(&mk, a.pool_K, (uint64_t)rows, D, box);  // 16-bit elements, copied as they are
  if (st == GFST_OK) st = make_bf16_map(&mv, a.pool_V, (uint64_t)rows, D, box);
  if (st != GFST_OK) return st;
  const int grid = sms < kAttnMaxGrid ? sms : kAttnMaxGrid;
  return attn_launch("prefix_attention_tc_kernel", kern, grid, kThreads, smem, stream, mk, mv, a, rows);
}

}  // namespace

// Whatever this kernel can compute it computes sooner than the FP32 units, down to
// the smallest call (2 requests behind 64 tokens, d = 64: 10.5 us for 16.9; 64
// behind 8192, d = 128: 47.6 for 505; 16 of up to 32,767 tokens: 140 for 432).
bool prefix_attention_tc_takes(const AttnArgs& a, int dtype) {
  return (dtype == GFST_BF16 || dtype == GFST_F16) && a.d == a.dv && (a.d == 64 || a.d == 128) &&
         ((a.L >= 8 && kKeys % a.L == 0) || a.L % kKeys == 0) && a.n_blocks * a.H * a.L < (1LL << 31) - kKeys &&
         a.scale_log2 > 0.f;  // the row maximum is taken before scaling
}

int launch_attn_tc_error(int status, cudaStream_t stream) {
  attn_tc_error_kernel<<<1, 1, 0, stream>>>(status);
  return check_launch("attn_tc_error_kernel");
}

int launch_prefix_attention_tc(const AttnArgs& a, int dtype, int sms, cudaStream_t stream) {
  const bool f16 = dtype == GFST_F16;
  if (a.d == 64) return f16 ? launch<64, true>(a, sms, stream) : launch<64, false>(a, sms, stream);
  return f16 ? launch<128, true>(a, sms, stream) : launch<128, false>(a, sms, stream);
}

}  // namespace gfst
