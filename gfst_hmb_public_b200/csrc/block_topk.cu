// C-ABI entry of the coarse block retrieval (score + top-k).
#include <mutex>

#include "block_topk.cuh"

namespace gfst {
namespace {

using TakeError = int (*)(int, unsigned int*);
constexpr TakeError kErrorWords[] = {take_device_error, take_readout_error,  take_commit_error, take_score_error,
                                     take_scan_error,   take_attn_fma_error, take_attn_tc_error};
constexpr int kNumErrorWords = sizeof(kErrorWords) / sizeof(kErrorWords[0]);
__device__ unsigned int g_error_words[kNumErrorWords];  // as the last check took them
std::mutex g_error_mutex;                               // one check at a time

}  // namespace
}  // namespace gfst

extern "C" int gfst_block_topk(const void* Q, const void* Ksum, int64_t n_streams, int n_queries, int n_blocks,
                               int n_blocks_stride, int d, int k, int dtype, float* top_scores, int32_t* top_idx,
                               cudaStream_t stream) {
  using namespace gfst;
  GFST_REQUIRE(n_streams >= 0 && n_queries >= 0 && n_blocks >= 0, GFST_ERR_ARG, "negative size");
  GFST_REQUIRE(n_blocks_stride >= n_blocks, GFST_ERR_ARG, "n_blocks_stride %d < n_blocks %d", n_blocks_stride,
               n_blocks);
  GFST_REQUIRE(k >= 1 && k <= 32, GFST_ERR_SHAPE, "k=%d outside [1, 32]", k);
  GFST_REQUIRE(d >= 1 && d <= 256, GFST_ERR_SHAPE, "d=%d outside [1, 256]", d);
  GFST_REQUIRE(dtype == GFST_F32 || dtype == GFST_BF16, GFST_ERR_DTYPE, "unsupported dtype %d", dtype);
  if (n_streams == 0 || n_queries == 0) return GFST_OK;
  GFST_REQUIRE(Q && top_scores && top_idx && (Ksum || n_blocks == 0), GFST_ERR_ARG, "null buffer");
  if (dtype == GFST_BF16)
    return block_topk_tc(Q, Ksum, n_streams, n_queries, n_blocks, n_blocks_stride, d, k, top_scores, top_idx,
                         stream);
  return block_topk_simt(Q, Ksum, n_streams, n_queries, n_blocks, n_blocks_stride, d, k, dtype, top_scores,
                         top_idx, stream);
}

extern "C" int gfst_debug_bounded_wait(int64_t cycles, cudaStream_t stream) {
  GFST_REQUIRE(cycles >= 1 && cycles <= 2000000000LL, GFST_ERR_ARG, "cycles=%lld outside [1, 2e9]",
               (long long)cycles);
  return gfst::launch_bounded_wait_probe((long long)cycles, stream);
}

extern "C" int gfst_debug_attention_error(int tensor_cores, int status, cudaStream_t stream) {
  GFST_REQUIRE(status == GFST_ERR_ARG || status == GFST_ERR_ALIGN || status == GFST_ERR_TIMEOUT, GFST_ERR_ARG,
               "status %d is none that an attention kernel records", status);
  return tensor_cores ? gfst::launch_attn_tc_error(status, stream) : gfst::launch_attn_fma_error(status, stream);
}

extern "C" int gfst_check_device_errors(int clear) {
  // every stream of the current device, the library's non-blocking ones included
  const cudaError_t se = cudaDeviceSynchronize();
  GFST_REQUIRE(se == cudaSuccess, GFST_ERR_DEVICE, "cudaDeviceSynchronize: %s", cudaGetErrorString(se));
  // All words by one copy: a copy a word took 14 us each.
  std::lock_guard<std::mutex> lock(gfst::g_error_mutex);
  void* at = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&at, gfst::g_error_words);
  for (int i = 0; e == cudaSuccess && i < gfst::kNumErrorWords; ++i) {
    const int st = gfst::kErrorWords[i](clear, static_cast<unsigned int*>(at) + i);
    if (st != GFST_OK) return st;
  }
  unsigned int words[gfst::kNumErrorWords];
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(words, gfst::g_error_words, sizeof(words));
  GFST_REQUIRE(e == cudaSuccess, GFST_ERR_DEVICE, "reading the device error words: %s", cudaGetErrorString(e));
  // the first word that holds a failure; a bad table entry, read as zeros, only
  // where no word does
  unsigned int v = 0;
  for (const unsigned int w : words)
    if (v == 0 || (v == GFST_ERR_ARG && w != 0)) v = w;
  if (v == GFST_ERR_ALIGN) {
    gfst::set_last_error("a kernel found its shared memory misaligned (device error word %u)", v);
    return (int)v;
  }
  if (v == GFST_ERR_ARG) {
    gfst::set_last_error("a block table entry outside the pool was read (device error word %u)", v);
    return (int)v;
  }
  if (v != 0) {
    gfst::set_last_error("a kernel gave up a bounded wait (device error word %u)", v);
    return (int)v;
  }
  return GFST_OK;
}
