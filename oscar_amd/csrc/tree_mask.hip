// Ancestor masks of drafted trees (gfx950).
//
// see(i) = {i} + see(parent(i)).  With jump_0 = parent and see_0(i) = {i}:
//   see_{k+1}(i) = see_k(i) | see_k(jump_k(i)),   jump_{k+1}(i) = jump_k(jump_k(i)),
// so that after k rounds a node sees 2^k - 1 generations above it.  One workgroup a request,
// masks and jumps in LDS; the rounds end when no node has a jump left.  Within a round masks are
// read and written in place: what a node reads of another's, before or after that one's own
// round, are ancestors, and at least those of the round before.
//
// Latency: ceil(log2(depth)) rounds of two barriers.  2.9 us for one tree of 16 nodes, 5.2 for 8
// of 32 or 12 of up to 64 (the last dispatch's end included); a walk up the parents would take a
// dependent access for each generation.
#include "common.h"

#include "../../include/oscar_operators.h"

namespace oscar {

namespace {

constexpr int kMostNodes = 1024;
constexpr int kThreads = 256;
constexpr int kOwn = kMostNodes / kThreads;  // nodes of a thread at most
constexpr int kRoot = -1, kDead = -2;        // jumps that end: past a root, and below no parent

__global__ __launch_bounds__(kThreads) void tree_mask_kernel(oscarop_tree_args_v1 A) {
  const int tid = threadIdx.x, threads = blockDim.x, words = (int)A.mask_words;
  extern __shared__ uint64_t s_see[];              // [max_nodes][words]
  int* s_jump = (int*)(s_see + A.max_nodes * words);  // [max_nodes]
  const int64_t rows = A.num_tokens;
  const int64_t end = A.num_reqs > 0 ? A.query_start_loc[A.num_reqs] : 0;
  if ((int)blockIdx.x >= A.num_reqs) {
    // the rows of no request
    const int64_t first = A.num_reqs > 0 ? A.query_start_loc[0] : 0;
    const int64_t step = (int64_t)(gridDim.x - A.num_reqs) * threads;
    for (int64_t i = (int64_t)(blockIdx.x - A.num_reqs) * threads + tid; i < rows; i += step) {
      if (i >= first && i < end) continue;
      for (int w = 0; w < words; ++w) A.mask[i * words + w] = 0;
      A.depths[i] = -1;
    }
    return;
  }
  const int64_t a = A.query_start_loc[blockIdx.x], b = A.query_start_loc[blockIdx.x + 1];
  if (b <= a) return;
  if (a < 0 || b > rows || b - a > A.max_nodes) {
    for (int64_t i = (a < 0 ? 0 : a) + tid; i < (b < rows ? b : rows); i += threads) {
      for (int w = 0; w < words; ++w) A.mask[i * words + w] = 0;
      A.depths[i] = -1;
    }
    return;
  }
  const int n = (int)(b - a);
  for (int i = tid; i < n; i += threads) {
    const int p = A.parents[a + i];
    s_jump[i] = p < -1 || p >= i ? kDead : p;
    for (int w = 0; w < words; ++w) s_see[i * words + w] = w == i >> 6 ? 1ull << (i & 63) : 0;
  }
  __syncthreads();
  for (;;) {
    int next[kOwn], any = 0;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int i = tid + k * threads;
      next[k] = kRoot;
      if (i >= n) continue;
      const int j = s_jump[i];
      next[k] = j;
      if (j < 0) continue;
      any = 1;
      for (int w = 0; w <= j >> 6; ++w) s_see[i * words + w] |= s_see[j * words + w];
      next[k] = s_jump[j];
    }
    if (!__syncthreads_or(any)) break;
#pragma unroll
    for (int k = 0; k < kOwn; ++k)
      if (tid + k * threads < n) s_jump[tid + k * threads] = next[k];
    __syncthreads();
  }
  for (int i = tid; i < n; i += threads) {
    const bool dead = s_jump[i] == kDead;
    int depth = -1;
    for (int w = 0; w < words; ++w) {
      const uint64_t see = dead ? 0 : s_see[i * words + w];
      depth += __popcll(see);
      A.mask[(a + i) * words + w] = (int64_t)see;
    }
    A.depths[a + i] = depth;
  }
}

}  // namespace

}  // namespace oscar

using namespace oscar;

extern "C" int oscarop_tree_mask_v1(const oscarop_tree_args_v1* args, void* stream) {
  if (!args) return fail(-22, "oscarop_tree_mask_v1: null args");
  const oscarop_tree_args_v1& a = *args;
  if (a.num_reqs < 0 || a.num_reqs > 0xffff || a.num_tokens < 0 || a.num_tokens > 1 << 30)
    return fail(-22, "oscarop_tree_mask_v1: requests or rows out of range");
  if (a.max_nodes < 1 || a.max_nodes > kMostNodes || a.mask_words != (a.max_nodes + 63) / 64)
    return fail(-22, "oscarop_tree_mask_v1: max_nodes must lie in [1, %d], with a word for each 64", kMostNodes);
  if (a.num_tokens == 0) return 0;
  if (!a.parents || !a.mask || !a.depths || (a.num_reqs > 0 && !a.query_start_loc))
    return fail(-22, "oscarop_tree_mask_v1: missing pointer");
  // rows of no request: one workgroup, more where they may be many
  const unsigned rest = (unsigned)(1 + (a.num_tokens > 16384 ? 31 : 0));
  const int threads = a.max_nodes <= 64 ? 64 : kThreads;
  const size_t lds = (size_t)a.max_nodes * (8 * a.mask_words + 4);
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)tree_mask_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return fail(-5, "oscarop_tree_mask_v1: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(tree_mask_kernel, dim3(a.num_reqs + rest), dim3(threads), lds, (hipStream_t)stream, a);
  OSCAR_CHECK_LAUNCH("tree_mask_kernel");
  return 0;
}
