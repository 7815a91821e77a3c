// spec.cu -- what follows a pass over drafted tokens: the walk that accepts a
// path of each sequence's tree, and the compaction of the int8 KV cache to
// that path.  reef decodes one token at a time and has neither (the
// definitions are this file's).
//
// A tree is parents[t] (t < drafts <= 64): the drafted token that t follows,
// an earlier one (parents[t] < t), or -1.  Node 0 is the root: the last
// token already chosen, whose keys the pass adds to the cache as row len; the
// other nodes' rows follow it.
//
// tree_accept: from cur = 0, next cur = the lowest c > cur with parents[c] =
// cur and tokens[c] = chosen[cur], until there is none; the nodes passed are
// the path, chosen[cur] of its last node the token that follows.  At most 64
// steps of two compares and two votes by one warp: bound by the launch (1.6 us for one
// tree of 8, 2.3 us for 512 of 64; cold 2.0 and 3.2).
//
// kv_compact_i8: row len + i := row len + path[i], i < accepted, for K, V and
// their scales, in every layer and KV head.  One CTA owns the rows of one
// (layer, sequence, KV head) and holds them all in registers (2 x 64 rows of
// 128 bytes at most: 4 KiB per warp) before it writes any, so a path may be in
// any order and name a row twice.  Rows already in their place are neither
// read nor written.  264 bytes a row, read and written once; a CTA has few of them,
// so one round trip to HBM bounds it: 2.5 us for 32 heads of one sequence (cold 2.8), 8.6
// us for 16 layers x 32 sequences x 8 heads (18.4 MB of rows, 2.1 TB/s of 6.5; cold 11.4).
#include "common.cuh"
#include "ops.h"

namespace reef {

namespace {

constexpr int kCThreads = 128;
constexpr int kCVecs = 2 * kMaxDrafts * 8 / kCThreads;  // 16-byte pieces per thread

__global__ void __launch_bounds__(128)
    tree_accept_kernel(int batch, int drafts, const int* __restrict__ draft_lens,
                       const int* __restrict__ parents, const int* __restrict__ tokens,
                       const int* __restrict__ chosen, int* __restrict__ path,
                       int* __restrict__ accepted, int* __restrict__ next) {
  const int b = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (b >= batch) return;
  const long long row = static_cast<long long>(b) * drafts;
  const int d = draft_lens == nullptr ? drafts : min(max(draft_lens[b], 0), drafts);
  // lane l holds nodes l and l + 32
  int par[2], tok[2], cho[2], mine[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int t = lane + 32 * j;
    par[j] = t >= d ? -2 : (parents == nullptr ? t - 1 : parents[row + t]);
    tok[j] = t < d ? tokens[row + t] : 0;
    cho[j] = t < d ? chosen[row + t] : 0;
    mine[j] = -1;  // path[t]
  }
  int cur = 0, n = 0, follow = -1;
  while (cur >= 0 && cur < d) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (lane + 32 * j == n) mine[j] = cur;
    ++n;
    const int c0 = __shfl_sync(0xffffffffu, cho[0], cur & 31);
    const int c1 = __shfl_sync(0xffffffffu, cho[1], cur & 31);
    follow = cur < 32 ? c0 : c1;
    const unsigned lo = __ballot_sync(0xffffffffu, lane > cur && par[0] == cur && tok[0] == follow);
    const unsigned hi =
        __ballot_sync(0xffffffffu, lane + 32 > cur && par[1] == cur && tok[1] == follow);
    cur = lo != 0 ? __ffs(static_cast<int>(lo)) - 1
                  : (hi != 0 ? __ffs(static_cast<int>(hi)) + 31 : -1);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (lane + 32 * j < drafts) path[row + lane + 32 * j] = mine[j];
  if (lane == 0) {
    accepted[b] = n;
    next[b] = follow;
  }
}

__global__ void __launch_bounds__(kCThreads)
    kv_compact_kernel(int batch, int heads_kv, int max_len, int drafts,
                      const int* __restrict__ lens, const int* __restrict__ path,
                      const int* __restrict__ accepted, int8_t* k_cache, float* k_scale,
                      int8_t* v_cache, float* v_scale, int* new_lens, int* err) {
  __shared__ int src[kMaxDrafts];
  const int tid = threadIdx.x;
  const unsigned pair = blockIdx.x;  // (layer, sequence, KV head)
  const int h = static_cast<int>(pair % static_cast<unsigned>(heads_kv));
  const int b = static_cast<int>(pair / static_cast<unsigned>(heads_kv) % static_cast<unsigned>(batch));
  const int len = lens[b], n = accepted[b];
  // (with the two above in one round trip, whether needed or not)
  const int p = tid < drafts ? path[static_cast<long long>(b) * drafts + tid] : 0;
  bool bad = len < 0 || len > max_len || n < 0 || n > drafts || len > max_len - n;
  if (!bad && tid < n) {
    src[tid] = p;
    bad = p < 0 || p >= drafts || p >= max_len - len;
  }
  // a bad sequence is left as it is; every CTA that works on it sees the same
  if (__syncthreads_or(bad)) {
    if (tid == 0 && h == 0 && pair < static_cast<long long>(batch) * heads_kv) {
      record_error(err, kDevBadPosition);
      new_lens[b] = len;
    }
    return;
  }
  if (tid == 0 && h == 0 && pair < static_cast<long long>(batch) * heads_kv) new_lens[b] = len + n;
  const long long row0 = static_cast<long long>(pair) * max_len + len;
  uint4 v[kCVecs];
  const int total = 2 * n * 8;  // 16-byte pieces: K's rows, then V's
#pragma unroll
  for (int j = 0; j < kCVecs; ++j) {
    const int i = tid + j * kCThreads;
    if (i >= total) continue;
    const int r = (i >> 3) % n, s = src[r];
    if (s == r) continue;
    const int8_t* c = i >> 3 < n ? k_cache : v_cache;
    v[j] = *reinterpret_cast<const uint4*>(c + (row0 + s) * 128 + (i & 7) * 16);
  }
  float sc = 0.0f;
  const int sr = tid < 2 * n ? tid % n : 0;
  const bool moves = tid < 2 * n && src[sr] != sr;
  if (moves) sc = (tid < n ? k_scale : v_scale)[row0 + src[sr]];
  __syncthreads();  // every row is held before any is written
#pragma unroll
  for (int j = 0; j < kCVecs; ++j) {
    const int i = tid + j * kCThreads;
    if (i >= total) continue;
    const int r = (i >> 3) % n;
    if (src[r] == r) continue;
    int8_t* c = i >> 3 < n ? k_cache : v_cache;
    *reinterpret_cast<uint4*>(c + (row0 + r) * 128 + (i & 7) * 16) = v[j];
  }
  if (moves) (tid < n ? k_scale : v_scale)[row0 + sr] = sc;
}

}  // namespace

int tree_accept(int batch, int drafts, const int* draft_lens, const int* parents,
                const int* tokens, const int* chosen, int* path, int* accepted, int* next,
                cudaStream_t stream) {
  tree_accept_kernel<<<(batch + 3) / 4, 128, 0, stream>>>(batch, drafts, draft_lens, parents,
                                                          tokens, chosen, path, accepted, next);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

int kv_compact_i8(long long layers, int batch, int heads_kv, int max_len, int drafts,
                  const int* lens, const int* path, const int* accepted, int8_t* k_cache,
                  float* k_scale, int8_t* v_cache, float* v_scale, int* new_lens,
                  cudaStream_t stream) {
  kv_compact_kernel<<<static_cast<unsigned>(layers * batch * heads_kv), kCThreads, 0, stream>>>(
      batch, heads_kv, max_len, drafts, lens, path, accepted, k_cache, k_scale, v_cache, v_scale,
      new_lens, device_error_ptr());
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace reef
