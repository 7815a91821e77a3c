// sample.cu -- token sampling with temperature, top-k, top-p and min-p from
// given random numbers, next to lm_head.cu's greedy argmax (reef chooses
// greedily only; this build's own definition).
//
// Per row of n logits x, with temperature T and a uniform number u in [0, 1):
//   w_i = exp((x_i - max x) / T)
//   order: by value, largest first, equal values by index
//   kept: the first top_k of the order; of those the shortest prefix whose
//     mass reaches top_p of theirs (rank r stays while the mass before it is <
//     top_p * total; the first always stays); of those w_i >= min_p
//   token: the first index, in index order, at which the running sum of the
//     kept w exceeds u times their total; prob: its w over that total.
// A NaN logit counts as -inf and weighs nothing; with +inf among the logits
// only those weigh (1 each).  T not above 0: the first largest logit.
//
// Exactness.  A draw lands next to a border between two tokens often enough
// (a vocabulary has 1e5 borders) that sums in float would choose wrongly for
// one row in a few dozen.  So w is computed in double and held as a 64-bit
// integer, round(w * 2^43): sums of up to 2^20 of them are exact, hence the
// same in any order, and nothing depends on the schedule.  The rounding moves a
// border by 2^-44 * sqrt(n), about 2e-11 of the largest weight.
//
// A cluster of C CTAs owns a row: each keeps its slice of the logits in shared
// memory, so the row is read from HBM once however many passes follow.  The
// kept set is always "key > cut, or key = cut and index <= cut_index" of the
// order-preserving 32-bit key of x, so top-k and top-p are radix selections
// (11 + 11 + 10 bits) over counts or masses, histograms summed over the cluster
// through distributed shared memory.
#include "common.cuh"
#include "ops.h"

#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

namespace cg = cooperative_groups;

namespace reef {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr double kOne = 8796093022208.0;  // 2^43, the weight 1
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // key_of(-inf)
constexpr int kMaxResident = 184 * 1024;      // bytes of logits a CTA keeps

typedef unsigned long long u64;

struct SampleArgs {
  int n;
  int slice;     // elements per CTA of the cluster
  int resident;  // of them, kept in shared memory
  const float* logits;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  uint32_t* index;
  float* prob;
};

struct Shared {
  uint32_t lo[kBins], hi[kBins];  // this CTA's histogram (hi: masses only)
  u64 sum[kBins];                 // the cluster's
  u64 slot[2][kMaxCluster];       // one value of every CTA
  u64 warp[kWarps];
  u64 pick[2];                    // a result of one thread for all
  u64 found;                      // a result of one CTA for all
};

// Order-preserving key: x < y exactly when key_of(x) < key_of(y); -0 equals
// +0, NaN is taken as -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (isnan(x)) return kKeyNegInf;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Row {
  const float* x;   // this CTA's slice, global
  const float* sm;  // its resident part
  int resident, count;
  int first;        // index of its first element in the row
  uint32_t max_key;
  double top, rcp_t;
  __device__ __forceinline__ uint32_t key(int i) const {
    return key_of(i < resident ? sm[i] : __ldg(x + i));
  }
  // exp((x - max) / T), 1 for the maximum itself
  __device__ __forceinline__ double weight(uint32_t k) const {
    if (k == max_key) return 1.0;
    if (k == kKeyNegInf) return 0.0;
    return exp((static_cast<double>(value_of(k)) - top) * rcp_t);
  }
  __device__ __forceinline__ u64 fixed(uint32_t k) const {
    return __double2ull_rn(weight(k) * kOne);
  }
};

// the elements that stay: key > cut, or key = cut and index <= cut_index
struct Cut {
  uint32_t key;
  int index;
  __device__ __forceinline__ bool keeps(uint32_t k, int i) const {
    return k > key || (k == key && i <= index);
  }
};

struct Ctx {
  cg::cluster_group cluster;
  Shared* s;
  int rank, ranks, tid, warp, lane, flip;
  // Warp w's part of the slice: a contiguous run, so that the warps' sums are
  // prefix sums in index order.
  __device__ __forceinline__ void run_of(const Row& r, int& i0, int& i1) const {
    const int per = (r.count + kWarps - 1) / kWarps;
    i0 = min(r.count, warp * per);
    i1 = min(r.count, i0 + per);
  }
  // Every CTA's value to every CTA: v of CTA c in slot(c) after it.
  __device__ __forceinline__ const u64* exchange(u64 v) {
    flip ^= 1;
    if (tid < ranks) cluster.map_shared_rank(s, tid)->slot[flip][rank] = v;
    cluster.sync();
    return s->slot[flip];
  }
};

// Sum of f(key, index) over the row's elements; s->warp holds this CTA's per
// warp, slot its cluster's per CTA.
template <typename F>
__device__ __forceinline__ u64 row_sum(Ctx& c, const Row& r, F f, const u64** slot) {
  int i0, i1;
  c.run_of(r, i0, i1);
  u64 v = 0;
  for (int i = i0 + c.lane; i < i1; i += 32) v += f(r.key(i), r.first + i);
  v = warp_sum(v);
  if (c.lane == 0) c.s->warp[c.warp] = v;
  __syncthreads();
  u64 mine = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) mine += c.s->warp[w];
  *slot = c.exchange(mine);
  u64 all = 0;
  for (int k = 0; k < c.ranks; ++k) all += (*slot)[k];
  return all;
}

// After row_sum(f): the first element, in index order, at which the running
// sum exceeds `target` (< the total).  True in the one lane that found it.
template <typename F>
__device__ __forceinline__ bool locate(Ctx& c, const Row& r, F f, const u64* slot, u64 target,
                                       int* at, uint32_t* at_key) {
  for (int k = 0; k < c.rank; ++k) {
    if (target < slot[k]) return false;  // an earlier CTA has it
    target -= slot[k];
  }
  if (target >= slot[c.rank]) return false;
  for (int w = 0; w < c.warp; ++w) {
    if (target < c.s->warp[w]) return false;
    target -= c.s->warp[w];
  }
  if (target >= c.s->warp[c.warp]) return false;
  int i0, i1;
  c.run_of(r, i0, i1);
  for (int i = i0; i < i1; i += 32) {
    const uint32_t k = i + c.lane < i1 ? r.key(i + c.lane) : 0u;
    const u64 v = i + c.lane < i1 ? f(k, r.first + i + c.lane) : 0ull;
    u64 run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 t = __shfl_up_sync(0xffffffffu, run, o);
      if (c.lane >= o) run += t;
    }
    const unsigned past = __ballot_sync(0xffffffffu, run > target);
    if (past != 0) {
      *at = r.first + i + c.lane;
      *at_key = k;
      return c.lane == __ffs(static_cast<int>(past)) - 1;
    }
    target -= __shfl_sync(0xffffffffu, run, 31);
  }
  return false;
}

// One level of a selection: of the elements that `cut` keeps and whose key
// agrees with `prefix` above bit shift + bits, the histogram of the next `bits`
// bits; finds, from the largest bin down, the bin at which the running sum
// reaches `target` (1 <= target <= the total).  Returns the bin, and in
// *before the sum of the bins above it.
template <bool kMass>
__device__ __forceinline__ uint32_t select_level(Ctx& c, const Row& r, const Cut& cut,
                                                 uint32_t prefix, int shift, int bits, u64 target,
                                                 u64* before) {
  Shared* s = c.s;
  const int bins = 1 << bits;
  for (int i = c.tid; i < bins; i += kThreads) {
    s->lo[i] = 0;
    if (kMass) s->hi[i] = 0;
  }
  __syncthreads();
  const int above = shift + bits;
  for (int i = c.tid; i < r.count; i += kThreads) {
    const uint32_t k = r.key(i);
    if (above < 32 && (k >> above) != (prefix >> above)) continue;
    if (!cut.keeps(k, r.first + i)) continue;
    const uint32_t bin = (k >> shift) & (bins - 1);
    if (kMass) {  // a 64-bit add of two 32-bit ones: the carry goes on, the order is free
      const u64 v = r.fixed(k);
      const uint32_t vl = static_cast<uint32_t>(v), vh = static_cast<uint32_t>(v >> 32);
      uint32_t carry = 0;
      if (vl != 0) carry = atomicAdd(&s->lo[bin], vl) > ~vl;
      if (vh + carry != 0) atomicAdd(&s->hi[bin], vh + carry);
    } else {
      atomicAdd(&s->lo[bin], 1u);
    }
  }
  c.cluster.sync();  // every CTA's histogram is done
  const int per = bins / c.ranks;
  for (int i = c.rank * per + c.tid; i < (c.rank + 1) * per; i += kThreads) {
    u64 v = 0;
    for (int k = 0; k < c.ranks; ++k) {
      const Shared* o = c.cluster.map_shared_rank(s, k);
      v += o->lo[i] + (kMass ? static_cast<u64>(o->hi[i]) << 32 : 0ull);
    }
    for (int k = 0; k < c.ranks; ++k) c.cluster.map_shared_rank(s, k)->sum[i] = v;
  }
  c.cluster.sync();  // every CTA has the cluster's
  // thread t's bins, from the largest down: [bins - (t + 1) * m, bins - t * m)
  const int m = bins / kThreads;  // 2 or 4
  u64 own = 0;
  for (int j = 0; j < m; ++j) own += s->sum[bins - 1 - (c.tid * m + j)];
  u64 run = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, run, o);
    if (c.lane >= o) run += t;
  }
  if (c.lane == 31) s->warp[c.warp] = run;
  __syncthreads();
  run -= own;
  for (int w = 0; w < c.warp; ++w) run += s->warp[w];
  if (run < target && target <= run + own) {
    for (int j = 0; j < m; ++j) {
      const int b = bins - 1 - (c.tid * m + j);
      const u64 v = s->sum[b];
      if (target <= run + v) {
        s->pick[0] = static_cast<u64>(b);
        s->pick[1] = run;
        break;
      }
      run += v;
    }
  }
  __syncthreads();
  *before = s->pick[1];
  return static_cast<uint32_t>(s->pick[0]);
}

// The shortest prefix of the kept order whose sum (count or mass) reaches
// `target` (1 <= target <= the kept total), as a tighter cut.
template <bool kMass>
__device__ __forceinline__ Cut select(Ctx& c, const Row& r, Cut cut, u64 target) {
  u64 before = 0;
  uint32_t key = select_level<kMass>(c, r, cut, 0, 21, 11, target, &before) << 21;
  target -= before;
  key |= select_level<kMass>(c, r, cut, key, 10, 11, target, &before) << 10;
  target -= before;
  key |= select_level<kMass>(c, r, cut, key, 0, 10, target, &before);
  target -= before;
  // of the elements equal to key, the first `ties` stay
  u64 ties = target;
  if (kMass) {
    const u64 w = r.fixed(key);
    ties = w > 0 ? (target + w - 1) / w : 1;
  }
  const u64* slot;
  auto tie = [&](uint32_t k, int i) -> u64 { return k == key && cut.keeps(k, i) ? 1ull : 0ull; };
  row_sum(c, r, tie, &slot);
  int at;
  uint32_t at_key;
  if (locate(c, r, tie, slot, ties - 1, &at, &at_key))
    for (int k = 0; k < c.ranks; ++k)
      c.cluster.map_shared_rank(c.s, k)->found = static_cast<u64>(at);
  c.cluster.sync();
  return Cut{key, static_cast<int>(c.s->found)};
}

__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Ctx c{cg::this_cluster()};
  c.s = reinterpret_cast<Shared*>(raw);
  float* sm = reinterpret_cast<float*>(raw + sizeof(Shared));
  c.rank = static_cast<int>(c.cluster.block_rank());
  c.ranks = static_cast<int>(c.cluster.num_blocks());
  c.tid = threadIdx.x;
  c.warp = c.tid >> 5;
  c.lane = c.tid & 31;
  c.flip = 0;
  const long long row = blockIdx.x / c.ranks;
  Row r;
  r.first = min(a.n, c.rank * a.slice);
  r.count = min(a.n, (c.rank + 1) * a.slice) - r.first;
  r.x = a.logits + row * a.n + r.first;
  r.sm = sm;
  r.resident = min(r.count, a.resident);
  r.max_key = 0;

  // ---- the row's maximum and the first index that has it
  u64 best = 0;  // key << 32 | ~index: the largest is the first largest logit
  for (int i = c.tid; i < r.count; i += kThreads) {
    const float x = __ldg(r.x + i);
    if (i < r.resident) sm[i] = x;
    const u64 v = (static_cast<u64>(key_of(x)) << 32) | ~static_cast<uint32_t>(r.first + i);
    best = v > best ? v : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 v = __shfl_xor_sync(0xffffffffu, best, o);
    best = v > best ? v : best;
  }
  if (c.lane == 0) c.s->warp[c.warp] = best;
  c.cluster.sync();  // (also: every CTA of the cluster has started)
#pragma unroll
  for (int w = 0; w < kWarps; ++w) best = c.s->warp[w] > best ? c.s->warp[w] : best;
  const u64* slot = c.exchange(best);
  for (int k = 0; k < c.ranks; ++k) best = slot[k] > best ? slot[k] : best;
  r.max_key = static_cast<uint32_t>(best >> 32);
  const uint32_t first_max = ~static_cast<uint32_t>(best);

  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  const bool none = r.max_key == kKeyNegInf;
  // every CTA of the cluster takes the same branch (row-wide values only)
  if (none || !(t > 0.0f)) {
    if (c.rank == 0 && c.tid == 0) {
      a.index[row] = none ? 0xffffffffu : first_max;
      if (a.prob != nullptr) a.prob[row] = none ? 0.0f : 1.0f;
    }
    c.cluster.sync();  // no CTA leaves while another may write its slots
    return;
  }
  r.top = static_cast<double>(value_of(r.max_key));
  r.rcp_t = 1.0 / static_cast<double>(t);

  // ---- the kept set
  Cut cut{0u, 0x7fffffff};
  const int k = a.top_k != nullptr ? a.top_k[row] : 0;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  const float mp = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  if (k > 0 && k < a.n) cut = select<false>(c, r, cut, static_cast<u64>(k));
  if (p < 1.0f) {
    auto kept = [&](uint32_t key, int i) { return cut.keeps(key, i) ? r.fixed(key) : 0ull; };
    const u64 all = row_sum(c, r, kept, &slot);
    const double want = ceil(static_cast<double>(p) * static_cast<double>(all));
    u64 target = want > 1.0 ? static_cast<u64>(want) : 1ull;
    target = target < all ? target : all;
    cut = select<true>(c, r, cut, target);
  }
  const double least = mp > 0.0f ? fmin(static_cast<double>(mp), 1.0) : 0.0;
  auto kept = [&](uint32_t key, int i) -> u64 {
    if (!cut.keeps(key, i)) return 0ull;
    const double w = r.weight(key);
    return w >= least ? __double2ull_rn(w * kOne) : 0ull;
  };

  // ---- the draw
  const u64 all = row_sum(c, r, kept, &slot);
  const float u = a.u[row];
  u64 target = u > 0.0f ? static_cast<u64>(fmin(static_cast<double>(u), 1.0) *
                                           static_cast<double>(all))
                        : 0ull;
  target = target < all ? target : all - 1;
  int at;
  uint32_t at_key;
  if (locate(c, r, kept, slot, target, &at, &at_key)) {
    a.index[row] = static_cast<uint32_t>(at);
    if (a.prob != nullptr)
      a.prob[row] = static_cast<float>(r.weight(at_key) * kOne / static_cast<double>(all));
  }
  c.cluster.sync();
}

}  // namespace

int sample_f32(long long rows, int n, const float* logits, const float* temperature,
               const int* top_k, const float* top_p, const float* min_p, const float* u,
               uint32_t* index, float* prob, cudaStream_t stream) {
  // Enough CTAs per row that its slices fit on chip, and more while the GPU
  // has SMs to spare and a slice stays above 4096 logits.
  int c = 1;
  const long long fit = kMaxResident / 4;
  while (c < kMaxCluster && (n > c * fit || (rows * c * 2 <= num_sms() && n > c * 8192))) c *= 2;
  SampleArgs a{};
  a.n = n;
  a.slice = (n + c - 1) / c;
  a.resident = static_cast<int>(std::min<long long>(a.slice, fit));
  a.logits = logits;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.u = u;
  a.index = index;
  a.prob = prob;
  const size_t smem = sizeof(Shared) + static_cast<size_t>(a.resident) * 4;
  static bool opted[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return kErrCuda;
  if (!opted[dev]) {
    if (cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(sizeof(Shared)) + kMaxResident) != cudaSuccess)
      return kErrCuda;
    opted[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * c));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(c);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, sample_kernel, a) != cudaSuccess) return kErrCuda;
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace reef
