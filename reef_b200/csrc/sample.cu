// sample.cu -- token sampling with temperature, top-k, top-p and min-p from
// given random numbers, next to lm_head.cu's greedy argmax (reef chooses
// greedily only; the definition is this file's).
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
// one row in a few dozen.  So w is held as a 64-bit integer, w * 2^43 rounded:
// sums of up to 2^20 of them are exact, hence the same in any order, and nothing
// depends on the schedule.  Weights from 2^-27 up ("heavy") are computed in
// double; the others are below 2^16 units, and float with the constants in two
// terms is off by 0.05 of one there (the exponent's one rounding, 2^-21, and 2 ulp of
// ex2; at 2^-20 it would be 6 units).  So an integer is off by 0.55 at most.  Logits that
// differ make a border move by about 2^-44 * sqrt(n) of the largest weight; equal ones
// share their rounding, and n of them move it by 0.55 n units at most.
//
// Passes.  A cluster of C CTAs owns a row: each keeps its slice of the logits in
// shared memory (one bulk copy), so the row is read from HBM once however many passes
// follow.  The first finds the maximum.  Then
//   no filter, top-p: every weight is taken once, into the sums of the warps (in index
//     order, so the draw is a prefix sum) and for top-p into a histogram of masses
//     over 1024 equal steps of what top-p may keep last, which weighs more than
//     (1 - top_p) * total / n (the excluded ones are at most n and weigh less).
//     The step at the border is known then, and what lies in it or above is listed.
//   top-k: what lies above a bound is listed: the k-th largest of the maxima of
//     groups of eight logits, from a histogram that the first pass makes on the way.
//   min-p alone: what may weigh enough is listed.
// A list short enough goes to one CTA, which ends the row alone: two elements to a
// thread, or one (256 of them) by comparing each with each, in one go.
// The kept set is always "x > value, or x = value and index <= index": a
// histogram (counts or masses, summed over the cluster through distributed shared
// memory) gives the step in which the last kept one lies, and the few elements of
// that step are compared with each other.  Where steps do not help (all values alike, infinities, a list
// that does not fit) a radix selection over the order-preserving 32-bit key
// takes its place.
//
// What bounds it: 131 MB of logits (256 rows of 128000) would take 20 us to read; no
// filter takes 141 us, top-p 248 (cold 260).  Two CTAs of 512 threads fill an SM's
// shared memory and registers, and each row's chain is 15 to 35 us long: the copy and
// the maximum 4, the weights 10 (50 instructions each where every second one is
// heavy; with the histogram 15), then half a dozen steps of 1 to 4 us that end in a
// cluster barrier; per instruction issued (0.51 a cycle and scheduler, seven warps) a warp
// stands 4 cycles at barriers and for the memory order they give, 2.5 at fixed latencies,
// 2.5 at loads and the tables.  A single row of 50257 with top-k: 14 us (cold 19), all of
// it that chain.
// Measured and dropped: two elements to an instruction (no change), the four adds of
// a thread into the histogram in flight at once (3 % slower), the list weighed in a
// pass of its own and the histogram in another (341).  Heavy from 2^-27 up instead of
// from 2^-20, where float is not enough, costs nothing but where most of a vocabulary
// weighs between the two (256 x 128000, no filter: 117 -> 140).
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
constexpr int kBins = 1024;
constexpr int kMaxCluster = 8;
constexpr int kSlice = 16384;   // logits per CTA: two CTAs fit on an SM
constexpr int kList = 1016;     // of a warp's run (1024 at that slice) that are listed
constexpr int kGather = 1024;   // of a row that one CTA takes over
constexpr int kNear = kThreads; // elements of one step, over the cluster
constexpr int kFew = 256;       // candidates of a row that are compared each with each
constexpr int kMaxResident = 168 * 1024;      // bytes of logits a CTA keeps
constexpr double kOne = 8796093022208.0;      // 2^43, the weight 1
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // key_of(-inf)

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
  int* err;
};

struct alignas(16) Shared {
  union {
    uint32_t hist[2 * kBins];  // this CTA's histogram: masses as low and high words, or counts
    struct {                   // or the elements of one step, a part for each CTA
      u64 w[kNear];
      float x[kNear];
      int index[kNear];
    } near;
  };
  union {
    u64 sum[kBins];            // the cluster's histogram
    uint32_t count[2 * kBins];
    struct {                   // or the row's list, gathered in CTA 0
      float x[kGather];
      int index[kGather];
    } all;
  };
  uint16_t list[kWarps][kList];  // elements of a warp's run, in index order
  int listed[kWarps];
  int near_n[kMaxCluster];
  u64 slot[2][2][kMaxCluster];   // two values of every CTA
  double exp2_of[16];            // 2^(j / 16), one to a pair of banks
  u64 warp[kWarps], part[kWarps];
  u64 pick[2];                   // a result of one thread for all
  u64 found;                     // a result of one CTA for all
  double ready[3];               // 1 / T, log2 of top-p's bound, T ln(min-p)
  uint64_t loaded;               // mbarrier: the slice is in shared memory
};

// By name, not through pointers in structs: a pointer that a function is handed is
// generic, and loads and atomics through it cost half as much again.
extern __shared__ __align__(16) uint8_t g_smem[];
__device__ __forceinline__ Shared* shared() { return reinterpret_cast<Shared*>(g_smem); }
// the resident part of this CTA's slice
__device__ __forceinline__ float* resident_part() {
  return reinterpret_cast<float*>(g_smem + sizeof(Shared));
}

// Order-preserving key: x < y exactly when key_of(x) < key_of(y); -0 equals
// +0, NaN is taken as -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(fmaxf(x, -INFINITY) + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
// the least value whose key starts with these bits
__device__ __forceinline__ float floor_of(uint32_t key) {
  return key <= kKeyNegInf ? -INFINITY : value_of(key);
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// inclusive prefix sum over the lanes
__device__ __forceinline__ u64 warp_prefix(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

struct Row {
  const float* x;   // this CTA's slice, global, from a 16-byte boundary on
  int resident, count;  // elements of it in shared memory, and in all
  int first;        // index of its first element in the row (below 0: not of the row, -inf)
  float top;        // the row's maximum
  bool plain;       // magnitudes at which light() holds
  float heavy;      // values from here up weigh 2^-27 or (barely) less
  float least;      // values below weigh nothing
  double c, rcp_t, per_bit;  // log2(e) / T, 1 / T, T ln 2
  float c_hi, c_lo, k_hi, k_lo;  // c, and top * c - 43, in two terms
  __device__ __forceinline__ float at(int i) const { return i < resident ? resident_part()[i] : __ldg(x + i); }
  // exp((x - top) / T), 1 for the maximum itself, 0 for -inf and NaN
  __device__ __forceinline__ double weight(float v) const {
    if (v == top) return 1.0;
    if (!(v > -INFINITY) || top == INFINITY) return 0.0;
    return exp((static_cast<double>(v) - static_cast<double>(top)) * rcp_t);
  }
  // weight * 2^43 of a value below `heavy`: under 2^16.  log2 of it is v * c -
  // (top * c - 43), one fma that rounds once (2^-21 below 16), plus what the second
  // terms add (2^-10 at most), taken to first order.
  __device__ __forceinline__ uint32_t light(float v) const {
    v = fmaxf(v, least);  // (-inf and NaN too)
    const float e = __fmaf_rn(v, c_lo, -k_lo);
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(__fmaf_rn(v, c_hi, -k_hi)));
    w *= __fmaf_rn(e, 0.69314718f, 1.0f);
    return __float_as_uint(w + 8388608.0f) & 0x7fffffu;  // the integer next to it
  }
  // weight * 2^43
  __device__ __forceinline__ u64 fixed(float v) const {
    if (!plain) return __double2ull_rn(weight(v) * kOne);
    if (!(v >= heavy)) return light(v);
    return full(v);
  }
  // weight * 2^43 of a value not far below `heavy` (of a row that is plain)
  __device__ __forceinline__ u64 full(float v) const {
    // 2^t = 2^(n / 16) * 2^r, |r| <= 1/32: a table, and the series of e^(r ln 2)
    // to the sixth power (2^-51 of it is left out)
    const double t = (static_cast<double>(v) - static_cast<double>(top)) * c;
    const double kShift = 422212465065984.0;  // 1.5 * 2^48: a sum's last bit is 1/16
    const double m = t + kShift;
    const int n = __double2loint(m);
    const double r = t - (m - kShift);
    double q = __fma_rn(r, 0x1.430912f86c786p-13, 0x1.5d87fe78a6730p-10);
    q = __fma_rn(q, r, 0x1.3b2ab6fba4e77p-7);
    q = __fma_rn(q, r, 0x1.c6b08d704a0bfp-5);
    q = __fma_rn(q, r, 0x1.ebfbdff82c58ep-3);
    q = __fma_rn(q, r, 0x1.62e42fefa39efp-1);
    const double s = shared()->exp2_of[n & 15];
    const double w = __fma_rn(q * r, s, s);  // in [2^-1, 2), times 2^(n >> 4)
    const double up = __hiloint2double(__double2hiint(w) + (((n >> 4) + 43) << 20),
                                       __double2loint(w));
    // the integer next to it, from the low bits of a sum with 2^52
    return static_cast<u64>(__double_as_longlong(up + 4503599627370496.0)) & 0xfffffffffffffull;
  }
  // a value that weighs a little less than 2^log2w
  __device__ __forceinline__ float below_top(double log2w) const {
    const double d = log2w * per_bit;
    return static_cast<float>(top + d - 1e-6 * (fabs(d) + fabsf(top)));
  }
};

// the elements that stay: x > value, or x = value and index <= index
struct Cut {
  float value;
  int index;
  __device__ __forceinline__ bool keeps(float v, int i) const {
    return v > value || (v == value && i <= index);
  }
};

// How a pass goes over the row: every element of the slice; the elements
// listed; or, in the one CTA that took the row over, the gathered list.
enum Mode : int { kAll, kListed, kGathered };

struct Ctx {
  cg::cluster_group cluster;
  int rank, ranks, tid, warp, lane, flip;
  Mode mode;
  int gathered;
  __device__ __forceinline__ void sync() const {
    if (ranks == 1) __syncthreads();
    else cluster.sync();
  }
  __device__ __forceinline__ Shared* of(int k) const {
    return ranks == 1 ? shared() : cluster.map_shared_rank(shared(), k);
  }
  // Warp w's part of the slice (or gathered list): a contiguous run, so that
  // the warps' sums are prefix sums in index order.
  __device__ __forceinline__ int run_length(int count) const {
    return ((count + kWarps - 1) / kWarps + 3) & ~3;
  }
  __device__ __forceinline__ void run_of(int count, int& i0, int& i1) const {
    const int per = run_length(count);
    i0 = min(count, warp * per);
    i1 = min(count, i0 + per);
  }
  // four neighbours of the slice (i divides by 4), -inf from i1 on (up to which the
  // run goes: a multiple of 4, or the slice's end, behind which -inf stands)
  __device__ __forceinline__ float4 four(const Row& r, int i, int i1) const {
    if (i < min(i1, r.resident)) return *reinterpret_cast<const float4*>(resident_part() + i);
    if (i >= i1) return make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    return make_float4(r.at(i), i + 1 < i1 ? r.at(i + 1) : -INFINITY,
                       i + 2 < i1 ? r.at(i + 2) : -INFINITY, i + 3 < i1 ? r.at(i + 3) : -INFINITY);
  }
  // f(x, index) for the elements of the warp's run
  template <typename F>
  __device__ __forceinline__ void each(const Row& r, F f) const {
    int i0, i1;
    if (mode == kAll) {
      run_of(r.count, i0, i1);
      for (int i = i0 + lane; i < i1; i += 32) f(r.at(i), r.first + i);
    } else if (mode == kListed) {
      for (int j = lane; j < shared()->listed[warp]; j += 32) {
        const int i = shared()->list[warp][j];
        f(r.at(i), r.first + i);
      }
    } else {
      run_of(gathered, i0, i1);
      for (int j = i0 + lane; j < i1; j += 32) f(shared()->all.x[j], shared()->all.index[j]);
    }
  }
  // Two values of every CTA to every CTA: of CTA k in [0][k] and [1][k] after it.
  __device__ __forceinline__ u64 (*exchange(u64 v, u64 w = 0))[kMaxCluster] {
    flip ^= 1;
    if (tid < ranks) {
      Shared* o = of(tid);
      o->slot[flip][0][rank] = v;
      o->slot[flip][1][rank] = w;
    }
    sync();
    return shared()->slot[flip];
  }
};

// this CTA's sum of the warps' values, in s->warp after it
__device__ __forceinline__ u64 block_sum(const Ctx& c, u64 v) {
  v = warp_sum(v);
  if (c.lane == 0) shared()->warp[c.warp] = v;
  __syncthreads();
  u64 mine = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) mine += shared()->warp[w];
  return mine;
}

// Sum of f(x, index) over the row's elements; s->warp holds this CTA's per
// warp, slot its cluster's per CTA.
template <typename F>
__device__ __forceinline__ u64 row_sum(Ctx& c, const Row& r, F f, const u64** slot) {
  u64 v = 0;
  c.each(r, [&](float x, int i) { v += f(x, i); });
  *slot = c.exchange(block_sum(c, v))[0];
  u64 all = 0;
  for (int k = 0; k < c.ranks; ++k) all += (*slot)[k];
  return all;
}

// Lists the elements from `least` up (above -inf) and counts them.  Whether every
// warp's list fits.
__device__ __noinline__ bool build(Ctx& ctx, const Row& row, float least, int* count) {
  const Ctx c = ctx;
  const Row r = row;
  Shared* s = shared();
  uint16_t* list = s->list[c.warp];
  int i0, i1, n = 0;
  c.run_of(r.count, i0, i1);
  const unsigned below = (1u << c.lane) - 1;
  for (int i = i0; i < i1; i += 128) {
    const int j = i + 4 * c.lane;
    const float4 v4 = c.four(r, j, i1);
    const float v[4] = {v4.x, v4.y, v4.z, v4.w};
    // (most of the time none is there)
    if (!__any_sync(0xffffffffu, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= least)) continue;
    unsigned ballot[4];
    int at = n;
#pragma unroll
    for (int e = 0; e < 4; ++e) ballot[e] = __ballot_sync(0xffffffffu, v[e] >= least);
#pragma unroll
    for (int e = 0; e < 4; ++e) at += __popc(ballot[e] & below);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (v[e] >= least) {
        if (at < kList) list[at] = static_cast<uint16_t>(j + e);
        ++at;
      }
      n += __popc(ballot[e]);
    }
  }
  if (c.lane == 0) s->listed[c.warp] = n;
  __syncthreads();
  int total = 0;
  bool fits = r.count <= 65536;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    total += s->listed[w];
    fits = fits && s->listed[w] <= kList;
  }
  const u64* got = ctx.exchange(fits ? static_cast<u64>(total) : ~0ull)[0];
  *count = 0;
  for (int k = 0; k < c.ranks; ++k) {
    fits = fits && got[k] != ~0ull;
    *count += static_cast<int>(got[k]);
  }
  return fits;
}

// After build: the row goes on with the list alone, in CTA 0 if it is short
// (false in the others: they are done), else in every CTA.
__device__ __noinline__ bool gather(Ctx& c, const Row& r, int count) {
  Shared* s = shared();
  if (count > kGather) {
    c.mode = kListed;
    return true;
  }
  int at = 0;
  for (int k = 0; k < c.rank; ++k) at += static_cast<int>(s->slot[c.flip][0][k]);
  for (int w = 0; w < c.warp; ++w) at += s->listed[w];
  Shared* o = c.of(0);
  for (int j = c.lane; j < s->listed[c.warp]; j += 32) {
    const int i = s->list[c.warp][j];
    o->all.x[at + j] = r.at(i);
    o->all.index[at + j] = r.first + i;
  }
  c.sync();
  c.mode = kGathered;
  c.gathered = count;
  c.ranks = 1;
  return c.rank == 0;
}

// After row_sum(f): the first element, in index order, at which the running
// sum exceeds `target` (< the total).  True in the one lane that found it.
// The CTA that has it goes over its warp's run again with all warps.
template <typename F>
__device__ __forceinline__ bool locate(Ctx& c, const Row& r, F f, const u64* slot, u64 target,
                                       int* at, float* at_x) {
  for (int k = 0; k < c.rank; ++k) {
    if (target < slot[k]) return false;  // an earlier CTA has it
    target -= slot[k];
  }
  if (target >= slot[c.rank]) return false;
  int w = 0;
  for (; w < kWarps - 1 && target >= shared()->warp[w]; ++w) target -= shared()->warp[w];
  int i0 = 0, i1 = shared()->listed[w];
  if (c.mode != kListed) {
    const int count = c.mode == kAll ? r.count : c.gathered;
    const int per = c.run_length(count);
    i0 = min(count, w * per);
    i1 = min(count, i0 + per);
  }
  const int per = (i1 - i0 + kWarps - 1) / kWarps;
  auto element = [&](int j, float* x, int* index) {
    if (c.mode == kGathered) {
      *x = shared()->all.x[j];
      *index = shared()->all.index[j];
    } else {
      const int i = c.mode == kListed ? shared()->list[w][j] : j;
      *x = r.at(i);
      *index = r.first + i;
    }
  };
  i1 = min(i1, i0 + (c.warp + 1) * per);
  i0 = min(i1, i0 + c.warp * per);
  float x = 0.0f;
  int index = 0;
  u64 v = 0;
  for (int j = i0 + c.lane; j < i1; j += 32) {
    element(j, &x, &index);
    v += f(x, index);
  }
  v = warp_sum(v);
  if (c.lane == 0) shared()->part[c.warp] = v;
  __syncthreads();
  for (int k = 0; k < c.warp; ++k) {
    if (target < shared()->part[k]) return false;
    target -= shared()->part[k];
  }
  if (target >= shared()->part[c.warp]) return false;
  for (int i = i0; i < i1; i += 32) {
    u64 run = 0;
    if (i + c.lane < i1) {
      element(i + c.lane, &x, &index);
      run = f(x, index);
    }
    run = warp_prefix(run, c.lane);
    const unsigned past = __ballot_sync(0xffffffffu, run > target);
    if (past != 0) {
      *at = index;
      *at_x = x;
      return c.lane == __ffs(static_cast<int>(past)) - 1;
    }
    target -= __shfl_sync(0xffffffffu, run, 31);
  }
  return false;
}

// Thread t's share of a histogram is its bins [bins - (t + 1) * m, bins - t *
// m); of(b) is the sum in bin b.  Finds, from the largest bin down, the bin at
// which the running sum reaches `target` (>= 1), and the sum of the bins above
// it; false if it never does.
template <typename Of>
__device__ __forceinline__ bool scan_bins(const Ctx& c, int bins, u64 target, Of of, int* bin,
                                          u64* before) {
  Shared* s = shared();
  const int m = bins / kThreads;
  u64 own = 0;
  for (int j = 0; j < m; ++j) own += of(bins - 1 - (c.tid * m + j));
  u64 run = warp_prefix(own, c.lane);
  if (c.lane == 31) s->warp[c.warp] = run;
  if (c.tid == 0) s->pick[0] = ~0ull;
  __syncthreads();
  run -= own;
  for (int w = 0; w < c.warp; ++w) run += s->warp[w];
  if (run < target && target <= run + own) {
    for (int j = 0; j < m; ++j) {
      const int b = bins - 1 - (c.tid * m + j);
      const u64 v = of(b);
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
  *bin = static_cast<int>(s->pick[0]);
  return s->pick[0] != ~0ull;
}

// Equal steps of the range from `least` up to the row's maximum.  Rounding is
// monotone, and so are the steps.
struct Steps {
  float least, scale;
  __device__ __forceinline__ Steps(float from, float top)
      : least(from), scale((kBins - 0.25f) / (top - from)) {}
  __device__ __forceinline__ bool part() const { return scale > 0.0f && scale < 1e30f; }
  __device__ __forceinline__ int bin(float x) const {  // of x from `least` up
    return min(kBins - 1, static_cast<int>((x - least) * scale));
  }
  // a little less than what lies in bin b
  __device__ __forceinline__ float below(int b, float top) const {
    return least + static_cast<float>(b) / scale -
           1e-6f * (top - least + fabsf(least) + fabsf(top));
  }
};

// A mass into this CTA's histogram: a 64-bit add of two 32-bit ones (the carry goes
// on, the order is free).
__device__ __forceinline__ void add_mass(int b, u64 v) {
  const uint32_t low = static_cast<uint32_t>(v);
  const uint32_t high = static_cast<uint32_t>(v >> 32) +
                        (atomicAdd(&shared()->hist[b], low) > ~low ? 1u : 0u);
  if (high != 0) atomicAdd(&shared()->hist[kBins + b], high);
}

// The CTAs' histograms (counts or masses; all done) added up, and scan_bins: every
// CTA gets the same answer.
template <bool kMass>
__device__ __noinline__ bool scan_cluster(const Ctx& ctx, u64 target, int* bin, u64* before) {
  const Ctx c = ctx;
  Shared* s = shared();
  auto local = [&](const Shared* o, int b) -> u64 {
    return o->hist[b] + (kMass ? static_cast<u64>(o->hist[kBins + b]) << 32 : 0ull);
  };
  if (c.ranks == 1)
    return scan_bins(c, kBins, target, [&](int b) { return local(s, b); }, bin, before);
  const int per = kBins / c.ranks;
  for (int i = c.rank * per + c.tid; i < (c.rank + 1) * per; i += kThreads) {
    u64 v = 0;
    for (int k = 0; k < c.ranks; ++k) v += local(c.of(k), i);
    for (int k = 0; k < c.ranks; ++k) c.of(k)->sum[i] = v;
  }
  c.sync();  // every CTA has the cluster's
  return scan_bins(c, kBins, target, [&](int b) { return s->sum[b]; }, bin, before);
}

// One histogram of the cluster: bin_of(x, index) is an element's bin, or -1.
// As scan_bins.
template <bool kMass, typename BinOf>
__device__ __forceinline__ bool histogram(const Ctx& c, const Row& r, BinOf bin_of, u64 target,
                                          int* bin, u64* before) {
  Shared* s = shared();
  for (int i = c.tid; i < (kMass ? 2 : 1) * kBins; i += kThreads) s->hist[i] = 0;
  __syncthreads();
  c.each(r, [&](float x, int i) {
    const int b = bin_of(x, i);
    if (b < 0) return;
    if (kMass) add_mass(b, r.fixed(x));
    else atomicAdd(&s->hist[b], 1u);
  });
  c.sync();
  return scan_cluster<kMass>(c, target, bin, before);
}

// The mass of a row that is plain: s->warp holds this CTA's per warp, slot the
// cluster's per CTA, as after row_sum; with kHist also this CTA's histogram of the
// elements from steps.least up.  A warp that has no heavy (no light) one among
// 128 neighbours leaves out what is for those.
template <bool kHist>
__device__ __noinline__ u64 weigh(Ctx& ctx, const Row& row, const Steps& st, const u64** slot) {
  const Ctx c = ctx;
  const Row r = row;
  const Steps steps = st;
  Shared* s = shared();
  if (kHist) {
    for (int i = c.tid; i < 2 * kBins; i += kThreads) s->hist[i] = 0;
    __syncthreads();
  }
  int i0, i1;
  c.run_of(r.count, i0, i1);
  u64 sum = 0;
  for (int i = i0; i < i1; i += 128) {
    const float4 v4 = c.four(r, i + 4 * c.lane, i1);
    const float v[4] = {v4.x, v4.y, v4.z, v4.w};
    const float hi = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
    const bool all4 = v[0] >= r.heavy && v[1] >= r.heavy && v[2] >= r.heavy && v[3] >= r.heavy;
    u64 w[4] = {0, 0, 0, 0};
    if (__any_sync(0xffffffffu, hi >= r.heavy)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = r.full(fmaxf(v[e], r.least));
    }
    if (!__all_sync(0xffffffffu, all4)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t l = r.light(v[e]);
        w[e] = v[e] >= r.heavy ? w[e] : l;
      }
    }
    sum += (w[0] + w[1]) + (w[2] + w[3]);
    if (kHist) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v[e] >= steps.least) add_mass(steps.bin(v[e]), w[e]);
    }
  }
  *slot = ctx.exchange(block_sum(c, sum))[0];
  u64 all = 0;
  for (int k = 0; k < c.ranks; ++k) all += (*slot)[k];
  return all;
}

// Of the elements of step `bin` that `cut` keeps, the shortest prefix of the order
// whose sum (count or mass) reaches `target` (>= 1), as a tighter cut.  False, with
// the cut as it was, where they are too many.
template <bool kMass>
__device__ __noinline__ bool select_near(const Ctx& ctx, const Row& row, Cut* cut_io,
                                         const Steps& st, int bin, u64 target) {
  const Ctx c = ctx;
  const Row r = row;
  const Cut cut = *cut_io;
  const Steps steps = st;
  Shared* s = shared();
  if (c.tid == 0) s->near_n[c.rank] = 0;
  __syncthreads();
  // the elements of that step to every CTA, each into its own part
  const int room = kNear / c.ranks;
  c.each(r, [&](float x, int i) {
    if (!(x >= steps.least) || steps.bin(x) != bin || !cut.keeps(x, i)) return;
    const int at = atomicAdd(&s->near_n[c.rank], 1);
    if (at >= room) return;
    for (int k = 0; k < c.ranks; ++k) {
      Shared* o = c.of(k);
      o->near.x[c.rank * room + at] = x;
      o->near.index[c.rank * room + at] = i;
    }
  });
  __syncthreads();
  if (c.tid < c.ranks && c.tid != c.rank) c.of(c.tid)->near_n[c.rank] = s->near_n[c.rank];
  c.sync();
  // side by side: the parts of several CTAs in `all` (which only a row that one CTA
  // took over uses)
  bool fits = true;
  int total = 0, mine = -1;
  for (int k = 0; k < c.ranks; ++k) {
    const int n = s->near_n[k];
    fits = fits && n <= room;
    if (c.tid >= total && c.tid < total + n) mine = k * room + c.tid - total;
    total += n;
  }
  if (!fits) return false;
  const float* xs = c.ranks > 1 ? s->all.x : s->near.x;
  const int* at = c.ranks > 1 ? s->all.index : s->near.index;
  if (mine >= 0) {
    const float x = s->near.x[mine];
    s->near.w[c.tid] = kMass ? r.fixed(x) : 1ull;
    if (c.ranks > 1) {
      s->all.x[c.tid] = x;
      s->all.index[c.tid] = s->near.index[mine];
    }
  }
  __syncthreads();
  // what comes before each in the order, by as many neighbouring threads as there are
  int each = 1;
  while (each < 32 && 2 * each * total <= kThreads) each *= 2;
  const int e = c.tid / each;
  if (e - c.lane / each < total) {  // (whole warps)
    const float x = e < total ? xs[e] : 0.0f;
    const int index = e < total ? at[e] : 0;
    u64 run = 0;
    for (int j = c.tid % each; j < total; j += each) {
      const float y = xs[j];
      if (y > x || (y == x && at[j] < index)) run += s->near.w[j];
    }
    for (int o = 1; o < each; o *= 2) run += __shfl_xor_sync(0xffffffffu, run, o);
    if (e < total && c.tid % each == 0 && run < target && target <= run + s->near.w[e])
      s->found = (static_cast<u64>(__float_as_uint(x)) << 32) | static_cast<uint32_t>(index);
  }
  __syncthreads();
  *cut_io = Cut{__uint_as_float(static_cast<uint32_t>(s->found >> 32)),
                static_cast<int>(static_cast<uint32_t>(s->found))};
  return true;
}

// Of the elements that `cut` keeps from `least` up (finite), the shortest
// prefix of the order whose sum reaches `target`, as a tighter cut.  False, with the
// cut as it was, where equal steps do not part them.
template <bool kMass>
__device__ __forceinline__ bool select_steps(const Ctx& c, const Row& r, Cut* cut, float least,
                                             u64 target) {
  const Steps steps(least, r.top);
  if (!steps.part()) return false;
  int bin;
  u64 before;
  auto bin_of = [&](float x, int i) {
    return x >= least && cut->keeps(x, i) ? steps.bin(x) : -1;
  };
  return histogram<kMass>(c, r, bin_of, target, &bin, &before) &&
         select_near<kMass>(c, r, cut, steps, bin, target - before);
}

// select_steps by radix, for any values: ten bits of the key at a time (the
// last ten overlap), then the first so many of the elements equal to it.
template <bool kMass>
__device__ __noinline__ void select_radix(Ctx& c, const Row& r, Cut* cut_io, float least,
                                          u64 target) {
  const Cut cut = *cut_io;
  uint32_t key = 0;
#pragma unroll 1
  for (int above = 32; above > 0; above = above > 10 ? above - 10 : 0) {
    const int shift = above > 10 ? above - 10 : 0;
    auto bin_of = [&](float x, int i) {
      x = fmaxf(x, -INFINITY);  // NaN
      if (!(x >= least) || !cut.keeps(x, i)) return -1;
      const uint32_t k = key_of(x);
      if (above < 32 && (k >> above) != (key >> above)) return -1;
      return static_cast<int>((k >> shift) & (kBins - 1));
    };
    int bin;
    u64 before;
    histogram<kMass>(c, r, bin_of, target, &bin, &before);
    target -= before;
    key = (key & ~((kBins - 1u) << shift)) | (static_cast<uint32_t>(bin & (kBins - 1)) << shift);
  }
  const float value = value_of(key);
  u64 ties = target;
  if (kMass) {
    const u64 w = r.fixed(value);
    ties = w > 0 ? (target + w - 1) / w : 1;
  }
  const u64* slot;
  auto tie = [&](float x, int i) -> u64 {
    x = fmaxf(x, -INFINITY);
    return x == value && cut.keeps(x, i) ? 1ull : 0ull;
  };
  row_sum(c, r, tie, &slot);
  int at;
  float at_x;
  if (locate(c, r, tie, slot, ties - 1, &at, &at_x))
    for (int k = 0; k < c.ranks; ++k) c.of(k)->found = static_cast<u64>(at);
  c.sync();
  *cut_io = Cut{value, static_cast<int>(shared()->found)};
}

// A token's share of the kept mass: from the integer where it has 30 bits, else anew
// (exp in double takes one thread a microsecond).
__device__ __forceinline__ float share(const Row& r, float x, u64 w, u64 all) {
  const double mine = w >> 30 != 0 ? static_cast<double>(w) : r.weight(x) * kOne;
  return static_cast<float>(mine / static_cast<double>(all));
}

// u times the total, below it
__device__ __forceinline__ u64 drawn(float u, u64 all) {
  const u64 at = u > 0.0f ? static_cast<u64>(fmin(static_cast<double>(u), 1.0) *
                                             static_cast<double>(all))
                          : 0ull;
  return at < all ? at : all - 1;
}

// The rest of a row whose candidates (all that any filter may keep, in index
// order) are one to a thread: the ranks and the masses ahead of each by comparing
// with every other, then the draw by a prefix sum.  k: 0 is off; keeps_min(x)
// says what min-p keeps.
template <typename KeepsMin>
__device__ __forceinline__ void finish_few(const Ctx& c, const Row& r, int k, float p,
                                           KeepsMin keeps_min, float u, uint32_t* index,
                                           float* prob) {
  Shared* s = shared();
  // as many neighbouring threads to an element as there are, two at least, for a part
  // of the others each
  int each = 2;
  while (each < 32 && 2 * each * c.gathered <= kThreads) each *= 2;
  const int e = c.tid / each, part = c.tid % each;
  const bool have = e < c.gathered;
  const float x = have ? s->all.x[e] : 0.0f;
  u64 w = have && part == 0 ? r.fixed(x) : 0ull;
  if (have && part == 0) s->near.w[e] = w;
  if (c.tid < 3) {  // (behind them, ahead of none)
    s->all.x[c.gathered + c.tid] = -INFINITY;
    s->near.w[c.gathered + c.tid] = 0;
  }
  __syncthreads();
  // the elements ahead in the order: how many, and for top-p their mass (they come
  // before this one, so top-k keeps them if it keeps this one)
  int rank = 0;
  u64 ahead = 0;
  if (have && p < 1.0f) {
    for (int j = 4 * part; j < c.gathered; j += 4 * each) {
      const float4 y4 = *reinterpret_cast<const float4*>(&s->all.x[j]);
      const float y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool before = y[q] > x || (y[q] == x && j + q < e);
        rank += before;
        ahead += before ? s->near.w[j + q] : 0ull;
      }
    }
  } else if (have && k > 0) {
#pragma unroll 2
    for (int j = 4 * part; j < c.gathered; j += 4 * each) {
      const float4 y4 = *reinterpret_cast<const float4*>(&s->all.x[j]);
      const float y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) rank += y[q] > x || (y[q] == x && j + q < e);
    }
  }
  for (int o = 1; o < each; o *= 2) {
    rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (p < 1.0f) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
  }
  if (k > 0 && rank >= k) w = 0;
  const u64 mass = block_sum(c, w);
  // kept: mass ahead < p * total, as integers
  if (p < 1.0f && rank > 0 &&
      static_cast<double>(ahead) >= ceil(static_cast<double>(p) * static_cast<double>(mass)))
    w = 0;
  if (w != 0 && !keeps_min(x)) w = 0;
  __syncthreads();  // (s->warp has been read)
  const u64 all = block_sum(c, w);
  const u64 target = drawn(u, all);
  u64 run = warp_prefix(w, c.lane) - w;
  for (int i = 0; i < c.warp; ++i) run += s->warp[i];
  if (run <= target && target < run + w) {  // (w is 0 but in an element's first thread)
    *index = static_cast<uint32_t>(s->all.index[e]);
    if (prob != nullptr)
      *prob = share(r, x, w, all);
  }
}

// The rest of a row for top-p (and min-p) in the one CTA that has gathered the
// elements from step `bin` up, in index order, two to a thread: those above the step
// stay, those in it while the mass ahead of them is below `target` (`before` is that
// of the steps above), and the draw is a prefix sum.  False where too many lie in the
// step.
template <typename KeepsMin>
__device__ __forceinline__ bool finish_steps(const Ctx& c, const Row& r, const Steps& steps,
                                             int bin, u64 before, u64 target, KeepsMin keeps_min,
                                             float u, uint32_t* index, float* prob) {
  static_assert(kGather == 2 * kThreads, "two to a thread");
  Shared* s = shared();
  if (c.tid == 0) s->near_n[0] = 0;
  __syncthreads();
  float x[2];
  u64 w[2];
  bool near[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int j = 2 * c.tid + e;
    x[e] = j < c.gathered ? s->all.x[j] : -INFINITY;
    const int b = x[e] >= steps.least ? steps.bin(x[e]) : -1;
    near[e] = b == bin;
    w[e] = b >= bin ? r.fixed(x[e]) : 0ull;
    if (near[e]) {
      const int at = atomicAdd(&s->near_n[0], 1);
      if (at < kNear) {
        s->near.x[at] = x[e];
        s->near.index[at] = j;
        s->near.w[at] = w[e];
      }
    }
  }
  __syncthreads();
  const int n = s->near_n[0];
  if (n > kNear) {
    __syncthreads();  // everyone has read the count, which select_near begins by clearing
    return false;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (near[e]) {
      u64 ahead = before;
      for (int j = 0; j < n; ++j) {
        const float y = s->near.x[j];
        if (y > x[e] || (y == x[e] && s->near.index[j] < 2 * c.tid + e)) ahead += s->near.w[j];
      }
      if (ahead >= target) w[e] = 0;
    }
    if (w[e] != 0 && !keeps_min(x[e])) w[e] = 0;
  }
  const u64 own = w[0] + w[1];
  u64 run = warp_prefix(own, c.lane);
  if (c.lane == 31) s->warp[c.warp] = run;
  __syncthreads();
  u64 all = 0;
  run -= own;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < c.warp) run += s->warp[i];
    all += s->warp[i];
  }
  const u64 at = drawn(u, all);
  if (run <= at && at < run + own) {
    const int e = at < run + w[0] ? 0 : 1;
    *index = static_cast<uint32_t>(s->all.index[2 * c.tid + e]);
    if (prob != nullptr)
      *prob = share(r, x[e], w[e], all);
  }
  return true;
}

__global__ void __launch_bounds__(kThreads, 2) sample_kernel(SampleArgs a) {
  Ctx c{cg::this_cluster()};
  Shared* s = shared();
  float* sm = resident_part();
  c.rank = static_cast<int>(c.cluster.block_rank());
  c.ranks = static_cast<int>(c.cluster.num_blocks());
  c.tid = threadIdx.x;
  c.warp = c.tid >> 5;
  c.lane = c.tid & 31;
  c.flip = 0;
  c.mode = kAll;
  c.gathered = 0;
  const long long row = blockIdx.x / c.ranks;
  // The slices begin on 16-byte boundaries: rank 0's with up to three elements that
  // are not of the row.
  const float* x = a.logits + row * a.n;
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
  Row r;
  r.first = c.rank * a.slice - shift;
  r.count = max(0, min(a.n - r.first, a.slice));
  r.x = x + r.first;
  r.resident = min(r.count, a.resident);
  const int lo = min(c.rank == 0 ? shift : 0, r.resident);
  const int al = min((lo + 3) & ~3, r.resident), ah = max(al, r.resident & ~3);
  if (c.tid == 0) {
    mbar_init(&s->loaded, 1);
    fence_barrier_init();
    mbar_arrive_expect_tx(&s->loaded, (ah - al) * 4);
    if (ah > al) bulk_load(sm + al, r.x + al, (ah - al) * 4, &s->loaded);
  }
  if (c.tid < 4) {  // what stands before and behind whole pieces, and the padding
    if (c.tid < lo) sm[c.tid] = -INFINITY;
    if (lo + c.tid < al) sm[lo + c.tid] = __ldg(r.x + lo + c.tid);
    if (ah + c.tid < ((r.resident + 3) & ~3))
      sm[ah + c.tid] = ah + c.tid < r.resident ? __ldg(r.x + ah + c.tid) : -INFINITY;
  }
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  const float mp = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  const float u = a.u[row];
  int k = a.top_k != nullptr ? a.top_k[row] : 0;
  if (k >= a.n || !(t > 0.0f)) k = 0;

  // (every CTA of the cluster takes the same branches: row-wide values only)
  if (k > 0)
    for (int i = c.tid; i < 2 * kBins; i += kThreads) s->hist[i] = 0;
  if (c.tid < 16 && t > 0.0f) s->exp2_of[c.tid] = exp2(c.tid / 16.0);
  __syncthreads();
  // the others have started when the wait below ends: nothing is written to them before
  if (c.ranks > 1) cg::this_cluster().barrier_arrive();

  // what does not need the logits, while they come (one thread each: a double's
  // logarithm in all of them costs as much as a pass over the slice).
  // What top-p keeps last weighs more than (1 - p) / n of the total (what it leaves
  // out is n at most, and weighs less), which is 1 at least; half of that, for the
  // roundings on the way.
  const double least = mp > 0.0f ? fmin(static_cast<double>(mp), 1.0) : 0.0;
  if (c.tid == 32) s->ready[0] = 1.0 / static_cast<double>(t);
  if (c.tid == 64 && p < 1.0f)
    s->ready[1] = log2(0.5 * (1.0 - static_cast<double>(fmaxf(p, 0.0f))) / a.n);
  if (c.tid == 96 && least > 0.0) s->ready[2] = log(least) * static_cast<double>(t);

  // ---- the row's maximum, and for top-k the histogram of the maxima of groups of
  // eight logits
  mbar_wait(&s->loaded, 0, a.err, kDevTimeoutFull);
  float top = -INFINITY;  // (fmaxf passes NaN over)
  for (int i = 4 * c.tid; i < r.resident; i += 8 * kThreads) {
    const float4 v = *reinterpret_cast<const float4*>(sm + i);
    float m = fmaxf(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), -INFINITY);
    if (i + 4 * kThreads < r.resident) {
      const float4 w = *reinterpret_cast<const float4*>(sm + i + 4 * kThreads);
      m = fmaxf(m, fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)));
    }
    if (k > 0) atomicAdd(&s->hist[key_of(m) >> 21], 1u);
    top = fmaxf(top, m);
  }
  for (int i = r.resident + c.tid; i < r.count; i += kThreads) {
    const float v = fmaxf(__ldg(r.x + i), -INFINITY);
    if (k > 0) atomicAdd(&s->hist[key_of(v) >> 21], 1u);
    top = fmaxf(top, v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (c.lane == 0) s->warp[c.warp] = key_of(top);
  __syncthreads();
  r.rcp_t = s->ready[0];
  u64 best = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) best = s->warp[w] > best ? s->warp[w] : best;
  if (c.ranks > 1) cg::this_cluster().barrier_wait();
  const u64* slot = c.exchange(best)[0];
  for (int j = 0; j < c.ranks; ++j) best = slot[j] > best ? slot[j] : best;
  top = value_of(static_cast<uint32_t>(best));
  r.top = top;

  if (top == -INFINITY) {
    if (c.rank == 0 && c.tid == 0) {
      a.index[row] = 0xffffffffu;
      if (a.prob != nullptr) a.prob[row] = 0.0f;
    }
    return;  // (nobody reads or writes another CTA after the exchange)
  }
  int at;
  float at_x;
  if (!(t > 0.0f)) {  // greedy: the first that equals the maximum
    auto first = [&](float x, int) -> u64 { return x == top ? 1ull : 0ull; };
    row_sum(c, r, first, &slot);
    if (locate(c, r, first, slot, 0, &at, &at_x)) {
      a.index[row] = static_cast<uint32_t>(at);
      if (a.prob != nullptr) a.prob[row] = 1.0f;
    }
    return;
  }
  r.per_bit = 0.6931471805599453 * static_cast<double>(t);
  r.c = 1.4426950408889634 * r.rcp_t;
  r.c_hi = static_cast<float>(r.c);
  r.c_lo = static_cast<float>(r.c - static_cast<double>(r.c_hi));
  const double k2 = static_cast<double>(top) * r.c - 43.0;
  r.k_hi = static_cast<float>(k2);
  r.k_lo = static_cast<float>(k2 - static_cast<double>(r.k_hi));
  r.plain = fabs(k2) < 8192.0 && fabsf(top) < 1e30f && t < 1e30f && t > 1e-30f;
  r.heavy = r.below_top(-27.0);
  r.least = r.below_top(-60.0);

  // min-p in float but next to the border, in double there
  float sure = INFINITY, out = -INFINITY;  // x from `sure` up stays, below `out` not
  if (least > 0.0 && r.plain) {
    const double x = static_cast<double>(top) + s->ready[2];
    const double slack = 1e-6 * (fabs(x) + fabs(static_cast<double>(top)) + 1e-6);
    sure = static_cast<float>(x + slack);
    out = static_cast<float>(x - slack);
  }
  auto keeps_min = [&](float x) {
    return least == 0.0 || x >= sure || (!(x < out) && r.weight(x) >= least);
  };
  uint32_t* const index = a.index + row;
  float* const prob = a.prob != nullptr ? a.prob + row : nullptr;

  // ---- the kept set
  Cut cut{-INFINITY, 0x7fffffff};
  u64 mass = 0;
  int count = 0;
  if (k > 0) {
    // the histogram of the groups' maxima, summed over the cluster
    u64 before;
    int bin;
    bool ok;
    if (c.ranks == 1) {
      ok = scan_bins(c, 2 * kBins, k, [&](int b) -> u64 { return s->hist[b]; }, &bin, &before);
    } else {
      const int per = 2 * kBins / c.ranks;
      for (int i = c.rank * per + c.tid; i < (c.rank + 1) * per; i += kThreads) {
        uint32_t v = 0;
        for (int j = 0; j < c.ranks; ++j) v += c.of(j)->hist[i];
        for (int j = 0; j < c.ranks; ++j) c.of(j)->count[i] = v;
      }
      c.sync();
      ok = scan_bins(c, 2 * kBins, k, [&](int b) -> u64 { return s->count[b]; }, &bin, &before);
    }
    // k groups have their maximum, so k logits lie, from here up
    const float from = ok ? floor_of(static_cast<uint32_t>(bin) << 21) : -INFINITY;
    ok = from > -INFINITY && build(c, r, from, &count);
    if (ok && !gather(c, r, count)) return;
    if (c.mode == kGathered && c.gathered <= kFew)
      return finish_few(c, r, k, p, keeps_min, u, index, prob);
    if (!ok || !select_steps<false>(c, r, &cut, from, static_cast<u64>(k)))
      select_radix<false>(c, r, &cut, from, static_cast<u64>(k));
  }
  bool summed = false;  // s->warp and slot hold the sums of all
  if (p < 1.0f) {
    const Steps steps(r.below_top(s->ready[1]), top);
    if (k == 0 && r.plain && steps.part()) {
      mass = weigh<true>(c, r, steps, &slot);
      summed = true;
    } else {
      mass = row_sum(c, r, [&](float x, int i) { return cut.keeps(x, i) ? r.fixed(x) : 0ull; },
                     &slot);
    }
    const double want = ceil(static_cast<double>(p) * static_cast<double>(mass));
    const u64 target = want > 1.0 ? static_cast<u64>(want) : 1ull;
    if (target < mass) {
      bool done = false;
      float from = cut.value;
      if (summed) {
        summed = false;
        int bin;
        u64 before;
        if (scan_cluster<true>(c, target, &bin, &before)) {
          from = steps.below(bin, top);
          if (build(c, r, from, &count) && !gather(c, r, count)) return;
          if (c.mode == kGathered && finish_steps(c, r, steps, bin, before, target, keeps_min, u,
                                                  index, prob))
            return;
          done = select_near<true>(c, r, &cut, steps, bin, target - before);
        }
      } else {
        if (r.plain)
          from = fmaxf(from,
                       r.below_top(log2(0.5 * static_cast<double>(mass - target) / (a.n * kOne))));
        done = c.mode != kAll && from > -INFINITY && select_steps<true>(c, r, &cut, from, target);
      }
      if (!done) select_radix<true>(c, r, &cut, from, target);
    }
    summed = summed && least == 0.0;
  }
  auto kept = [&](float x, int i) -> u64 {
    return cut.keeps(x, i) && keeps_min(x) ? r.fixed(x) : 0ull;
  };

  // ---- the draw
  u64 all = mass;
  if (c.mode == kAll && r.plain && k == 0 && !(p < 1.0f)) {
    if (least > 0.0) {  // what min-p may keep is listed
      if (build(c, r, out, &count) && !gather(c, r, count)) return;
      if (c.mode == kGathered && c.gathered <= kFew)
        return finish_few(c, r, 0, 1.0f, keeps_min, u, index, prob);
    } else {  // every element counts
      all = weigh<false>(c, r, Steps(0.0f, 1.0f), &slot);
      summed = true;
    }
  }
  if (!summed) all = row_sum(c, r, kept, &slot);
  const u64 target = drawn(u, all);
  if (locate(c, r, kept, slot, target, &at, &at_x)) {
    *index = static_cast<uint32_t>(at);
    if (prob != nullptr)
      *prob = share(r, at_x, r.fixed(at_x), all);
  }
}

}  // namespace

int sample_f32(long long rows, int n, const float* logits, const float* temperature,
               const int* top_k, const float* top_p, const float* min_p, const float* u,
               uint32_t* index, float* prob, cudaStream_t stream) {
  // Slices of 16384 logits (two CTAs to an SM), and smaller ones while the GPU
  // has SMs to spare.
  int c = 1;
  const long long fit = kMaxResident / 4;
  while (c < kMaxCluster && (n > c * kSlice || (rows * c * 2 <= num_sms() && n > c * 4096))) c *= 2;
  SampleArgs a{};
  a.n = n;
  a.slice = ((n + 3 + c - 1) / c + 3) & ~3;  // (up to three elements before the row)
  a.resident = static_cast<int>(std::min<long long>(a.slice, fit));
  a.logits = logits;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.u = u;
  a.index = index;
  a.prob = prob;
  a.err = device_error_ptr();
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
