// tree_attn.cu -- int8 attention of drafted tokens over the int8 KV cache
// (the pass that checks a tree of drafts; reef decodes one token at a time,
// so the definition is this file's).
//
// Sequence b has len committed keys and d drafted tokens, whose keys and
// values stand in the cache right behind them, at rows len + t.  Query (t,
// head) sees every committed key and, of the drafted ones, its own and its
// ancestors' (parents[t] is the drafted token that t follows, an earlier one,
// or -1; without parents, t - 1):
//   s_j = (q . k_j) * (q_scale * sm_scale * k_scale_j),  p = softmax(s),
//   out = sum_j p_j * v_scale_j * v_j.
// The G = heads_q / heads_kv heads of one KV head and the d drafts share its
// keys: G * d query rows read each cache byte once (up to a tile of 8 * NT rows
// at a time).
//
// Work is cut into segments (sequence, KV head, tile of query rows) and these
// into units of 128 keys, counted from the lengths on the device; every CTA of
// one wave takes the same number of units, so sequences of any lengths load the
// SMs alike.  A segment that one CTA covers is written straight to out;
// one that several share leaves a partial (max, sum, O) in each, at most two per
// CTA, which a second kernel joins in the order of the keys.
//
// The output is fp32 and meant to be.  V's codes are exact in f16; P takes the
// key's V scale in, P' = 2^(s - m + log2 v_scale + 11) <= 2^15 with m the
// running maximum of s + log2 v_scale, and goes into the product as two f16
// terms, head and remainder (22 bits together, where one f16 leaves 11), with
// fp32 sums; the softmax sum takes P' / v_scale.  Two kernels:
//
// Up to 16 query rows, tree_mma_kernel: meant to be bound by the cache's bytes.  K
// and V tiles by TMA through a ring; warp w owns keys [16w, 16w + 16) of every
// tile with its own running maximum, S^T = K . q^T by int8 mma.sync, O^T = V^T .
// P^T by f16 mma.sync (the rows are the n = 8 side, so few are padding).
//
// More rows, tree_tc_kernel: tcgen05 with a tile of 128 query rows, bound by
// the latency of the softmax warps, which go through their steps together (S in
// int8, P'.V twice in f16 leave the tensor pipe busy for a fifth).  Scores go into two TMEM tiles in turn, so that the
// next are there before the softmax of one ends; two warpgroups share a tile, a
// thread holding half of a query row's 128 scores; P' overwrites the scores (its
// heads in the first 64 columns, the rests in the last) and the product reads it
// there.  Another warpgroup turns V's codes into f16, [key][dim] as they stand: the
// product takes B with the dims contiguous.  The tensor pipe truncates when it adds
// to O (1.4e-5 of the result over 16k keys), so every six tiles O is added to a
// second accumulator by the softmax threads, with rounding, and begins anew (5 of
// 175 us over 16k keys).
//
// Up to 64 query rows (of a KV head), the tile of 128 holds them two or four times:
// each copy takes its own keys of every tile of 128 and zeros for the others' P', so
// that all warps have work (64 x 8 drafts, 8 heads on one: 53 -> 41 us); the copies share
// the maxima and add up at the end.
//
// Measured (a call in a graph of them, inputs in L2 where they fit; with everything cold
// in brackets): 4 drafts over 499 keys, 32 heads of their own, 8.7 us (8.7), which is the
// launch and three round trips (lengths, queries, keys).  64 sequences over up to 4096
// keys, 8 heads on one: 1 draft each (70 MB of cache) 26 us, 2 drafts 35, 8 drafts (ragged,
// 54 MB) 35 (39), of which 11 are the shares, the first loads, the epilogues and the join.
// Two sequences over 16301 keys, 64 drafts, 64 heads on 8 (68.5 Gflop): 178 us (188), 0.38
// Pflop/s of products or 0.77 with the rests; a tile takes 5000 cycles, of which the
// tensor pipe is busy for 1100.  What holds it is latency: a scheduler has two softmax
// warps, a converter and one that mostly waits, and issues in 0.48 of its cycles (0.42 for
// 64 x 8).  Per instruction issued, warps stand 2.0 cycles at loads from TMEM and waits
// for barriers in memory, 1.6 at the fixed latencies of arithmetic, 1.4 at the barrier on
// which all eight softmax warps meet once a tile: they read scales, take exponentials and
// wait for scores at the same time.  Left out for a measurement, the loads of the scales
// save 27 us, the rests 11, the exponentials 4.  Up to 32 rows a tile takes 2500 cycles.
// Measured and dropped: quarter rows in four warpgroups
// (they spill; with two copies they do not, and 64 x 8 takes 42 us: what a warp does
// once a tile counts twice as often), scores taken a tile ahead, a barrier per pair of
// warps, scores in fragments of 16 x 8 (a quarter of the loads of scales, but 184 us), O
// moved by the converters.
#include "attn_mma.cuh"
#include "common.cuh"
#include "ops.h"

#include <cuda_fp16.h>

#include <algorithm>

namespace reef {

namespace {

constexpr int kTThreads = 256;  // eight warps
constexpr int kTWarps = kTThreads / 32;
constexpr int kTileKeys = 128;  // keys per unit
constexpr int kMaxBatch = kMaxTreeBatch;  // a CTA holds every sequence's length
constexpr int kPartRow = 132;     // floats per row of a partial: m, l, 2 unused, O[128]
constexpr int kMaxTileRows = 16;  // query rows per segment (tree_mma_kernel)
constexpr int kTcRows = 128;      // the same (tree_tc_kernel)
constexpr int kMaxCtasPerSm = 2;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 4.0f;   // the maximum is raised when a score passes it by more (log2)
constexpr float kLift = 11.0f;  // log2 of P' at the maximum
// A V scale below counts as 0, and stands for its key in P' and the softmax sum.  P' <=
// 2^15 over it, 2^24 times, must stay below 2^128; and the P' of such a key, beside scales
// of up to 2^48, above 2^-126 down to 2^-25 of their weight (11 - 64 - 48 - 25).
constexpr float kNoScale = 0x1p-64f;

struct TreeArgs {
  int batch, drafts, heads_q, heads_kv, max_len;
  int group;   // query heads per KV head
  int rows;    // group * drafts
  int qtiles;  // segments per (sequence, KV head)
  int ctas;
  int per_cta;           // 1: a segment per CTA, nothing to join; 0: equal shares of the units
  float sm_scale;
  const int8_t* q8;      // [B][T][Hq][128]
  const float* q_scale;  // [B][T][Hq]
  const float* k_scale;  // [B][Hkv][max_len]
  const float* v_scale;
  const int* lens;        // [B]
  const int* draft_lens;  // [B] or null
  const int* parents;     // [B][T] or null
  float* part;            // [ctas][2][tile rows][kPartRow]
  int4* meta;             // [ctas]: what the CTA's units cover, see Meta
  float* out;             // [B][T][Hq][128]
  int* err;
};

// meta[c]: x first segment, y 1 when it began in an earlier CTA, z last
// segment, w not 0 when it goes on in the next CTA: its query rows (of the KV head,
// live). x = -1 for a CTA without units.
template <int kStages>
struct TLayout {  // shared memory layout (bytes from a 1024-aligned base)
  static constexpr int kKV = 2 * kTileKeys * 128;  // K then V, int8 [128][128] SW128
  static constexpr int kScales = kStages * kKV;    // per stage ks[128], vs[128]
  static constexpr int kWarpM = kScales + kStages * 1024;  // m[8][16], then l[8][16]
  static constexpr int kAnc = kWarpM + 2 * kTWarps * kMaxTileRows * 4;  // u64[64]
  static constexpr int kPar = kAnc + kMaxDrafts * 8;                    // int[64]
  static constexpr int kPre = kPar + kMaxDrafts * 4;                    // int[batch + 1]
  static constexpr int kBars = kPre + (kMaxBatch + 4) * 4;              // full[], empty[]
  static constexpr int kEnd = kBars + 2 * kStages * 8;
  static constexpr int kBytes = kEnd + 1024;  // + alignment slack
};
static_assert(TLayout<3>::kBars % 8 == 0 && TLayout<3>::kAnc % 8 == 0, "aligned");
static_assert(TLayout<3>::kBytes <= 232448 / 2 - 1024, "two CTAs per SM");
static_assert(TLayout<6>::kBytes <= 232448 - 1024, "one CTA per SM");
static_assert(kTWarps * 8 * 128 * 4 <= TLayout<3>::kKV, "eight rows merge inside a stage");

// two f32 -> f16 pair, the first in the low half
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// p - h, in one step (the difference is exact)
__device__ __forceinline__ float less_half(float p, uint32_t h) {
  float d;
  asm("{.reg .b16 m; mov.b16 m, 0xBC00; fma.rn.f32.f16 %0, %1, m, %2;}"  // h * -1 + p
      : "=f"(d) : "h"(static_cast<uint16_t>(h)), "f"(p));
  return d;
}
// what the pair leaves of them, as another pair
__device__ __forceinline__ uint32_t rest_of(float lo, float hi, uint32_t pair) {
  return half2_of(less_half(lo, pair), less_half(hi, pair >> 16));
}

// two f32 in a register pair, and arithmetic on both at once
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two int8 codes with their sign bits flipped, each under the exponent byte
// 0x64, i.e. the f16 values code + 1152 -> the codes, exactly
__device__ __forceinline__ uint32_t unbias(uint32_t x) {
  const uint32_t bias = 0x64806480u;  // 1152
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x),
                            *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&v);
}
// split_biased's pairs without the bias: the codes themselves
__device__ __forceinline__ void split_codes(uint32_t w, uint32_t& even, uint32_t& odd) {
  split_biased(w, even, odd);
  even = unbias(even);
  odd = unbias(odd);
}

// log2 and reciprocal of a V scale (2^-22 off at most); of one that counts as
// 0, of kNoScale instead (its codes are taken as zeros).  The reciprocal is
// finite whatever the scale, so a masked key's P' = 0 times it is 0.
__device__ __forceinline__ float scale_log2(float vs) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaxf(vs, kNoScale)));
  return vs == vs ? y : vs;
}
__device__ __forceinline__ float scale_rcp(float vs) {
  return __frcp_rn(fmaxf(vs, kNoScale));
}

// d of sequence b, 0 when it has none or its rows do not fit in the cache
__device__ __forceinline__ int drafts_of(const TreeArgs& a, int b, int len, bool* bad) {
  const int d = a.draft_lens == nullptr ? a.drafts : min(a.draft_lens[b], a.drafts);
  *bad = len < 0 || len > a.max_len || d > a.max_len - len;
  return *bad || d < 0 ? 0 : d;
}

// pre[b] = 128-key tiles of the sequences before b (all threads of the block);
// returns after a barrier
template <int kThreads>
__device__ __forceinline__ void count_tiles(const TreeArgs& a, int* pre, int* scratch) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kPer = (kMaxBatch + kThreads - 1) / kThreads;
  const int b0 = tid * kPer;
  int t[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    t[i] = 0;
    if (b0 + i < a.batch) {
      const int len = a.lens[b0 + i];
      bool bad;
      const int d = drafts_of(a, b0 + i, len, &bad);
      if (d > 0) t[i] = (len + d + kTileKeys - 1) / kTileKeys;
      if (bad && blockIdx.x == 0) record_error(a.err, kDevBadPosition);
    }
    sum += t[i];
  }
  int run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += v;
  }
  if (lane == 31) scratch[warp] = run;
  __syncthreads();
  run -= sum;
  for (int w = 0; w < warp; ++w) run += scratch[w];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (b0 + i < a.batch) pre[b0 + i] = run;
    run += t[i];
    if (b0 + i == a.batch - 1) pre[a.batch] = run;
  }
  __syncthreads();
}

// What a segment's beginning and end take, in units: 3 measured best at 8 to 512
// query rows (against none: 64 x 8 drafts over up to 4k keys 38.6 -> 37.1 us, 2 x 64 over
// 16k 177 -> 173), 2 and 4 a little behind.
constexpr int kCost = 3;

// A unit's place: sequence, (KV head, tile of query rows), tile of keys.
struct Place {
  int b, hq, tile, tiles;
};

// The first unit of CTA `cta` and how many it has.  With a segment per CTA the
// sequence's length alone says so; otherwise every sequence's does (count_tiles:
// all threads come here).
template <int kThreads>
__device__ __forceinline__ Place share_of(const TreeArgs& a, int cta, int* pre, int* scratch,
                                          int* nunits) {
  const int per_seq = a.heads_kv * a.qtiles;
  Place p{};
  if (a.per_cta) {
    p.b = cta / per_seq;
    p.hq = cta % per_seq;
    const int len = a.lens[p.b];
    bool bad;
    const int d = drafts_of(a, p.b, len, &bad);
    if (bad && p.hq == 0 && threadIdx.x == 0) record_error(a.err, kDevBadPosition);
    p.tiles = d > 0 ? (len + d + kTileKeys - 1) / kTileKeys : 0;
    *nunits = p.tiles;
    __syncthreads();  // (as count_tiles: what the caller wrote before is in)
    return p;
  }
  count_tiles<kThreads>(a, pre, scratch);
  // Equal shares of a line on which kCost that stand for a segment's beginning come
  // before its units.  An even lane looks for the share's first unit, an odd one for the
  // next share's.
  const int batch = a.batch, lane = threadIdx.x & 31;
  const long long all = (static_cast<long long>(pre[batch]) + batch * kCost) * per_seq;
  const long long v = all * (cta + (lane & 1)) / a.ctas;
  int lo = 0, hi = batch - 1;  // the last sequence that begins at v or before
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((static_cast<long long>(pre[mid]) + mid * kCost) * per_seq <= v) lo = mid;
    else hi = mid - 1;
  }
  const long long off = v - (static_cast<long long>(pre[lo]) + lo * kCost) * per_seq;
  p.b = lo;
  p.tiles = pre[lo + 1] - pre[lo];
  const unsigned each = static_cast<unsigned>(p.tiles) + kCost;
  p.hq = off >> 32 == 0 ? static_cast<int>(static_cast<unsigned>(off) / each)
                        : static_cast<int>(off / each);
  p.tile = max(0, static_cast<int>(off - static_cast<long long>(p.hq) * each) - kCost);
  const long long before =
      static_cast<long long>(pre[lo]) * per_seq + static_cast<long long>(p.hq) * p.tiles + p.tile;
  *nunits = static_cast<int>(__shfl_sync(0xffffffffu, before, 1) -
                             __shfl_sync(0xffffffffu, before, 0));
  p.b = __shfl_sync(0xffffffffu, p.b, 0);
  p.hq = __shfl_sync(0xffffffffu, p.hq, 0);
  p.tile = __shfl_sync(0xffffffffu, p.tile, 0);
  p.tiles = __shfl_sync(0xffffffffu, p.tiles, 0);
  if (*nunits > 0 && p.tiles == 0) {  // the next sequence that has any
    p.hq = p.tile = 0;
    do {
      ++p.b;
      p.tiles = pre[p.b + 1] - pre[p.b];
    } while (p.tiles == 0);
  }
  return p;
}

__device__ __forceinline__ void next_unit(const int* pre, int batch, int per_seq, Place& p) {
  if (++p.tile < p.tiles) return;
  p.tile = 0;
  if (++p.hq < per_seq) return;
  p.hq = 0;
  do {
    ++p.b;
    p.tiles = p.b < batch ? pre[p.b + 1] - pre[p.b] : 1;
  } while (p.tiles == 0);
}

// NT: query rows of a segment / 8; with two the accumulators take 237 registers, and
// one CTA per SM with a ring twice as deep (41 us for 16 x 4 drafts, 4 heads each
// of 8 KV heads, 2k keys) beats two that spill (50 us): what the ring leaves of the
// L1 is too little for spills.
template <int NT, int kStages, int kPerSm>
__global__ void __launch_bounds__(kTThreads, kPerSm)
    tree_mma_kernel(const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap, TreeArgs a) {
  using TL = TLayout<kStages>;
  constexpr int kRows = 8 * NT;
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) &
                                           ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + TL::kBars);
  uint64_t* empty = full + kStages;
  float* warp_m = reinterpret_cast<float*>(sm + TL::kWarpM);  // [8][16]
  float* warp_l = warp_m + kTWarps * kMaxTileRows;            // [8][16]
  unsigned long long* anc = reinterpret_cast<unsigned long long*>(sm + TL::kAnc);
  int* par = reinterpret_cast<int*>(sm + TL::kPar);
  int* pre = reinterpret_cast<int*>(sm + TL::kPre);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, tig = lane & 3;
  const int cta = blockIdx.x;

  if (tid == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kTWarps);
    }
    fence_barrier_init();
  }
  pdl_wait();
  pdl_trigger();  // the joining kernel waits for this grid's completion
  const int per_seq = a.heads_kv * a.qtiles;
  int nunits;
  Place at = share_of<kTThreads>(a, cta, pre, par, &nunits);  // (publishes the mbarriers too)
  if (nunits == 0) {
    if (tid == 0 && !a.per_cta) a.meta[cta] = make_int4(-1, 0, -1, 0);
    return;
  }
  Place ahead = at;  // next unit to issue (thread 0)
  const int first_seg = at.b * per_seq + at.hq;
  const bool first_cut = at.tile > 0;

  auto issue = [&](int j) {
    const int s = j % kStages;
    const int pair = ahead.b * a.heads_kv + ahead.hq / a.qtiles;
    const int key0 = ahead.tile * kTileKeys;
    // scales: whole 16-byte groups inside the row (max_len % 4 == 0)
    const int n4 = min(kTileKeys, a.max_len - key0);
    const long long srow = static_cast<long long>(pair) * a.max_len + key0;
    uint8_t* kv = sm + s * TL::kKV;
    float* sc = reinterpret_cast<float*>(sm + TL::kScales + s * 1024);
    mbar_arrive_expect_tx(&full[s], static_cast<uint32_t>(2 * kTileKeys * 128 + 2 * n4 * 4));
    tma_load_3d(kv, &kmap, &full[s], 0, key0, pair);
    tma_load_3d(kv + kTileKeys * 128, &vmap, &full[s], 0, key0, pair);
    bulk_load(sc, a.k_scale + srow, n4 * 4, &full[s]);
    bulk_load(sc + kTileKeys, a.v_scale + srow, n4 * 4, &full[s]);
    if (j + 1 < nunits) next_unit(pre, a.batch, per_seq, ahead);
  };
  int issued = 0;  // units issued (thread 0)
  if (tid == 0)
    for (; issued < kStages && issued < nunits; ++issued) issue(issued);

  const float base = a.sm_scale * kLog2e;
  const int wk = warp * 16;  // this warp's first key in a tile
  // fragment rows of this lane in the ldmatrix loads (keys wk + [0, 16))
  const int frow = wk + ((lane >> 3) & 1) * 8 + (lane & 7);

  // per-segment state; rows nt*8 + 2 tig + {0, 1} of the tile are this
  // thread's columns (see decode_attn.cu for the fragments)
  uint32_t qb[4][NT][2];
  float qsc[NT][2];
  float o[8][NT][4];
  float m[NT][2], l[NT][2];
  int len = 0, d = 0, row0 = 0;
  long long qbase = 0;  // row (b, t = 0, first head of the KV head) of q and out
  bool ok = true;
  int waited = 0;  // units whose stage thread 0 saw complete

  // query row r of the segment's KV head -> row of q8 / q_scale / out
  auto qrow = [&](int r) {
    const int t = r / a.group;
    return qbase + static_cast<long long>(t) * a.heads_q + (r - t * a.group);
  };

  for (int j = 0; j < nunits; ++j) {
    const int s = j % kStages;
    if (j == 0 || at.tile == 0) {  // a new segment: its tree, q, a fresh state
      const int hkv = at.hq / a.qtiles;
      row0 = (at.hq % a.qtiles) * kRows;
      qbase = static_cast<long long>(at.b) * a.drafts * a.heads_q + hkv * a.group;
      // every load at once (all drafts' rows are there, whoever is live): one round trip
      len = a.lens[at.b];
      int up = 0;
      if (a.parents != nullptr && tid < a.drafts)
        up = a.parents[static_cast<long long>(at.b) * a.drafts + tid];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = row0 + nt * 8 + g;
        const uint32_t* q32 =
            reinterpret_cast<const uint32_t*>(a.q8) + (r < a.rows ? qrow(r) * 32 : 0);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          qb[ks][nt][0] = q32[8 * ks + tig];
          qb[ks][nt][1] = q32[8 * ks + 4 + tig];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int rc = row0 + nt * 8 + 2 * tig + e;
          qsc[nt][e] = a.q_scale[rc < a.rows ? qrow(rc) : 0];
          m[nt][e] = -INFINITY;
          l[nt][e] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][nt][e] = 0.0f;
      }
      bool bad;
      d = drafts_of(a, at.b, len, &bad);
      if (tid < a.drafts) par[tid] = up;
      __syncthreads();
      if (tid < d) {
        unsigned long long bits = (2ull << tid) - 1;  // a chain
        if (a.parents != nullptr) {
          bits = 0;
          for (int t = tid; t >= 0;) {  // strictly downwards: it ends
            bits |= 1ull << t;
            const int p = par[t];
            t = p < t ? p : -1;
          }
        }
        anc[tid] = bits;
      }
      const int live = d * a.group;  // rows past it are computed as zeros
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          if (row0 + nt * 8 + g >= live) qb[ks][nt][0] = qb[ks][nt][1] = 0u;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          qsc[nt][e] = row0 + nt * 8 + 2 * tig + e < live ? qsc[nt][e] * base : 0.0f;
      }
      __syncthreads();  // anc is in
    }
    if (ok) ok = mbar_wait(&full[s], (j / kStages) & 1, a.err, kDevTimeoutFull);
    ok = __all_sync(0xffffffffu, ok);  // what follows is the whole warp's, also after a timeout
    if (ok && tid == 0) waited = j + 1;
    const int key0 = at.tile * kTileKeys + wk;  // this warp's first key
    if (ok && key0 < len + d) {
      const uint8_t* kv = sm + s * TL::kKV;
      const float* ksc = reinterpret_cast<const float*>(sm + TL::kScales + s * 1024);
      // ---- S^T = K . q^T: rows keys wk + g (c 0, 1), wk + g + 8 (c 2, 3)
      int c[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[nt][e] = 0;
      const uint32_t kb = smem_u32(kv);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint32_t ka[4];
        ldsm_x4(kb + sw128(frow, 2 * ks + (lane >> 4)), ka);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_s8_16832(c[nt], ka, qb[ks][nt][0], qb[ks][nt][1]);
      }
      // ---- scores in log2 units.  Committed keys are seen by every row; a
      // drafted key by the rows whose ancestors it is among.  A key that no
      // row may see brings neither its score nor its scales in.
      const bool edge = key0 + 16 > len;
      const int n_lo = key0 + g - len, n_hi = n_lo + 8;  // drafted token, < 0: committed
      const float ks_lo = ksc[wk + g], ks_hi = ksc[wk + g + 8];
      const float vs_lo = n_lo < d ? ksc[kTileKeys + wk + g] : 0.0f;
      const float vs_hi = n_hi < d ? ksc[kTileKeys + wk + g + 8] : 0.0f;
      const float lv_lo = scale_log2(vs_lo), lv_hi = scale_log2(vs_hi);
      const float rv_lo = scale_rcp(vs_lo), rv_hi = scale_rcp(vs_hi);
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sc[nt][0] = fmaf(small_i2f(c[nt][0]) * qsc[nt][0], ks_lo, lv_lo);
        sc[nt][1] = fmaf(small_i2f(c[nt][1]) * qsc[nt][1], ks_lo, lv_lo);
        sc[nt][2] = fmaf(small_i2f(c[nt][2]) * qsc[nt][0], ks_hi, lv_hi);
        sc[nt][3] = fmaf(small_i2f(c[nt][3]) * qsc[nt][1], ks_hi, lv_hi);
        if (edge) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int t = (row0 + nt * 8 + 2 * tig + e) / a.group;
            const unsigned long long bits = t < d ? anc[t] : 0ull;
            if (n_lo >= 0 && (n_lo >= d || ((bits >> n_lo) & 1ull) == 0)) sc[nt][e] = -INFINITY;
            if (n_hi >= 0 && (n_hi >= d || ((bits >> n_hi) & 1ull) == 0))
              sc[nt][e + 2] = -INFINITY;
          }
        }
      }
      // ---- the running maximum, raised only when a score passes it by more
      // than 2^kLazy
      bool need = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) need |= fmaxf(sc[nt][e], sc[nt][e + 2]) > m[nt][e] + kLazy;
      if (__any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(sc[nt][e], sc[nt][e + 2]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const bool up = x > m[nt][e] + kLazy;
            const float al = up ? fast_exp2(m[nt][e] - x) : 1.0f;  // 0 from -inf
            if (up) m[nt][e] = x;
            l[nt][e] *= al;
#pragma unroll
            for (int cc = 0; cc < 8; ++cc) {
              o[cc][nt][e] *= al;
              o[cc][nt][e + 2] *= al;
            }
          }
      }
      // ---- P', its sum without the V scale, and its two f16 terms, transposed
      // into the B operand
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float r0 = (m[nt][0] == -INFINITY ? 0.0f : m[nt][0]) - kLift;
        const float r1 = (m[nt][1] == -INFINITY ? 0.0f : m[nt][1]) - kLift;
        float p0 = fast_exp2(sc[nt][0] - r0), p1 = fast_exp2(sc[nt][1] - r1);
        float p2 = fast_exp2(sc[nt][2] - r0), p3 = fast_exp2(sc[nt][3] - r1);
        l[nt][0] = fmaf(p2, rv_hi, fmaf(p0, rv_lo, l[nt][0]));
        l[nt][1] = fmaf(p3, rv_hi, fmaf(p1, rv_lo, l[nt][1]));
        if (vs_lo < kNoScale) p0 = p1 = 0.0f;
        if (vs_hi < kNoScale) p2 = p3 = 0.0f;
        const uint32_t h0 = half2_of(p0, p1), h1 = half2_of(p2, p3);
        ph[nt][0] = movmatrix_t(h0);
        ph[nt][1] = movmatrix_t(h1);
        pl[nt][0] = movmatrix_t(rest_of(p0, p1, h0));
        pl[nt][1] = movmatrix_t(rest_of(p2, p3, h1));
      }
      // ---- O^T += V^T . P^T; ldmatrix .trans matrices (keys wk + [0, 8),
      // chunk 2cc), (keys wk + [8, 16), chunk 2cc), then 2cc + 1
      const uint32_t vb = smem_u32(kv + kTileKeys * 128);
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        uint32_t r[4];
        ldsm_x4_t(vb + sw128(frow, 2 * cc + (lane >> 4)), r);
        uint32_t va[4], vc[4];
        split_codes(r[0], va[0], va[1]);
        split_codes(r[1], va[2], va[3]);
        split_codes(r[2], vc[0], vc[1]);
        split_codes(r[3], vc[2], vc[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // the tile's own sum, then one rounded add: the tensor cores' adds
          // truncate, and a long row of them would show
          float t0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, t1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma_f16_16816(t0, va, pl[nt][0], pl[nt][1]);
          mma_f16_16816(t1, vc, pl[nt][0], pl[nt][1]);
          mma_f16_16816(t0, va, ph[nt][0], ph[nt][1]);
          mma_f16_16816(t1, vc, ph[nt][0], ph[nt][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[2 * cc][nt][e] += t0[e];
            o[2 * cc + 1][nt][e] += t1[e];
          }
        }
      }
    }
    // ---- release the stage; thread 0 refills it once every warp has (after
    // the merge below when this unit ends a segment: the merge uses it)
    const bool ends = at.tile + 1 == at.tiles;
    const bool last = j + 1 == nunits || ends;
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
    if (tid == 0 && ok && !last && j + kStages < nunits) {
      ok = mbar_wait(&empty[s], (j / kStages) & 1, a.err, kDevTimeoutEmpty);
      if (ok) issue(issued++);
    }

    // ---- end of the segment in this CTA: merge the eight warps, eight rows
    // at a time.  Each warp weighs its state by 2^(m_w - max) and writes it to
    // its own slot; the slots are summed in warp order.
    if (last) {
      // whole here (and written out), or cut: its first tiles elsewhere
      // (slot 0), or only its last (slot 1)
      const int seg = at.b * per_seq + at.hq;
      const bool cut_before = seg == first_seg && first_cut;
      const bool whole = ends && !cut_before;
      float* slot = a.part + (static_cast<long long>(cta) * 2 + (cut_before ? 0 : 1)) * kRows *
                                 kPartRow;
      if (j + 1 == nunits && tid == 0 && !a.per_cta)
        a.meta[cta] = make_int4(first_seg, first_cut ? 1 : 0, seg, ends ? 0 : d * a.group);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = l[nt][e];
          x += __shfl_xor_sync(0xffffffffu, x, 4);
          x += __shfl_xor_sync(0xffffffffu, x, 8);
          x += __shfl_xor_sync(0xffffffffu, x, 16);
          l[nt][e] = x;
          if (g == 0) warp_m[warp * kMaxTileRows + nt * 8 + 2 * tig + e] = m[nt][e];
        }
      __syncthreads();  // every warp's m is in, and every warp is done with stage s
      float ws[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int rr = nt * 8 + 2 * tig + e;
          float mx = -INFINITY;
#pragma unroll
          for (int w = 0; w < kTWarps; ++w) mx = fmaxf(mx, warp_m[w * kMaxTileRows + rr]);
          ws[nt][e] = m[nt][e] == -INFINITY ? 0.0f : exp2f(m[nt][e] - mx);
          if (g == 0) warp_l[warp * kMaxTileRows + rr] = l[nt][e] * ws[nt][e];
        }
      float* mrg = reinterpret_cast<float*>(sm + s * TL::kKV);
      float* mine = mrg + warp * 8 * 128;  // [8][128]
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int cc = 0; cc < 8; ++cc)
            *reinterpret_cast<float2*>(mine + (2 * tig + e) * 128 + 16 * cc + 2 * g) =
                make_float2(o[cc][nt][e] * ws[nt][e], o[cc][nt][e + 2] * ws[nt][e]);
        __syncthreads();
        for (int i = tid; i < 8 * 128; i += kTThreads) {
          const int rr = nt * 8 + (i >> 7), dim = i & 127;
          float acc = 0.0f, ls = 0.0f;
#pragma unroll
          for (int w = 0; w < kTWarps; ++w) {
            acc += mrg[w * 8 * 128 + i];
            ls += warp_l[w * kMaxTileRows + rr];
          }
          if (whole) {
            const int r = row0 + rr;
            if (r < d * a.group) a.out[qrow(r) * 128 + dim] = acc / ls;
          } else {
            float* prow = slot + rr * kPartRow;
            prow[4 + dim] = acc;
            if (dim == 0) {
              float mx = -INFINITY;
#pragma unroll
              for (int w = 0; w < kTWarps; ++w) mx = fmaxf(mx, warp_m[w * kMaxTileRows + rr]);
              prow[0] = mx;
              prow[1] = ls;
            }
          }
        }
        __syncthreads();  // the merge area (and, after the last, warp_m / warp_l) is free
      }
      if (tid == 0 && ok && j + kStages < nunits) {  // the refill held back above
        fence_proxy_async_smem();  // the merge's stores before the copy's writes
        ok = mbar_wait(&empty[s], (j / kStages) & 1, a.err, kDevTimeoutEmpty);
        if (ok) issue(issued++);
      }
    }
    if (j + 1 < nunits) next_unit(pre, a.batch, per_seq, at);
  }
  // copies still in flight land before exit (only after a timeout can any
  // remain)
  if (tid == 0 && !ok) {
    for (int j = waited; j < issued; ++j)
      mbar_wait(&full[j % kStages], (j / kStages) & 1, a.err, kDevTimeoutDrain);
  }
}

// ---- more rows: tcgen05 -----------------------------------------------------------

constexpr int kParts = 2;       // softmax warpgroups: parts of a row
constexpr int kCols = kTileKeys / kParts;  // keys of a row that a thread holds
constexpr int kSoftmax = 128 * kParts;     // their threads
constexpr int kCThreads = 256 + kSoftmax;  // and the control and converter warpgroups
// Registers: 128 a thread at launch; the control warpgroup drops to 72 and the
// converters to 88, each softmax warpgroup rises to 176.
constexpr uint32_t kRegsControl = 72, kRegsConvert = 88, kRegsSoftmax = 176;
static_assert(kRegsControl + kRegsConvert + kParts * kRegsSoftmax <= 65536 / 128,
              "register split exceeds the launch allocation");
constexpr int kFlushTiles = 6;  // tiles (and one more at the end) whose adds O takes
constexpr int kKStages = 4;     // K tiles in flight (int8, 16 KiB)
constexpr int kVStages = 3;     // V tiles in flight (the same)

struct CL {  // shared memory layout (bytes from a 1024-aligned base)
  static constexpr int kQ = 0;                            // int8 [128][128] SW128
  static constexpr int kK = 16384;                        // kKStages x 16 KiB
  static constexpr int kV = kK + kKStages * 16384;        // kVStages x 16 KiB
  // 2 x f16 [2 dim halves][128 keys][64] SW128
  static constexpr int kVf = kV + kVStages * 16384;
  // [2 tiles][warps][ks, log2 vs, 1 / vs][kCols]
  static constexpr int kScales = kVf + 2 * 32768;
  static constexpr int kML = kScales + 2 * kSoftmax / 32 * 3 * kCols * 4;  // [2 tiles][parts][128]
  static constexpr int kPar = kML + 2 * kSoftmax * 4;         // int[64]
  static constexpr int kPre = kPar + kMaxDrafts * 4;      // int[batch + 1]
  static constexpr int kKeep = kPre + (kMaxBatch + 4) * 4;  // int[8][softmax threads]
  static constexpr int kBars = kKeep + 8 * kSoftmax * 4;
  static constexpr int kNumBars = 9 + 2 * kKStages + 2 * kVStages + 4;
  static constexpr int kTmemSlot = kBars + kNumBars * 8;
  static constexpr int kBytes = kTmemSlot + 16 + 1024;
};
static_assert(CL::kBytes <= 232448, "one CTA per SM");
static_assert(CL::kBars % 8 == 0, "aligned");

// B operand with N contiguous (128-byte swizzle): 64 values of N to a 128-byte
// row of one k, rows of 8 k 1024 bytes together and those back to back (stride
// byte offset), the next 64 of N 16384 bytes on (leading byte offset).
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(16384u >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

// a load that stays where it is written (a plain one would sink to its use)
__device__ __forceinline__ float load_now(const float* p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

// a word put aside in shared memory while registers are short
__device__ __forceinline__ void put_aside(uint32_t at, int v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v));
}
__device__ __forceinline__ int take_back(uint32_t at) {
  int v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}

// A CTA's tiles of one segment.
struct Piece {
  Place at;  // its first tile
  int n;     // tiles
};
__device__ __forceinline__ Piece piece_at(const Place& at, int left) {
  return Piece{at, min(at.tiles - at.tile, left)};
}
__device__ __forceinline__ void next_piece(const int* pre, int batch, int per_seq, Place& at,
                                           int n, int& left) {
  left -= n;
  at.tile += n - 1;
  if (left > 0) next_unit(pre, batch, per_seq, at);
}

template <int kCopies>
__global__ void __launch_bounds__(kCThreads, 1)
    tree_tc_kernel(const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, TreeArgs a) {
  // (each copy takes its share of a tile's; adding zeros loses nothing)
  constexpr int kFlush = kFlushTiles * kCopies;
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) &
                                           ~static_cast<uintptr_t>(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sm + CL::kBars);  // the segment's Q is in
  uint64_t* o_free = q_full + 1;    // its accumulator has been read
  uint64_t* drain = q_full + 2;
  uint64_t* p_full = q_full + 3;    // [2] P' of an even / odd tile is in its S_x
  uint64_t* s_full = q_full + 5;    // [2] S_x done
  uint64_t* o_done = q_full + 7;    // [2] the tile's product is in O
  uint64_t* k_full = q_full + 9;
  uint64_t* k_empty = k_full + kKStages;
  uint64_t* v_full = k_empty + kKStages;
  uint64_t* v_empty = v_full + kVStages;
  uint64_t* f_full = v_empty + kVStages;  // [2] f16 V
  uint64_t* f_empty = f_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + CL::kTmemSlot);
  int* par = reinterpret_cast<int*>(sm + CL::kPar);
  int* pre = reinterpret_cast<int*>(sm + CL::kPre);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x;
  int* err = a.err;
  if (tid == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    mbar_init(q_full, kSoftmax);
    mbar_init(o_free, kSoftmax);
    mbar_init(drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&o_done[i], 1);
      mbar_init(&p_full[i], kSoftmax);
      mbar_init(&f_full[i], 4);
      mbar_init(&f_empty[i], 1);
    }
    for (int i = 0; i < kKStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < kVStages; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 4);
    }
    fence_barrier_init();
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  int nunits;
  Place at = share_of<kCThreads>(a, cta, pre, par, &nunits);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // columns: S_0 [0, 128), S_1 [128, 256), O [256, 384), the second accumulator
  // [384, 512)
  const uint32_t tS = tmem, tO = tmem + 256, tSum = tmem + 384;

  const int per_seq = a.heads_kv * a.qtiles;
  int left = nunits;
  const int first_seg = at.b * per_seq + at.hq;
  const bool first_cut = at.tile > 0;
  if (nunits == 0 && tid == 0 && !a.per_cta) a.meta[cta] = make_int4(-1, 0, -1, 0);

  if (warp < 4) {
    setmaxnreg_dec<kRegsControl>();
    if (warp == 0 && lane < 2) {
      // ---------------- TMA: lane 0 the K ring, lane 1 the V ring ----------------
      const int stages = lane == 0 ? kKStages : kVStages;
      uint64_t* full = lane == 0 ? k_full : v_full;
      uint64_t* empty = lane == 0 ? k_empty : v_empty;
      const CUtensorMap* map = lane == 0 ? &kmap : &vmap;
      uint8_t* ring = sm + (lane == 0 ? CL::kK : CL::kV);
      int issued = 0;
      for (; issued < nunits; ++issued) {
        const int s = issued % stages;
        if (!mbar_wait(&empty[s], ((issued / stages) & 1) ^ 1u, err, kDevTimeoutEmpty)) break;
        mbar_arrive_expect_tx(&full[s], 16384);
        tma_load_3d(ring + s * 16384, map, &full[s], 0, at.tile * kTileKeys,
                    at.b * a.heads_kv + at.hq / a.qtiles);
        if (issued + 1 < nunits) next_unit(pre, a.batch, per_seq, at);
      }
      // copies in flight land before exit
      for (int j = issued > stages ? issued - stages : 0; j < issued; ++j)
        mbar_wait(&full[j % stages], (j / stages) & 1, err, kDevTimeoutDrain);
    } else if (warp == 1 && lane == 0 && nunits > 0) {
      // ---------------- MMA ----------------
      constexpr uint32_t kIdescS = idesc_i8(128, 128);
      constexpr uint32_t kIdescO = idesc_f16(128, 128, true);
      const uint32_t sq = smem_u32(sm + CL::kQ);
      int kc = 0, tc = 0;  // K tiles multiplied, tiles' products issued
      bool ok = true;
      auto issue_s = [&] {  // the next K tile against Q into its S_x
        const int s = kc % kKStages, x = kc & 1;
        if (!mbar_wait(&k_full[s], (kc / kKStages) & 1, err, kDevTimeoutFull)) return false;
        tc_fence_after();
        const uint32_t sk = smem_u32(sm + CL::kK + s * 16384);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_i8(tS + x * 128, smem_desc_k_sw128(sq + kk * 32), smem_desc_k_sw128(sk + kk * 32),
                 kIdescS, kk > 0 ? 1u : 0u);
        mma_commit(&s_full[x]);
        mma_commit(&k_empty[s]);
        ++kc;
        return true;
      };
      for (int piece = 0; left > 0 && ok; ++piece) {
        const Piece w = piece_at(at, left);
        ok = mbar_wait(q_full, piece & 1, err, kDevTimeoutFull);
        if (ok) ok = issue_s();
        if (ok && w.n > 1) ok = issue_s();
        for (int j = 0; j < w.n && ok; ++j, ++tc) {
          const int x = tc & 1;
          // (the softmax may be a tile ahead of this thread, hence two p_full)
          ok = mbar_wait(&p_full[x], (tc >> 1) & 1, err, kDevTimeoutFull) &&
               mbar_wait(&f_full[x], (tc >> 1) & 1, err, kDevTimeoutFull) &&
               (j > 0 || piece == 0 || mbar_wait(o_free, (piece - 1) & 1, err, kDevTimeoutAccEmpty));
          if (!ok) break;
          tc_fence_after();
          const bool fresh = j == 0 || (j % kFlush == 0 && j + 1 < w.n);
          const uint32_t sv = smem_u32(sm + CL::kVf + x * 32768);
#pragma unroll
          for (int kk = 0; kk < 16; ++kk)  // 16 keys a step: 8 columns of the heads, then the rests
            mma_f16_tmem_a(tO, tS + x * 128 + kk * 8, smem_desc_mn_sw128(sv + (kk & 7) * 2048),
                           kIdescO, (!fresh || kk > 0) ? 1u : 0u);
          mma_commit(&f_empty[x]);
          mma_commit(&o_done[x]);
          // (the pipe runs in order: S_x is overwritten once the product has read it)
          if (j + 2 < w.n) ok = issue_s();
        }
        next_piece(pre, a.batch, per_seq, at, w.n, left);
      }
      mma_commit(drain);
      mbar_wait(drain, 0, err, kDevTimeoutDrain);
    }
  } else if (warp < 8) {
    setmaxnreg_dec<kRegsConvert>();
    // ---------------- V's codes to f16: thread t takes key t of every tile ----------------
    const int t = tid - 128;
    bool ok = true;
    auto scale = [&] {  // of the tile at `at`
      const int key = at.tile * kTileKeys + t;
      return key < a.max_len ? __ldg(a.v_scale + (static_cast<long long>(at.b) * a.heads_kv +
                                                  at.hq / a.qtiles) * a.max_len + key)
                             : 0.0f;
    };
    float vs = nunits > 0 ? scale() : 0.0f;
    for (int j = 0; j < nunits; ++j) {
      const int s = j % kVStages, f = j & 1;
      const bool zero = vs < kNoScale;
      if (j + 1 < nunits) {  // a tile ahead
        next_unit(pre, a.batch, per_seq, at);
        vs = scale();
      }
      if (ok) ok = mbar_wait(&v_full[s], (j / kVStages) & 1, err, kDevTimeoutFull);
      const uint8_t* row = sm + CL::kV + s * 16384 + t * 128;
      uint8_t* out = sm + CL::kVf + f * 32768 + t * 128;
      uint4 v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = *reinterpret_cast<const uint4*>(row + ((c ^ (t & 7)) << 4));
      if (ok) ok = mbar_wait(&f_empty[f], ((j >> 1) & 1) ^ 1u, err, kDevTimeoutEmpty);
#pragma unroll
      for (int c = 0; c < 8; ++c) {  // 16 dims: two 16-byte pieces of f16
        const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
        uint32_t u[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t x = zero ? 0x80808080u : w[e] ^ 0x80808080u;
          u[2 * e] = unbias(__byte_perm(x, 0x64646464u, 0x4140));
          u[2 * e + 1] = unbias(__byte_perm(x, 0x64646464u, 0x4342));
        }
        uint8_t* o = out + (c >> 2) * 16384;
        const int p = (c & 3) * 2;
        *reinterpret_cast<uint4*>(o + ((p ^ (t & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
        *reinterpret_cast<uint4*>(o + (((p + 1) ^ (t & 7)) << 4)) =
            make_uint4(u[4], u[5], u[6], u[7]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v_empty[s]);
        mbar_arrive(&f_full[f]);
      }
    }
  } else {
    setmaxnreg_inc<kRegsSoftmax>();
    // -------- softmax: thread (x, t) has query row t % kRows and kKeys keys of every tile
    constexpr int kRows = kTcRows / kCopies;   // query rows of the tile
    constexpr int kKeys = kCols / kCopies;     // a thread's keys: every copy takes its own
    constexpr int kLaneKeys = kKeys < 32 ? 1 : kKeys / 32;  // of which a lane stages the scales
    const int x = (warp - 8) >> 2;
    const int t = (warp & 3) * 32 + lane;  // == TMEM lane
    const int tr = t % kRows, chunk = t / kRows * kParts + x;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    float* scw0 = reinterpret_cast<float*>(sm + CL::kScales) + (warp - 8) * 3 * kCols;  // of 2
    float* ml = reinterpret_cast<float*>(sm + CL::kML);  // [2][kParts][128]
    const float base = a.sm_scale * kLog2e;
    int tc = 0;  // tiles done
    bool ok = true;
    // What the segments' ends need alone waits in shared memory, so that the loop over
    // the tiles has registers enough
    const uint32_t keep = smem_u32(sm + CL::kKeep) + (tid - 256) * 4;
    constexpr int kNext = kSoftmax * 4;
    put_aside(keep + 6 * kNext, first_cut ? -1 - first_seg : first_seg);
    while (left > 0) {
      const int ntiles = piece_at(at, left).n;
      put_aside(keep, at.b);
      put_aside(keep + kNext, at.hq);
      put_aside(keep + 2 * kNext, at.tile);
      put_aside(keep + 3 * kNext, at.tiles);
      put_aside(keep + 4 * kNext, left);
      // every load at once (all drafts' rows are there, whoever is live): one round trip
      const int b = at.b, hkv = at.hq / a.qtiles;
      const int len = a.lens[b];
      const int r = (at.hq % a.qtiles) * kTcRows + tr;  // query row of the KV head
      const int node = r / a.group;
      // row of q8, q_scale and out
      const int qrow = (b * a.drafts + node) * a.heads_q + hkv * a.group + (r - node * a.group);
      const int mine = tid - 256;
      int up = 0;
      if (a.parents != nullptr && mine < a.drafts)
        up = a.parents[static_cast<long long>(b) * a.drafts + mine];
      uint4 v[8 / kParts];  // this part of the row of Q
      float amul = 0.0f;
      {
        const uint4* src = reinterpret_cast<const uint4*>(a.q8) + static_cast<long long>(qrow) * 8 +
                           8 / kParts * x;
        const bool there = r < a.rows;
#pragma unroll
        for (int c = 0; c < 8 / kParts; ++c) v[c] = there ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
        if (there) amul = a.q_scale[qrow];
      }
      const int keys0 = at.tile * kTileKeys + kKeys * chunk;  // this part's first key
      const float* ksp = a.k_scale + (static_cast<long long>(b) * a.heads_kv + hkv) * a.max_len;
      const float* vsp = a.v_scale + (ksp - a.k_scale);
      float nk[kLaneKeys], nv[kLaneKeys];
      // loads this lane's keys of tile i (past the cache's end, where nobody looks,
      // the last one's: without a branch, the loads run on)
      auto scales = [&](int i) {
#pragma unroll
        for (int k = 0; k < kLaneKeys; ++k) {
          const int key = min(keys0 + i * kTileKeys + 32 * k + lane % kKeys, a.max_len - 1);
          nk[k] = load_now(ksp + key);
          nv[k] = load_now(vsp + key);
        }
      };
      scales(0);
      bool bad;
      const int d = drafts_of(a, b, len, &bad);
      const bool live = r < d * a.group;
      put_aside(keep + 5 * kNext, live ? qrow : -1);
      put_aside(keep + 7 * kNext, d * a.group);
      amul = live ? amul * base : 0.0f;
      if (mine < a.drafts) par[mine] = up;
      {
        uint8_t* q = sm + CL::kQ + t * 128;
#pragma unroll
        for (int c = 0; c < 8 / kParts; ++c)
          *reinterpret_cast<uint4*>(q + (((c + 8 / kParts * x) ^ (t & 7)) << 4)) =
              live ? v[c] : make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
      named_barrier(1, kSoftmax);
      unsigned long long bits = 0;  // the drafted tokens that this row sees
      if (live) {
        if (a.parents == nullptr) {
          bits = (2ull << node) - 1;
        } else {
          for (int i = node; i >= 0;) {  // strictly downwards: it ends
            bits |= 1ull << i;
            const int p = par[i];
            i = p < i ? p : -1;
          }
        }
      }
      // a warp without a live row (as its partners in the other parts) only keeps
      // the barriers going
      const bool idle = !__any_sync(0xffffffffu, live);
      auto stage = [&](int n) {  // and hands them to the warp, as the n-th tile's
        float* scw = scw0 + (n & 1) * (kSoftmax / 32 * 3 * kCols);
        __syncwarp();
        if (kKeys >= 32 || lane < kKeys) {
#pragma unroll
          for (int k = 0; k < kLaneKeys; ++k) {
            scw[32 * k + lane] = nk[k];
            scw[kCols + 32 * k + lane] = scale_log2(nv[k]);
            scw[2 * kCols + 32 * k + lane] = scale_rcp(nv[k]);
          }
        }
        __syncwarp();
      };
      f32x2 s[kKeys / 2];
      const f32x2 lift = pack2(-12582912.0f, -12582912.0f), am = pack2(amul, amul);
      float mt0, mt1;
      // scores of 16 keys (chunk h of tile i, the n-th) in log2 units, with the key's
      // V scale (small_i2f's steps, two at a time)
      auto scores = [&](int i, int n, int h, const uint32_t (&acc)[16]) {
        const float* scw = scw0 + (n & 1) * (kSoftmax / 32 * 3 * kCols);
        const ulonglong2* k4 = reinterpret_cast<const ulonglong2*>(scw);
        const ulonglong2* lv4 = reinterpret_cast<const ulonglong2*>(scw + kCols);
        // (step by step over the chunk, so that its elements cover each other's
        // latencies)
        f32x2 v[8], k[8], lv[8];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const ulonglong2 a2 = k4[h * 4 + (e >> 1)], b2 = lv4[h * 4 + (e >> 1)];
          k[e] = a2.x;
          k[e + 1] = a2.y;
          lv[e] = b2.x;
          lv[e + 1] = b2.y;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v[e] = pack2(__uint_as_float(acc[2 * e] + 0x4B400000u),
                       __uint_as_float(acc[2 * e + 1] + 0x4B400000u));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = add2(v[e], lift);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = mul2(v[e], am);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[h * 8 + e] = fma2(v[e], k[e], lv[e]);
        const int over = keys0 + i * kTileKeys + 16 * h - len;  // key e: drafted token over + e
        if (over + 16 > 0) {
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float f0, f1;
            unpack2(s[h * 8 + (e >> 1)], f0, f1);
            const int q = over + e;
            if (q >= 0 && (q >= kMaxDrafts || ((bits >> q) & 1ull) == 0)) f0 = -INFINITY;
            if (q >= -1 && (q + 1 >= kMaxDrafts || ((bits >> (q + 1)) & 1ull) == 0)) f1 = -INFINITY;
            s[h * 8 + (e >> 1)] = pack2(f0, f1);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float f0, f1, f2, f3;
          unpack2(s[h * 8 + e], f0, f1);
          unpack2(s[h * 8 + e + 1], f2, f3);
          mt0 = max3(mt0, f0, f1);
          mt1 = max3(mt1, f2, f3);
        }
      };
      auto wait_s = [&](int n) {  // S of the n-th tile
        if (ok) ok = mbar_wait(&s_full[n & 1], (n >> 1) & 1, err, kDevTimeoutAccFull);
        ok = __all_sync(0xffffffffu, ok);  // reconverge before warp-collective tcgen05.ld
        tc_fence_after();
      };
      float m = -INFINITY, l = 0.0f;
      float carry = 1.0f;  // the second accumulator's scale to the new maxima
      int i = 0, flush = kFlush;  // the tile, and the one before whose product O is moved
      for (;;) {
        const int stop = min(ntiles - 1, flush);
        for (;; ++i, ++tc) {
          const uint32_t tSx = tS + (tc & 1) * 128 + lane_off;
          stage(tc);
          scales(i + 1);
          mt0 = mt1 = -INFINITY;
          wait_s(tc);
          if (!idle) {
            uint32_t acc[kKeys / 16][16];
#pragma unroll
            for (int h = 0; h < kKeys / 16; ++h)
              tmem_ld_32x32b_x16(tSx + chunk * kKeys + h * 16, acc[h]);
            tmem_ld_wait();
#pragma unroll
            for (int h = 0; h < kKeys / 16; ++h) scores(i, tc, h, acc[h]);
          }
          // the other parts' maxima; after the barrier every part's scores are in
          // registers, so P' may overwrite them
          float mt = fmaxf(mt0, mt1);
          float* mrow = ml + (tc & 1) * kSoftmax;
          mrow[x * 128 + t] = mt;
          named_barrier(1, kSoftmax);
          if (!idle) {
#pragma unroll
            for (int k = 0; k < kParts * kCopies; ++k)
              mt = fmaxf(mt, mrow[k % kParts * 128 + k / kParts * kRows + tr]);
            // The rescale is warp-collective, so the warp decides (and its partners
            // alike): when any row passes its maximum, every row moves to its own.
            float alpha = 1.0f;
            bool rescale = false;
            if (__any_sync(0xffffffffu, mt > m + kLazy)) {
              const float m_new = fmaxf(m, mt);
              alpha = m == -INFINITY ? 0.0f : fast_exp2(m - m_new);
              m = m_new;
              rescale = i > 0;
              carry *= alpha;
            }
            const float nm = kLift - (m == -INFINITY ? 0.0f : m);
            const f32x2 nm2 = pack2(nm, nm);
            const ulonglong2* rv4 = reinterpret_cast<const ulonglong2*>(
                scw0 + (tc & 1) * (kSoftmax / 32 * 3 * kCols) + 2 * kCols);
            f32x2 ls0 = 0, ls1 = 0;  // (0.0f, 0.0f)
#pragma unroll
            for (int h = 0; h < kKeys / 16; ++h) {  // 16 keys: 8 columns of heads, 8 of rests
              uint32_t hi[8], lo[8];
              f32x2 p[8], rv[8];
              float f0[8], f1[8];
#pragma unroll
              for (int e = 0; e < 8; e += 2) {
                const ulonglong2 a2 = rv4[h * 4 + (e >> 1)];
                rv[e] = a2.x;
                rv[e + 1] = a2.y;
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) unpack2(add2(s[h * 8 + e], nm2), f0[e], f1[e]);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                f0[e] = fast_exp2(f0[e]);
                f1[e] = fast_exp2(f1[e]);
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                hi[e] = half2_of(f0[e], f1[e]);
                p[e] = pack2(f0[e], f1[e]);
              }
#pragma unroll
              for (int e = 0; e < 8; e += 2) {
                ls0 = fma2(p[e], rv[e], ls0);
                ls1 = fma2(p[e + 1], rv[e + 1], ls1);
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) lo[e] = rest_of(f0[e], f1[e], hi[e]);
              tmem_st_32x32b_x8(tSx + chunk * (kKeys / 2) + h * 8, hi);
              tmem_st_32x32b_x8(tSx + 64 + chunk * (kKeys / 2) + h * 8, lo);
            }
            if constexpr (kCopies > 1) {  // P' of the other copies' keys: heads or rests
              const uint32_t zeros[16] = {};
#pragma unroll
              for (int k = 1; k < kCopies; ++k)
#pragma unroll
                for (int h = 0; h < kKeys; h += 16)
                  tmem_st_32x32b_x16(tSx + 64 * x + (t / kRows + k) % kCopies * kKeys + h, zeros);
            }
            {
              float f0, f1;
              unpack2(add2(ls0, ls1), f0, f1);
              l = fmaf(l, alpha, f0 + f1);
            }
            if (rescale) {  // this part of O, once the products so far are in it
              if (ok)
                ok = mbar_wait(&o_done[(tc - 1) & 1], ((tc - 1) >> 1) & 1, err, kDevTimeoutAccFull);
              ok = __all_sync(0xffffffffu, ok);
              tc_fence_after();
#pragma unroll 1
              for (int c = 8 / kParts * x; c < 8 / kParts * (x + 1); ++c) {
                uint32_t o[16];
                tmem_ld_32x32b_x16(tO + lane_off + c * 16, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st_32x32b_x16(tO + lane_off + c * 16, o);
              }
            }
            tmem_st_wait();
            tc_fence_before();
          }
          if (i == stop) break;
          mbar_arrive(&p_full[tc & 1]);
        }
        // P' of tile i is there; O goes to the second accumulator before its product,
        // or after it if it is the last
        const bool last = i == ntiles - 1;
        if (last) {
          mbar_arrive(&p_full[tc & 1]);
          ++tc;
        }
        if (ok) ok = mbar_wait(&o_done[(tc - 1) & 1], ((tc - 1) >> 1) & 1, err, kDevTimeoutAccFull);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        if (ntiles > kFlush + 1 && !idle) {
#pragma unroll 1
          for (int c = 0; c < 128 / kParts; c += 8) {
            const uint32_t col = tO + lane_off + 128 / kParts * x + c;
            uint32_t o[8], q[8];
            tmem_ld_32x32b_x8(col, o);
            if (flush > kFlush) tmem_ld_32x32b_x8(col + 128, q);
            tmem_ld_wait();
            if (flush > kFlush) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                o[e] = __float_as_uint(fmaf(__uint_as_float(q[e]), carry, __uint_as_float(o[e])));
            }
            tmem_st_32x32b_x8(col + 128, o);
          }
          tmem_st_wait();
          tc_fence_before();
          carry = 1.0f;
        }
        if (last) break;
        mbar_arrive(&p_full[tc & 1]);
        ++i, ++tc, flush += kFlush;
      }
      // ---- the segment's end in this CTA
      float* lrow = ml + (tc & 1) * kSoftmax;  // (the other buffer may still be read)
      lrow[x * 128 + t] = l;
      named_barrier(1, kSoftmax);  // every product is done (Q is free), the sums in
      tc_fence_after();
      float lsum = 0.0f;
#pragma unroll
      for (int k = 0; k < kParts * kCopies; ++k)
        lsum += lrow[k % kParts * 128 + k / kParts * kRows + tr];
      const int home = take_back(keep + 5 * kNext), cut = take_back(keep + 6 * kNext);
      at = Place{take_back(keep), take_back(keep + kNext), take_back(keep + 2 * kNext),
                 take_back(keep + 3 * kNext)};
      left = take_back(keep + 4 * kNext);
      const Piece w = piece_at(at, left);
      const int seg = at.b * per_seq + at.hq;
      const bool ends = w.at.tile + w.n == w.at.tiles;
      const bool cut_before = cut == -1 - seg;
      const bool whole = ends && !cut_before;
      // 16 columns at a time through this warp's part of Q's buffer, so that four
      // lanes write 64 bytes of one row
      float* part = a.part + (static_cast<long long>(cta) * 2 + (cut_before ? 0 : 1)) * kTcRows *
                                 kPartRow;
      float4* stg = reinterpret_cast<float4*>(sm + CL::kQ + (warp - 8) * 2048);  // [32 rows][4]
      const uint32_t from = w.n > kFlush + 1 ? tSum : tO;
      if constexpr (kCopies == 1) {
        if (!idle) {
          const float scale = whole ? 1.0f / lsum : 1.0f;
          const int dst_row = home < 0 ? -1 : whole ? home : t;  // row of out or of the partial
#pragma unroll 1
          for (int c = 8 / kParts * x; c < 8 / kParts * (x + 1); ++c) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(from + lane_off + c * 16, o);
            tmem_ld_wait();
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e)
              stg[lane * 4 + (e ^ ((lane >> 1) & 3))] = make_float4(
                  __uint_as_float(o[4 * e]) * scale, __uint_as_float(o[4 * e + 1]) * scale,
                  __uint_as_float(o[4 * e + 2]) * scale, __uint_as_float(o[4 * e + 3]) * scale);
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int row = 8 * k + (lane >> 2), e = lane & 3;
              const int to = __shfl_sync(0xffffffffu, dst_row, row);
              const float4 v = stg[row * 4 + (e ^ ((row >> 1) & 3))];
              if (to >= 0) {
                float* dst = whole ? a.out + static_cast<long long>(to) * 128
                                   : part + static_cast<long long>(to) * kPartRow + 4;
                *reinterpret_cast<float4*>(dst + c * 16 + 4 * e) = v;
              }
            }
          }
        }
      } else {
        // The copies' sums are one another's rest: all stage their 16 columns, then
        // every warp adds up kRows / 4 rows.
        constexpr int kOwn = kRows / 4;
        const int row0 = (warp & 3) * kOwn + (lane >> 2), e4 = lane & 3;
        int to[kOwn / 8];        // rows of out, or -1
        float scale[kOwn / 8];
#pragma unroll
        for (int k = 0; k < kOwn / 8; ++k) {
          to[k] = take_back(smem_u32(sm + CL::kKeep) + 5 * kNext + (row0 + 8 * k) * 4);
          float all = 0.0f;
#pragma unroll
          for (int q = 0; q < kParts * kCopies; ++q)
            all += lrow[q % kParts * 128 + q / kParts * kRows + row0 + 8 * k];
          scale[k] = whole ? 1.0f / all : 1.0f;
        }
#pragma unroll 1
        for (int c = 8 / kParts * x; c < 8 / kParts * (x + 1); ++c) {
          uint32_t o[16];
          tmem_ld_32x32b_x16(from + lane_off + c * 16, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 4; ++e)
            stg[lane * 4 + (e ^ ((lane >> 1) & 3))] =
                make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                            __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
          named_barrier(1, kSoftmax);
#pragma unroll
          for (int k = 0; k < kOwn / 8; ++k) {
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int q = 0; q < kCopies; ++q) {
              const int src = q * kRows + row0 + 8 * k;  // its lane
              const float4 p = reinterpret_cast<const float4*>(
                  sm + CL::kQ + (4 * x + (src >> 5)) * 2048)[(src & 31) * 4 + (e4 ^ ((src >> 1) & 3))];
              v = make_float4(v.x + p.x, v.y + p.y, v.z + p.z, v.w + p.w);
            }
            if (to[k] >= 0) {
              float* dst = whole ? a.out + static_cast<long long>(to[k]) * 128
                                 : part + static_cast<long long>(row0 + 8 * k) * kPartRow + 4;
              *reinterpret_cast<float4*>(dst + c * 16 + 4 * e4) =
                  make_float4(v.x * scale[k], v.y * scale[k], v.z * scale[k], v.w * scale[k]);
            }
          }
          named_barrier(1, kSoftmax);
        }
      }
      if (!whole && x == 0 && t < kRows) {
        part[t * kPartRow] = m;
        part[t * kPartRow + 1] = lsum;
      }
      tc_fence_before();
      mbar_arrive(o_free);
      if (left == w.n && tid == 256 && !a.per_cta)
        a.meta[cta] = make_int4(cut < 0 ? -1 - cut : cut, cut < 0 ? 1 : 0, seg,
                                ends ? 0 : take_back(keep + 7 * kNext));
      next_piece(pre, a.batch, per_seq, at, w.n, left);
      named_barrier(1, kSoftmax);  // Q's buffer is free again
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Joins the partials of the segments that several CTAs share.  Block (c, i):
// the segment that CTA c leaves unfinished after beginning it, query rows
// [8i, 8i + 8) of it, one warp each (a lane holds four dims).  The CTAs that follow
// are looked at 32 at a time, a lane each; the partials are added in their
// order, i.e. the keys'.
__global__ void __launch_bounds__(256) tree_join_kernel(TreeArgs a, int tile_rows) {
  pdl_wait();
  pdl_trigger();
  const int c = blockIdx.x, rr = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int4 none = make_int4(-1, 0, -1, 0);
  int4 mk = c + lane < a.ctas ? a.meta[c + lane] : none;
  // c's own part is its slot 1, the others' their slot 0.  What two or three CTAs share
  // is on its way before it is known to be needed (all of it lies in the workspace).
  const long long step = static_cast<long long>(2) * tile_rows * kPartRow;  // one CTA
  const float* row = a.part + static_cast<long long>(rr) * kPartRow;
  const float* own = row + c * step + static_cast<long long>(tile_rows) * kPartRow;
  const float* one = lane == 0 ? own : row + min(c + lane, a.ctas - 1) * step;
  float2 ml = make_float2(0.0f, 0.0f);
  if (lane < 4) ml = *reinterpret_cast<const float2*>(one);
  const float4 v_own = reinterpret_cast<const float4*>(own + 4)[lane];
  const float4 v_next =
      reinterpret_cast<const float4*>(row + min(c + 1, a.ctas - 1) * step + 4)[lane];
  const int4 first = make_int4(__shfl_sync(0xffffffffu, mk.x, 0), __shfl_sync(0xffffffffu, mk.y, 0),
                               __shfl_sync(0xffffffffu, mk.z, 0), __shfl_sync(0xffffffffu, mk.w, 0));
  // unfinished at the end of c, and begun in c
  if (first.x < 0 || first.w == 0 || (first.z == first.x && first.y != 0)) return;
  const int seg = first.z;
  const int per_seq = a.heads_kv * a.qtiles;
  const int b = seg / per_seq, hq = seg % per_seq;
  const int r = (hq % a.qtiles) * tile_rows + rr;
  if (r >= first.w) return;
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int k0 = c; k0 < a.ctas; k0 += 32) {
    if (k0 > c) mk = k0 + lane < a.ctas ? a.meta[k0 + lane] : none;
    // lanes of the segment up to the CTA in which it ends (CTAs without units lie
    // between)
    const bool self = k0 + lane == c, mine = self || mk.x == seg;
    const unsigned end = __ballot_sync(0xffffffffu, mine && !self && (mk.z != seg || mk.w == 0));
    unsigned in = __ballot_sync(0xffffffffu, mine);
    if (end != 0) in &= (2u << (__ffs(static_cast<int>(end)) - 1)) - 1;
    const float* p = row + (k0 + lane) * step +
                     (self ? static_cast<long long>(tile_rows) * kPartRow : 0);
    float pm = -INFINITY, pl = 0.0f;
    if (in >> lane & 1u) {
      if (k0 > c || lane >= 4) ml = *reinterpret_cast<const float2*>(p);
      pm = ml.x;
      pl = ml.y;
    }
    float mx = fmaxf(m, pm);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
    // a CTA whose keys this row does not see has m = -inf
    const float w0 = m == -INFINITY ? 0.0f : exp2f(m - mx);
    const float w = pm == -INFINITY ? 0.0f : exp2f(pm - mx);
    pl *= w;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) pl += __shfl_xor_sync(0xffffffffu, pl, s);
    l = l * w0 + pl;
    o = make_float4(o.x * w0, o.y * w0, o.z * w0, o.w * w0);
    m = mx;
#pragma unroll 4
    for (unsigned left = in; left != 0; left &= left - 1) {
      const int k = __ffs(static_cast<int>(left)) - 1;
      const float wk = __shfl_sync(0xffffffffu, w, k);
      const float* q = row + (k0 + k) * step +
                       (k0 + k == c ? static_cast<long long>(tile_rows) * kPartRow : 0);
      const float4 v = k0 + k == c       ? v_own
                       : k0 + k == c + 1 ? v_next
                                         : reinterpret_cast<const float4*>(q + 4)[lane];
      o = make_float4(fmaf(v.x, wk, o.x), fmaf(v.y, wk, o.y), fmaf(v.z, wk, o.z),
                      fmaf(v.w, wk, o.w));
    }
    if (end != 0) break;
  }
  const int t = r / a.group;
  const long long at = (static_cast<long long>(b) * a.drafts + t) * a.heads_q +
                       hq / a.qtiles * a.group + (r - t * a.group);
  reinterpret_cast<float4*>(a.out + at * 128)[lane] =
      make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
}

// A segment per CTA where the cache holds few tiles of keys: what the shares and
// the join cost (4 us) is more than those tiles one after the other.  Else one
// wave of CTAs with equal shares, and the join.  alone: the most tiles for the
// first.
int launch_tree(void (*kernel)(CUtensorMap, CUtensorMap, TreeArgs), int threads, int smem,
                int per_sm, int tile_rows, int alone, const CUtensorMap& km,
                const CUtensorMap& vm, TreeArgs& a, cudaStream_t st) {
  a.qtiles = (a.rows + tile_rows - 1) / tile_rows;
  const long long segs = static_cast<long long>(a.batch) * a.heads_kv * a.qtiles;
  const int tiles = (a.max_len + kTileKeys - 1) / kTileKeys;
  a.per_cta = tiles <= alone;
  a.ctas = static_cast<int>(
      a.per_cta ? segs
                : std::min<long long>(static_cast<long long>(per_sm) * num_sms(), segs * tiles));
  if (int rc = launch_k(kernel, dim3(static_cast<unsigned>(a.ctas)), dim3(threads), smem, st, km,
                        vm, a))
    return rc;
  if (a.per_cta) return kOk;
  PdlScope pdl;
  return launch_k(tree_join_kernel,
                  dim3(static_cast<unsigned>(a.ctas), std::min(tile_rows, (a.rows + 7) / 8 * 8) / 8),
                  dim3(256), 0, st, a, tile_rows);
}

// The kernels' shared memory, asked for once per device.
bool opt_in() {
  static bool done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return false;
  if (!done[dev]) {
    const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    done[dev] = cudaFuncSetAttribute(tree_mma_kernel<1, 3, 2>, attr, TLayout<3>::kBytes) == cudaSuccess &&
                cudaFuncSetAttribute(tree_mma_kernel<2, 6, 1>, attr, TLayout<6>::kBytes) == cudaSuccess &&
                cudaFuncSetAttribute(tree_tc_kernel<4>, attr, CL::kBytes) == cudaSuccess &&
                cudaFuncSetAttribute(tree_tc_kernel<2>, attr, CL::kBytes) == cudaSuccess &&
                cudaFuncSetAttribute(tree_tc_kernel<1>, attr, CL::kBytes) == cudaSuccess;
  }
  return done[dev];
}

}  // namespace

size_t tree_attn_workspace_bytes() {
  const size_t ctas = static_cast<size_t>(kMaxCtasPerSm) * num_sms();
  const size_t rows = std::max<size_t>(ctas * kMaxTileRows, num_sms() * kTcRows);
  return rows * 2 * kPartRow * sizeof(float) + ctas * sizeof(int4);
}

int tree_attn_i8(const TreeProblem& p, cudaStream_t st) {
  TreeArgs a{};
  a.batch = p.batch;
  a.drafts = p.drafts;
  a.heads_q = p.heads_q;
  a.heads_kv = p.heads_kv;
  a.max_len = p.max_len;
  a.group = p.heads_q / p.heads_kv;
  a.rows = a.group * p.drafts;
  a.sm_scale = p.sm_scale;
  a.q8 = p.q8;
  a.q_scale = p.q_scale;
  a.k_scale = p.k_scale;
  a.v_scale = p.v_scale;
  a.lens = p.lens;
  a.draft_lens = p.draft_lens;
  a.parents = p.parents;
  const size_t ctas = static_cast<size_t>(kMaxCtasPerSm) * num_sms();
  a.meta = static_cast<int4*>(p.workspace);
  a.part = reinterpret_cast<float*>(a.meta + ctas);
  a.out = p.out;
  a.err = device_error_ptr();
  // K and V as [pairs][max_len][128] int8, 128-key boxes with the 128-byte
  // swizzle (rows past max_len read as zeros)
  CUtensorMap km, vm;
  const long long seg = static_cast<long long>(p.max_len) * 128;
  const int pairs = p.batch * p.heads_kv;
  if (int rc = make_tma_3d_i8(&km, p.k_cache, p.max_len, 128, 128, pairs, seg, 128, kTileKeys))
    return rc;
  if (int rc = make_tma_3d_i8(&vm, p.v_cache, p.max_len, 128, 128, pairs, seg, 128, kTileKeys))
    return rc;
  if (!opt_in()) return kErrCuda;
  if (a.rows <= 8)
    return launch_tree(tree_mma_kernel<1, 3, 2>, kTThreads, TLayout<3>::kBytes, 2, 8, 4, km, vm, a,
                       st);
  if (a.rows <= 16)
    return launch_tree(tree_mma_kernel<2, 6, 1>, kTThreads, TLayout<6>::kBytes, 1, 16, 4, km, vm, a,
                       st);
  if (a.rows <= 32)
    return launch_tree(tree_tc_kernel<4>, kCThreads, CL::kBytes, 1, kTcRows, 2, km, vm, a, st);
  if (a.rows <= 64)
    return launch_tree(tree_tc_kernel<2>, kCThreads, CL::kBytes, 1, kTcRows, 2, km, vm, a, st);
  return launch_tree(tree_tc_kernel<1>, kCThreads, CL::kBytes, 1, kTcRows, 2, km, vm, a, st);
}

}  // namespace reef
