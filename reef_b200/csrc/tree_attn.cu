// tree_attn.cu -- int8 attention of drafted tokens over the int8 KV cache
// (the pass that checks a tree of drafts; reef decodes one token at a time,
// so this is this build's own definition).
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
// Within a CTA: K and V tiles by TMA through a 3-stage ring; warp w owns keys
// [16w, 16w + 16) of every tile with its own running maximum, S^T = K . q^T by
// int8 mma, O^T = V^T . P^T by bf16 mma.  The output is fp32 and meant to be:
// V's codes are exact in bf16, and P times the key's V scale goes in as two
// bf16 terms, head and remainder (16 bits of it together, a relative error
// of 2^-17 at most, where a single f16 P leaves 2^-12), with fp32 sums.
#include "attn_mma.cuh"
#include "common.cuh"
#include "ops.h"

#include <cuda_bf16.h>

#include <algorithm>

namespace reef {

namespace {

constexpr int kTThreads = 256;  // eight warps
constexpr int kTWarps = kTThreads / 32;
constexpr int kTileKeys = 128;  // keys per unit
constexpr int kStages = 3;
constexpr int kMaxBatch = kMaxTreeBatch;  // a CTA holds every sequence's length
constexpr int kPartRow = 132;     // floats per row of a partial: m, l, 2 unused, O[128]
constexpr int kMaxTileRows = 32;  // query rows per segment
constexpr int kMaxCtasPerSm = 2;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 4.0f;  // log2 of the largest P before its maximum is raised

struct TreeArgs {
  int batch, drafts, heads_q, heads_kv, max_len;
  int group;   // query heads per KV head
  int rows;    // group * drafts
  int qtiles;  // segments per (sequence, KV head)
  int ctas;
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
// segment, w 1 when it goes on in the next CTA; x = -1 for a CTA without
// units.
struct TL {  // shared memory layout (bytes from a 1024-aligned base)
  static constexpr int kKV = 2 * kTileKeys * 128;  // K then V, int8 [128][128] SW128
  static constexpr int kScales = kStages * kKV;    // per stage ks[128], vs[128]
  static constexpr int kWarpM = kScales + kStages * 1024;  // m[8][32], then l[8][32]
  static constexpr int kAnc = kWarpM + 2 * kTWarps * kMaxTileRows * 4;  // u64[64]
  static constexpr int kPar = kAnc + kMaxDrafts * 8;                    // int[64]
  static constexpr int kPre = kPar + kMaxDrafts * 4;                    // int[batch + 1]
  static constexpr int kBars = kPre + (kMaxBatch + 4) * 4;              // full[], empty[]
  static constexpr int kEnd = kBars + 2 * kStages * 8;
  static constexpr int kBytes = kEnd + 1024;  // + alignment slack
};
static_assert(TL::kBars % 8 == 0 && TL::kAnc % 8 == 0, "aligned");
static_assert(TL::kBytes <= 232448 / 2 - 1024, "two CTAs per SM");
static_assert(kTWarps * 8 * 128 * 4 <= TL::kKV, "eight rows merge inside a stage");

// two f32 -> bf16 pair, the first in the low half
__device__ __forceinline__ uint32_t bf2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float bf_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// D (16x8 f32) += A (16x16 bf16, row) x B (16x8 bf16, col)
__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A word of an ldmatrix .trans over int8 pairs: bytes (k, d), (k, d + 1),
// (k + 1, d), (k + 1, d + 1).  Out: the bf16 pairs {(k, d), (k + 1, d)} and
// {(k, d + 1), (k + 1, d + 1)}, exact: under the exponent byte 0x43 the low
// seven bits of a code read 128 + (code & 127), its sign bit alone 128 or
// 256, and their difference is the code.
__device__ __forceinline__ uint32_t bf16_codes(uint32_t x) {
  const uint32_t p = x & 0xff7fff7fu, n = x & 0xff80ff80u;
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&p),
                                   *reinterpret_cast<const __nv_bfloat162*>(&n));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void split_codes(uint32_t w, uint32_t& even, uint32_t& odd) {
  even = bf16_codes(__byte_perm(w, 0x43434343u, 0x4240));
  odd = bf16_codes(__byte_perm(w, 0x43434343u, 0x4341));
}

// d of sequence b, 0 when it has none or its rows do not fit in the cache
__device__ __forceinline__ int drafts_of(const TreeArgs& a, int b, int len, bool* bad) {
  const int d = a.draft_lens == nullptr ? a.drafts : min(a.draft_lens[b], a.drafts);
  *bad = len < 0 || len > a.max_len || d > a.max_len - len;
  return *bad || d < 0 ? 0 : d;
}

// pre[b] = 128-key tiles of the sequences before b (all threads; B <= 2048:
// eight sequences per thread); returns after a barrier
__device__ __forceinline__ void count_tiles(const TreeArgs& a, int* pre, int* scratch) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kPer = kMaxBatch / kTThreads;
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

// A unit's place: sequence, (KV head, tile of query rows), tile of keys.
struct Place {
  int b, hq, tile, tiles;
};
__device__ __forceinline__ Place place_of(const int* pre, int batch, int per_seq, long long u) {
  int lo = 0, hi = batch - 1;  // the last b with pre[b] * per_seq <= u and tiles
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (static_cast<long long>(pre[mid]) * per_seq <= u) lo = mid;
    else hi = mid - 1;
  }
  Place p;
  p.b = lo;
  p.tiles = pre[lo + 1] - pre[lo];
  const long long rem = u - static_cast<long long>(pre[lo]) * per_seq;
  p.hq = static_cast<int>(rem / p.tiles);
  p.tile = static_cast<int>(rem % p.tiles);
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

// NT: query rows of a segment / 8
template <int NT>
__global__ void __launch_bounds__(kTThreads, NT > 2 ? 1 : 2)
    tree_mma_kernel(const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap, TreeArgs a) {
  constexpr int kRows = 8 * NT;
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) &
                                           ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + TL::kBars);
  uint64_t* empty = full + kStages;
  float* warp_m = reinterpret_cast<float*>(sm + TL::kWarpM);  // [8][32]
  float* warp_l = warp_m + kTWarps * kMaxTileRows;            // [8][32]
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
  count_tiles(a, pre, par);  // (its barriers also publish the mbarriers)

  const int per_seq = a.heads_kv * a.qtiles;
  const long long units = static_cast<long long>(pre[a.batch]) * per_seq;
  const long long u0 = units * cta / a.ctas, u1 = units * (cta + 1) / a.ctas;
  const int nunits = static_cast<int>(u1 - u0);
  if (nunits == 0) {
    if (tid == 0) a.meta[cta] = make_int4(-1, 0, -1, 0);
    return;
  }
  Place at = place_of(pre, a.batch, per_seq, u0);
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
    next_unit(pre, a.batch, per_seq, ahead);
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
      len = a.lens[at.b];
      bool bad;
      d = drafts_of(a, at.b, len, &bad);
      qbase = static_cast<long long>(at.b) * a.drafts * a.heads_q + hkv * a.group;
      if (a.parents != nullptr && tid < d)
        par[tid] = a.parents[static_cast<long long>(at.b) * a.drafts + tid];
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
        const int r = row0 + nt * 8 + g;
        const uint32_t* q32 = reinterpret_cast<const uint32_t*>(a.q8) + (r < live ? qrow(r) * 32 : 0);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          qb[ks][nt][0] = r < live ? q32[8 * ks + tig] : 0u;
          qb[ks][nt][1] = r < live ? q32[8 * ks + 4 + tig] : 0u;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int rc = row0 + nt * 8 + 2 * tig + e;
          qsc[nt][e] = rc < live ? a.q_scale[qrow(rc)] * base : 0.0f;
          m[nt][e] = -INFINITY;
          l[nt][e] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][nt][e] = 0.0f;
      }
      __syncthreads();  // anc is in
    }
    if (ok) ok = mbar_wait(&full[s], (j / kStages) & 1, a.err, kDevTimeoutFull);
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
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sc[nt][0] = small_i2f(c[nt][0]) * qsc[nt][0] * ks_lo;
        sc[nt][1] = small_i2f(c[nt][1]) * qsc[nt][1] * ks_lo;
        sc[nt][2] = small_i2f(c[nt][2]) * qsc[nt][0] * ks_hi;
        sc[nt][3] = small_i2f(c[nt][3]) * qsc[nt][1] * ks_hi;
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
      // ---- P = 2^(s - m) (summed unscaled), times the key's V scale, as a
      // bf16 head and remainder, transposed into the B operand
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float r0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0];
        const float r1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1];
        float p0 = fast_exp2(sc[nt][0] - r0), p1 = fast_exp2(sc[nt][1] - r1);
        float p2 = fast_exp2(sc[nt][2] - r0), p3 = fast_exp2(sc[nt][3] - r1);
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        // 0 * a scale that is not finite stays 0: a masked key adds nothing
        p0 = p0 == 0.0f ? 0.0f : p0 * vs_lo;
        p1 = p1 == 0.0f ? 0.0f : p1 * vs_lo;
        p2 = p2 == 0.0f ? 0.0f : p2 * vs_hi;
        p3 = p3 == 0.0f ? 0.0f : p3 * vs_hi;
        const uint32_t h0 = bf2(p0, p1), h1 = bf2(p2, p3);
        ph[nt][0] = movmatrix_t(h0);
        ph[nt][1] = movmatrix_t(h1);
        pl[nt][0] = movmatrix_t(bf2(p0 - bf_lo(h0), p1 - bf_hi(h0)));
        pl[nt][1] = movmatrix_t(bf2(p2 - bf_lo(h1), p3 - bf_hi(h1)));
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
          mma_bf16_16816(o[2 * cc][nt], va, ph[nt][0], ph[nt][1]);
          mma_bf16_16816(o[2 * cc + 1][nt], vc, ph[nt][0], ph[nt][1]);
          mma_bf16_16816(o[2 * cc][nt], va, pl[nt][0], pl[nt][1]);
          mma_bf16_16816(o[2 * cc + 1][nt], vc, pl[nt][0], pl[nt][1]);
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
      if (j + 1 == nunits && tid == 0)
        a.meta[cta] = make_int4(first_seg, first_cut ? 1 : 0, seg, ends ? 0 : 1);
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
    next_unit(pre, a.batch, per_seq, at);
  }
  // copies still in flight land before exit (only after a timeout can any
  // remain)
  if (tid == 0 && !ok) {
    for (int j = waited; j < issued; ++j)
      mbar_wait(&full[j % kStages], (j / kStages) & 1, a.err, kDevTimeoutDrain);
  }
}

// Joins the partials of the segments that several CTAs share.  Block (c, i):
// the segment that CTA c leaves unfinished after beginning it, query rows
// [8i, 8i + 8) of it, one warp each (a lane holds four dims); the partials are
// taken in the CTAs' order, i.e. the keys'.
__global__ void __launch_bounds__(256) tree_join_kernel(TreeArgs a, int tile_rows) {
  pdl_wait();
  pdl_trigger();
  const int c = blockIdx.x, rr = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int4 first = a.meta[c];
  // unfinished at the end of c, and begun in c
  if (first.x < 0 || first.w == 0 || (first.z == first.x && first.y != 0)) return;
  const int seg = first.z;
  const int per_seq = a.heads_kv * a.qtiles;
  const int b = seg / per_seq, hq = seg % per_seq;
  bool bad;
  const int d = drafts_of(a, b, a.lens[b], &bad);
  const int r = (hq % a.qtiles) * tile_rows + rr;
  if (r >= d * a.group) return;
  const long long step = static_cast<long long>(2) * tile_rows * kPartRow;  // one CTA
  const float* p = a.part + c * step + (static_cast<long long>(tile_rows) + rr) * kPartRow;
  float m = p[0], l = p[1];
  float4 o = reinterpret_cast<const float4*>(p + 4)[lane];
  p = a.part + c * step + static_cast<long long>(rr) * kPartRow;  // slot 0 from here on
  for (int k = c + 1; k < a.ctas; ++k) {
    const int4 mk = a.meta[k];
    p += step;
    if (mk.x < 0) continue;  // a CTA without units
    // a CTA whose keys this row does not see has m = -inf
    const float mx = fmaxf(m, p[0]);
    const float w0 = m == -INFINITY ? 0.0f : exp2f(m - mx);
    const float w1 = p[0] == -INFINITY ? 0.0f : exp2f(p[0] - mx);
    const float4 v = reinterpret_cast<const float4*>(p + 4)[lane];
    l = l * w0 + p[1] * w1;
    o = make_float4(o.x * w0 + v.x * w1, o.y * w0 + v.y * w1, o.z * w0 + v.z * w1,
                    o.w * w0 + v.w * w1);
    m = mx;
    if (mk.z != seg || mk.w == 0) break;  // it ends there
  }
  const int t = r / a.group;
  const long long row = (static_cast<long long>(b) * a.drafts + t) * a.heads_q +
                        hq / a.qtiles * a.group + (r - t * a.group);
  reinterpret_cast<float4*>(a.out + row * 128)[lane] =
      make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
}

template <int NT>
int launch_tree(const CUtensorMap& km, const CUtensorMap& vm, TreeArgs& a, cudaStream_t st) {
  static int per_sm[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return kErrCuda;
  if (per_sm[dev] == 0) {
    int n = 0;
    if (cudaFuncSetAttribute(tree_mma_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             TL::kBytes) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, tree_mma_kernel<NT>, kTThreads,
                                                      TL::kBytes) != cudaSuccess ||
        n <= 0)
      return kErrCuda;
    per_sm[dev] = std::min(n, kMaxCtasPerSm);
  }
  a.qtiles = (a.rows + 8 * NT - 1) / (8 * NT);
  // one wave, and no more CTAs than the cache has room for units
  const long long most = static_cast<long long>(a.batch) * a.heads_kv * a.qtiles *
                         ((a.max_len + kTileKeys - 1) / kTileKeys);
  a.ctas = static_cast<int>(std::min<long long>(static_cast<long long>(per_sm[dev]) * num_sms(),
                                                most));
  if (int rc = launch_k(tree_mma_kernel<NT>, dim3(static_cast<unsigned>(a.ctas)), dim3(kTThreads),
                        TL::kBytes, st, km, vm, a))
    return rc;
  PdlScope pdl;
  return launch_k(tree_join_kernel, dim3(static_cast<unsigned>(a.ctas), NT), dim3(256), 0, st,
                  a, 8 * NT);
}

}  // namespace

size_t tree_attn_workspace_bytes() {
  const size_t ctas = static_cast<size_t>(kMaxCtasPerSm) * num_sms();
  return ctas * 2 * kMaxTileRows * kPartRow * sizeof(float) + ctas * sizeof(int4);
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
  if (a.rows <= 8) return launch_tree<1>(km, vm, a, st);
  if (a.rows <= 16) return launch_tree<2>(km, vm, a, st);
  return launch_tree<4>(km, vm, a, st);
}

}  // namespace reef
