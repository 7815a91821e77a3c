// verify.cpp -- the Llama layer on drafted tokens: the decode step with `drafts`
// new tokens per sequence, each seeing the committed cache rows, itself and its
// ancestors in the sequence's tree.  Everything but the cache append and the
// attention is the decode step's own (layer.cpp), on batch * drafts rows.  Llama-70B's
// TP = 8 shard over 4096 cached rows: 64 x 1 94 us (the decode step: 86, whose attention
// rounds P to f16 and begins its loads before the append ends), 16 x 8 102, 64 x 2 114.
#include "comm.h"
#include "layer.h"

#include <algorithm>

using namespace reef;

namespace {

// the decode step's description of the same layer, a row per drafted token.  Its o and
// down projections are row-parallel: weights, x and y of the all-gather plan are others.
bool rows_of(const reef_b200_llama_layer* L, size_t drafts, reef_b200_llama_layer* rows) {
  if (L == nullptr || drafts == 0 || drafts > static_cast<size_t>(kMaxDrafts) || L->batch == 0 ||
      L->batch > 128 ||
      (comm_world(reinterpret_cast<Comm*>(L->comm)) > 1 && L->tp_mode != REEF_B200_TP_ALLREDUCE))
    return false;
  *rows = *L;
  rows->batch = L->batch * drafts;  // <= 128, checked with the rest of it
  return true;
}

struct Verify final : DecodeHooks {
  const reef_b200_llama_layer* L;
  int drafts, max_len;
  const int32_t *lens, *draft_lens, *parents;
  int8_t* kc;
  float* ks;
  int8_t* vc;
  float* vs;
  void* workspace;  // the attention's
  int append(const int32_t* part, int splits, const float* xs, int8_t* q8, float* qs, int*,
             cudaStream_t st) override {
    return draft_rope_append_partials(
        static_cast<int>(L->batch), drafts, static_cast<int>(L->heads_q),
        static_cast<int>(L->heads_kv), max_len, L->rope_base, lens, draft_lens, parents, part,
        splits, xs, L->s_qkv, q8, qs, kc, ks, vc, vs, st);
  }
  int attend(const int8_t* q8, const float* qs, const int*, float*, float* out,
             cudaStream_t st) override {
    TreeProblem p{};
    p.batch = static_cast<int>(L->batch);
    p.drafts = drafts;
    p.heads_q = static_cast<int>(L->heads_q);
    p.heads_kv = static_cast<int>(L->heads_kv);
    p.max_len = max_len;
    p.sm_scale = 0.08838834764831845f;  // 1 / sqrt(128)
    p.q8 = q8;
    p.q_scale = qs;
    p.k_cache = kc;
    p.k_scale = ks;
    p.v_cache = vc;
    p.v_scale = vs;
    p.lens = lens;
    p.draft_lens = draft_lens;
    p.parents = parents;
    p.workspace = workspace;
    p.out = out;
    return tree_attn_i8(p, st);
  }
};

size_t up256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

}  // namespace

extern "C" {

size_t reef_b200_llama_verify_workspace_bytes(const reef_b200_llama_layer* layer, size_t drafts,
                                              size_t max_len) {
  reef_b200_llama_layer rows;
  if (!rows_of(layer, drafts, &rows) || max_len % 4 != 0) return 0;
  const size_t decode = decode_run_bytes(&rows, max_len);
  return decode == 0 ? 0 : up256(decode) + tree_attn_workspace_bytes();
}

int reef_b200_llama_verify_forward(const reef_b200_llama_layer* layer, size_t drafts,
                                   const float* x, float* y, const int32_t* lens,
                                   const int32_t* draft_lens, const int32_t* parents,
                                   int8_t* k_cache, float* k_scale, int8_t* v_cache,
                                   float* v_scale, size_t max_len, void* workspace,
                                   size_t workspace_bytes, reef_b200_stream_t stream) {
  reef_b200_llama_layer rows;
  if (!rows_of(layer, drafts, &rows) || !x || !y || !lens || !k_cache || !k_scale || !v_cache ||
      !v_scale || !workspace)
    return REEF_B200_ERR_INVALID;
  if (max_len % 4 != 0 || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 ||
      (reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) % 16 != 0)
    return REEF_B200_ERR_ALIGNMENT;
  if (int rc = check_device()) return rc;
  const size_t decode = up256(decode_run_bytes(&rows, max_len));
  if (decode == 0 || workspace_bytes < decode + tree_attn_workspace_bytes())
    return REEF_B200_ERR_INVALID;
  Verify hooks;
  hooks.L = layer;
  hooks.drafts = static_cast<int>(drafts);
  hooks.max_len = static_cast<int>(max_len);
  hooks.lens = lens;
  hooks.draft_lens = draft_lens;
  hooks.parents = parents;
  hooks.kc = k_cache;
  hooks.ks = k_scale;
  hooks.vc = v_cache;
  hooks.vs = v_scale;
  hooks.workspace = static_cast<uint8_t*>(workspace) + decode;
  return decode_run(&rows, x, y, max_len, workspace, decode, hooks,
                    reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
