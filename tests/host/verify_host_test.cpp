// verify_host_test.cpp -- test infrastructure: drives the Llama layer on drafted
// tokens (reef_b200/csrc/verify.cpp over layer.cpp's decode step) at TP = world
// on the CPU, threads as ranks, over the stand-ins in fake_cuda_nccl.cpp and
// fake_ops.cpp and three of its own below.  Prints one "ok <case>" line per
// passing case, "FAIL ..." lines otherwise; exits non-zero on any failure.
//
// Under the all-reduce plan every call returns OK, every rank issues the same
// collectives in the same order, and what the attention and the cache append
// are given lies inside the buffers (the stand-ins write all of it, under
// AddressSanitizer).  A layer of the all-gather plan, whose w_o, w_down and x
// are laid out by output rows and columns, is refused.
#include "comm.h"
#include "reef_b200.h"

#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <thread>
#include <vector>

using namespace reef;

extern "C" void fake_set_rank(int r);
extern "C" int fake_violations();
extern "C" int fake_live_allocations();

namespace {

std::atomic<int> g_fail{0}, g_appends{0}, g_attends{0};

#define CHECK_EQ(a, b)                                                                      \
  do {                                                                                      \
    const long long va = static_cast<long long>(a), vb = static_cast<long long>(b);         \
    if (va != vb) {                                                                         \
      std::fprintf(stderr, "FAIL %s:%d: %s == %s (%lld vs %lld)\n", __FILE__, __LINE__, #a, \
                   #b, va, vb);                                                             \
      ++g_fail;                                                                             \
    }                                                                                       \
  } while (0)

}  // namespace

namespace reef {

int draft_rope_append_partials(int batch, int drafts, int heads_q, int heads_kv, int max_len,
                               float, const int* lens, const int* draft_lens, const int* parents,
                               const int32_t*, int, const float*, const float*, int8_t* q8,
                               float* q_scale, int8_t* k_cache, float* k_scale, int8_t* v_cache,
                               float* v_scale, cudaStream_t) {
  ++g_appends;
  const size_t rows = static_cast<size_t>(batch) * drafts * heads_q;
  std::memset(q8, 1, rows * 128);
  std::memset(q_scale, 1, rows * sizeof(float));
  for (int b = 0; b < batch; ++b) {
    CHECK_EQ(lens[b], 7 + b);
    CHECK_EQ(draft_lens[b], drafts);
    CHECK_EQ(parents[b * drafts], -1);
    for (int h = 0; h < heads_kv; ++h) {
      const size_t row = (static_cast<size_t>(b) * heads_kv + h) * max_len + lens[b];
      std::memset(k_cache + row * 128, 1, drafts * 128);
      std::memset(v_cache + row * 128, 1, drafts * 128);
      std::memset(k_scale + row, 1, drafts * sizeof(float));
      std::memset(v_scale + row, 1, drafts * sizeof(float));
    }
  }
  return kOk;
}
size_t tree_attn_workspace_bytes() { return 123456; }
int tree_attn_i8(const TreeProblem& p, cudaStream_t) {
  ++g_attends;
  std::memset(p.workspace, 2, tree_attn_workspace_bytes());
  std::memset(p.out, 3, static_cast<size_t>(p.batch) * p.drafts * p.heads_q * 128 * sizeof(float));
  // (the append's rows are where the attention reads them)
  for (int b = 0; b < p.batch; ++b)
    for (int t = 0; t < p.drafts * p.heads_q; ++t)
      CHECK_EQ(p.q8[(static_cast<size_t>(b) * p.drafts * p.heads_q + t) * 128], 1);
  return kOk;
}

}  // namespace reef

namespace {

alignas(1024) unsigned char g_dummy[1024];

reef_b200_llama_layer layer_for(int world, Comm* c, int mode, size_t batch) {
  reef_b200_llama_layer L{};
  L.batch = batch;
  L.seq = 8;
  L.hidden = 1024;
  L.heads_q = 32 / world;
  L.heads_kv = 8 / world;
  L.head_dim = 128;
  L.ffn = 2816 / world;
  L.rms_eps = 1e-5f;
  L.rope_base = 10000.0f;
  const auto* f = reinterpret_cast<const float*>(g_dummy);
  const auto* w = reinterpret_cast<const int8_t*>(g_dummy);
  L.attn_norm = L.mlp_norm = L.s_qkv = L.s_o = L.s_gu = L.s_down = f;
  L.w_qkv = L.w_o = L.w_gu = L.w_down = w;
  L.comm = reinterpret_cast<reef_b200_comm*>(c);
  L.tp_mode = mode;
  return L;
}

template <typename T>
T* make(size_t n) {
  return static_cast<T*>(std::aligned_alloc(256, (n * sizeof(T) + 255) / 256 * 256));
}

void run_ranks(int world, const std::function<void(int)>& f) {
  std::vector<std::thread> th;
  for (int r = 0; r < world; ++r)
    th.emplace_back([&f, r] {
      fake_set_rank(r);
      f(r);
    });
  for (auto& t : th) t.join();
}

// One call; `need` what the workspace query says (0: the call's own status says more).
int verify(const reef_b200_llama_layer& L, size_t drafts, size_t* need) {
  const size_t max_len = 256, cache = L.batch * L.heads_kv * max_len, rows = L.batch * drafts;
  *need = reef_b200_llama_verify_workspace_bytes(&L, drafts, max_len);
  const size_t bytes = *need != 0 ? *need : 1 << 20;
  auto *kc = make<int8_t>(cache * 128), *vc = make<int8_t>(cache * 128);
  auto *ks = make<float>(cache), *vs = make<float>(cache);
  auto *x = make<float>(rows * L.hidden), *y = make<float>(rows * L.hidden);
  std::vector<int32_t> lens, drafted(L.batch, static_cast<int32_t>(drafts)), parents(rows, -1);
  for (size_t b = 0; b < L.batch; ++b) lens.push_back(static_cast<int32_t>(7 + b));
  auto* ws = make<uint8_t>(bytes);
  std::memset(ws, 0, bytes);
  const int rc = reef_b200_llama_verify_forward(&L, drafts, x, y, lens.data(), drafted.data(),
                                                parents.data(), kc, ks, vc, vs, max_len, ws, bytes,
                                                nullptr);
  if (*need != 0)  // a byte less is refused
    CHECK_EQ(reef_b200_llama_verify_forward(&L, drafts, x, y, lens.data(), drafted.data(),
                                            parents.data(), kc, ks, vc, vs, max_len, ws,
                                            reef_b200_llama_verify_workspace_bytes(&L, drafts, max_len) -
                                                256 - reef::tree_attn_workspace_bytes(),
                                            nullptr),
             REEF_B200_ERR_INVALID);
  for (void* p : {static_cast<void*>(kc), static_cast<void*>(vc), static_cast<void*>(ks),
                  static_cast<void*>(vs), static_cast<void*>(x), static_cast<void*>(y),
                  static_cast<void*>(ws)})
    std::free(p);
  return rc;
}

void world_case(int world) {
  std::vector<unsigned char> id(comm_unique_id_bytes());
  fake_set_rank(0);
  CHECK_EQ(comm_unique_id(id.data(), id.size()), kOk);
  std::vector<Comm*> comms(world, nullptr);
  run_ranks(world,
            [&](int r) { CHECK_EQ(comm_init(r, world, id.data(), 5.0, &comms[r]), kOk); });
  for (Comm* c : comms)
    if (c == nullptr) return;
  g_appends = g_attends = 0;
  const size_t shapes[][2] = {{1, 1}, {3, 5}, {2, 64}, {16, 8}, {128, 1}};  // batch, drafts
  run_ranks(world, [&](int r) {
    for (const auto& s : shapes) {
      size_t need = 0;
      CHECK_EQ(verify(layer_for(world, comms[r], REEF_B200_TP_ALLREDUCE, s[0]), s[1], &need),
               REEF_B200_OK);
      CHECK_EQ(need != 0, 1);
      const reef_b200_llama_layer L = layer_for(world, comms[r], REEF_B200_TP_ALLGATHER, s[0]);
      CHECK_EQ(verify(L, s[1], &need), REEF_B200_ERR_INVALID);
      CHECK_EQ(need, 0);
    }
    size_t need = 1;  // more rows than the decode step's GEMMs take
    CHECK_EQ(verify(layer_for(world, comms[r], REEF_B200_TP_ALLREDUCE, 16), 9, &need),
             REEF_B200_ERR_INVALID);
    CHECK_EQ(need, 0);
  });
  CHECK_EQ(g_appends.load(), 5 * world);
  CHECK_EQ(g_attends.load(), 5 * world);
  run_ranks(world, [&](int r) { CHECK_EQ(comm_destroy(comms[r]), kOk); });
  CHECK_EQ(fake_violations(), 0);
  CHECK_EQ(fake_live_allocations(), 0);
}

}  // namespace

int main() {
  for (int world : {2, 4, 8}) {
    const int before = g_fail.load();
    world_case(world);
    if (g_fail.load() == before) std::printf("ok verify world %d\n", world);
  }
  const int before = g_fail.load();
  size_t need = 0;  // alone, the plan says nothing
  CHECK_EQ(verify(layer_for(1, nullptr, REEF_B200_TP_ALLGATHER, 3), 5, &need), REEF_B200_OK);
  if (g_fail.load() == before) std::printf("ok verify alone\n");
  std::fflush(stdout);
  return g_fail.load() == 0 ? 0 : 1;
}
