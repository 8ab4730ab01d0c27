// Host-side AddressSanitizer run of the paged cache's entry points (kv_paged.hip, attn_paged.hip), built and run by tools/asan_host.sh beside
// abi_host_asan.cpp: argument checks, the plan with its workspace sizes over many geometries, calls that have nothing to do. No call below
// reaches a kernel launch.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <memory>
#include "../../include/vividmed_hip.h"

static int fails = 0;
#define EXPECT(call, want)                                                                  \
  do {                                                                                      \
    const int got__ = (call);                                                               \
    if (got__ != (want)) { std::printf("FAIL %s -> %d (want %d)\n", #call, got__, (want)); ++fails; } \
  } while (0)

int main() {
  char* const any = reinterpret_cast<char*>(uintptr_t{1} << 20);      // an aligned address that is never followed
  // each struct in an allocation of exactly its size: a read behind it is reported
  auto c = std::make_unique<vm_paged_kv>();
  auto a = std::make_unique<vm_attn_paged_args>();
  auto bytes = std::make_unique<int64_t>(-1);
  std::memset(c.get(), 0, sizeof *c);
  std::memset(a.get(), 0, sizeof *a);
  int32_t* const i32 = reinterpret_cast<int32_t*>(any);
  float* const f = reinterpret_cast<float*>(any);

  EXPECT(vm_attn_paged_workspace(nullptr, bytes.get()), VM_ERR_BAD_ARG);
  EXPECT(vm_attn_paged_workspace(a.get(), nullptr), VM_ERR_BAD_ARG);
  EXPECT(vm_attn_paged_workspace(a.get(), bytes.get()), VM_ERR_BAD_ARG);               // an empty struct
  EXPECT(vm_attn_paged_bf16(nullptr, nullptr), VM_ERR_BAD_ARG);
  EXPECT(vm_attn_paged_bf16(a.get(), nullptr), VM_ERR_BAD_ARG);
  EXPECT(vm_kv_append_paged_bf16(nullptr, any, 1024, i32, i32, i32, f, f, 10, 4, 4, any, 512, nullptr, nullptr), VM_ERR_BAD_ARG);
  EXPECT(vm_kv_append_paged_bf16(c.get(), any, 1024, i32, i32, i32, f, f, 10, 4, 4, any, 512, nullptr, nullptr), VM_ERR_BAD_ARG);
  EXPECT(vm_kv_evict_paged_bf16(nullptr, f, 200, 100, 100, i32, i32 + 64, 3, 3, 64, 8, f + 64, 200, 100, i32 + 128, i32, nullptr), VM_ERR_BAD_ARG);

  const int sizes[] = {1, 2, 15, 16, 17, 31, 33, 255, 256, 257, 4097, 100000};
  int planned = 0;
  for (int hd : {32, 64, 96, 128})
    for (int page : {16, 48, 64, 1024})
      for (int group : {1, 3, 16, 17})
        for (int n_seq : {0, 1, 7, 300})
          for (int new_tokens : sizes)
            for (int kv : sizes)
              for (int weights : {0, 1}) {
                const int hk = 2, cols = (kv + page - 1) / page, rows = n_seq * new_tokens, heads = hk * group;
                c->k_pages = c->v_pages = any; c->ld_page = (int64_t)hk * page * hd; c->n_pages = 4; c->page_size = page;
                c->block_table = i32; c->ld_table = c->max_pages = cols; c->n_seq = n_seq; c->n_kv_heads = hk; c->head_dim = hd;
                a->cache = *c;
                a->q = a->out = any; a->ldq = a->ldo = (int64_t)heads * hd; a->cu_q = a->kv_lens = i32; a->lse = f; a->ld_lse = a->n_rows = rows;
                a->max_q = new_tokens; a->max_kv = kv; a->n_heads = heads; a->scale = 0.1f;
                a->weights = weights ? f : nullptr; a->weights_out = weights ? f : nullptr;
                a->w_cols = weights ? cols * page : 0; a->ldw_head = a->ldwo_head = a->w_cols; a->ldw_seq = a->ldwo_seq = hk * (int64_t)a->w_cols;
                const bool legal = hd != 96 && page != 48;
                *bytes = -1;
                EXPECT(vm_attn_paged_workspace(a.get(), bytes.get()), legal ? VM_OK : VM_ERR_UNSUPPORTED);
                if (!legal) {
                  EXPECT(vm_attn_paged_bf16(a.get(), nullptr), VM_ERR_UNSUPPORTED);
                } else if (*bytes > 0) {                                              // without its workspace the call ends before a launch
                  a->workspace = nullptr; a->workspace_bytes = 0;
                  EXPECT(vm_attn_paged_bf16(a.get(), nullptr), VM_ERR_BAD_ARG);
                  a->workspace = any; a->workspace_bytes = *bytes - 1;
                  EXPECT(vm_attn_paged_bf16(a.get(), nullptr), VM_ERR_BAD_ARG);
                  ++planned;
                } else if (n_seq == 0) {
                  EXPECT(vm_attn_paged_bf16(a.get(), nullptr), VM_OK);                // no sample: nothing to do
                }
                EXPECT(*bytes < 0 ? legal : 0, 0);
              }
  EXPECT(planned > 1000 ? 0 : 1, 0);
  c->head_dim = 128; c->page_size = 64; c->ld_page = 2 * 64 * 128; c->ld_table = c->max_pages = 3; c->n_seq = 2;
  EXPECT(vm_kv_append_paged_bf16(c.get(), any, 1024, i32, i32, i32, f, f, 10, 0, 4, any, 512, nullptr, nullptr), VM_OK);                // no rows
  EXPECT(vm_kv_append_paged_bf16(c.get(), any, 1016, i32, i32, i32, f, f, 10, 4, 4, any, 512, nullptr, nullptr), VM_ERR_BAD_ARG);       // rows overlap
  EXPECT(vm_kv_evict_paged_bf16(c.get(), f, 200, 100, 100, i32, i32, 3, 3, 64, 8, f + 64, 200, 100, i32 + 128, i32, nullptr), VM_ERR_BAD_ARG);      // in place
  EXPECT(vm_kv_evict_paged_bf16(c.get(), f, 200, 100, 100, i32, i32 + 64, 1, 1, 65, 8, f + 64, 200, 100, i32 + 128, i32, nullptr), VM_ERR_BAD_ARG);     // no place for 65
  c->n_seq = 0;
  EXPECT(vm_kv_evict_paged_bf16(c.get(), f, 200, 100, 100, i32, i32 + 64, 3, 3, 64, 8, f + 64, 200, 100, i32 + 128, i32, nullptr), VM_OK);
  std::printf("%s: %d failed checks, %d plans (paged cache)\n", fails ? "FAILED" : "OK", fails, planned);
  return fails ? 1 : 0;
}
