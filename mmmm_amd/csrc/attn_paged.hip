// Attention of a chunk of new tokens over the paged KV cache (generation path): one token, a follow-up question or a whole prompt.
// Stands for the attention calls of /root/reference/mmmm/models/cogvlm/modeling_cogvlm.py:113-141 where K and V come from the cache.
//
// Query rows of one kv head are taken together: row r of (sample b, kv head hk) is query i = r / G of head hk G + r % G (G heads share the
// kv head), so grouped heads read K and V once. Query i sees the tokens j <= L - n + i.
#include "paged.hpp"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct AttnPagedP {
  PagedKV c;
  const unsigned short* q; int64_t ldq;
  const int32_t* cu; const int32_t* kv_lens; const int32_t* row_of_pos;
  unsigned short* out; int64_t ldo;
  float* lse; int64_t ld_lse;
  int n_rows, n_seq, n_heads, G;
  int max_q, max_kv;
  float scale;
  const float* w_in; float* w_out; int64_t ldw_seq, ldw_head, ldwo_seq, ldwo_head; int w_cols;
};

// what one sample brings, read from the device and held inside the buffers' bounds
struct SeqInfo { int p0, nq, len; };
__device__ __forceinline__ SeqInfo seq_info(const AttnPagedP& p, int b) {
  SeqInfo s;
  s.p0 = max(0, min(p.cu[b], p.n_rows));
  const int p1 = max(s.p0, min(p.cu[b + 1], p.n_rows));
  s.nq = p1 - s.p0;
  s.len = max(0, (int)min((int64_t)p.kv_lens[b], (int64_t)p.c.max_pages << p.c.shift));
  return s;
}
__device__ __forceinline__ int phys_row(const AttnPagedP& p, int pos) {      // packed row of a position, -1: none
  const int r = p.row_of_pos ? p.row_of_pos[pos] : pos;
  return (unsigned)r < (unsigned)p.n_rows ? r : -1;
}

// ----------------------------------------------------------------------------- one wave per query row (the plain form of the kernel)
template <int HD>
__global__ __launch_bounds__(256) void attn_paged_row_k(const AttnPagedP p) {
  __shared__ float sp[4][64];
  __shared__ float sq[4][HD];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = blockIdx.x * 4 + wave, hk = blockIdx.y, b = blockIdx.z;
  const SeqInfo s = seq_info(p, b);
  const int i = r / p.G, h = hk * p.G + r % p.G;
  if (i >= s.nq) return;
  const int row = phys_row(p, s.p0 + i);
  if (row < 0) return;
  const int lim = min(s.len - s.nq + i, s.len - 1);
  for (int d = lane; d < HD; d += 64) sq[wave][d] = bf2f(p.q[row * p.ldq + h * HD + d]);
  __builtin_amdgcn_wave_barrier();
  const float sc = p.scale * LOG2E;
  float m = -INFINITY, l = 0.f, o[(HD + 63) / 64] = {0.f};
  for (int j0 = 0; j0 <= lim; j0 += 64) {
    const int j = j0 + lane;
    float sco = -INFINITY;
    if (j <= lim) {
      const int page = p.c.table[b * p.c.ld_table + (j >> p.c.shift)];
      if (page_ok(page, p.c.n_pages)) {
        const unsigned short* k = p.c.k + page_row(page, p.c.ld_page, hk, j & p.c.mask, p.c.shift, HD);
        float a = 0.f;
        for (int d = 0; d < HD; ++d) a = fmaf(sq[wave][d], bf2f(k[d]), a);
        sco = a * sc;
      }
    }
    const float mn = fmaxf(m, wave_max(sco)), base = mn == -INFINITY ? 0.f : mn;
    const float corr = exp2f(m - base), e = exp2f(sco - base);
    m = mn;
    l = l * corr + wave_sum(e);
    sp[wave][lane] = e;
    __builtin_amdgcn_wave_barrier();
    for (int t = 0; t < (HD + 63) / 64; ++t) o[t] *= corr;
    for (int jj = 0; jj < 64 && j0 + jj <= lim; ++jj) {
      const int page = p.c.table[b * p.c.ld_table + ((j0 + jj) >> p.c.shift)];
      if (!page_ok(page, p.c.n_pages)) continue;
      const unsigned short* v = p.c.v + page_row(page, p.c.ld_page, hk, (j0 + jj) & p.c.mask, p.c.shift, HD);
      const float e2 = sp[wave][jj];
      for (int t = 0; t < (HD + 63) / 64; ++t)
        if (lane + 64 * t < HD) o[t] = fmaf(e2, bf2f(v[lane + 64 * t]), o[t]);
    }
    __builtin_amdgcn_wave_barrier();
  }
  for (int t = 0; t < (HD + 63) / 64; ++t)
    if (lane + 64 * t < HD) p.out[row * p.ldo + h * HD + lane + 64 * t] = f2bf(l > 0.f || l != l ? o[t] / l : 0.f);
  if (lane == 0) p.lse[h * p.ld_lse + s.p0 + i] = l > 0.f || l != l ? (m + log2f(l)) * LN2 : -INFINITY;
}

// one wave per 64 tokens of (sample, kv head): the lane's token against every query row
template <int HD>
__global__ __launch_bounds__(64) void attn_paged_weights_k(const AttnPagedP p) {
  const int lane = threadIdx.x, j = blockIdx.x * 64 + lane, hk = blockIdx.y, b = blockIdx.z;
  const SeqInfo s = seq_info(p, b);
  if (blockIdx.x * 64 >= min(s.len, p.w_cols)) return;
  const float sc = p.scale * LOG2E;
  int page = -1;
  if (j < s.len) page = p.c.table[b * p.c.ld_table + (j >> p.c.shift)];
  const bool ok = page_ok(page, p.c.n_pages);
  const unsigned short* k = p.c.k + (ok ? page_row(page, p.c.ld_page, hk, j & p.c.mask, p.c.shift, HD) : 0);
  float sum = 0.f;
  for (int i = 0; i < s.nq; ++i) {
    const int row = phys_row(p, s.p0 + i);
    if (row < 0) continue;
    for (int g = 0; g < p.G; ++g) {
      const int h = hk * p.G + g;
      const float l2 = p.lse[h * p.ld_lse + s.p0 + i] * LOG2E;
      if (!ok || j > s.len - s.nq + i) continue;
      float a = 0.f;
      for (int d = 0; d < HD; ++d) a = fmaf(bf2f(p.q[row * p.ldq + h * HD + d]), bf2f(k[d]), a);
      sum += exp2f(a * sc - l2);
    }
  }
  if (j < min(s.len, p.w_cols)) p.w_out[b * p.ldwo_seq + hk * p.ldwo_head + j] = p.w_in[b * p.ldw_seq + hk * p.ldw_head + j] + sum;
}

int fill(const vm_attn_paged_args* a, AttnPagedP& p) {
  if (!a) return VM_ERR_BAD_ARG;
  const int rc = paged_cache(&a->cache, p.c);
  if (rc != VM_OK) return rc;
  if (a->n_rows < 0 || a->n_heads <= 0 || a->n_heads % p.c.n_kv_heads || a->max_q < 0 || a->max_kv < 0) return VM_ERR_BAD_ARG;
  if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return VM_ERR_BAD_ARG;
  if (a->cache.n_seq > 65535 || p.c.n_kv_heads > 65535) return VM_ERR_UNSUPPORTED;
  const int64_t width = (int64_t)a->n_heads * a->cache.head_dim;
  if ((a->ldq & 7) || (a->ldo & 7) || a->ldq < width || a->ldo < width || a->ld_lse < a->n_rows) return VM_ERR_BAD_ARG;
  if (misaligned16(a->q) || misaligned16(a->out)) return VM_ERR_BAD_ARG;
  if (a->n_rows > 0 && (!a->q || !a->out || !a->lse)) return VM_ERR_BAD_ARG;
  if (a->cache.n_seq > 0 && (!a->cu_q || !a->kv_lens)) return VM_ERR_BAD_ARG;
  if (a->weights_out && (!a->weights || a->w_cols <= 0 || a->ldw_head < a->w_cols || a->ldwo_head < a->w_cols || a->ldw_seq < 0 || a->ldwo_seq < 0)) return VM_ERR_BAD_ARG;
  if ((int64_t)a->max_q * (a->n_heads / p.c.n_kv_heads) > 0x7FFFFFFF - 4096) return VM_ERR_UNSUPPORTED;
  p.q = (const unsigned short*)a->q; p.ldq = a->ldq; p.cu = a->cu_q; p.kv_lens = a->kv_lens; p.row_of_pos = a->row_of_pos;
  p.out = (unsigned short*)a->out; p.ldo = a->ldo; p.lse = a->lse; p.ld_lse = a->ld_lse;
  p.n_rows = a->n_rows; p.n_seq = a->cache.n_seq; p.n_heads = a->n_heads; p.G = a->n_heads / p.c.n_kv_heads;
  p.max_q = a->max_q < a->n_rows ? a->max_q : a->n_rows;
  const int64_t cap = (int64_t)p.c.max_pages << p.c.shift;
  p.max_kv = a->max_kv < cap ? a->max_kv : (int)cap;
  p.scale = a->scale;
  p.w_in = a->weights; p.w_out = a->weights_out; p.ldw_seq = a->ldw_seq; p.ldw_head = a->ldw_head;
  p.ldwo_seq = a->ldwo_seq; p.ldwo_head = a->ldwo_head; p.w_cols = a->w_cols;
  return VM_OK;
}

}  // namespace

extern "C" {

int vm_attn_paged_workspace(const vm_attn_paged_args* args_host, int64_t* bytes_host) {
  AttnPagedP p;
  if (!bytes_host) return VM_ERR_BAD_ARG;
  const int rc = fill(args_host, p);
  if (rc != VM_OK) return rc;
  *bytes_host = 0;
  return VM_OK;
}

int vm_attn_paged_bf16(const vm_attn_paged_args* args_host, void* stream) {
  AttnPagedP p;
  const int rc = fill(args_host, p);
  if (rc != VM_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (p.n_seq == 0) return VM_OK;
  const int hd = args_host->cache.head_dim;
  if (p.max_q > 0) {
    const dim3 grid((p.max_q * p.G + 3) / 4, p.c.n_kv_heads, p.n_seq);
    if (hd == 128) hipLaunchKernelGGL(attn_paged_row_k<128>, grid, dim3(256), 0, st, p);
    else if (hd == 64) hipLaunchKernelGGL(attn_paged_row_k<64>, grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL(attn_paged_row_k<32>, grid, dim3(256), 0, st, p);
    VM_LAUNCH_CHECK();
  }
  if (p.w_out && p.max_kv > 0) {
    const dim3 grid((p.max_kv + 63) / 64, p.c.n_kv_heads, p.n_seq);
    if (hd == 128) hipLaunchKernelGGL(attn_paged_weights_k<128>, grid, dim3(64), 0, st, p);
    else if (hd == 64) hipLaunchKernelGGL(attn_paged_weights_k<64>, grid, dim3(64), 0, st, p);
    else hipLaunchKernelGGL(attn_paged_weights_k<32>, grid, dim3(64), 0, st, p);
    VM_LAUNCH_CHECK();
  }
  return VM_OK;
}

}  // extern "C"
