// Paged KV cache of the generation path: storing new tokens (with the rotary positions of q and k) and eviction by received attention
// weight. Replaces, for a paged cache, the rotary call and the torch.cat of /root/reference/mmmm/models/cogvlm/modeling_cogvlm.py:246-262.
#include "paged.hpp"

namespace {

// ----------------------------------------------------------------------------- append
// q'[t] = R(pos_t) q[t], K[page, row] = R(pos_t) k[t], V[page, row] = v[t];  R on the halves (x1, x2): (x1 c1 - x2 s1, x2 c2 + x1 s2),
// fp32, rounded to bf16 once. HBM-bound: every qkv element is read once and written once. One workgroup takes 256 / tpr rows; a thread
// owns one 8-element chunk index of the half head and walks the heads, so its 32 table values are loaded once per row and not per head.
// 4 x 4609 tokens, 32 heads of width 128: 140 us, 752 MB, 5.4 TB/s (a 2 GiB copy reaches 4.9); one token of eight samples: 3.9 us, the launch.
struct AppendP {
  const unsigned short* qkv; int64_t ld;
  const int32_t* row_seq; const int32_t* row_index; const int32_t* row_pos;
  const float* cos; const float* sin; int n_pos;
  const int32_t* nrows_dev; int rows;
  int n_heads, n_seq;
  unsigned short* q_out; int64_t ldq;
  int tpr;                    // threads per row (power of two, <= 256)
  PagedKV c;
};

template <int HD>
__global__ __launch_bounds__(256) void kv_append_k(const AppendP p) {
  constexpr int CPH = HD / 16;                    // 8-element chunks of a half head
  int rows = p.rows;
  if (p.nrows_dev) rows = min(rows, *p.nrows_dev);
  const int row = blockIdx.x * (256 / p.tpr) + threadIdx.x / p.tpr;
  if (row >= rows) return;
  const int t = threadIdx.x & (p.tpr - 1);
  const int ch = t & (CPH - 1), hl = t / CPH, hstep = p.tpr / CPH;
  const int pos = max(0, min(p.row_pos[row], p.n_pos - 1));
  const int seq = p.row_seq[row], idx = p.row_index[row];
  int64_t dst = -1;                               // element offset of (page, head 0, row), or -1: nothing is stored
  if ((unsigned)seq < (unsigned)p.n_seq && idx >= 0 && (idx >> p.c.shift) < p.c.max_pages) {
    const int page = p.c.table[seq * p.c.ld_table + (idx >> p.c.shift)];
    if (page_ok(page, p.c.n_pages)) dst = page_row(page, p.c.ld_page, 0, idx & p.c.mask, p.c.shift, HD);
  }
  const int64_t head_ld = (int64_t)HD << p.c.shift;
  float c1[8], s1[8], c2[8], s2[8];
  {
    const float* cr = p.cos + (int64_t)pos * HD + ch * 8;
    const float* sr = p.sin + (int64_t)pos * HD + ch * 8;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      *reinterpret_cast<f32x4_t*>(c1 + e) = *reinterpret_cast<const f32x4_t*>(cr + e);
      *reinterpret_cast<f32x4_t*>(s1 + e) = *reinterpret_cast<const f32x4_t*>(sr + e);
      *reinterpret_cast<f32x4_t*>(c2 + e) = *reinterpret_cast<const f32x4_t*>(cr + HD / 2 + e);
      *reinterpret_cast<f32x4_t*>(s2 + e) = *reinterpret_cast<const f32x4_t*>(sr + HD / 2 + e);
    }
  }
  const unsigned short* src = p.qkv + (int64_t)row * p.ld + ch * 8;
  const int H = p.n_heads, Hk = p.c.n_kv_heads, total = H + 2 * Hk;
  for (int h = hl; h < total; h += hstep) {
    const u16x8_t a = *reinterpret_cast<const u16x8_t*>(src + h * HD);
    const u16x8_t b = *reinterpret_cast<const u16x8_t*>(src + h * HD + HD / 2);
    u16x8_t oa = a, ob = b;
    if (h < H + Hk) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x1 = bf2f(a[e]), x2 = bf2f(b[e]);
        oa[e] = f2bf(x1 * c1[e] - x2 * s1[e]);
        ob[e] = f2bf(x2 * c2[e] + x1 * s2[e]);
      }
    }
    unsigned short* d;
    if (h < H) {
      d = p.q_out + (int64_t)row * p.ldq + h * HD;
    } else {
      if (dst < 0) continue;
      const bool is_v = h >= H + Hk;
      d = const_cast<unsigned short*>(is_v ? p.c.v : p.c.k) + dst + (h - H - (is_v ? Hk : 0)) * head_ld;
    }
    *reinterpret_cast<u16x8_t*>(d + ch * 8) = oa;
    *reinterpret_cast<u16x8_t*>(d + HD / 2 + ch * 8) = ob;
  }
}

// ----------------------------------------------------------------------------- eviction
// One workgroup per (sample, kv head) picks the tokens that stay: the `budget` best by (key descending, index ascending), where the key
// is 2^32 - 1 for the `recent` newest tokens, an order-preserving image of the weight for the others (NaN lowest, -0 = +0) and 0 for
// tokens of absent pages, which never stay. The threshold key is found digit by digit (11 + 11 + 10 bits, histogram in LDS) — exact,
// whatever the distribution; then every thread takes a run of consecutive tokens, one scan of the (above, at the threshold) counts gives
// each its place, and the first of those AT the threshold stay. The keys are read and made once and held in LDS (up to EV_LDS_KEYS; beyond
// that they are made again in each pass). Latency-bound: three histogram rounds and four scans of a few hundred cycles (9 us for 600 tokens, 16 us for
// 256 times 4609; the first form, which made the keys again in every round: 52 and 57 us).
constexpr int EV_THREADS = 1024, EV_WAVES = EV_THREADS / 64;

__device__ __forceinline__ unsigned weight_key(float w) {
  if (w != w) return 1u;
  if (w == 0.f) w = 0.f;
  const unsigned u = __builtin_bit_cast(unsigned, w);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

struct EvictP {
  const float* w; float* w_new; int64_t ldw_seq, ldw_head, ldn_seq, ldn_head; int w_cols;
  const int32_t* lens; int32_t* new_lens;
  const int32_t* new_table; int64_t ld_new; int new_pages;
  int32_t* kept; int budget, recent, lds_keys;
  int move_here, log_chunks;  // small budgets: kv_evict_select_k moves the rows itself; log2 of the 16-byte pieces of a row
  PagedKV c;
};

__device__ __forceinline__ unsigned evict_key(const EvictP& p, const float* w, const int32_t* table, int j, int newest) {
  if (!page_ok(table[j >> p.c.shift], p.c.n_pages)) return 0u;
  return j >= newest ? 0xFFFFFFFFu : weight_key(w[j]);
}

constexpr int EV_LDS_KEYS = 32768;

// exclusive scan of a pair of counts over the workgroup; `total`: the sums. Two barriers.
__device__ __forceinline__ uint2 block_scan2(uint2 v, uint2 (*ws)[EV_WAVES], uint2& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint2 x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned a = __shfl_up(x.x, o, 64), b = __shfl_up(x.y, o, 64);
    if (lane >= o) { x.x += a; x.y += b; }
  }
  if (lane == 63) (*ws)[wave] = x;
  __syncthreads();
  uint2 before = {0, 0};
  total = {0, 0};
#pragma unroll
  for (int i = 0; i < EV_WAVES; ++i) {
    const uint2 w = (*ws)[i];
    if (i < wave) { before.x += w.x; before.y += w.y; }
    total.x += w.x;
    total.y += w.y;
  }
  __syncthreads();
  return {before.x + x.x - v.x, before.y + x.y - v.y};
}

// 16 bytes of the row that becomes token j from old token i, K and V, at element e of the row
__device__ __forceinline__ void evict_move(const EvictP& p, int hk, int b, int j, int i, int e, int head_dim) {
  if ((j >> p.c.shift) >= p.new_pages) return;
  const int src = p.c.table[b * p.c.ld_table + (i >> p.c.shift)], dst = p.new_table[b * p.ld_new + (j >> p.c.shift)];
  if (!page_ok(src, p.c.n_pages) || !page_ok(dst, p.c.n_pages)) return;
  const int64_t s = page_row(src, p.c.ld_page, hk, i & p.c.mask, p.c.shift, head_dim) + e, d = page_row(dst, p.c.ld_page, hk, j & p.c.mask, p.c.shift, head_dim) + e;
  if (s == d) return;
  const u16x8_t kv = *reinterpret_cast<const u16x8_t*>(p.c.k + s), vv = *reinterpret_cast<const u16x8_t*>(p.c.v + s);
  *reinterpret_cast<u16x8_t*>(const_cast<unsigned short*>(p.c.k) + d) = kv;
  *reinterpret_cast<u16x8_t*>(const_cast<unsigned short*>(p.c.v) + d) = vv;
}

// The most rows that kv_evict_select_k moves itself: one launch less (8 rows 10.4 -> 9.1 us, 128 rows 10.7 -> 10.4, of 16 x 32 heads 27 -> 25); above it
// the one workgroup of a cache is too few (192 rows: 11.1 us in two launches).
constexpr int EV_MOVE = 128;

__global__ __launch_bounds__(EV_THREADS) void kv_evict_select_k(const EvictP p) {
  extern __shared__ unsigned keys[];              // min(n, EV_LDS_KEYS) of them
  __shared__ unsigned hist[2048];
  __shared__ unsigned found[2];
  __shared__ uint2 ws[EV_WAVES];
  __shared__ int stay[EV_MOVE];
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int cap = (int)min((int64_t)p.c.max_pages << p.c.shift, (int64_t)p.w_cols);
  const int n = max(0, min(p.lens[b], cap));
  const int newest = n - min(p.recent, n);
  const float* w = p.w + b * p.ldw_seq + hk * p.ldw_head;
  float* wn = p.w_new + b * p.ldn_seq + hk * p.ldn_head;
  const int32_t* table = p.c.table + b * p.c.ld_table;
  int32_t* kept = p.kept + ((int64_t)b * p.c.n_kv_heads + hk) * p.budget;
  const bool in_lds = n <= p.lds_keys;
  auto key_of = [&](int j) -> unsigned { return in_lds ? keys[j] : evict_key(p, w, table, j, newest); };
  // ---- threshold
  unsigned prefix = 0, pmask = 0;
  int want = 0, keep = 0;                         // how many of the keys that share the prefix stay
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    hist[tid] = hist[tid + EV_THREADS] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += EV_THREADS) {
      unsigned key;
      if (pass == 0) {
        key = evict_key(p, w, table, j, newest);
        if (in_lds) keys[j] = key;
      } else {
        key = key_of(j);
      }
      if (key != 0 && (key & pmask) == prefix) atomicAdd(&hist[(key >> shift) & ((1 << bits) - 1)], 1u);
    }
    __syncthreads();
    // bins in descending order, two per thread: the one that holds the want-th largest key
    const unsigned h0 = hist[2047 - 2 * tid], h1 = hist[2046 - 2 * tid];
    uint2 all;
    const unsigned above = block_scan2({h0 + h1, 0}, &ws, all).x;
    if (pass == 0) keep = want = min((int)all.x, p.budget);
    if (above < (unsigned)want && (unsigned)want <= above + h0 + h1) {
      const bool second = (unsigned)want > above + h0;
      found[0] = 2047 - 2 * tid - (second ? 1 : 0);
      found[1] = above + (second ? h0 : 0);
    }
    __syncthreads();
    if (want > 0) {
      prefix |= found[0] << shift;
      want -= (int)found[1];
    }
    pmask |= ((1u << bits) - 1) << shift;
  }
  // ---- survivors in index order
  if (keep > 0) {
    const int run = ((n + EV_THREADS - 1) / EV_THREADS) | 1;        // odd: no LDS bank conflicts between the threads' runs
    const int j0 = min(tid * run, n), j1 = min(j0 + run, n);
    uint2 c = {0, 0}, all;
    for (int j = j0; j < j1; ++j) {
      const unsigned key = key_of(j);
      c.x += key > prefix;
      c.y += key == prefix;
    }
    const uint2 before = block_scan2(c, &ws, all);
    unsigned eq = before.y, at = before.x + min(eq, (unsigned)want);
    for (int j = j0; j < j1; ++j) {
      const unsigned key = key_of(j);
      const bool tie = key == prefix;
      if (key > prefix || (tie && eq < (unsigned)want)) {
        kept[at] = j;
        wn[at] = w[j];
        if (p.move_here) stay[at] = j;
        ++at;
      }
      eq += tie;
    }
  }
  for (int j = keep + tid; j < p.budget; j += EV_THREADS) kept[j] = -1;
  for (int j = keep + tid; j < p.w_cols; j += EV_THREADS) wn[j] = 0.f;      // the next tokens of this sample start at zero
  if (hk == 0 && tid == 0) p.new_lens[b] = keep;
  if (p.move_here) {
    __syncthreads();
    for (int x = tid; x < keep << p.log_chunks; x += EV_THREADS) {
      const int j = x >> p.log_chunks;
      evict_move(p, hk, b, j, stay[j], (x & ((1 << p.log_chunks) - 1)) * 8, 8 << p.log_chunks);
    }
  }
}

// the rows that stay, K and V, into the sample's new pages: HD / 8 lanes per row, 16 bytes each. HBM-bound: 8 x 32 heads x 1152 rows of width 128,
// 302 MB, 65 us, 4.6 TB/s.
template <int HD>
__global__ __launch_bounds__(256) void kv_evict_move_k(const EvictP p) {
  constexpr int LPR = HD / 8, RPB = 256 / LPR;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int j = blockIdx.x * RPB + threadIdx.x / LPR, e = (threadIdx.x & (LPR - 1)) * 8;
  if (j >= p.budget) return;
  const int i = p.kept[((int64_t)b * p.c.n_kv_heads + hk) * p.budget + j];
  if (i >= 0) evict_move(p, hk, b, j, i, e, HD);
}

}  // namespace

extern "C" {

int vm_kv_append_paged_bf16(const vm_paged_kv* cache_host, const void* qkv, int64_t ld, const int32_t* row_seq, const int32_t* row_index,
                            const int32_t* row_pos, const float* cos_tab, const float* sin_tab, int n_pos, int rows, int n_heads,
                            void* q_out, int64_t ldq, const int32_t* nrows_dev, void* stream) {
  AppendP p;
  const int rc = paged_cache(cache_host, p.c);
  if (rc != VM_OK) return rc;
  if (rows < 0 || n_heads <= 0 || n_pos <= 0) return VM_ERR_BAD_ARG;
  if (rows == 0) return VM_OK;                    // (rows without a sample still have a rotated q)
  if (!qkv || !row_seq || !row_index || !row_pos || !cos_tab || !sin_tab || !q_out) return VM_ERR_BAD_ARG;
  const int hd = cache_host->head_dim, total = n_heads + 2 * p.c.n_kv_heads;
  if (misaligned16(qkv) || misaligned16(q_out) || misaligned16(cos_tab) || misaligned16(sin_tab) || (ld & 7) || (ldq & 7)) return VM_ERR_BAD_ARG;
  if (ld < (int64_t)total * hd || ldq < (int64_t)n_heads * hd) return VM_ERR_BAD_ARG;
  p.qkv = (const unsigned short*)qkv; p.ld = ld; p.row_seq = row_seq; p.row_index = row_index; p.row_pos = row_pos;
  p.cos = cos_tab; p.sin = sin_tab; p.n_pos = n_pos; p.nrows_dev = nrows_dev; p.rows = rows; p.n_heads = n_heads; p.n_seq = cache_host->n_seq;
  p.q_out = (unsigned short*)q_out; p.ldq = ldq;
  p.tpr = hd / 16;
  while (p.tpr < 256 && p.tpr < total * (hd / 16)) p.tpr *= 2;
  const dim3 grid((rows + 256 / p.tpr - 1) / (256 / p.tpr));
  hipStream_t st = (hipStream_t)stream;
  if (hd == 128) hipLaunchKernelGGL(kv_append_k<128>, grid, dim3(256), 0, st, p);
  else if (hd == 64) hipLaunchKernelGGL(kv_append_k<64>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(kv_append_k<32>, grid, dim3(256), 0, st, p);
  VM_LAUNCH_CHECK();
  return VM_OK;
}

int vm_kv_evict_paged_bf16(const vm_paged_kv* cache_host, const float* weights, int64_t ldw_seq, int64_t ldw_head, int w_cols,
                           const int32_t* kv_lens, const int32_t* new_table, int64_t ld_new_table, int new_pages, int budget, int recent,
                           float* new_weights, int64_t ldn_seq, int64_t ldn_head, int32_t* new_lens, int32_t* kept, void* stream) {
  EvictP p;
  const int rc = paged_cache(cache_host, p.c);
  if (rc != VM_OK) return rc;
  if (budget <= 0 || recent < 0 || recent > budget || w_cols <= 0 || new_pages <= 0 || ld_new_table < new_pages) return VM_ERR_BAD_ARG;
  if (ldw_head < w_cols || ldn_head < w_cols || ldw_seq < 0 || ldn_seq < 0) return VM_ERR_BAD_ARG;
  const int64_t most = (int64_t)p.c.max_pages << p.c.shift;
  const int cols = (int)(most < w_cols ? most : w_cols);
  if ((int64_t)new_pages << p.c.shift < (budget < cols ? budget : cols)) return VM_ERR_BAD_ARG;      // who stays has a place
  if (cache_host->n_seq == 0) return VM_OK;
  if (cache_host->n_seq > 65535 || p.c.n_kv_heads > 65535) return VM_ERR_UNSUPPORTED;
  if (!weights || !kv_lens || !new_table || !new_weights || !new_lens || !kept) return VM_ERR_BAD_ARG;
  if (weights == new_weights || kv_lens == new_lens || cache_host->block_table == new_table) return VM_ERR_BAD_ARG;      // out of place
  p.w = weights; p.w_new = new_weights; p.ldw_seq = ldw_seq; p.ldw_head = ldw_head; p.ldn_seq = ldn_seq; p.ldn_head = ldn_head; p.w_cols = w_cols;
  p.lens = kv_lens; p.new_lens = new_lens; p.new_table = new_table; p.ld_new = ld_new_table; p.new_pages = new_pages;
  p.kept = kept; p.budget = budget; p.recent = recent;
  hipStream_t st = (hipStream_t)stream;
  static std::atomic<uint64_t> set{0};
  if (!allow_lds((const void*)kv_evict_select_k, EV_LDS_KEYS * 4, set)) return VM_ERR_LAUNCH;
  p.lds_keys = cols < EV_LDS_KEYS ? cols : EV_LDS_KEYS;
  p.log_chunks = cache_host->head_dim == 128 ? 4 : cache_host->head_dim == 64 ? 3 : 2;
  p.move_here = budget <= EV_MOVE;
  hipLaunchKernelGGL(kv_evict_select_k, dim3(p.c.n_kv_heads, cache_host->n_seq), dim3(EV_THREADS), p.lds_keys * 4, st, p);
  VM_LAUNCH_CHECK();
  if (p.move_here) return VM_OK;
  const int hd = cache_host->head_dim, rpb = 256 / (hd / 8);
  const dim3 grid((budget + rpb - 1) / rpb, p.c.n_kv_heads, cache_host->n_seq);
  if (hd == 128) hipLaunchKernelGGL(kv_evict_move_k<128>, grid, dim3(256), 0, st, p);
  else if (hd == 64) hipLaunchKernelGGL(kv_evict_move_k<64>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(kv_evict_move_k<32>, grid, dim3(256), 0, st, p);
  VM_LAUNCH_CHECK();
  return VM_OK;
}

}  // extern "C"
