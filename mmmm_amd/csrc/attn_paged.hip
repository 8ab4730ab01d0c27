// Attention of a chunk of new tokens over the paged KV cache (generation path): one token, a follow-up question or a whole prompt.
// Stands for the attention calls of /root/reference/mmmm/models/cogvlm/modeling_cogvlm.py:113-141 where K and V come from the cache.
//
// Query rows of one kv head are taken together: row r of (sample b, kv head hk) is query i = r / G of head hk G + r % G (G heads share the
// kv head), so grouped heads read K and V once. Query i sees the tokens j <= L - n + i.
#include "paged.hpp"
#include "vm_tile.hpp"

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
  // split form: n_split key splits; workspace of s_rows query rows per (sample, kv head)
  int n_split, s_rows, s_ld;
  int n_tiles, n_wg;          // tile form: row tiles per (sample, kv head), workgroups
  int w_blocks;               // weigh_k: 128-token blocks per (sample, kv head)
  float* part;                // [.., s_rows, n_split, hd + 4]: max, sum, -, -, O
  float* s_ws;                // [.., s_rows, s_ld] scores (log2 domain), if the received weights are asked for
  int join_blocks;            // attn_paged_join_k: workgroups (x) that join rows; those behind them count
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

// ----------------------------------------------------------------------------- few query rows: keys split over waves and workgroups
// HBM-bound: K and V of a sample are read once (4 hd bytes per token and kv head), the arithmetic is small beside it. A wave owns 16 query
// rows and walks blocks of 32 keys:
//   S^T[key][row] = K Q^T with v_mfma_f32_16x16x32_bf16: a lane loads its 16-byte pieces of K straight from the page as the A operand (K never
//   touches LDS); the row sits on the lane (ln = lane & 15), so the running maximum and sum are per-lane scalars plus two lane swaps;
//   O^T[d][row] += V^T P^T: V goes page -> registers -> the wave's own 8 KiB of LDS and comes back transposed (ds_read_b64_tr_b16); the two
//   stacked score tiles ARE the B operand. P is taken as two bf16 terms (its rounding and what that left out: 16 significant bits), the
//   second product costs matrix time that the loads leave idle, and the only rounding the result sees is its own.
// The next block's K and V are in flight while one is computed; page numbers are fetched two blocks ahead through the scalar cache.
// A workgroup has eight waves, each a key stream of its own (one workgroup per CU: 8 x 16 KiB in flight); they meet in LDS, and if the keys
// were split over workgroups too the partial (max, sum, O) of each goes to the workspace and attn_paged_join_k joins them in a fixed order.
// Measured beside four waves a workgroup and two of them per CU: 32 x 16384 grouped 281 us (5.8 TB/s) / 285 us, 8 x 4609 92 / 91 us.
constexpr int SP_WAVES = 8;
constexpr int SP_ROWS = 16;                        // query rows (queries x heads of the group) of the form

__device__ __forceinline__ void swap16(float& a, float& b) { asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ void swap32(float& a, float& b) { asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ float max_over_g(float x) {        // maximum over the lanes that share lane & 15
  float a = x, b = x;
  swap16(a, b);
  a = b = fmaxf(a, b);
  asm volatile("" : "+v"(a), "+v"(b));
  swap32(a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float sum_over_g(float x) {
  float a = x, b = x;
  swap16(a, b);
  a = b = a + b;
  asm volatile("" : "+v"(a), "+v"(b));
  swap32(a, b);
  return a + b;
}
// Values that are not finite, in a tile that only some rows see: the matrix product would carry them into the rows that do not (0 x inf, 0 x NaN).
// Such a tile is multiplied with them as zeros, and the rows that see them get their share one key at a time.
__device__ __forceinline__ bool none_finite2(unsigned m) { return (m >> 16) >= 0x7F80u || (m & 0xFFFFu) >= 0x7F80u; }
__device__ __forceinline__ unsigned max2(unsigned m, unsigned x) {          // two 16-bit magnitudes at a time
  typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, m), __builtin_bit_cast(u16x2_t, x & 0x7FFF7FFFu)));
}
__device__ __forceinline__ unsigned finite2(unsigned x) {
  if ((x & 0x7F80u) == 0x7F80u) x &= 0xFFFF0000u;
  if ((x & 0x7F800000u) == 0x7F800000u) x &= 0x0000FFFFu;
  return x;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

template <int HD>
struct KVBlock {                                    // 32 keys of one kv head on their way through a wave
  static constexpr int KS = HD / 32, CPR = HD / 8, RPI = 64 / CPR, NV = 32 / RPI;
  i32x4_t k[2][KS], v[NV];
};

// the two page numbers of a 32-key block (pages of 16 rows end inside it); -1 behind the last key
struct PagePair { int a, b; };
__device__ __forceinline__ PagePair block_pages(const AttnPagedP& p, table_ptr table, int j0, int kv_end) {
  PagePair r = {-1, -1};
  if (j0 < kv_end) r.a = table[j0 >> p.c.shift];
  if (j0 + 16 < kv_end) r.b = table[(j0 + 16) >> p.c.shift];
  if (!page_ok(r.a, p.c.n_pages)) r.a = -1;
  if (!page_ok(r.b, p.c.n_pages)) r.b = -1;
  return r;
}

template <int HD>
__device__ __forceinline__ void load_block(const AttnPagedP& p, KVBlock<HD>& x, PagePair pg, int hk, int j0, int kv_end, int lane) {
  typedef KVBlock<HD> B;
  const int ln = lane & 15, g = lane >> 4;
  const i32x4_t zero = {0, 0, 0, 0};
#pragma unroll
  for (int jj = 0; jj < 2; ++jj) {
    const int page = jj ? pg.b : pg.a, row = (j0 + 16 * jj) & p.c.mask;
    const unsigned short* kb = p.c.k + page_row(page < 0 ? 0 : page, p.c.ld_page, hk, row, p.c.shift, HD) + ln * HD + 8 * g;
#pragma unroll
    for (int s = 0; s < B::KS; ++s) x.k[jj][s] = page < 0 ? zero : *reinterpret_cast<const i32x4_t*>(kb + 32 * s);
  }
#pragma unroll
  for (int i = 0; i < B::NV; ++i) {
    const int r = i * B::RPI + lane / B::CPR;        // row of the block
    const int page = r < 16 ? pg.a : pg.b, row = (j0 + r) & p.c.mask;
    x.v[i] = zero;                                   // rows behind the last token that is seen hold anything: they count as zeros
    if (page >= 0 && j0 + r < kv_end)
      x.v[i] = *reinterpret_cast<const i32x4_t*>(p.c.v + page_row(page, p.c.ld_page, hk, row, p.c.shift, HD) + (lane & (B::CPR - 1)) * 8);
  }
}

// The received weight of token j from the scores that the query rows left behind (log2 domain) and the log2 of their sums, the rows in their order.
__device__ __forceinline__ void count(const AttnPagedP& p, const SeqInfo& s, int b, int hk, int R, int j, const float* l2) {
  float sum = 0.f;
  // the first row of a query that sees the token: its scores, and those of all later rows, were stored by the wave that walked the block
  // (max_q bounds it before the product: R fits 32 bits, the number of rows behind a long sample need not). A page that is not there: nothing.
  const int first = page_ok(p.c.table[b * p.c.ld_table + (j >> p.c.shift)], p.c.n_pages) ? min(max(0, j - (s.len - s.nq)), p.max_q) * p.G : R;
  const float* sc = p.s_ws + ((int64_t)b * p.c.n_kv_heads + hk) * p.s_rows * p.s_ld + j;
  float x[SP_ROWS];
#pragma unroll
  for (int r = 0; r < SP_ROWS; ++r) x[r] = r >= first && r < R ? sc[(int64_t)r * p.s_ld] : -INFINITY;
#pragma unroll
  for (int r = 0; r < SP_ROWS; ++r)
    if (r >= first && r < R && l2[r] != -INFINITY) sum += fast_exp2(x[r] - l2[r]);
  p.w_out[b * p.ldwo_seq + hk * p.ldwo_head + j] = p.w_in[b * p.ldw_seq + hk * p.ldw_head + j] + sum;
}

template <int HD>
__global__ __launch_bounds__(SP_WAVES * 64, 2) void attn_paged_split_k(const AttnPagedP p) {
  typedef KVBlock<HD> B;
  constexpr int KW = SP_WAVES;
  constexpr int ND = HD / 16;
  __shared__ __attribute__((aligned(1024))) char smem[SP_WAVES][32 * ROWB];
  __shared__ float red[SP_WAVES][2][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, g = lane >> 4;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int split = blockIdx.x;
  const SeqInfo s = seq_info(p, b);
  const int R = min(min(s.nq, p.max_q) * p.G, SP_ROWS);
  if (R <= 0) {                                      // no new token: the weights stay what they are
    if (p.s_ws && p.n_split == 1)
      for (int j = threadIdx.x; j < min(s.len, min(p.w_cols, p.s_ld)); j += SP_WAVES * 64) count(p, s, b, hk, 0, j, red[0][0]);
    return;
  }
  const int r = ln;
  const bool live = r < R;
  const int i = live ? r / p.G : 0, h = hk * p.G + (live ? r - i * p.G : 0);
  const int prow = live ? phys_row(p, s.p0 + i) : -1;
  const int lim = live ? s.len - s.nq + i : -1;      // last token this row sees
  const int lim_min = s.len - s.nq;
  const int kv_end = max(0, s.len - s.nq + (R - 1) / p.G + 1);
  // this workgroup's blocks
  const int nblk = (kv_end + 31) / 32, per = (nblk + p.n_split - 1) / p.n_split;
  const int blk0 = min(split * per, nblk), blk1 = min(blk0 + per, nblk);

  bf16x8_t qf[B::KS];
#pragma unroll
  for (int t = 0; t < B::KS; ++t) {
    i32x4_t v = {0, 0, 0, 0};
    if (prow >= 0) v = *reinterpret_cast<const i32x4_t*>(p.q + prow * p.ldq + h * HD + 32 * t + 8 * g);
    qf[t] = __builtin_bit_cast(bf16x8_t, v);
  }
  f32x4_t o[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) o[t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const float sc = p.scale * LOG2E;
  const table_ptr table = table_of(p.c, b);
  char* tv = smem[wave];
  float* srow = p.s_ws ? p.s_ws + (((int64_t)b * p.c.n_kv_heads + hk) * p.s_rows + r) * p.s_ld : nullptr;

  KVBlock<HD> cur, nxt;
  int blk = blk0 + wave;
  PagePair pg = block_pages(p, table, blk * 32, kv_end);
  if (blk < blk1) load_block<HD>(p, cur, pg, hk, blk * 32, kv_end, lane);
  PagePair pg1 = block_pages(p, table, (blk + KW) * 32, kv_end);
  for (; blk < blk1; blk += KW) {
    const PagePair pg2 = block_pages(p, table, (blk + 2 * KW) * 32, kv_end);
    if (blk + KW < blk1) load_block<HD>(p, nxt, pg1, hk, (blk + KW) * 32, kv_end, lane);
    const int j0 = blk * 32;
    f32x4_t sa[2];
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      sa[jj] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < B::KS; ++t) sa[jj] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, cur.k[jj][t]), qf[t], sa[jj], 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) sa[jj][e] *= sc;
    }
    bool strange = false;
    if (j0 + 31 > lim_min || pg.a < 0 || pg.b < 0) {
#pragma unroll
      for (int jj = 0; jj < 2; ++jj)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((jj ? pg.b : pg.a) < 0 || j0 + 16 * jj + 4 * g + e > lim) sa[jj][e] = -INFINITY;
      unsigned most = 0;
#pragma unroll
      for (int t = 0; t < B::NV; ++t)
#pragma unroll
        for (int w = 0; w < 4; ++w) most = max2(most, __builtin_bit_cast(u32x4_t, cur.v[t])[w]);
      strange = __builtin_amdgcn_ballot_w64(none_finite2(most)) != 0;
    }
    if (srow && live) {
#pragma unroll
      for (int jj = 0; jj < 2; ++jj)
        if (j0 + 16 * jj + 4 * g < p.s_ld) *reinterpret_cast<f32x4_t*>(srow + j0 + 16 * jj + 4 * g) = sa[jj];
    }
    // V -> LDS while the scores settle
#pragma unroll
    for (int t = 0; t < B::NV; ++t) {
      u32x4_t v = __builtin_bit_cast(u32x4_t, cur.v[t]);
      if (__builtin_expect(strange, 0)) {
#pragma unroll
        for (int w = 0; w < 4; ++w) v[w] = finite2(v[w]);
      }
      *reinterpret_cast<u32x4_t*>(tv + tile_off16(t * B::RPI + lane / B::CPR, lane & (B::CPR - 1))) = v;
    }
    float mx = fmaxf(fmaxf(fmaxf(sa[0][0], sa[0][1]), fmaxf(sa[0][2], sa[0][3])), fmaxf(fmaxf(sa[1][0], sa[1][1]), fmaxf(sa[1][2], sa[1][3])));
    mx = max_over_g(mx);
    if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
      const float mn = fmaxf(m, mx), alpha = fast_exp2(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][e] *= alpha;
    }
    const float base = m == -INFINITY ? 0.f : m;
    u16x8_t hi, lo;
#pragma unroll
    for (int jj = 0; jj < 2; ++jj)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = fast_exp2(sa[jj][e] - base);
        l += x;
        hi[4 * jj + e] = f2bf(x);
        lo[4 * jj + e] = f2bf(x - bf2f(hi[4 * jj + e]));
      }
    const bf16x8_t ph = __builtin_bit_cast(bf16x8_t, hi), pl = __builtin_bit_cast(bf16x8_t, lo);
#pragma unroll
    for (int t = 0; t < ND; ++t) {
      const bf16x8_t vf = frag16_tr(tv, 0, t, lane);
      o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, ph, o[t], 0, 0, 0);
      o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl, o[t], 0, 0, 0);
    }
    if (__builtin_expect(strange, 0)) {
#pragma unroll
      for (int t = 0; t < B::NV; ++t)
        *reinterpret_cast<i32x4_t*>(tv + tile_off16(t * B::RPI + lane / B::CPR, lane & (B::CPR - 1))) = cur.v[t];
#pragma unroll
      for (int jj = 0; jj < 2; ++jj)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = fast_exp2(sa[jj][e] - base);
          for (int gg = 0; gg < 4; ++gg) {                          // key 16 jj + 4 gg + e of the block: its weight for this lane's row
            const float w = __shfl(x, ln + 16 * gg, 64);
            const bool sees = __shfl(sa[jj][e], ln + 16 * gg, 64) != -INFINITY;
#pragma unroll
            for (int t = 0; t < ND; ++t) {
              const u16x4_t v = *reinterpret_cast<const u16x4_t*>(tv + tile_off16(16 * jj + 4 * gg + e, 2 * t + (g >> 1)) + 8 * (g & 1));
#pragma unroll
              for (int c = 0; c < 4; ++c)
                if (sees && (v[c] & 0x7F80) == 0x7F80) o[t][c] = fmaf(w, bf2f(v[c]), o[t][c]);
            }
          }
        }
    }
    cur = nxt;
    pg = pg1;
    pg1 = pg2;
  }
  l = sum_over_g(l);
  // ---- the key streams meet in LDS: each wave adds up its share of O^T, in the order of the streams
  if (g == 0) { red[wave][0][ln] = m; red[wave][1][ln] = l; }
  __syncthreads();
  {
    float mm = m;
#pragma unroll
    for (int k = 0; k < KW; ++k) mm = fmaxf(mm, red[k][0][ln]);
    const float base = mm == -INFINITY ? 0.f : mm, f = fast_exp2(m - base);
    l = 0.f;
#pragma unroll
    for (int k = 0; k < KW; ++k) l += red[k][1][ln] * fast_exp2(red[k][0][ln] - base);
    m = mm;
    float* slab = reinterpret_cast<float*>(smem[wave]);          // O^T of this wave, [d][row]
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) slab[(16 * t + 4 * g + e) * 16 + ln] = o[t][e] * f;
  }
  __syncthreads();
  if (live && wave < ND) {
    f32x4_t x = {0.f, 0.f, 0.f, 0.f};              // the wave's 16 columns
#pragma unroll
    for (int k = 0; k < KW; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += reinterpret_cast<const float*>(smem[k])[(16 * wave + 4 * g + e) * 16 + ln];
    const bool writes_row = wave == 0 && g == 0;
    if (p.n_split == 1) {
      const bool some = !(l == 0.f);
      const float inv = some ? 1.f / l : 0.f;
      if (prow >= 0) {
        const u16x4_t w = {f2bf(x[0] * inv), f2bf(x[1] * inv), f2bf(x[2] * inv), f2bf(x[3] * inv)};
        *reinterpret_cast<u16x4_t*>(p.out + prow * p.ldo + h * HD + 16 * wave + 4 * g) = some ? w : (u16x4_t){0, 0, 0, 0};
      }
      if (writes_row) {
        const float l2 = some && prow >= 0 ? m + log2f(l) : -INFINITY;
        p.lse[h * p.ld_lse + s.p0 + i] = l2 * LN2;
        red[0][0][ln] = l2;
      }
    } else {
      float* part = p.part + ((((int64_t)b * p.c.n_kv_heads + hk) * p.s_rows + r) * p.n_split + split) * (HD + 4);
      if (writes_row) { part[0] = m; part[1] = l; }
      *reinterpret_cast<f32x4_t*>(part + 4 + 16 * wave + 4 * g) = x;
    }
  }
  if (p.s_ws && p.n_split == 1) {                   // nothing to join: the received weights at once
    __syncthreads();
    for (int j = threadIdx.x; j < min(s.len, min(p.w_cols, p.s_ld)); j += SP_WAVES * 64) count(p, s, b, hk, R, j, red[0][0]);
  }
}

// joins the key splits of a query row: out = sum_k 2^(m_k - m) O_k / sum_k 2^(m_k - m) l_k, the splits in their order. HD / 4 lanes per row, 16 bytes
// each. Latency-bound for a few rows (4 us of which the launch is most): the partial results are asked for four splits at a time and before anything
// is known about the sample (a row that does not exist reads its own piece of the workspace and throws it away). 32 x 512 rows in four splits,
// 35 MB: 8 us (one wave per row, 4 bytes a lane and split: 11).
template <int HD>
__global__ __launch_bounds__(256) void attn_paged_join_k(const AttnPagedP p) {
  constexpr int LPR = HD / 4, RPB = 256 / LPR, U = 4;                // lanes per row, rows per workgroup
  const int hk = blockIdx.y, b = blockIdx.z;
  const int n = p.n_split;
  if ((int)blockIdx.x >= p.join_blocks) {            // split form with received weights: the other workgroups take 256 tokens each
    __shared__ float l2s[SP_ROWS];
    const SeqInfo s = seq_info(p, b);
    const int R = min(min(s.nq, p.max_q) * p.G, SP_ROWS), j = ((int)blockIdx.x - p.join_blocks) * 256 + threadIdx.x, t = threadIdx.x;
    if (t < R) {
      const float* part = p.part + (((int64_t)b * p.c.n_kv_heads + hk) * p.s_rows + t) * n * (HD + 4);
      float m = -INFINITY, l = 0.f;
      for (int k = 0; k < n; ++k) m = fmaxf(m, part[(int64_t)k * (HD + 4)]);
      const float base = m == -INFINITY ? 0.f : m;
      for (int k = 0; k < n; ++k) l += fast_exp2(part[(int64_t)k * (HD + 4)] - base) * part[(int64_t)k * (HD + 4) + 1];
      l2s[t] = !(l == 0.f) && phys_row(p, s.p0 + t / p.G) >= 0 ? m + log2f(l) : -INFINITY;
    }
    __syncthreads();
    if (j < min(s.len, min(p.w_cols, p.s_ld))) count(p, s, b, hk, R, j, l2s);
    return;
  }
  const int r = blockIdx.x * RPB + threadIdx.x / LPR, sub = threadIdx.x & (LPR - 1), d = 4 * sub;
  const int64_t slot = ((int64_t)b * p.c.n_kv_heads + hk) * p.s_rows + min(r, p.s_rows - 1);
  const float* part = p.part + slot * n * (HD + 4);
  struct Piece { float m[U], l[U]; f32x4_t o[U]; } x;
  auto load = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* q = part + (int64_t)min(k0 + u, n - 1) * (HD + 4);
      const f32x2_t ml = *reinterpret_cast<const f32x2_t*>(q);
      x.m[u] = ml[0];
      x.l[u] = ml[1];
      x.o[u] = *reinterpret_cast<const f32x4_t*>(q + 4 + d);
    }
  };
  load(0);
  float m = -INFINITY;
  for (int k = sub; k < n; k += LPR) m = fmaxf(m, part[(int64_t)k * (HD + 4)]);
#pragma unroll
  for (int k = 1; k < LPR; k <<= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
  const SeqInfo s = seq_info(p, b);
  if (r >= min(s.nq, p.max_q) * p.G) return;
  const int i = r / p.G, h = hk * p.G + r % p.G, prow = phys_row(p, s.p0 + i);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < n; k += U) {
    if (k > 0) load(k);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k + u >= n) break;
      const float f = fast_exp2(x.m[u] - base);
      l += f * x.l[u];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(f, x.o[u][e], o[e]);
    }
  }
  const bool some = !(l == 0.f);
  const float inv = some ? 1.f / l : 0.f, l2 = some && prow >= 0 ? m + log2f(l) : -INFINITY;
  if (prow >= 0) {
    const u16x4_t w = {f2bf(o[0] * inv), f2bf(o[1] * inv), f2bf(o[2] * inv), f2bf(o[3] * inv)};
    *reinterpret_cast<u16x4_t*>(p.out + prow * p.ldo + h * HD + d) = some ? w : (u16x4_t){0, 0, 0, 0};
  }
  if (sub == 0) p.lse[h * p.ld_lse + s.p0 + i] = l2 * LN2;
}

}  // namespace
#include "attn_paged_tile.hpp"
namespace {

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

// ----------------------------------------------------------------------------- which form, and its workspace
struct Plan { bool split; int64_t part, s_ws, bytes; };

Plan plan(AttnPagedP& p, int hd) {
  Plan a = {};
  const int64_t rows = (int64_t)p.max_q * p.G, heads = (int64_t)p.n_seq * p.c.n_kv_heads;
  // 16 rows are what the split form's matrix tile holds. Beyond it the tile form wins although most of its 256 rows are empty: 4 x 17 queries
  // over 2086 tokens 31 us beside 37 us (two row tiles a workgroup), 17 x 4 heads over 8704 26 beside 45, 64 queries 37 beside 53.
  a.split = rows <= SP_ROWS;
  p.n_split = 1; p.s_rows = (int)rows; p.s_ld = (p.max_kv + 31) / 32 * 32;
  p.part = p.s_ws = nullptr;
  p.join_blocks = (int)((rows * hd + 1023) / 1024);
  p.n_tiles = p.n_wg = 0;
  if (rows == 0 || heads == 0) return a;
  if (!a.split) {
    p.n_tiles = (int)((rows + apt::QB - 1) / apt::QB);
    const int64_t wgs = heads * p.n_tiles, want = (256 + wgs - 1) / wgs, most = (p.max_kv + 511) / 512;
    p.n_split = (int)(want < most ? want : most);
    if (p.n_split < 1) p.n_split = 1;
    if (p.n_split > 1) a.bytes = heads * rows * p.n_split * (hd + 4) * 4;
    p.n_wg = wgs * p.n_split > 0x7FFFFF00 ? -1 : (int)(wgs * p.n_split);
    return a;
  }
  // one workgroup per CU, two rounds (ragged lengths): 512, and 64 keys for a wave at least
  const int64_t want = (512 + heads - 1) / heads, most = (p.max_kv + 64 * SP_WAVES - 1) / (64 * SP_WAVES);
  p.n_split = (int)(want < most ? want : most);
  if (p.n_split < 1) p.n_split = 1;
  int64_t at = 0;
  if (p.n_split > 1) { a.part = at; at += heads * rows * p.n_split * (hd + 4) * 4; }
  if (p.w_out) { a.s_ws = at; at += heads * rows * p.s_ld * 4; }
  a.bytes = at;
  return a;
}

template <int HD>
void launch_split(const AttnPagedP& p, hipStream_t st) {
  hipLaunchKernelGGL(attn_paged_split_k<HD>, dim3(p.n_split, p.c.n_kv_heads, p.n_seq), dim3(SP_WAVES * 64), 0, st, p);
  const int count_blocks = p.w_out ? (p.max_kv + 255) / 256 : 0;
  if (p.n_split > 1) hipLaunchKernelGGL(attn_paged_join_k<HD>, dim3(p.join_blocks + count_blocks, p.c.n_kv_heads, p.n_seq), dim3(256), 0, st, p);
}

// workgroups of the tile form: eight XCDs, each as many as the longest piece of the list (tile_k: whole caches where the list is short)
int64_t tile_grid(const AttnPagedP& p) {
  const int64_t caches = (int64_t)p.n_seq * p.c.n_kv_heads, even = ((int64_t)p.n_wg + 7) / 8, whole = (caches + 7) / 8 * p.n_tiles * p.n_split;
  return 8 * (whole > even ? whole : even);
}

template <int HD>
int launch_weigh(AttnPagedP& p, hipStream_t st) {
  p.w_blocks = (p.max_kv + 127) / 128;
  const int64_t caches = ((int64_t)p.n_seq * p.c.n_kv_heads + 7) / 8 * 8;
  if (caches * p.w_blocks > 0x7FFFFF00) return VM_ERR_UNSUPPORTED;
  // four sets of waves per workgroup take a CU's LDS: where the workgroups do not even fill the chip once
  if (caches * p.w_blocks <= 256 && (int64_t)p.max_q * p.G > 128) {
    static std::atomic<uint64_t> set{0};
    if (!allow_lds((const void*)apt::weigh_k<HD, 4>, 4 * sizeof(apt::WeighLds), set)) return VM_ERR_LAUNCH;
    hipLaunchKernelGGL((apt::weigh_k<HD, 4>), dim3((unsigned)(caches * p.w_blocks)), dim3(1024), 4 * sizeof(apt::WeighLds), st, p);
  } else {
    hipLaunchKernelGGL((apt::weigh_k<HD, 1>), dim3((unsigned)(caches * p.w_blocks)), dim3(256), sizeof(apt::WeighLds), st, p);
  }
  VM_LAUNCH_CHECK();
  return VM_OK;
}

template <int HD>
int launch_tile(AttnPagedP& p, hipStream_t st) {
  static std::atomic<uint64_t> set{0};
  if (!allow_lds((const void*)apt::tile_k<HD>, apt::RING_LDS, set)) return VM_ERR_LAUNCH;
  hipLaunchKernelGGL(apt::tile_k<HD>, dim3((unsigned)tile_grid(p)), dim3(apt::NW * 64), apt::RING_LDS, st, p);
  if (p.n_split > 1) hipLaunchKernelGGL(attn_paged_join_k<HD>, dim3(p.join_blocks, p.c.n_kv_heads, p.n_seq), dim3(256), 0, st, p);
  VM_LAUNCH_CHECK();
  return p.w_out && p.max_kv > 0 ? launch_weigh<HD>(p, st) : VM_OK;
}

}  // namespace

extern "C" {

int vm_attn_paged_workspace(const vm_attn_paged_args* args_host, int64_t* bytes_host) {
  AttnPagedP p;
  if (!bytes_host) return VM_ERR_BAD_ARG;
  const int rc = fill(args_host, p);
  if (rc != VM_OK) return rc;
  *bytes_host = plan(p, args_host->cache.head_dim).bytes;
  return VM_OK;
}

int vm_attn_paged_bf16(const vm_attn_paged_args* args_host, void* stream) {
  AttnPagedP p;
  const int rc = fill(args_host, p);
  if (rc != VM_OK) return rc;
  // the weights of many rows need the queries once more
  if (p.w_out && p.n_rows > 0 && args_host->out == args_host->q) return VM_ERR_BAD_ARG;
  hipStream_t st = (hipStream_t)stream;
  const int hd = args_host->cache.head_dim;
  const Plan a = plan(p, hd);
  if (a.bytes > 0 && (!args_host->workspace || args_host->workspace_bytes < a.bytes || misaligned16(args_host->workspace))) return VM_ERR_BAD_ARG;
  if (p.n_seq == 0) return VM_OK;
  char* ws = (char*)args_host->workspace;
  if (a.split && p.max_q > 0) {
    if (p.n_split > 1) p.part = (float*)(ws + a.part);
    if (p.w_out) { p.s_ws = (float*)(ws + a.s_ws); }
    if (hd == 128) launch_split<128>(p, st);
    else if (hd == 64) launch_split<64>(p, st);
    else launch_split<32>(p, st);
    VM_LAUNCH_CHECK();
    return VM_OK;
  }
  if (p.max_q > 0) {
    if (p.n_wg < 0) return VM_ERR_UNSUPPORTED;
    if (p.n_split > 1) p.part = (float*)(ws + a.part);
    if (hd == 128) return launch_tile<128>(p, st);
    if (hd == 64) return launch_tile<64>(p, st);
    return launch_tile<32>(p, st);
  }
  return p.w_out && p.max_kv > 0 ? launch_weigh<32>(p, st) : VM_OK;      // no new token anywhere: the weights stay what they are
}

}  // extern "C"
