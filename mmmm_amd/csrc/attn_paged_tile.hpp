// attn_paged.hip, the form for many query rows: 32 query rows per wave on v_mfma_f32_32x32x16_bf16, 8 waves = 256 rows per workgroup.
//
// The pipeline is the one of attn32_fwd.hpp (scores transposed so that a query sits on the MFMA column and its softmax is in-lane; four
// clusters per 64-key tile between raw barriers, the two waves of a SIMD one cluster apart; K and V by LDS-DMA into three-slot rings retired
// by counted vmcnt). What the cache changes:
//  * a 64-key tile may lie in up to four pages. The unit of the DMA is the 8-row group a wave stages: it never crosses a page (page size
//    >= 16), its page number is one scalar load, fetched two tiles ahead, and the buffer descriptor is made for exactly that group — base in 64
//    bits, extent = the rows that exist — so rows behind the last token and pages that are not there arrive as zeros without a compare;
//  * rows are (query, head of the group) pairs: grouped heads fill the tile together and read K and V once;
//  * the causal limit of a row is any token, not its own position: the last two tiles of a wave may need the mask, and a row may see nothing
//    (scores at -inf, a base of 0 while the maximum is -inf);
//  * with fewer than one workgroup per CU the keys are split over workgroups too (partial results joined by attn_paged_join_k);
//  * V^T fragments are read in two assembly statements of 16 ds_read_b64_tr_b16 that end in their own wait.
// Matrix-bound in theory (4 hd operations per visible pair), in fact by the softmax between the two products and the barriers between the clusters:
// 4 x 4609 tokens, 32 heads of width 128: 585-603 us on three boxes, 785-810 TFLOP/s of the visible pairs, matrix pipes busy 0.39 of the time, waves
// waiting 0.38 of theirs; 512 tokens over 8704: 96 us with the join, 740 TFLOP/s. Measured and not taken: 64 rows per wave and four waves (half the LDS reads, but the
// registers of two row sets: 680 us beside 583-607); V read untransposed, which would be wrong, gains 3 % — its transposed reads are not what costs.
#pragma once
#include <type_traits>
#include "attn32_tile.hpp"

namespace apt {

using a32::TILE;
using a32::NW;
using a32::NS;
using a32::SLAB;
using a32::SLAB_PITCH;
using a32::RING_LDS;
constexpr int QB = NW * 32;                     // query rows per workgroup
// The running maximum is raised with every tile that exceeds it, so a row's largest probability is exactly 1 and its bf16 rounding nothing. Raising it
// only beyond a step of 5 (log2 units) would spare most of the rescaling, but then the largest probability is any number up to 2^5 and rounded like the
// others: error against 64 bits 0.0021 of the output beside 0.0018 (512 new over 8704; the same in 32 bits throughout: 0.0017), for 100 beside 107 us,
// and 551 beside 585 us on 4 x 4609.

typedef __attribute__((address_space(3))) void* lds_vptr_t;

// eight transposed fragments, complete on return (offsets: 4096 per 16 rows, 512 per 32 columns)
template <int O0, int O1, int O2, int O3, int O4, int O5, int O6, int O7>
__device__ __forceinline__ void ld_tr8(unsigned a, unsigned b, bf16x8_t* f) {
  s16x4_t l0, l1, l2, l3, l4, l5, l6, l7, h0, h1, h2, h3, h4, h5, h6, h7;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16 offset:%18\n\tds_read_b64_tr_b16 %8, %17 offset:%18\n\t"
      "ds_read_b64_tr_b16 %1, %16 offset:%19\n\tds_read_b64_tr_b16 %9, %17 offset:%19\n\t"
      "ds_read_b64_tr_b16 %2, %16 offset:%20\n\tds_read_b64_tr_b16 %10, %17 offset:%20\n\t"
      "ds_read_b64_tr_b16 %3, %16 offset:%21\n\tds_read_b64_tr_b16 %11, %17 offset:%21\n\t"
      "ds_read_b64_tr_b16 %4, %16 offset:%22\n\tds_read_b64_tr_b16 %12, %17 offset:%22\n\t"
      "ds_read_b64_tr_b16 %5, %16 offset:%23\n\tds_read_b64_tr_b16 %13, %17 offset:%23\n\t"
      "ds_read_b64_tr_b16 %6, %16 offset:%24\n\tds_read_b64_tr_b16 %14, %17 offset:%24\n\t"
      "ds_read_b64_tr_b16 %7, %16 offset:%25\n\tds_read_b64_tr_b16 %15, %17 offset:%25\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(l0), "=&v"(l1), "=&v"(l2), "=&v"(l3), "=&v"(l4), "=&v"(l5), "=&v"(l6), "=&v"(l7), "=&v"(h0), "=&v"(h1), "=&v"(h2), "=&v"(h3), "=&v"(h4),
        "=&v"(h5), "=&v"(h6), "=&v"(h7)
      : "v"(a), "v"(b), "n"(O0), "n"(O1), "n"(O2), "n"(O3), "n"(O4), "n"(O5), "n"(O6), "n"(O7)
      : "memory");
  const s16x4_t lo[8] = {l0, l1, l2, l3, l4, l5, l6, l7}, hi[8] = {h0, h1, h2, h3, h4, h5, h6, h7};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo[i], hi[i], 0, 1, 2, 3, 4, 5, 6, 7));
}
template <int O0, int O1, int O2, int O3>
__device__ __forceinline__ void ld_tr4(unsigned a, unsigned b, bf16x8_t* f) {
  s16x4_t l0, l1, l2, l3, h0, h1, h2, h3;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%10\n\tds_read_b64_tr_b16 %4, %9 offset:%10\n\t"
      "ds_read_b64_tr_b16 %1, %8 offset:%11\n\tds_read_b64_tr_b16 %5, %9 offset:%11\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:%12\n\tds_read_b64_tr_b16 %6, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %3, %8 offset:%13\n\tds_read_b64_tr_b16 %7, %9 offset:%13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(l0), "=&v"(l1), "=&v"(l2), "=&v"(l3), "=&v"(h0), "=&v"(h1), "=&v"(h2), "=&v"(h3)
      : "v"(a), "v"(b), "n"(O0), "n"(O1), "n"(O2), "n"(O3)
      : "memory");
  const s16x4_t lo[4] = {l0, l1, l2, l3}, hi[4] = {h0, h1, h2, h3};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo[i], hi[i], 0, 1, 2, 3, 4, 5, 6, 7));
}
// the V^T fragments of a tile: f[m * ND + b] = rows 16 m .. + 15, columns 32 b .. + 31
template <int ND>
__device__ __forceinline__ void ld_v(unsigned a, unsigned b, bf16x8_t* f) {
  if constexpr (ND == 4) {
    ld_tr8<0, 512, 1024, 1536, 4096, 4608, 5120, 5632>(a, b, f);
    ld_tr8<8192, 8704, 9216, 9728, 12288, 12800, 13312, 13824>(a, b, f + 8);
  } else if constexpr (ND == 2) {
    ld_tr8<0, 512, 4096, 4608, 8192, 8704, 12288, 12800>(a, b, f);
  } else {
    ld_tr4<0, 4096, 8192, 12288>(a, b, f);
  }
}

// maximum of a lane's 32 scores. Assembly: fmaxf() of MFMA results costs a canonicalising instruction per operand. The statement waits out
// the matrix pipe itself (v_mfma_f32_32x32x16: 16 passes) and its operands are read only behind the wait.
__device__ __forceinline__ float max32(const f32x16_t (&S)[2]) {
  float m0, m1, m2, m3;
  asm("s_nop 15\n\ts_nop 3\n\t"
      "v_max3_f32 %0, %4, %5, %6\n\tv_max3_f32 %1, %8, %9, %10\n\tv_max3_f32 %2, %12, %13, %14\n\tv_max3_f32 %3, %16, %17, %18\n\t"
      "v_max_f32 %0, %0, %7\n\tv_max_f32 %1, %1, %11\n\tv_max_f32 %2, %2, %15\n\tv_max_f32 %3, %3, %19"
      : "=&v"(m0), "=&v"(m1), "=&v"(m2), "=&v"(m3)
      : "v"(S[0][0]), "v"(S[0][1]), "v"(S[0][2]), "v"(S[0][3]), "v"(S[0][4]), "v"(S[0][5]), "v"(S[0][6]), "v"(S[0][7]), "v"(S[0][8]), "v"(S[0][9]),
        "v"(S[0][10]), "v"(S[0][11]), "v"(S[0][12]), "v"(S[0][13]), "v"(S[0][14]), "v"(S[0][15]));
  asm("v_max3_f32 %0, %0, %4, %5\n\tv_max3_f32 %1, %1, %8, %9\n\tv_max3_f32 %2, %2, %12, %13\n\tv_max3_f32 %3, %3, %16, %17\n\t"
      "v_max3_f32 %0, %0, %6, %7\n\tv_max3_f32 %1, %1, %10, %11\n\tv_max3_f32 %2, %2, %14, %15\n\tv_max3_f32 %3, %3, %18, %19\n\t"
      "v_max3_f32 %0, %0, %1, %2\n\tv_max_f32 %0, %0, %3"
      : "+v"(m0), "+v"(m1), "+v"(m2), "+v"(m3)
      : "v"(S[1][0]), "v"(S[1][1]), "v"(S[1][2]), "v"(S[1][3]), "v"(S[1][4]), "v"(S[1][5]), "v"(S[1][6]), "v"(S[1][7]), "v"(S[1][8]), "v"(S[1][9]),
        "v"(S[1][10]), "v"(S[1][11]), "v"(S[1][12]), "v"(S[1][13]), "v"(S[1][14]), "v"(S[1][15]));
  return m0;
}

// end of a cluster (attn32_tile.hpp) with any count
template <int VM>
__device__ __forceinline__ void cluster_end() {
  if constexpr (VM >= 0) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(VM) : "memory");
  else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

// what a wave needs to stage its 8-row group of a tile
template <int HD>
struct Stager {
  static constexpr int PW = HD > 64 ? 2 : 1;     // DMA instructions per group: 64 columns each
  int voff[PW];                                  // byte offset inside the group, or out of every descriptor's reach
  int64_t head;                                  // element offset of (kv head, row 0) inside a page
  __device__ __forceinline__ void init(int hk, int shift, int wave, int lane) {
    const int row = 8 * wave + ((lane >> 2) & 7);
    head = ((int64_t)hk << shift) * HD;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int chunk = 4 * (2 * i + (lane >> 5)) + ((lane & 3) ^ ((row >> 2) & 3));      // the image's XOR goes onto the source chunk
      voff[i] = chunk * 8 < HD ? ((lane >> 2) & 7) * HD * 2 + chunk * 16 : 0x7FFFFFF0;
    }
  }
  // where the wave's group of tile t lies in both pools, and how many bytes of it are there
  struct Group { uint64_t at; int bytes; };
  __device__ __forceinline__ Group group(const PagedKV& c, int page, int t, int kv_end, int wave) const {
    const int tok = 64 * t + 8 * wave;
    const bool ok = page_ok(page, c.n_pages);
    const int there = max(0, min(8, kv_end - tok)), rows = ok ? there : 0;      // selects, no branch
    const uint64_t at = (uint64_t)(unsigned)(ok ? page : 0) * (uint64_t)c.ld_page + (uint64_t)head + (unsigned)((tok & c.mask) * HD);
    return {at * 2, __builtin_amdgcn_readfirstlane(rows * HD * 2)};
  }
  __device__ __forceinline__ void stage(const unsigned short* pool, const Group& g, char* tile, int wave) const {
    const uint64_t at = (uint64_t)pool + g.at;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)at), hi = __builtin_amdgcn_readfirstlane((unsigned)(at >> 32));
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(((uint64_t)hi << 32) | lo), 0, g.bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < PW; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_vptr_t)(tile + (2 * wave + i) * 1024), 16, voff[i], 0, 0, 0);
  }
};

template <int HD>
__global__ __launch_bounds__(NW * 64, 2) void tile_k(const AttnPagedP p) {
  typedef Stager<HD> St;
  constexpr int KS = HD / 16;                 // k-steps of the score product
  constexpr int ND = HD / 32;                 // 32-row d-tiles of O^T
  constexpr int PW = St::PW;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5;
  // ---- which tile. Workgroups id and id + 8 share an XCD (one L2 each): every XCD takes a contiguous piece of the list, in which the samples
  // of a kv head lie side by side (few caches: spread them instead). Long lists go cache by cache, longest row tile first, so that the tiles
  // of one cache meet in one L2; lists of a few rounds go row tile by row tile, the long ones of all caches first, so that the rounds end
  // together.
  int lin;
  {
    const int id = blockIdx.x, xcd = id & 7, slot = id >> 3, caches = p.n_seq * p.c.n_kv_heads;
    lin = id;
    if (caches >= 16 && p.n_wg <= 1024) {
      const int share = (caches + 7) >> 3, first = xcd * share, mine = max(0, min(share, caches - first)) * p.n_split;
      if (slot >= mine * p.n_tiles) return;
      const int tl = slot / mine, q = slot - tl * mine;
      lin = ((first + q / p.n_split) * p.n_tiles + tl) * p.n_split + q % p.n_split;
    } else if (caches >= 16) {
      const int share = (p.n_wg + 7) >> 3;
      if (slot >= share) return;
      lin = xcd * share + slot;
    }
    if (lin >= p.n_wg) return;
  }
  const int split = lin % p.n_split, rest = lin / p.n_split;
  const int tile = p.n_tiles - 1 - rest % p.n_tiles, hs = rest / p.n_tiles;
  const int b = hs % p.n_seq, hk = hs / p.n_seq;
  const SeqInfo s = seq_info(p, b);
  const int R = min(s.nq, p.max_q) * p.G, row0 = tile * QB;
  if (row0 >= R) return;
  const int past = s.len - s.nq;
  const int qw = row0 + wave * 32;                                 // this wave's first row
  const bool wave_live = qw < R;
  const int r = qw + (lane & 31);
  const bool live = r < R;
  const int qi = live ? r / p.G : 0, h = hk * p.G + (live ? r - qi * p.G : 0);
  const int prow = live ? phys_row(p, s.p0 + qi) : -1;
  const int lim = live ? past + qi : -1;                           // last token the row sees (may be negative: none)
  const int lim_lo = past + min(qw, R - 1) / p.G, lim_hi = past + min(qw + 31, R - 1) / p.G;
  const int kv_end = max(0, past + (min(row0 + QB, R) - 1) / p.G + 1);
  const int nt_all = (kv_end + 63) / 64, per = (nt_all + p.n_split - 1) / p.n_split;
  const int t0 = min(split * per, nt_all), t1 = min(t0 + per, nt_all), nt = t1 - t0;
  const int t_w = wave_live && lim_hi >= 0 ? min(t1, lim_hi / 64 + 1) : t0;      // tiles [t0, t_w) are this wave's
  const bool late = wave >= NW / 2;

  // the range's entries in the table, 64 of them at once: asked for here, looked at behind the first tiles' DMA
  const int e0 = nt > 0 ? 64 * t0 >> p.c.shift : 0, e1 = nt > 0 ? (min(64 * t1, kv_end) - 1) >> p.c.shift : 0;
  const int entry = p.c.table[b * p.c.ld_table + min(e0 + lane, e1)];

  bf16x8_t qf[KS];
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    i32x4_t v = {0, 0, 0, 0};
    if (prow >= 0) v = *reinterpret_cast<const i32x4_t*>(p.q + prow * p.ldq + h * HD + 16 * k + 8 * hf);
    qf[k] = __builtin_bit_cast(bf16x8_t, v);
  }
  f32x16_t o[ND];
#pragma unroll
  for (int b2 = 0; b2 < ND; ++b2)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[b2][e] = 0.f;
  const float sc = p.scale * LOG2E;
  int strange = 0x7FFFFFFF;                                        // first tile in which a value that is not finite was taken as zero
  float msc = -INFINITY, base = 0.f, l_run = 0.f;                  // running maximum (log2 domain), what is subtracted, this half's sum

  const table_ptr table = table_of(p.c, b);
  if (nt > 0) {
    // the page of this wave's group of tile t, read two tiles before the first use, so that the scalar load is never waited for
    auto page_of = [&](int t) -> int { return table_at(table, __builtin_amdgcn_readfirstlane(min(64 * t + 8 * wave, kv_end - 1) >> p.c.shift)); };
    char* const kring = smem;
    char* const vring = smem + NS * TILE;
    St st;
    st.init(hk, p.c.shift, wave, lane);
    // DMA order per wave (PW instructions a group): K(0) V(0) V(1) K(1); c0(u) issues V(u+2), c1(u) issues K(u+2). At the end of c0(u) V(u)
    // must have landed (V(u+1) K(u+1) V(u+2) may fly: vmcnt(3 PW)), at the end of c2(u) K(u+1) (V(u+2) K(u+2): vmcnt(2 PW)).
    // the queries were asked for before the tiles: they have arrived when the first of those is waited for (said here, so that no wait for them
    // stands inside the loop)
    auto arrived = [&]() {
#pragma unroll
      for (int k = 0; k < KS; ++k) asm volatile("" : "+v"(qf[k]));
    };
    const int pga = page_of(t0), pgb = page_of(t0 + 1);
    int pgc = page_of(t0 + 2);
    asm volatile("" : "+s"(pgc));                                  // (no page number is on its way into the loop: nothing there waits for one)
    typename St::Group grp = st.group(p.c, pga, t0, kv_end, wave);
    st.stage(p.c.k, grp, kring, wave);
    st.stage(p.c.v, grp, vring, wave);
    if (nt > 1) {
      grp = st.group(p.c, pgb, t0 + 1, kv_end, wave);
      st.stage(p.c.v, grp, vring + TILE, wave);
      st.stage(p.c.k, grp, kring + TILE, wave);
      arrived();
      cluster_end<3 * PW>();
    } else {
      arrived();
      cluster_end<0>();
    }
    if (late) cluster_end<-1>();
    bool bad = !page_ok(entry, p.c.n_pages);
    for (int i = e0 + 64 + lane; i <= e1; i += 64) bad |= !page_ok(p.c.table[b * p.c.ld_table + i], p.c.n_pages);
    const bool gaps = __builtin_amdgcn_ballot_w64(bad) != 0;       // some page of the range is not there
    const char* const kb0 = kring + a32::row_base(lane, 0);
    const char* const kb1 = kring + a32::row_base(lane, 1);
    const unsigned vbA = (unsigned)(size_t)(vring + a32::tr_base(lane, 0)), vbB = (unsigned)(size_t)(vring + a32::tr_base(lane, 1));
    f32x16_t S[2];
    bf16x8_t kv[(4 * ND > 2 * KS) ? 4 * ND : 2 * KS];              // the K fragments of a tile, then its V fragments
    int s0 = 0, s1 = TILE, s2 = 2 * TILE;
    for (int u = 0; u < nt; ++u) {
      const int t = t0 + u;
      const bool on = t < t_w;
      const bool more1 = u + 1 < nt, more2 = u + 2 < nt;
      const int pgd = page_of(t + 3);                              // (here it arrives under the LDS reads, whose wait is its wait)
      // ---- c0: K fragments -> registers; DMA of V(u+2)
      if (on) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) kv[kt * KS + ks] = a32::ld_row(((ks & 1) ? kb1 : kb0) + s0, 8192 * kt + 512 * (ks >> 1));
      }
      if (more2) {
        grp = st.group(p.c, pgc, t + 2, kv_end, wave);
        st.stage(p.c.v, grp, vring + s2, wave);
      }
      if (more2) cluster_end<3 * PW>(); else if (more1) cluster_end<2 * PW>(); else cluster_end<0>();
      // ---- c1: S^T = K Q^T; DMA of K(u+2)
      if (on) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          f32x16_t acc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) acc = a32::mfma32(kv[kt * KS + ks], qf[ks], acc);
          S[kt] = acc;
        }
      }
      if (more2) st.stage(p.c.k, grp, kring + s2, wave);
      pgc = pgd;
      cluster_end<-1>();
      // ---- c2: V fragments -> registers, mask, maximum, rescale
      if (on) {
        ld_v<ND>(vbA + s0, vbB + s0, kv);
        const int kv0 = 64 * t;
        if (__builtin_expect(kv0 + 63 > lim_lo || gaps, 0)) {
          bool ok[4] = {true, true, true, true};                   // 16 keys of one page each
          if (gaps) {
#pragma unroll
            for (int i = 0; i < 4; ++i) ok[i] = page_ok(table_at(table, __builtin_amdgcn_readfirstlane(min(kv0 + 16 * i, kv_end - 1) >> p.c.shift)), p.c.n_pages);
          }
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              S[kt][e] = ok[2 * kt + (e >> 3)] && kv0 + 32 * kt + acc_row(e, hf) <= lim ? S[kt][e] : -INFINITY;
          unsigned most = 0;
#pragma unroll
          for (int i = 0; i < 4 * ND; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) most = max2(most, __builtin_bit_cast(u32x4_t, kv[i])[w]);
          if (__builtin_expect(__builtin_amdgcn_ballot_w64(none_finite2(most)) != 0, 0)) {
            strange = min(strange, t);
#pragma unroll
            for (int i = 0; i < 4 * ND; ++i) {
              u32x4_t x = __builtin_bit_cast(u32x4_t, kv[i]);
#pragma unroll
              for (int w = 0; w < 4; ++w) x[w] = finite2(x[w]);
              kv[i] = __builtin_bit_cast(bf16x8_t, x);
            }
          }
        }
        float ma = max32(S), mb = ma;
        a32::swap_halves(ma, mb);
        const float mxs = fmaxf(ma, mb) * sc;
        if (__builtin_amdgcn_ballot_w64(mxs > msc) != 0) {
          const float mn = fmaxf(msc, mxs);
          base = mn == -INFINITY ? 0.f : mn;
          const float alpha = fast_exp2(msc - base);               // 0 while nothing was seen
          msc = mn;
          l_run *= alpha;
#pragma unroll
          for (int b2 = 0; b2 < ND; ++b2)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[b2][e] *= alpha;
        }
      }
      if (more2) cluster_end<2 * PW>(); else cluster_end<0>();
      // ---- c3: O^T += V^T P^T, the next 16 keys' exponentials beside it
      if (on) {
        float rs0 = 0.f, rs1 = 0.f;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          u16x8_t w;
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const int e = 8 * (m & 1) + j;
            const float e0 = fast_exp2(fmaf(S[m >> 1][e], sc, -base)), e1 = fast_exp2(fmaf(S[m >> 1][e + 1], sc, -base));
            w[j] = f2bf(e0);
            w[j + 1] = f2bf(e1);
            rs0 += e0;
            rs1 += e1;
          }
          const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, w);
#pragma unroll
          for (int b2 = 0; b2 < ND; ++b2) o[b2] = a32::mfma32(kv[m * ND + b2], pf, o[b2]);
        }
        l_run += rs0 + rs1;
      }
      cluster_end<-1>();
      { const int x = s0; s0 = s1; s1 = s2; s2 = x; }
    }
    if (!late) cluster_end<-1>();                // every LDS read is over: the slabs may overlay the rings
  }

  if (!wave_live) return;
  if (__builtin_expect(strange < t_w, 0)) {
    for (int j = 64 * strange; j < min(64 * t_w, kv_end); ++j) {
      const int page = table[__builtin_amdgcn_readfirstlane(j >> p.c.shift)];
      if (!page_ok(page, p.c.n_pages)) continue;
      const int64_t at = page_row(page, p.c.ld_page, hk, j & p.c.mask, p.c.shift, HD);
      bool odd = false;
#pragma unroll 1
      for (int c = 0; c < HD / 8; ++c) {
        const u16x4_t v = *reinterpret_cast<const u16x4_t*>(p.c.v + at + 8 * c + 4 * hf);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (v[e] & 0x7F80) == 0x7F80;
      }
      if (__builtin_amdgcn_ballot_w64(odd) == 0) continue;
      float dot = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u16x8_t kr = *reinterpret_cast<const u16x8_t*>(p.c.k + at + 16 * ks + 8 * hf), qr = __builtin_bit_cast(u16x8_t, qf[ks]);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(bf2f(kr[e]), bf2f(qr[e]), dot);
      }
      float da = dot, db = dot;
      a32::swap_halves(da, db);
      const float w = fast_exp2(fmaf(da + db, sc, -base));
#pragma unroll
      for (int b2 = 0; b2 < ND; ++b2)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const u16x4_t v = *reinterpret_cast<const u16x4_t*>(p.c.v + at + 32 * b2 + 8 * g4 + 4 * hf);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j <= lim && (v[e] & 0x7F80) == 0x7F80) o[b2][4 * g4 + e] = fmaf(w, bf2f(v[e]), o[b2][4 * g4 + e]);
        }
    }
  }
  {
    float a = l_run, c = l_run;
    a32::swap_halves(a, c);
    l_run = a + c;
  }
  if (p.n_split > 1) {
    if (!live) return;
    float* part = p.part + ((((int64_t)b * p.c.n_kv_heads + hk) * p.s_rows + r) * p.n_split + split) * (HD + 4);
    if (hf == 0) { part[0] = msc; part[1] = l_run; }
#pragma unroll
    for (int b2 = 0; b2 < ND; ++b2)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<f32x4_t*>(part + 4 + 32 * b2 + 8 * g4 + 4 * hf) = (f32x4_t){o[b2][4 * g4], o[b2][4 * g4 + 1], o[b2][4 * g4 + 2], o[b2][4 * g4 + 3]};
    return;
  }
  const bool some = !(l_run == 0.f);
  const float inv = some ? 1.f / l_run : 0.f;
  if (live && hf == 0) p.lse[h * p.ld_lse + s.p0 + qi] = some && prow >= 0 ? (msc + log2f(l_run)) * LN2 : -INFINITY;
  // O^T registers -> this wave's slab [32 rows][HD], then whole rows out
  char* slab = smem + wave * SLAB;
#pragma unroll
  for (int b2 = 0; b2 < ND; ++b2)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const u16x4_t w = {f2bf(o[b2][4 * g4] * inv), f2bf(o[b2][4 * g4 + 1] * inv), f2bf(o[b2][4 * g4 + 2] * inv), f2bf(o[b2][4 * g4 + 3] * inv)};
      *reinterpret_cast<u16x4_t*>(slab + (lane & 31) * SLAB_PITCH + (32 * b2 + 8 * g4 + 4 * hf) * 2) = w;
    }
  __builtin_amdgcn_wave_barrier();
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  constexpr int CPR = HD / 8;                    // 16-byte chunks per row
  const int64_t mine = prow >= 0 ? prow * p.ldo + h * HD : -1;     // where this lane's row goes
#pragma unroll
  for (int i = lane; i < 32 * CPR; i += 64) {
    const int rr = i / CPR, ch = i - rr * CPR;
    const int64_t at = __shfl(mine, rr, 64);
    if (at >= 0) *reinterpret_cast<i32x4_t*>(p.out + at + ch * 8) = *reinterpret_cast<const i32x4_t*>(slab + rr * SLAB_PITCH + ch * 16);
  }
}

// ----------------------------------------------------------------------------- received weights of a chunk
// w[j] += sum over the query rows of exp2(s q_r . k_j - l2_r): the scores once more (2 hd of the 4 hd operations of the attention itself;
// keeping them would be 4 bytes per row and token). A wave keeps 32 tokens as B operands in registers (straight from the page) and the
// workgroup's four waves walk the rows that see them, 64 at a time through LDS as A operands: a token sits on the lane, so its sum over the
// rows is in-lane — per tile first, then onto the running sum, halves last: a fixed order. Row numbers and lse are fetched two tiles ahead, the
// rows one tile ahead through registers. Bound by the latency of a tile (eight of them in a row for the earliest tokens of 456) and the vector work
// on the scores beside it: 8 x 456 tokens, 32 heads of width 128: 22 us (34 us at three workgroups per CU with the rows waited for in front of the
// products; 60 us with the rows straight from memory as B operands of each wave, bound by the L1's line rate).
// Few caches with many query rows (grouped heads) leave most CUs idle: there a workgroup has four such sets of four waves, each with every fourth
// tile of rows, and their sums meet in LDS, in order (5 x 433 tokens, 4 heads per kv head of 3, width 32: with the attention 50 -> 34 us;
// 4 x 2000, 8 heads for one, width 128: 369 -> 229; from 500 workgroups on
// it gains nothing).
struct WeighLds {
  char q[2][TILE];
  float l2[3][64];
  int lim[3][64];
  int64_t off[3][64];                                              // element offset of the row's query (no such row: 0, any query)
  int gap[4];                                                      // one of the tile's rows is no row
};

template <int HD, int SETS>
__global__ __launch_bounds__(256 * SETS, 4) void weigh_k(const AttnPagedP p) {
  constexpr int KS = HD / 16, CPR = HD / 8, NQ = CPR / 4;          // 16-byte chunks per row, chunks per thread and tile
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int set = SETS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  WeighLds& L = reinterpret_cast<WeighLds*>(smem)[set];
  const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hf = lane >> 5;
  // 128 tokens of one cache. The blocks of a cache differ in work (early tokens are seen by more rows) and share its queries: every XCD takes whole
  // caches where there are enough of them (blocks dealt out in order would give one XCD the early blocks of all: 8 x 456 with the attention 69 beside 68 us).
  int blk, hs;
  {
    const int id = blockIdx.x, caches = p.n_seq * p.c.n_kv_heads, slot = id >> 3;
    blk = caches >= 16 ? slot % p.w_blocks : id % p.w_blocks;
    hs = caches >= 16 ? (slot / p.w_blocks) * 8 + (id & 7) : id / p.w_blocks;
    if (hs >= caches) return;
  }
  const int hk = hs % p.c.n_kv_heads, b = hs / p.c.n_kv_heads;
  const SeqInfo s = seq_info(p, b);
  const int n = min(s.len, p.w_cols), jw = blk * 128, j0 = jw + wave * 32, j = j0 + (lane & 31);
  if (jw >= n) return;
  const int R = min(s.nq, p.max_q) * p.G, past = s.len - s.nq;
  bool there = false;
  bf16x8_t kf[KS];
  {
    int page = -1;
    if (j < n) page = p.c.table[b * p.c.ld_table + (j >> p.c.shift)];
    there = page_ok(page, p.c.n_pages);
    // (a token that is not there reads row 0 of the pool: its column of the product is thrown away)
    const unsigned short* kr = p.c.k + (there ? page_row(page, p.c.ld_page, hk, j & p.c.mask, p.c.shift, HD) : 0) + 8 * hf;
#pragma unroll
    for (int k = 0; k < KS; ++k) kf[k] = *reinterpret_cast<const bf16x8_t*>(kr + 16 * k);
  }
  const float sc = p.scale * LOG2E;
  float sum = 0.f;
  const int rs = min(max(0, jw - past), p.max_q) * p.G / 64 * 64;                // the first tile with a row that sees one of these tokens
  const int tiles = R > rs ? (R - rs + 63) / 64 : 0, mine = (tiles - set + SETS - 1) / SETS, steps = (tiles + SETS - 1) / SETS;
  auto row0 = [&](int u) { return rs + 64 * (set + SETS * u); };    // of this set's u-th tile
  struct Info { int r, i, h, row; float lse; };                    // as loaded: looked at when it is put into LDS, a tile later
  auto info = [&](int r) -> Info {
    Info x;
    x.r = r;
    const int rr = min(r, R - 1);
    x.i = p.G == 1 ? rr : rr / p.G;
    x.h = hk * p.G + rr - x.i * p.G;
    x.row = s.p0 + x.i;
    if (p.row_of_pos) x.row = p.row_of_pos[s.p0 + x.i];
    x.lse = p.lse[x.h * p.ld_lse + s.p0 + x.i];
    return x;
  };
  auto put = [&](int slot, const Info& x) {
    const bool ok = x.r < R && (unsigned)x.row < (unsigned)p.n_rows && x.lse != -INFINITY;
    L.off[slot][tid] = ok ? x.row * p.ldq + x.h * HD : 0;
    L.l2[slot][tid] = ok ? x.lse * LOG2E : INFINITY;               // no such row: exp2(. - inf) = 0
    L.lim[slot][tid] = ok ? past + x.i : -1;
    const bool gap = __builtin_amdgcn_ballot_w64(!ok) != 0;
    if (tid == 0) L.gap[slot] = gap;
  };
  i32x4_t qv[NQ];
  auto load_q = [&](int slot) {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int c = tid + 256 * i;
      qv[i] = *reinterpret_cast<const i32x4_t*>(p.q + L.off[slot][c / CPR] + (c % CPR) * 8);
    }
  };
  auto store_q = [&](char* tile) {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int c = tid + 256 * i, row = c / CPR, ch = c % CPR;
      *reinterpret_cast<i32x4_t*>(tile + 2048 * (row >> 3) + 512 * (ch >> 2) + 64 * (row & 7) + 16 * ((ch & 3) ^ ((row >> 2) & 3))) = qv[i];
    }
  };
  if (tiles > 0) {
    if (tid < 64) {
      const Info a = info(row0(0) + tid), c = info(row0(1) + tid);
      put(0, a);
      put(1, c);
    }
    __syncthreads();
    load_q(0);
    store_q(L.q[0]);
    __syncthreads();
  }
  const int rb0 = a32::row_base(lane, 0), rb1 = a32::row_base(lane, 1);
  // 64 rows against the wave's 32 tokens; edge: some rows do not see some of the tokens, or are no rows
  auto add = [&](const char* qt, int slot, auto edge) {
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int rt = 0; rt < 2; ++rt) {                               // (not unrolled: 128 registers, four workgroups per CU)
      f32x16_t acc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) acc = a32::mfma32(a32::ld_row(qt + 8192 * rt + ((k & 1) ? rb1 : rb0), 512 * (k >> 1)), kf[k], acc);
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        const int row = 32 * rt + 8 * g4 + 4 * hf;
        const f32x4_t l2 = *reinterpret_cast<const f32x4_t*>(&L.l2[slot][row]);
        i32x4_t lim;
        if constexpr (decltype(edge)::value) lim = *reinterpret_cast<const i32x4_t*>(&L.lim[slot][row]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = fast_exp2(fmaf(acc[4 * g4 + e], sc, -l2[e]));
          if constexpr (decltype(edge)::value) part[e] += j <= lim[e] ? x : 0.f;
          else part[e] += x;
        }
      }
    }
    sum += (part[0] + part[1]) + (part[2] + part[3]);
  };
#pragma unroll
  for (int k = 0; k < KS; ++k) asm volatile("" : "+v"(kf[k]));       // they are here: no wait for them in the loop, which would be one for the rows too
  int slot = 0;
  for (int u = 0; u < steps; ++u) {
    const int next = slot == 2 ? 0 : slot + 1, third = next == 2 ? 0 : next + 1;
    Info ahead;
    if (tid < 64) ahead = info(row0(u + 2) + tid);
    if (u + 1 < mine) load_q(next);
    const char* qt = L.q[u & 1];
    const int r_last = min(row0(u) + 63, R - 1);
    if (u < mine && past + r_last / p.G >= j0) {
      if (L.gap[slot] || past + row0(u) / p.G < j0 + 31) add(qt, slot, std::true_type{});
      else add(qt, slot, std::false_type{});
    }
    if (u + 1 < mine) store_q(L.q[(u + 1) & 1]);
    if (tid < 64) put(third, ahead);
    __syncthreads();
    slot = next;
  }
  float a = sum, c = sum;
  a32::swap_halves(a, c);
  a += c;
  if constexpr (SETS > 1) {
    float* const all = reinterpret_cast<float*>(L.q);               // (the last barrier is behind the last read)
    if (hf == 0) all[tid >> 6 << 5 | (lane & 31)] = a;
    __syncthreads();
    if (set > 0) return;
    for (int i = 1; i < SETS; ++i) a += reinterpret_cast<const float*>(reinterpret_cast<WeighLds*>(smem)[i].q)[tid >> 6 << 5 | (lane & 31)];
  }
  if (hf == 0 && j < n) p.w_out[b * p.ldwo_seq + hk * p.ldwo_head + j] = p.w_in[b * p.ldw_seq + hk * p.ldw_head + j] + (there ? a : 0.f);
}

}  // namespace apt
