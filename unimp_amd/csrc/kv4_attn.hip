// Attention of one new token per row over the 4-bit pages (kv4.h): o = softmax_j(scale q k_j + slope j) v_j over the row's cached tokens j < len
// (eval_rec.py:100-110 / eval_exp.py:103-113 / eval_img_gen.py:102-111: the cached decode step inside Flamingo.generate).
//
// One wave takes one page (32 tokens) at a time, everything on the matrix pipe, K and V never unpacked in LDS:
//   scores   S^T = K Q^T on v_mfma_scale_f32_16x16x128_f8f6f4: A = the page's K codes and scale bytes AS STORED (kv4.h: a lane's operand is one 16-byte load),
//            B = the queries in its 16 columns, each 32-dim block of a query as e4m3 hi + lo under a shared power-of-two scale.  A bf16 has 8 significant bits, e4m3 four:
//            hi + lo is exact for elements down to 2^-10 of the block's largest and within 2^-17 of that one below.
//   softmax  online, base 2, lane (column c, group g) holds tokens 16 h + 4 g + e of the page; the running reference point m lies 10 above the maximum when it moves, and moves
//            only when a score exceeds it (p of the largest score is 2^-10 ... 1), so the common page has no cross-lane step and no rescale.
//   range    p times V's scale and its sums stay in fp32 for every value that a page holds: p <= 1, scale <= 2^125, and V's codes enter the product times 2^-22 (the last division takes it
//            back), so 2^21 tokens (the widest table) of 6 2^125 make less than 2^127.  Downwards a p V below 2^-94 is subnormal there.
//   o^T     += V^T P^T on v_mfma_f32_16x16x32_bf16: A = V's nibbles through v_cvt_scalef32_pk_bf16_fp4 (exact), B = p times the token's V scale, which differs per 32 dims.
//            p is split in two bf16 (16 bits kept).  The scale blocks and the two halves are COLUMNS of B where the queries leave room: with one or two queries
//            (MODE 0) every column is another (query, block, half) and a lane prepares 8 values per page instead of 64; the tile of dims 16 i ... takes the
//            columns of its block and ignores the others.  MODE 1: (query, block) columns, the halves as two products; MODE 3: (query, half) columns, a product per block;
//            MODE 2: 16 queries, block and half as products.  Measured, 64 rows x 8 key heads x 128 dims of up to 8 000 tokens (all of 8 000), TB/s of pages: MODE 0 (1 or 2 queries
//            of a key head) 5.7 (5.5), MODE 1 (4) 5.5 (5.1), MODE 3 (8) 4.9 (4.9), where MODE 2 reads 4.5 (4.85), MODE 2 (16) 4.1 (4.6).
// Bound by the bytes of the pages, 17 / 32 of a byte per element, where there are many (a large read by torch reaches 5.75 TB/s here, this 5.7; the matrix pipe is a sixth busy), else by the chain
// length -> page id -> page -> join: one row of 469 tokens x 32 heads x 80 6.6 us, ten rows 8.1.
#include <type_traits>
#include "kv4.h"
#include "unimp_hip.h"

typedef __attribute__((ext_vector_type(8))) int i32x8;
#define KV4_TEAMS 4                    // rows of a workgroup on a beam group's tails
#define KV4_AHEAD 10.f                 // log2: how far m is set above the maximum
#define KV4_V_UNIT 0x1p-22f            // V's codes in the product; sums carry it to the end

struct Kv4AttnArgs {
  const bf16* q; long q_rs, q_hs; const uint8_t* pages; long n_pages; int kv_heads; const int32_t* tables; long t_stride; int width; const int32_t* lens;
  int rows, heads; float scale; const float* alibi; bf16* o; long o_rs, o_hs; int group; const int32_t* shared;
  int G, chunk, slots;                 // query heads of a key head; pages of a workgroup on a row's own columns; its partial slots
  int chunk_p, slots_p;                // the same for the columns that a group shares (slots_p = 0: no groups)
  float* ws;                           // null: a workgroup holds a row's whole range and writes o
};

template <int D, int MODE> struct Kv4Cols {
  static constexpr int NBP = D == 64 ? 2 : 4;                                     // scale blocks as columns (three of head dim 80 in four)
  static constexpr int VAR = MODE == 0 ? 2 * NBP : MODE == 1 ? NBP : MODE == 3 ? 2 : 1, Q = 16 / VAR;
};

template <int D> struct Kv4Frag {        // one page as a wave holds it
  u32x4 k[2]; u32x4 v0; u32x4 v1; uint32_t ks; u32x2 vs;
};

// slot i of a (row, head) in the workspace: [0, slots_p) the group's columns, then the row's own; hd sums, reference point, sum of exponentials
__device__ __forceinline__ float* kv4_partial(const Kv4AttnArgs& a, int D, int row, int head, int slot) {
  return a.ws + (((long)row * a.heads + head) * (a.slots_p + a.slots) + slot) * (D + 2);
}

// prefix: the columns that a group's rows share, for the queries of all of them; else one row's own columns.  NW waves share the pages of a chunk; TEAMS > 1
// (NW = 1): every wave of the workgroup has a row of its own.
template <int D, int MODE, int NW, int TEAMS, bool ALIBI, bool prefix>
__device__ __forceinline__ void kv4_attn_part(const Kv4AttnArgs& a) {
  using P = Kv4<D>;
  using CO = Kv4Cols<D, MODE>;
  constexpr int NI = P::NI;
  static_assert(TEAMS == 1 || NW == 1, "a team of several waves needs the workgroup's barrier");
  __shared__ float team_o[TEAMS][NW][CO::Q][D], team_m[TEAMS][NW][CO::Q], team_l[TEAMS][NW][CO::Q];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int team = TEAMS > 1 ? wave : 0, w = TEAMS > 1 ? 0 : wave, tid = TEAMS > 1 ? lane : threadIdx.x;
  float (&so)[NW][CO::Q][D] = team_o[team];
  float (&sm)[NW][CO::Q] = team_m[team];
  float (&sl)[NW][CO::Q] = team_l[team];
  const int kvh = blockIdx.x, slot = blockIdx.y, G = a.G;
  const int row = prefix ? ((int)blockIdx.z - (a.rows + KV4_TEAMS - 1) / KV4_TEAMS) * a.group : (int)blockIdx.z * TEAMS + team;
  if (row >= a.rows) return;
  const int chunk = prefix ? a.chunk_p : a.chunk, slots = prefix ? a.slots_p : a.slots;
  if (slot >= slots) return;
  const int nq = prefix ? a.group * G : G;
  const int qi = col / CO::VAR, var = col % CO::VAR;
  const int my_row = prefix ? row + min(qi / G, a.group - 1) : row, my_head = kvh * G + (qi < nq ? qi % G : 0);

  // queries: lane (c, g) holds dims 16 g ... and 64 + 16 g ... of column c's query (16 dims are inside the head or behind it).  Requested first: what is waited for in
  // order must not stand behind the pages.
  bf16x8 qu[4];
  {
    const bf16* qp = a.q + (long)my_row * a.q_rs + (long)my_head * a.q_hs;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bf16* part = qp + (64 * h + 16 * g < D ? 64 * h + 16 * g : 0);        // behind the head: loaded from its start, zeroed below (a masked load would end the others' flight)
      qu[2 * h] = *(const bf16x8*)part;
      qu[2 * h + 1] = *(const bf16x8*)(part + 8);
    }
  }
  const int shared = a.group > 1 ? min(max(a.shared[row / a.group], 0) / KV4_PAGE, a.width) : 0;
  // page ids of this wave: page c0 + w + NW k in lane k; where one chunk holds the whole row they are requested beside the lengths
  int ids = -1, c0 = prefix ? 0 : shared;
  auto load_ids = [&](int pages) { if (NW * lane + w < pages && c0 + w + NW * lane < a.width) ids = a.tables[(long)row * a.t_stride + c0 + w + NW * lane]; };
  if (slots == 1) load_ids(chunk);
  const int my_len = min(max(a.lens[my_row], 0), a.width * KV4_PAGE);
  int top = my_len;                                                               // the longest of the rows here
  if (prefix) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor(top, o, 16));
  }
  top = __builtin_amdgcn_readfirstlane(top);
  const int cols = (top + KV4_PAGE - 1) / KV4_PAGE;
  const int end = prefix ? min(shared, cols) : cols, nch = (max(end - c0, 0) + chunk - 1) / chunk;      // chunks in use
  int c1 = min(c0 + chunk, end);
  if (slots > 1) {                                                                // as many as there are, equally long
    const int ch = nch > 0 ? (end - c0 + nch - 1) / nch : 0;
    c0 += slot * ch;
    c1 = min(c0 + ch, end);
    load_ids(ch);
  }
  if (c0 >= c1 && a.ws) return;                                                   // nothing here (a row without tokens still gets its zeros)
  const int n = c1 > c0 + w ? (c1 - c0 - w + NW - 1) / NW : 0;                    // pages of this wave
  if (ids >= a.n_pages) ids = -1;

  // lanes of blocks behind the head, and the upper half of a 16-wide last block, hold whatever is there (the next bytes of the page): the query is zero in those dims
  const int gk = min(g, P::NB - 1), half_block = P::BLK_LAST < 32 && gk == P::NB - 1;
  const uint32_t k_at = 512 * gk + (half_block ? 8 : 16) * col, k_step = half_block ? 128 : 256, ks_at = P::KS + 32 * gk + 2 * col;
  const uint32_t v_at = P::VOFF + 4 * (g * D + col * NI), vs_at = P::VS + 8 * P::NB * g + 8 * min(MODE == 0 ? var >> 1 : MODE == 1 ? var : col & 3, P::NB - 1);
  auto page_of = [&](int k) { return a.pages + ((long)max(__builtin_amdgcn_readlane(ids, k), 0) * a.kv_heads + kvh) * P::BYTES; };
  // every lane's loads of page k, unconditional (past the last page: that one again, from the cache), so that the number in flight is known everywhere
  auto load = [&](Kv4Frag<D>& f, int k) {
    const uint8_t* page = page_of(min(k, n - 1));
    uint32_t k_off = k_at, ks_off = ks_at, v_off = v_at, vs_off = vs_at;
    // 32-bit offsets of this block: the page's address stays scalar.  Not beside a group's columns (40 rows of 4 096 shared tokens, 80 dims: 31.7 us, without 29.6)
    if (!prefix && TEAMS == 1) asm volatile("" : "+v"(k_off), "+v"(ks_off), "+v"(v_off), "+v"(vs_off));
    typedef __attribute__((ext_vector_type(4), aligned(8))) uint32_t u32x4h;
#pragma unroll
    for (int h = 0; h < 2; ++h) f.k[h] = *(const u32x4h*)(D == 80 ? page + (k_off + k_step * h) : page + k_off + 256 * h);
    f.ks = *(const uint16_t*)(page + ks_off);
    if constexpr (D == 80) {
      typedef __attribute__((ext_vector_type(4), aligned(4))) uint32_t u32x4u;
      f.v0 = *(const u32x4u*)(page + v_off); f.v1[0] = *(const uint32_t*)(page + v_off + 16);
    } else {
      f.v0 = *(const u32x4*)(page + v_off);
      if (D == 128) f.v1 = *(const u32x4*)(page + v_off + 16);
    }
    f.vs = *(const u32x2*)(page + vs_off);                                        // of the lane's block; MODE 2: of block col & 3
  };

  Kv4Frag<D> fa, fb;
  if (n > 0) {                                                                    // in this order: the loop counts them
    load(fa, 0);
    __builtin_amdgcn_sched_barrier(0);
    load(fb, 1);
    __builtin_amdgcn_sched_barrier(0);
  }

  i32x8 qh, ql;
  int sb;
  {
    int sx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[16];
      uint32_t mx = 0;
      const bool in = qi < nq && 64 * h + 16 * g < D;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        x[j] = in ? bf2f(qu[2 * h + (j >> 3)][j & 7]) : 0.f;
        mx = max(mx, __float_as_uint(x[j]) & 0x7fffffffu);
      }
      mx = max(mx, __shfl_xor(mx, 16, 64));                                       // the other half of the 32-dim block
      const int eb = (int)(mx >> 23), s = max(eb - 7, 1);
      sx[h] = eb == 255 ? 127 : s;
      const float inv = __uint_as_float((uint32_t)(254 - s) << 23);
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        int hi = 0, lo = 0;
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[j] * inv, x[j + 1] * inv, hi, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[j + 2] * inv, x[j + 3] * inv, hi, true);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[j] * inv - __builtin_amdgcn_cvt_f32_fp8(hi, 0), x[j + 1] * inv - __builtin_amdgcn_cvt_f32_fp8(hi, 1), lo, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[j + 2] * inv - __builtin_amdgcn_cvt_f32_fp8(hi, 2), x[j + 3] * inv - __builtin_amdgcn_cvt_f32_fp8(hi, 3), lo, true);
        qh[4 * h + j / 4] = eb == 255 ? 0x7f7f7f7f : hi;                          // an infinite or NaN query: its scores are NaN
        ql[4 * h + j / 4] = eb == 255 ? 0 : lo;
      }
    }
    // the scale operand's lane (c, t) carries block t: blocks 0, 1 are the first halves of groups 0, 2; blocks 2, 3 their second halves
    const int s0 = __shfl(sx[0], (g & 1) * 32 + col, 64), s1 = __shfl(sx[1], (g & 1) * 32 + col, 64);
    sb = g < 2 ? s0 : s1;
  }
  const float sc = a.scale * 1.4426950408889634f, slope = ALIBI ? a.alibi[my_head] * 1.4426950408889634f : 0.f;

  const uint32_t lo_mask = (MODE == 0 ? var & 1 : var) ? 0xffff0000u : 0u;
  f32x4 acc[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, mu = 0.f, l = 0.f;                                         // reference point; the same, 0 while there is none; sum of this lane's tokens

  auto compute = [&](const Kv4Frag<D>& f, int k) {
    const int c = c0 + w + NW * k;
    const int vis = __builtin_amdgcn_readlane(ids, k) < 0 ? 0 : my_len - c * KV4_PAGE;      // tokens of this page that the lane's query sees
    f32x4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const i32x8 ka = {(int)f.k[h][0], (int)f.k[h][1], (int)f.k[h][2], (int)f.k[h][3], 0, 0, 0, 0};
      const int ks = h ? (int)(f.ks >> 8) : (int)f.ks;
      f32x4 z = {0.f, 0.f, 0.f, 0.f};
      z = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(ka, qh, z, 4, 0, 0, ks, 0, sb);
      s[h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(ka, ql, z, 4, 0, 0, ks, 0, sb);
    }
    uint32_t vs0 = f.vs[0], vs1 = f.vs[1];
    float x[8];
    const float at = ALIBI ? (float)(c * KV4_PAGE + 4 * g - my_len + 1) : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = s[j >> 2][j & 3] * sc;
      if (ALIBI) x[j] = fmaf(slope, at + (float)(16 * (j >> 2) + (j & 3)), x[j]);
    }
    const bool part = __any(vis < KV4_PAGE);
    if (part) {                                                                   // the last page, or a hidden one
      int g4 = 4 * g;
      asm volatile("" : "+v"(g4));                                                // keeps these comparisons from living in registers across the loop
#pragma unroll
      for (int j = 0; j < 8; ++j) if (16 * (j >> 2) + g4 + (j & 3) >= vis) x[j] = -INFINITY;
    }
    const float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    if (__any(mx > m)) {
      float t = fmaxf(mx, __shfl_xor(mx, 16, 64));
      t = fmaxf(t, __shfl_xor(t, 32, 64));
      t = fmaxf(t + KV4_AHEAD, m);
      const float r = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - t);
      m = t; mu = t == -INFINITY ? 0.f : t;
      l *= r;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] *= r;
    }
    float hi[8];
    [[maybe_unused]] float lo[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float p = __builtin_amdgcn_exp2f(x[j] - mu);
      l += p;
      // pack() drops the lower half: p itself is the high part.  MODE 0 and 3: hi is the part that this lane's column holds
      if constexpr (MODE == 0 || MODE == 3) hi[j] = p - __uint_as_float(__float_as_uint(p) & lo_mask);
      else { hi[j] = p; lo[j] = p - __uint_as_float(__float_as_uint(p) & 0xffff0000u); }
    }
    auto pack = [](float a0, float a1) { return __builtin_amdgcn_perm(__float_as_uint(a1), __float_as_uint(a0), 0x07060302u); };      // upper halves
    auto vscale = [&](uint32_t d, int j) {                                        // byte j << 23; byte 255 (not a number): infinity, 0 x infinity = NaN
      uint32_t r;
      switch (j) {
        case 0: asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0" : "=v"(r) : "v"(23), "v"(d)); break;
        case 1: asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_1" : "=v"(r) : "v"(23), "v"(d)); break;
        case 2: asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_2" : "=v"(r) : "v"(23), "v"(d)); break;
        default: asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_3" : "=v"(r) : "v"(23), "v"(d));
      }
      return __uint_as_float(r);
    };
    auto value = [&](int i) {                                                     // operand of dims 16 i + col
      const uint32_t d = i < 4 ? f.v0[i & 3] : f.v1[i & 3];
      union { bf16x2 h[4]; bf16x8 v; } u;
      u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, KV4_V_UNIT, 0);
      u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, KV4_V_UNIT, 1);
      u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, KV4_V_UNIT, 2);
      u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, KV4_V_UNIT, 3);
      return u.v;
    };
    union B { uint32_t d[4]; bf16x8 v; };
    auto hide = [&](uint32_t& d0, uint32_t& d1) {                                 // scale bytes of tokens that are not there: 0, whatever memory holds
      if (part) {
        const int n0 = min(max(vis - 4 * g, 0), 4), n1 = min(max(vis - 16 - 4 * g, 0), 4);      // of four
        d0 &= (uint32_t)((1ull << (8 * n0)) - 1); d1 &= (uint32_t)((1ull << (8 * n1)) - 1);
      }
    };
    if constexpr (MODE == 0) {
      hide(vs0, vs1);
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = hi[j] * vscale(j < 4 ? vs0 : vs1, j & 3);
      B b;
#pragma unroll
      for (int j = 0; j < 4; ++j) b.d[j] = pack(y[2 * j], y[2 * j + 1]);
#pragma unroll
      for (int i = 0; i < NI; ++i) acc[i] = MFMA16(value(i), b.v, acc[i]);
    } else if constexpr (MODE == 1) {
      hide(vs0, vs1);
      B bh, bl;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s0 = vscale(j < 2 ? vs0 : vs1, 2 * j & 3), s1 = vscale(j < 2 ? vs0 : vs1, (2 * j + 1) & 3);
        bh.d[j] = pack(hi[2 * j] * s0, hi[2 * j + 1] * s1);
        bl.d[j] = pack(lo[2 * j] * s0, lo[2 * j + 1] * s1);
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) { const bf16x8 v = value(i); acc[i] = MFMA16(v, bh.v, acc[i]); acc[i] = MFMA16(v, bl.v, acc[i]); }
    } else {
      auto block = [&](auto BLK) {                                                // four lanes hold the four blocks' scales: taken from the neighbour (quad_perm)
        constexpr int blk = decltype(BLK)::value;
        uint32_t d0 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)vs0, blk * 0x55, 0xf, 0xf, true);
        uint32_t d1 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)vs1, blk * 0x55, 0xf, 0xf, true);
        hide(d0, d1);
        B bh, bl;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float s0 = vscale(j < 2 ? d0 : d1, 2 * j & 3), s1 = vscale(j < 2 ? d0 : d1, (2 * j + 1) & 3);
          bh.d[j] = pack(hi[2 * j] * s0, hi[2 * j + 1] * s1);
          if constexpr (MODE == 2) bl.d[j] = pack(lo[2 * j] * s0, lo[2 * j + 1] * s1);
        }
#pragma unroll
        for (int i = 2 * blk; i < 2 * blk + 2; ++i) if (i < NI) {
          const bf16x8 v = value(i);
          acc[i] = MFMA16(v, bh.v, acc[i]);
          if constexpr (MODE == 2) acc[i] = MFMA16(v, bl.v, acc[i]);
        }
      };
      block(std::integral_constant<int, 0>()); block(std::integral_constant<int, 1>());
      if constexpr (P::NB > 2) block(std::integral_constant<int, 2>());
      if constexpr (P::NB > 3) block(std::integral_constant<int, 3>());
    }
  };

  for (int k = 0; k + 1 < n; k += 2) {
    compute(fa, k);
    load(fa, k + 2);
    __builtin_amdgcn_sched_barrier(0);                                            // requested before the wait for the other page
    compute(fb, k + 1);
    load(fb, k + 3);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (n & 1) compute(fa, n - 1);

  // ---- join the waves: lane (c, g) holds dims 16 i + 4 g + e of column c
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    f32x4 x = acc[i];
    if constexpr (MODE == 0 || MODE == 3) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], 1, 64);                // the two halves of p
    }
    const bool mine = MODE == 0 ? var == 2 * (i >> 1) : MODE == 1 ? var == (i >> 1) : MODE == 3 ? var == 0 : true;
    if (mine && qi < nq) *(f32x4*)&so[w][qi][16 * i + 4 * g] = x;
  }
  if (var == 0 && g == 0) { sm[w][qi] = m; sl[w][qi] = l; }
  if constexpr (TEAMS > 1) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else __syncthreads();
  for (int x = tid; x < nq * D; x += 64 * NW) {
    const int qq = x / D, d = x - qq * D;
    float M = sm[0][qq];
#pragma unroll
    for (int i = 1; i < NW; ++i) M = fmaxf(M, sm[i][qq]);
    float L = 0.f, o = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const float e = __builtin_amdgcn_exp2f(sm[i][qq] - (M == -INFINITY ? 0.f : M));       // a wave without tokens: exp2(-infinity) = 0
      L = fmaf(sl[i][qq], e, L); o = fmaf(so[i][qq][d], e, o);
    }
    const int r = prefix ? row + qq / G : row, h = kvh * G + qq % G;
    if (a.ws) {
      float* p = kv4_partial(a, D, r, h, (prefix ? 0 : a.slots_p) + slot);
      p[d] = o;
      if (d == 0) { p[D] = M; p[D + 1] = L; }
    } else {
      a.o[r * a.o_rs + h * a.o_hs + d] = f2bf(L == 0.f ? 0.f : o / L * (1.f / KV4_V_UNIT));
    }
  }
}

template <int D, int MODE, int NW, bool ALIBI>
__global__ __launch_bounds__(64 * NW, D == 64 ? 4 : 1) void kv4_attn_kernel(Kv4AttnArgs a) { kv4_attn_part<D, MODE, NW, 1, ALIBI, false>(a); }

// beam groups: the first workgroups (z) take the rows' own columns, few pages each: a wave per row; the others a group's shared columns for up to 16 queries at once,
// in the mode that their number allows (GMODE; 8 prompts x 5 beams x 32 heads x 128 behind 4 096 shared tokens: MODE 3 41.7 us, MODE 2 44.3)
template <int D, int MODE, int GMODE, bool ALIBI>
__global__ __launch_bounds__(256) void kv4_attn_group_kernel(Kv4AttnArgs a) {
  if ((int)blockIdx.z >= (a.rows + KV4_TEAMS - 1) / KV4_TEAMS) kv4_attn_part<D, GMODE, 4, 1, ALIBI, true>(a);
  else kv4_attn_part<D, MODE, 1, KV4_TEAMS, ALIBI, false>(a);
}

// joins the partials of a (row, head): PARTS groups of threads, two dims to a thread, each an online pass over every PARTS-th slot (all loads independent: one
// memory latency), then the groups in order.  3 ... 5 us, nearly all of it launch and that latency
#define KV4_MAX_SLOTS 256                                                         // of a row's own columns, and of its group's
template <int D, int PARTS>
__global__ __launch_bounds__(PARTS * D / 2) void kv4_attn_merge_kernel(Kv4AttnArgs a) {
  __shared__ float so[PARTS][D], sm[PARTS], sl[PARTS];
  const int h = blockIdx.x, row = blockIdx.y, d = threadIdx.x % (D / 2) * 2, part = threadIdx.x / (D / 2);
  const int len = min(max(a.lens[row], 0), a.width * KV4_PAGE), cols = (len + KV4_PAGE - 1) / KV4_PAGE;
  int np = 0, sh = 0;
  if (a.slots_p) {
    int top = 0;                                                                  // a group's workgroups go as far as its longest row
    const int r0 = row / a.group * a.group;
#pragma unroll
    for (int j = 0; j < 16; ++j) top = max(top, a.lens[r0 + min(j, a.group - 1)]);
    top = min(top, a.width * KV4_PAGE);
    sh = min(max(a.shared[row / a.group], 0) / KV4_PAGE, a.width);
    np = min(sh, (top + KV4_PAGE - 1) / KV4_PAGE);
  }
  // chunks in use, as kv4_attn_part counts them: ceil(columns / chunk) of equal length, so the last of them may have none left
  auto used = [](int columns, int chunk) { const int k = (columns + chunk - 1) / chunk, ch = k > 0 ? (columns + k - 1) / k : 1; return (columns + ch - 1) / ch; };
  const int n0 = a.slots_p ? used(np, a.slots_p > 1 ? a.chunk_p : max(np, 1)) : 0, own = max(cols - sh, 0), n = n0 + used(own, a.slots > 1 ? a.chunk : max(own, 1));
  const float* base = kv4_partial(a, D, row, h, 0);
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll 4
  for (int i = part; i < n; i += PARTS) {
    const float* p = base + (i < n0 ? i : a.slots_p + i - n0) * (D + 2);
    const float2 st = *(const float2*)(p + D), po = *(const float2*)(p + d);
    const float t = fmaxf(m, st.x), u = t == -INFINITY ? 0.f : t;
    const float r = __builtin_amdgcn_exp2f(m - u), e = __builtin_amdgcn_exp2f(st.x - u);    // exp2(-infinity) = 0: nothing yet, or an empty partial
    l = fmaf(st.y, e, l * r); o0 = fmaf(po.x, e, o0 * r); o1 = fmaf(po.y, e, o1 * r);
    m = t;
  }
  if constexpr (PARTS > 1) {
    so[part][d] = o0; so[part][d + 1] = o1;
    if (d == 0) { sm[part] = m; sl[part] = l; }
    __syncthreads();
    if (part) return;
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) m = fmaxf(m, sm[i]);
    const float u = m == -INFINITY ? 0.f : m;
    l = o0 = o1 = 0.f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) { const float e = __builtin_amdgcn_exp2f(sm[i] - u); l = fmaf(sl[i], e, l); o0 = fmaf(so[i][d], e, o0); o1 = fmaf(so[i][d + 1], e, o1); }
  }
  bf16* o = a.o + row * a.o_rs + h * a.o_hs + d;
  o[0] = f2bf(l == 0.f ? 0.f : o0 / l * (1.f / KV4_V_UNIT)); o[1] = f2bf(l == 0.f ? 0.f : o1 / l * (1.f / KV4_V_UNIT));
}

struct Kv4Plan { int mode, gmode, nw, chunk, slots, group, chunk_p, slots_p; int64_t floats; };
static Kv4Plan kv4_plan(const unimp_kv4_attn_desc* d) {
  Kv4Plan p;
  auto clamp = [](long x, long lo, long hi) { return (int)(x < lo ? lo : x > hi ? hi : x); };
  auto mode = [&](int nq) { const int nbp = d->hd == 64 ? 2 : 4; return nq <= 8 / nbp ? 0 : nq <= 16 / nbp ? 1 : nq <= 8 ? 3 : 2; };
  const int G = d->heads / d->kv_heads;
  const long units = (long)d->rows * d->kv_heads;
  p.mode = mode(G);
  // groups cost a merge and pay by reading the shared columns once.  Measured (us, groups | every row for itself), 32 heads x 80, pages = rows x heads x columns: 10 beams, prompt 469
  // (5 120 pages) 10.6 | 7.4, 800 (8 320) 10.5 | 9.0, 1 024 (10 560) 10.7 | 10.0, 1 300 (13 440) 11.0 | 11.3, 4 096 (41 280) 15.4 | 21.6; 40 rows, prompt 128 (6 400) 10.3 | 7.8,
  // 300 (14 080) 11.7 | 11.5, 469 (20 480) 12.5 | 14.8, 4 096 28.8 | 58.1; 128 dims, 8 x 5 beams, prompt 1 024 (42 240) 20.6 | 21.4, 4 096 41.8 | 67.5.  The two sides meet between 13 000 and
  // 20 000 pages; from 8 192 up to there a group costs up to 1.5 us, with 4 query heads to a key head 6 (8 x 4 beams x 8 key heads x 128, prompt 1 024, 8 448 pages: 14.2 | 8.1)
  p.group = d->group > 1 && d->shared_len && d->rows % d->group == 0 && d->group * G <= 16 && d->width <= 16 * KV4_MAX_SLOTS && d->width * units >= 8192 ? d->group : 1;
  p.gmode = mode(p.group * G);
  // waves of a workgroup: eight where a row is one chunk and workgroups are few (128 pairs x 47 pages 8.5 us, two chunks of four waves 10.5; 512 pairs x 128 dims of up to 2 048 tokens:
  // four waves 15.8, eight 17.8), one where rows are short and many
  p.nw = p.mode >= 2 || p.group > 1 ? 4 : units <= 256 && d->width <= (units > 64 ? 48 : 32) ? 8 : units >= 1024 && d->width <= 16 ? 1 : 4;
  // 512 (row, key head) pairs and more: whole rows up to 2 048 tokens, 48 pages above (64 rows x 8 key heads of up to 8 000 tokens: 32 pages 52.1 us, 48 48.1, 64 53.9, 96 49.7).
  // Fewer: one chunk where a wave has few pages then (no merge: 8 query heads to a key head, 20 pages: 9.3 -> 8.2 us), else as many as make 512 workgroups of at least 16 pages
  // (128 pairs x 157 pages: 4 chunks 14.6 us, 5 16.6, 8 16.5; 256 x 50: 2 chunks 12.1, 3 13.4; 32 x 63: 4 chunks 8.1, 2 10.0)
  const int most = d->width <= 64 ? 64 : 48, least = p.nw == 8 ? 64 : d->width <= 32 ? 32 : 16, parts = units < 512 ? (int)(512 / (units > 0 ? units : 1)) : 1;
  p.chunk = clamp((d->width + parts - 1) / parts, least, most);
  p.chunk_p = p.slots_p = 0;
  if (p.group > 1) {
    p.chunk = 16;
    p.chunk_p = clamp((long)d->width * (units / p.group) / 512, 16, 64);
    p.slots_p = (d->width + p.chunk_p - 1) / p.chunk_p;
  }
  // longer chunks where a row would have more partials than the merge is made for (over 393 216 tokens at 48 pages); groups end at 16 KV4_MAX_SLOTS columns
  if (d->width > (long)KV4_MAX_SLOTS * p.chunk) p.chunk = (d->width + KV4_MAX_SLOTS - 1) / KV4_MAX_SLOTS;
  p.slots = d->width > 0 ? (d->width + p.chunk - 1) / p.chunk : 1;
  p.floats = p.group == 1 && p.slots == 1 ? 0 : (int64_t)d->rows * d->heads * (p.slots + p.slots_p) * (d->hd + 2);
  return p;
}
static int kv4_attn_check(const unimp_kv4_attn_desc* d) {
  if (d && (d->rows == 0 || d->heads == 0)) return UNIMP_OK;                        // empty tensors have no pointers
  if (!d || !d->q || !d->pages || (!d->tables && d->width) || !d->lens || !d->out) return unimp_set_error(UNIMP_ERR_ARG, "kv4_attn_decode: null pointer");
  if (d->kv_heads <= 0 || d->heads < 0 || d->heads % d->kv_heads || d->heads / d->kv_heads > 16 || d->width < 0 || d->width > 64 * 4 * KV4_MAX_SLOTS || d->rows < 0 || d->rows > 32767 ||
      d->heads > 65535 || d->n_pages <= 0)
    return unimp_set_error(UNIMP_ERR_SHAPE, "kv4_attn_decode: query heads a multiple of the key heads, at most 16 to one; at most 32767 rows, 65536 pages of a row; a pool with pages");
  if (d->hd != 64 && d->hd != 80 && d->hd != 128) return unimp_set_error(UNIMP_ERR_SHAPE, "kv4: head dim 64, 80 or 128");
  if ((((uintptr_t)d->pages | (uintptr_t)d->q) & 15) || ((d->q_row_stride | d->q_head_stride) & 7))
    return unimp_set_error(UNIMP_ERR_ALIGN, "kv4_attn_decode: 16-byte aligned pages and q, q strides multiples of 8 elements");
  return UNIMP_OK;
}

extern "C" int64_t unimp_kv4_attn_workspace(const unimp_kv4_attn_desc* d) { return kv4_attn_check(d) || !d->rows || !d->heads ? 0 : kv4_plan(d).floats; }

template <int D>
static void kv4_merge_launch(const Kv4AttnArgs& a, const Kv4Plan& p, hipStream_t s) {
  const dim3 grid(a.heads, a.rows);
  const int n = p.slots + p.slots_p;                                              // few slots, or enough (row, head) pairs to fill the chip with one wave each
  if (n <= 8 || (n <= 16 && (long)a.rows * a.heads >= 1024)) hipLaunchKernelGGL((kv4_attn_merge_kernel<D, 1>), grid, dim3(D / 2), 0, s, a);
  else hipLaunchKernelGGL((kv4_attn_merge_kernel<D, 8>), grid, dim3(4 * D), 0, s, a);
}
template <int D>
static void kv4_attn_launch(const Kv4AttnArgs& a, const Kv4Plan& p, hipStream_t s) {
  if (p.group > 1) {
    const dim3 grid(a.kv_heads, p.slots > p.slots_p ? p.slots : p.slots_p, (a.rows + KV4_TEAMS - 1) / KV4_TEAMS + a.rows / p.group);
#define KV4_G(M, GM)                                                                                         \
  do {                                                                                                       \
    if (a.alibi) hipLaunchKernelGGL((kv4_attn_group_kernel<D, M, GM, true>), grid, dim3(256), 0, s, a);      \
    else hipLaunchKernelGGL((kv4_attn_group_kernel<D, M, GM, false>), grid, dim3(256), 0, s, a);             \
  } while (0)
    // a row's own queries are at most half of the group's
    if (p.gmode != 2) {
      if constexpr (D == 64) { if (p.gmode == 0) KV4_G(0, 0); else KV4_G(0, 1); }
      else if (p.gmode == 0) KV4_G(0, 0);
      else if (p.gmode == 1) KV4_G(0, 1);
      else if (p.mode == 0) KV4_G(0, 3);
      else KV4_G(1, 3);
    } else if (p.mode == 0) KV4_G(0, 2);
    else if (p.mode == 1) KV4_G(1, 2);
    else if constexpr (D > 64) KV4_G(3, 2);
#undef KV4_G
    kv4_merge_launch<D>(a, p, s);
    return;
  }
  // key heads fastest: a row's chunks are of unequal use (the last ones mostly behind its end), and consecutive workgroups go to the eight dies in turn
  const dim3 grid(a.kv_heads, p.slots, a.rows);
#define KV4_L(M, W)                                                                                          \
  do {                                                                                                       \
    if (a.alibi) hipLaunchKernelGGL((kv4_attn_kernel<D, M, W, true>), grid, dim3(64 * W), 0, s, a);          \
    else hipLaunchKernelGGL((kv4_attn_kernel<D, M, W, false>), grid, dim3(64 * W), 0, s, a);                 \
  } while (0)
#define KV4_W(M)                                                                                             \
  do {                                                                                                       \
    if (p.nw == 8) KV4_L(M, 8); else if (p.nw == 4) KV4_L(M, 4); else KV4_L(M, 1); \
  } while (0)
  if (p.mode == 0) KV4_W(0);
  else if (p.mode == 1) KV4_W(1);
  else if (p.mode == 2) KV4_L(2, 4);
  else if constexpr (D > 64) KV4_L(3, 4);                                         // 5 ... 8 queries; of head dim 64 they are MODE 1
#undef KV4_W
#undef KV4_L
  if (a.ws) kv4_merge_launch<D>(a, p, s);
}

extern "C" int unimp_kv4_attn_decode(const unimp_kv4_attn_desc* d, float* workspace, void* stream) {
  const int rc = kv4_attn_check(d);
  if (rc) return rc;
  if (!d->rows || !d->heads) return UNIMP_OK;
  const Kv4Plan p = kv4_plan(d);
  if (p.floats && !workspace) return unimp_set_error(UNIMP_ERR_ARG, "kv4_attn_decode: workspace of unimp_kv4_attn_workspace floats");
  Kv4AttnArgs a{(const bf16*)d->q, d->q_row_stride, d->q_head_stride, (const uint8_t*)d->pages, d->n_pages, d->kv_heads, d->tables, d->table_stride, d->width, d->lens,
                d->rows, d->heads, d->scale, d->alibi_slopes, (bf16*)d->out, d->o_row_stride, d->o_head_stride, p.group, d->shared_len, d->heads / d->kv_heads, p.chunk, p.slots, p.chunk_p, p.slots_p,
                p.floats ? workspace : nullptr};
  switch (d->hd) {
    case 64: kv4_attn_launch<64>(a, p, (hipStream_t)stream); break;
    case 80: kv4_attn_launch<80>(a, p, (hipStream_t)stream); break;
    default: kv4_attn_launch<128>(a, p, (hipStream_t)stream);
  }
  return unimp_check_launch("kv4_attn_decode");
}
