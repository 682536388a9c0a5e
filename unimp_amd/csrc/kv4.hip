// Paged 4-bit K/V cache of a decode (F1: the past_key_values behind Flamingo.generate, eval_rec.py:100-110, eval_exp.py:103-113, eval_img_gen.py:102-111):
// quantise-and-write of prompt tokens, rotary embedding + append of a decode step's tokens, read-back as values, page tables and slots from the rows' lengths,
// and the beam reorder.  Layout of a page: kv4.h.  Attention over the pages: kv4_attn.hip.
//
// An MX block of x: e = floor(log2 max |x|) - 2 between -125 and 125, codes rne(x / 2^e) on e2m1, saturated at 6: 2^e code is exact in bf16, so what is read back is
// exactly what the attention multiplies.  All of these are bound by bytes; the arithmetic is a few instructions per element.
#include <type_traits>
#include "kv4.h"
#include "unimp_hip.h"

template <typename F> static int kv4_for_hd(int hd, F f) {
  switch (hd) {
    case 64: return f(std::integral_constant<int, 64>());
    case 80: return f(std::integral_constant<int, 80>());
    case 128: return f(std::integral_constant<int, 128>());
    default: return unimp_set_error(UNIMP_ERR_SHAPE, "kv4: head dim 64, 80 or 128");
  }
}
extern "C" int unimp_kv4_page_bytes(int hd) { return hd == 64 || hd == 80 || hd == 128 ? 32 * hd + 64 * ((hd + 31) / 32) : -1; }

// ------------------------------------------------------------------------------------------- runs of slots
// A RUN is a maximal stretch of consecutive rows whose slots are consecutive inside one page; a workgroup (chunk of 32 rows, some heads) owns the runs that START
// in its chunk (a run has at most 32 rows: it looks 31 rows ahead), so every row is moved once and every page is touched by one wave per run, whatever the
// alignment of the rows to the pages.  A run shorter than KV4_SHORT rows costs its latencies whatever its length: the rows of such runs are moved one by one, all of a chunk's
// at once.  Measured, 16 384 tokens x 32 heads x 80 dims in runs of 8 | 11 | 12 | 15, write: as rows 91 | 90 | 88 | 88 us, as runs 127 | 103 | 97 |
// 86; 33 requests of 1 or 2 tokens x 32 heads x 128, write and read back: 116 -> 16 us.  sl[KV4_BACK + i] = slot of row i0 + i, -1: none.
#define KV4_SHORT 12
#define KV4_BACK 12
#define KV4_SLOTS (KV4_BACK + 64)
__device__ __forceinline__ void kv4_load_slots(int64_t (&sl)[KV4_SLOTS], const int64_t* __restrict__ slots, long i0, long tokens, long n_pages) {
  if (threadIdx.x < KV4_SLOTS) {
    const long i = i0 - KV4_BACK + (int)threadIdx.x;
    const int64_t s = i >= 0 && i < tokens ? slots[i] : -1;
    sl[threadIdx.x] = s >= 0 && s < n_pages * KV4_PAGE ? s : -1;
  }
  __syncthreads();
}
// rows of a workgroup's chunk: 32; 8 where that leaves the chip empty (64 tokens x 32 heads x 128 in runs of 1: 19.5 -> 8.9 us, read 15.3 -> 8.0)
static int kv4_chunk_rows(int64_t tokens, int64_t blocks) { return (tokens + 31) / 32 * blocks <= 256 ? 8 : 32; }      // blocks: of heads, times layers
// a chunk's rows as bits: `few` belong to runs of less than KV4_SHORT rows, a longer run begins at `starts`, `none` have no slot; `links` go on where the row before ends
struct Kv4Rows { uint32_t few, starts, none, links; };
__device__ __forceinline__ Kv4Rows kv4_rows(const int64_t (&sl)[KV4_SLOTS], int rows) {
  const int lane = lane_id();
  const int64_t s = sl[lane];
  const uint64_t link = __ballot(lane > 0 && s >= 0 && (s & 31) && sl[max(lane - 1, 0)] + 1 == s);      // bit l: row i0 - KV4_BACK + l
  const int at = KV4_BACK + (lane & 31);
  const int back = __builtin_clzll(~(link << (63 - at))), on = __builtin_ctzll(~(link >> (at + 1)));   // link's lowest bit is 0, and its shifts bring zeros in
  const bool has = lane < rows && sl[at] >= 0, few = back + on + 1 < KV4_SHORT;
  Kv4Rows r;
  r.few = (uint32_t)__ballot(has && few);
  r.starts = (uint32_t)__ballot(has && !few && !back);
  r.none = (uint32_t)__ballot(lane < rows && !has);
  r.links = (uint32_t)(link >> KV4_BACK);
  return r;
}
// rows of the run that starts at row a
__device__ __forceinline__ int kv4_run(const int64_t (&sl)[KV4_SLOTS], int a) {
  const int64_t s0 = sl[KV4_BACK + a];
  const int lane = lane_id(), t0 = (int)(s0 & 31);
  const bool on = lane < 32 && t0 + lane < 32 && sl[KV4_BACK + a + (lane & 31)] == s0 + lane;      // lane 0: itself
  return __builtin_ctzll(~__ballot(on));
}
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}
// eight dwords of eight nibbles, turned round: out[i] nibble j = in[j] nibble i
__device__ __forceinline__ void kv4_turn8(uint32_t (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = x[i], b = x[i + 4];
    x[i] = __builtin_amdgcn_perm(b, a, 0x05040100u); x[i + 4] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  }
#pragma unroll
  for (int h = 0; h < 8; h += 4)
#pragma unroll
    for (int i = h; i < h + 2; ++i) {
      const uint32_t a = x[i], b = x[i + 2];
      x[i] = __builtin_amdgcn_perm(b, a, 0x06020400u); x[i + 2] = __builtin_amdgcn_perm(b, a, 0x07030501u);
    }
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint32_t a = x[i], b = x[i + 1], m = 0x0f0f0f0fu;
    x[i] = (a & m) | ((b << 4) & ~m); x[i + 1] = ((a >> 4) & m) | (b & ~m);
  }
}
__device__ __forceinline__ void wave_lds_fence() {                   // LDS of this wave's other lanes
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ------------------------------------------------------------------------------------------- write
// A wave per (run, head).  Four lanes hold an MX block of a token (16-byte loads, the block's maximum by two lane exchanges); V's codes turn round (8 tokens x 8 dims
// per lane) through LDS; the page is put together in LDS and leaves in 16-byte stores.  A run that does not fill its page writes its own bytes, and its nibbles of V dwords
// that other runs share by atomic and + or: the fields are disjoint, the result does not depend on the order.  Bound by its bytes (4 in, 17 / 16 out per element of k): 54 000 tokens
// in pages of 32 x 32 heads x 128: 237 us, 4.7 TB/s, where a large copy reaches 4.9; runs that share pages pay the atomics (16 384 tokens in runs of 16: 101 us, whole pages 41).
#define KV4_HEADS 4                                                  // heads of a workgroup; the head blocks of a chunk are neighbours in the grid (whole rows in flight)
template <int D>
__global__ __launch_bounds__(256, 4) void kv4_write_kernel(const bf16* __restrict__ k, const bf16* __restrict__ v, long k_ts, long k_hs, long v_ts, long v_hs,
                                                           uint8_t* __restrict__ pages, long n_pages, int heads, int head_blocks, int chunk_rows, const int64_t* __restrict__ slots, long tokens) {
  using P = Kv4<D>;
  constexpr int X = D / 8, TP = 16 / P::NB, PASSES = (32 + TP - 1) / TP;      // 8-dim pieces of a row; tokens of a pass (four lanes to a block)
  __shared__ int64_t sl[KV4_SLOTS];
  __shared__ __attribute__((aligned(16))) uint8_t image[4][P::BYTES];
  __shared__ uint32_t turn[4][32 * X];
  __shared__ int piece[4][32];
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quad = lane & 3;
  const int tl = (lane >> 2) / P::NB, b = (lane >> 2) - tl * P::NB, d = 32 * b + 8 * quad;      // this lane's token of a pass, block and dims
  const bool on = tl < TP && d < D;
  const long lane_k = tl * k_ts + d, lane_v = tl * v_ts + d;
  const long chunk = blockIdx.x / head_blocks, i0 = chunk * chunk_rows;
  const int h0 = (blockIdx.x - (unsigned)chunk * head_blocks) * KV4_HEADS, h1 = min(h0 + KV4_HEADS, heads);
  kv4_load_slots(sl, slots, i0, tokens, n_pages);
  uint8_t* im = image[w];
  uint32_t* tv = turn[w];
  // four lanes' 8 elements each of one block -> this lane's codes and the scale byte
  auto quantise = [](const bf16x8& u, int& sb) {
    float f[8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) { f[j] = bf2f(u[j]); m = max(m, __float_as_uint(f[j]) & 0x7fffffffu); }
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true));       // lane ^ 1
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true));       // lane ^ 2
    sb = kv4_scale_byte((int)(m >> 23));
    const float scale = __uint_as_float((uint32_t)(sb == 255 ? 127 : sb) << 23);
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[0], f[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[2], f[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[4], f[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, f[6], f[7], scale, 3);
    return sb == 255 ? 0u : r;
  };
  const Kv4Rows rows = kv4_rows(sl, chunk_rows);
  if (const uint32_t few = rows.few, links = rows.links; few) {
    constexpr bool PAIR = P::NI % 2 == 0;
    constexpr int U = PAIR ? D / 2 : D;
    const uint32_t quarter = (uint32_t)__ballot(lane < 32 && !(sl[KV4_BACK + (lane & 31)] & 3)) | 1u;      // row 0 and tokens 0, 4, ... of a page start a piece in any case
    const int n_pieces = __builtin_popcount(few & ~(links & ~quarter));
    for (int head = h0 + w; head < h1; head += 4) {
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        const long ts = kind ? v_ts : k_ts;
        const bf16* mine = (kind ? v + head * v_hs + lane_v : k + head * k_hs + lane_k) + i0 * ts;
        bf16x8 u[PASSES];
#pragma unroll
        for (int ps = 0; ps < PASSES; ++ps) {
          const int i = ps * TP + tl;
          u[ps] = bf16x8{};
          if (on && i < 32 && (few >> i & 1)) u[ps] = *(const bf16x8*)(mine + ps * TP * ts);
        }
#pragma unroll
        for (int ps = 0; ps < PASSES; ++ps) {
          if (!(few >> (ps * TP) & ((1u << TP) - 1))) continue;      // uniform
          const int i = ps * TP + tl;
          int sb;
          const uint32_t r = quantise(u[ps], sb);
          if (on && i < 32 && (few >> i & 1)) {
            const int64_t slot = sl[KV4_BACK + i];
            const int t = (int)(slot & 31);
            uint8_t* page = pages + ((slot >> 5) * heads + head) * (long)P::BYTES;
            if (!quad) page[kind ? P::vs_byte(t, b) : P::ks_byte(t, b)] = (uint8_t)sb;
            if (!kind) *(uint32_t*)(page + P::k_byte(t, b) + 4 * quad) = r;
            else tv[i * X + (d >> 3)] = r;
          }
        }
      }
      // V: up to four consecutive tokens share their dwords (a piece); consecutive lanes take consecutive dwords, two at a time where a token's dwords pair up
      if (lane < 32) {
        const uint32_t starts = few & ~(links & ~quarter);
        if (starts >> lane & 1) piece[w][__builtin_popcount(starts & ((1u << lane) - 1))] = lane | (__builtin_ctz(~((links & ~quarter & few) >> 1 >> lane)) + 1) << 8;
      }
      wave_lds_fence();
      const int units = n_pieces * U;
      for (int x = lane; x < units; x += 64) {
        const int pc = piece[w][x / U], first = pc & 255, len = pc >> 8, un = x % U;
        const int64_t slot = sl[KV4_BACK + first];
        const int t = (int)(slot & 31), sh = 4 * kv4_nibble(t);
        uint8_t* page = pages + ((slot >> 5) * heads + head) * (long)P::BYTES;
        const int dim = PAIR ? 32 * (un % (P::NI / 2)) + un / (P::NI / 2) : 16 * (un % P::NI) + un / P::NI;
        uint32_t lo = 0, hi = 0;
        for (int e = 0; e < len; ++e) {
          const uint32_t* row = tv + (first + e) * X;
          lo |= (row[dim >> 3] >> (4 * (dim & 7)) & 15u) << (4 * e);
          if (PAIR) hi |= (row[(dim >> 3) + 2] >> (4 * (dim & 7)) & 15u) << (4 * e);
        }
        const uint32_t mask = (0xffffu >> (16 - 4 * len)) << sh;
        if constexpr (PAIR) {
          unsigned long long* o = (unsigned long long*)(page + P::v_dword(t, dim));
          atomicAnd(o, ~(mask * 0x100000001ull)); atomicOr(o, (unsigned long long)(lo << sh) | (unsigned long long)(hi << sh) << 32);
        } else {
          uint32_t* o = (uint32_t*)(page + P::v_dword(t, dim));
          atomicAnd(o, ~mask); atomicOr(o, lo << sh);
        }
      }
      wave_lds_fence();
    }
  }
  for (uint32_t todo = rows.starts; todo; todo &= todo - 1) {
    const int a = __builtin_ctz(todo), n = __builtin_amdgcn_readfirstlane(kv4_run(sl, a));
    const int64_t s0 = uniform64(sl[KV4_BACK + a]);
    const int t0 = (int)(s0 & 31);
    const long row0 = i0 + a - t0;                                   // the row that page token 0 has or would have
    for (int head = h0 + w; head < h1; head += 4) {
      uint8_t* page = pages + ((s0 >> 5) * heads + head) * (long)P::BYTES;
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        const long ts = kind ? v_ts : k_ts;
        const bf16* src = (kind ? v + head * v_hs : k + head * k_hs) + row0 * ts;
        const bf16* mine = src + (kind ? lane_v : lane_k);
        bf16x8 u[PASSES];
#pragma unroll
        for (int ps = 0; ps < PASSES; ++ps) {                        // all loads of the half page first
          const int t = ps * TP + tl;
          u[ps] = bf16x8{};
          if (on && t >= t0 && t < t0 + n) u[ps] = *(const bf16x8*)(mine + ps * TP * ts);
        }
#pragma unroll
        for (int ps = 0; ps < PASSES; ++ps) {
          const int t = ps * TP + tl;
          int sb;
          const uint32_t r = quantise(u[ps], sb);
          if (on && t < 32) {
            if (!kind) *(uint32_t*)(im + P::k_byte(t, b) + 4 * quad) = r;
            else tv[t * X + (d >> 3)] = r;
            if (!quad) im[kind ? P::vs_byte(t, b) : P::ks_byte(t, b)] = (uint8_t)sb;
          }
        }
      }
      wave_lds_fence();
      if (4 * X == 64 || lane < 4 * X) {                             // lane: 8 tokens of group g, 8 dims
        const int g = lane / X, c8 = lane - g * X;
        uint32_t y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = tv[(16 * (j >> 2) + 4 * g + (j & 3)) * X + c8];
        kv4_turn8(y);
#pragma unroll
        for (int j = 0; j < 8; ++j) *(uint32_t*)(im + P::v_dword(4 * g, 8 * c8 + j)) = y[j];
      }
      wave_lds_fence();
      if (n == 32) {
#pragma unroll
        for (int x = lane * 16; x < P::BYTES; x += 1024) *(u32x4*)(page + x) = *(const u32x4*)(im + x);
      } else {
        for (int x = lane; x < n * X; x += 64) {
          const int t = t0 + x / X, c = (x % X) * 8, o = P::k_byte(t, c >> 5) + ((c & 31) >> 1);
          *(uint32_t*)(page + o) = *(const uint32_t*)(im + o);
        }
        for (int x = lane; x < n * 2 * P::NB; x += 64) {
          const int t = t0 + x / (2 * P::NB), bb = x % P::NB, o = x % (2 * P::NB) < P::NB ? P::ks_byte(t, bb) : P::vs_byte(t, bb);
          page[o] = im[o];
        }
        for (int x = lane; x < 4 * D; x += 64) {
          const int g = x / D;
          uint32_t mask = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) { const int t = 16 * (j >> 2) + 4 * g + (j & 3); if (t >= t0 && t < t0 + n) mask |= 15u << (4 * j); }
          uint32_t* o = (uint32_t*)(page + P::VOFF) + x;
          const uint32_t val = *((const uint32_t*)(im + P::VOFF) + x);
          if (mask == 0xffffffffu) *o = val;
          else if (mask) { atomicAnd(o, ~mask); atomicOr(o, val & mask); }
        }
      }
      wave_lds_fence();
    }
  }
}

extern "C" int unimp_kv4_write(const void* k, const void* v, int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs, void* pages, int64_t n_pages, int heads,
                               int hd, const int64_t* slots, int64_t tokens, void* stream) {
  if (tokens <= 0 || heads <= 0 || n_pages <= 0) return UNIMP_OK;
  if (!k || !v || !pages || !slots) return unimp_set_error(UNIMP_ERR_ARG, "kv4_write: null pointer");
  const int64_t hb = (heads + KV4_HEADS - 1) / KV4_HEADS;
  const int cr = kv4_chunk_rows(tokens, hb);
  if (heads > 65535 || (tokens + 31) / 32 * hb > 1 << 23) return unimp_set_error(UNIMP_ERR_SHAPE, "kv4_write: at most 65535 heads and 2^30 token heads");
  if (((k_ts | k_hs | v_ts | v_hs) & 7) || (((uintptr_t)k | (uintptr_t)v | (uintptr_t)pages) & 15))
    return unimp_set_error(UNIMP_ERR_ALIGN, "kv4_write: strides multiples of 8 elements, 16-byte aligned pointers");
  return kv4_for_hd(hd, [&](auto d) {
    hipLaunchKernelGGL((kv4_write_kernel<decltype(d)::value>), dim3((unsigned)((tokens + cr - 1) / cr * hb)), dim3(256), 0, (hipStream_t)stream, (const bf16*)k,
                       (const bf16*)v, (long)k_ts, (long)k_hs, (long)v_ts, (long)v_hs, (uint8_t*)pages, (long)n_pages, heads, (int)hb, cr, slots, (long)tokens);
    return unimp_check_launch("kv4_write");
  });
}

// ------------------------------------------------------------------------------------------- decode step: rotary embedding + append
// A wave per (row, head), two dims to a lane.  The rotation runs in 64 bits (two products of a bf16 and an fp32, exact there, and their sum): a code is decided next to a border, and
// k's codes are those of the given tables' rotation in 64 bits.  V's nibbles go in by atomics: two rows of a launch may write different tokens of one page.  A few rows are bound by
// three dependent steps (load, block maximum, write): 10 rows x 32 x 80 4.1 us.  Many rows are not, nor by bytes: 200 x 32 x 128 10.1 us for 7.6 MB, 258 vector instructions a wave (the
// codes' comparisons in 64 bits among them) on 6 waves a SIMD beside two atomics a lane.
__device__ __forceinline__ uint32_t kv4_code_f64(double x, double inv) {
  const double a = fabs(x) * inv;
  const uint32_t c = (a > 0.25) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0);
  return c | (x < 0.0 ? 8u : 0u);
}
template <int CTRL> __device__ __forceinline__ int kv4_dpp(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true); }
template <int D>
__global__ __launch_bounds__(256) void kv4_rope_append_kernel(const bf16* __restrict__ qkv, long row_stride, long head_stride, int q_off, int k_off, int v_off,
                                                              int rot, const float* __restrict__ cos_rows, const float* __restrict__ sin_rows,
                                                              bf16* __restrict__ q_out, uint8_t* __restrict__ pages, long n_pages, int heads,
                                                              const int64_t* __restrict__ slots) {
  using P = Kv4<D>;
  const int row = blockIdx.y, lane = lane_id(), head = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = 2 * lane;
  // V: dims 32 b + c and 32 b + 16 + c of lane (b, c) are neighbouring dwords: one 64-bit atomic for both (head dim 80: odd rows of dwords, two of 32 bits)
  constexpr bool PAIR = P::NI % 2 == 0;
  const int v_dim = PAIR ? 32 * (lane >> 4) + (lane & 15) : d;
  if (head >= heads) return;                                        // uniform over the wave
  const int64_t slot = slots[row];
  const bf16* base = qkv + (long)row * row_stride + (long)head * head_stride;
  double q[2] = {0, 0}, k[2] = {0, 0}, v[2] = {0, 0};
  if (d < D) {
    const int h = rot >> 1;
    const float* c = cos_rows + (long)row * h;
    const float* s = sin_rows + (long)row * h;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int e = d + j;
      q[j] = (double)bf2f(base[q_off + e]); k[j] = (double)bf2f(base[k_off + e]); v[j] = (double)bf2f(base[v_off + v_dim + 16 * j * PAIR + j * !PAIR]);
      if (e < rot) {
        const int i = e < h ? e : e - h, p = e < h ? e + h : e - h;
        const double cc = c[i], ss = s[i], q2 = (double)bf2f(base[q_off + p]), k2 = (double)bf2f(base[k_off + p]);
        q[j] = e < h ? q[j] * cc - q2 * ss : q[j] * cc + q2 * ss;
        k[j] = e < h ? k[j] * cc - k2 * ss : k[j] * cc + k2 * ss;
      }
    }
    bf16x2 o = {f2bf((float)q[0]), f2bf((float)q[1])};
    *(bf16x2*)(q_out + ((long)row * heads + head) * D + d) = o;
  }
  if (slot < 0 || slot >= n_pages * KV4_PAGE) return;               // uniform
  const int t = (int)(slot & 31);
  uint8_t* page = pages + ((slot >> 5) * heads + head) * (long)P::BYTES;
  uint32_t code[2][2]; int sb[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const double (&x)[2] = w ? v : k;
    // exponent field: floor(log2 |x|) + 1023, 2047 for infinity and NaN; its maximum over the 16 lanes of a block
    int e = max((int)((__double2hiint(x[0]) >> 20) & 0x7ff), (int)((__double2hiint(x[1]) >> 20) & 0x7ff));
    e = max(e, kv4_dpp<0xB1>(e)); e = max(e, kv4_dpp<0x4E>(e));     // lane ^ 1, ^ 2: quads agree
    e = max(e, kv4_dpp<0x141>(e)); e = max(e, kv4_dpp<0x140>(e));   // mirrored inside 8 and inside 16 lanes
    sb[w] = e == 2047 ? 255 : min(max(e - 1023 - 2, -125), 125) + 127;      // a rotation may leave bf16's range: saturated like any code above 6
    const double inv = __hiloint2double((1023 + 127 - sb[w]) << 20, 0);
#pragma unroll
    for (int j = 0; j < 2; ++j) code[w][j] = sb[w] == 255 ? 0u : kv4_code_f64(x[j], inv);
  }
  int kk = (int)((code[0][0] | (code[0][1] << 4)) << (8 * (lane & 3)));      // four lanes' K codes into one dword
  kk |= kv4_dpp<0xB1>(kk); kk |= kv4_dpp<0x4E>(kk);
  if (d < D) {
    if (!(lane & 3)) *(uint32_t*)(page + P::k_byte(t, d >> 5) + ((d & 31) >> 1)) = (uint32_t)kk;
    if (!(lane & 15)) { page[P::ks_byte(t, d >> 5)] = (uint8_t)sb[0]; page[P::vs_byte(t, d >> 5)] = (uint8_t)sb[1]; }
    const int sh = 4 * kv4_nibble(t);
    if constexpr (PAIR) {
      unsigned long long* o = (unsigned long long*)(page + P::v_dword(t, v_dim));
      const unsigned long long both = 0x100000001ull;
      atomicAnd(o, ~((15u << sh) * both)); atomicOr(o, (unsigned long long)(code[1][0] << sh) | (unsigned long long)(code[1][1] << sh) << 32);
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t* o = (uint32_t*)(page + P::v_dword(t, d + j));
        atomicAnd(o, ~(15u << sh)); atomicOr(o, code[1][j] << sh);
      }
    }
  }
}

extern "C" int unimp_kv4_rope_append(const void* qkv, int64_t row_stride, int64_t head_stride, int rows, int heads, int hd, int q_off, int k_off, int v_off, int rot,
                                     const float* cos_rows, const float* sin_rows, void* q_out, void* pages, int64_t n_pages, const int64_t* slots, void* stream) {
  if (rows <= 0 || heads <= 0) return UNIMP_OK;
  if (!qkv || !q_out || (!pages && n_pages > 0) || !slots || (rot && (!cos_rows || !sin_rows))) return unimp_set_error(UNIMP_ERR_ARG, "kv4_rope_append: null pointer");
  if (rot < 0 || (rot & 1) || rot > hd || rows > 65535) return unimp_set_error(UNIMP_ERR_SHAPE, "kv4_rope_append: rot even and at most the head dim, at most 65535 rows");
  if (((uintptr_t)pages & 15) || ((uintptr_t)q_out & 3)) return unimp_set_error(UNIMP_ERR_ALIGN, "kv4_rope_append: 16-byte aligned pages, 4-byte aligned q_out");
  return kv4_for_hd(hd, [&](auto d) {
    hipLaunchKernelGGL((kv4_rope_append_kernel<decltype(d)::value>), dim3((heads + 3) / 4, rows), dim3(256), 0, (hipStream_t)stream, (const bf16*)qkv, (long)row_stride,
                       (long)head_stride, q_off, k_off, v_off, rot, cos_rows, sin_rows, (bf16*)q_out, (uint8_t*)pages, (long)n_pages, heads, slots);
    return unimp_check_launch("kv4_rope_append");
  });
}

// ------------------------------------------------------------------------------------------- read back as values
// A wave per (run, head): every page is read once, whatever rows name its tokens.  K: a lane converts 8 dims of a token; V: a lane takes 8 tokens x 8 dims, turns the
// nibbles round in registers and stores 16 bytes of each token.  Bound by the bf16 rows that leave: 65 600 rows x 32 x 128, 1.3 GB: 232 us, 5.6 TB/s.
template <int D>
__global__ __launch_bounds__(256, 4) void kv4_read_kernel(const uint8_t* __restrict__ pages, long layer_stride, long n_pages, int heads, int head_blocks, int chunk_rows,
                                                          const int64_t* __restrict__ slots, long tokens, bf16* __restrict__ k, bf16* __restrict__ v) {
  using P = Kv4<D>;
  constexpr int X = D / 8, TP = 64 / X, PASSES = (32 + TP - 1) / TP;          // 8-dim pieces of a row; tokens of a pass
  __shared__ int64_t sl[KV4_SLOTS];
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tl = lane / X, d = (lane - tl * X) * 8, b = d >> 5;               // K: this lane's token of a pass and dims; V: tl = group g of 8 tokens
  const long chunk = blockIdx.x / head_blocks, i0 = chunk * chunk_rows;
  const int h0 = (blockIdx.x - (unsigned)chunk * head_blocks) * KV4_HEADS, h1 = min(h0 + KV4_HEADS, heads);
  kv4_load_slots(sl, slots, i0, tokens, n_pages);
  const long lo = (long)blockIdx.y * tokens;
  const long row = (long)heads * D;                                            // elements of an output row
  auto values = [](uint32_t c, uint32_t byte) {                                // eight codes as values
    const float sc = kv4_scale(byte);
    union { bf16x2 h[4]; bf16x8 v; } u;
    u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 0); u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 1);
    u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 2); u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 3);
    if (byte == 255u) { const uint32_t nn = 0x7fc07fc0u; u.h[0] = u.h[1] = u.h[2] = u.h[3] = __builtin_bit_cast(bf16x2, nn); }
    return u.v;
  };
  const Kv4Rows rows = kv4_rows(sl, chunk_rows);
  if (rows.none) {                                                   // no slots: rows of zeros
    const int per = (h1 - h0) * X, end = (int)min((long)chunk_rows, tokens - i0);
    for (int x = threadIdx.x; x < end * per; x += 256) if (rows.none >> (x / per) & 1) {
      const long o = (lo + i0 + x / per) * row + h0 * D + 8 * (x % per);
      *(bf16x8*)(k + o) = bf16x8{}; *(bf16x8*)(v + o) = bf16x8{};
    }
  }
  if (const uint32_t few = rows.few) {
    for (int head = h0 + w; head < h1; head += 4) {
#pragma unroll 2
      for (int ps = 0; ps < PASSES; ++ps) {
        if (!(few >> (ps * TP) & ((1u << TP) - 1))) continue;        // uniform
        const int i = ps * TP + tl;
        if (tl < TP && i < 32 && (few >> i & 1)) {
          const int64_t slot = sl[KV4_BACK + i];
          const int t = (int)(slot & 31), sh = 4 * kv4_nibble(t);
          const uint8_t* page = pages + (long)blockIdx.y * layer_stride + ((slot >> 5) * heads + head) * (long)P::BYTES;
          const long o = (lo + i0 + i) * row + head * D + d;
          const uint32_t c = *(const uint32_t*)(page + P::k_byte(t, b) + ((d & 31) >> 1)), ks = page[P::ks_byte(t, b)], vs = page[P::vs_byte(t, b)];
          uint32_t y = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) y |= (*(const uint32_t*)(page + P::v_dword(t, d + j)) >> sh & 15u) << (4 * j);
          *(bf16x8*)(k + o) = values(c, ks);
          *(bf16x8*)(v + o) = values(y, vs);
        }
      }
    }
  }
  for (uint32_t todo = rows.starts; todo; todo &= todo - 1) {
    const int a = __builtin_ctz(todo), n = __builtin_amdgcn_readfirstlane(kv4_run(sl, a));
    const int64_t s0 = uniform64(sl[KV4_BACK + a]);
    const int t0 = (int)(s0 & 31);
    for (int head = h0 + w; head < h1; head += 4) {
      const uint8_t* page = pages + (long)blockIdx.y * layer_stride + ((s0 >> 5) * heads + head) * (long)P::BYTES;
      const long o0 = (lo + i0 + a - t0) * row + head * D;           // output of the page's token 0
      uint32_t c[PASSES], ks[PASSES], y[8];
      u32x2 vs = {0, 0};
#pragma unroll
      for (int ps = 0; ps < PASSES; ++ps) {                          // the page's loads first
        const int t = ps * TP + tl;
        c[ps] = ks[ps] = 0;
        if (tl < TP && t < 32) { c[ps] = *(const uint32_t*)(page + P::k_byte(t, b) + ((d & 31) >> 1)); ks[ps] = page[P::ks_byte(t, b)]; }
      }
      if (tl < 4) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = *(const uint32_t*)(page + P::v_dword(4 * tl, d) + 4 * P::NI * j);
        vs = *(const u32x2*)(page + P::VS + 8 * P::NB * tl + 8 * b);
      }
#pragma unroll
      for (int ps = 0; ps < PASSES; ++ps) {
        const int t = ps * TP + tl;
        if (tl < TP && t >= t0 && t < t0 + n) *(bf16x8*)(k + o0 + ps * TP * row + (tl * (int)row + d)) = values(c[ps], ks[ps]);
      }
      if (tl < 4) {
        kv4_turn8(y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int t = 16 * (j >> 2) + 4 * tl + (j & 3);
          if (t >= t0 && t < t0 + n) *(bf16x8*)(v + o0 + (16 * (j >> 2) + (j & 3)) * row + (4 * tl * (int)row + d)) = values(y[j], (vs[j >> 2] >> (8 * (j & 3))) & 0xffu);
        }
      }
    }
  }
}

extern "C" int unimp_kv4_read(const void* pages, int64_t layer_stride, int layers, int64_t n_pages, int heads, int hd, const int64_t* slots, int64_t tokens, void* k,
                              void* v, void* stream) {
  if (tokens <= 0 || heads <= 0 || layers <= 0) return UNIMP_OK;
  if ((!pages && n_pages > 0) || !slots || !k || !v) return unimp_set_error(UNIMP_ERR_ARG, "kv4_read: null pointer");
  const int64_t hb = (heads + KV4_HEADS - 1) / KV4_HEADS;
  const int cr = kv4_chunk_rows(tokens, hb * layers);
  if (layers > 65535 || heads > 65535 || (tokens + 31) / 32 * hb > 1 << 23)
    return unimp_set_error(UNIMP_ERR_SHAPE, "kv4_read: at most 65535 layers and heads, 2^30 token heads");
  if (((uintptr_t)pages | (uintptr_t)k | (uintptr_t)v) & 15) return unimp_set_error(UNIMP_ERR_ALIGN, "kv4_read: 16-byte aligned pointers");
  return kv4_for_hd(hd, [&](auto d) {
    constexpr int D = decltype(d)::value;
    hipLaunchKernelGGL((kv4_read_kernel<D>), dim3((unsigned)((tokens + cr - 1) / cr * hb), layers), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)pages,
                       (long)layer_stride, (long)n_pages, heads, (int)hb, cr, slots, (long)tokens, (bf16*)k, (bf16*)v);
    return unimp_check_launch("kv4_read");
  });
}

// ------------------------------------------------------------------------------------------- page tables and slots from lengths
// What a row takes from the free list starts at the sum of what the rows before it take: every workgroup sums that itself (a handful of integer operations
// per row, from L2), so the whole step is one launch and nothing is exchanged between workgroups.  8 bytes per token: bound by its launch and three dependent memory
// latencies (lengths, table or free list, slots): 80 rows 5 us, 2 000 rows with 1 000 000 new tokens 10.8 us (9 MB).
struct PageRow { int need, begin; };                                // columns [begin, need) come from the free list
struct PageArgs {
  int32_t* tables; const int32_t *mapped, *cached, *fresh, *cover, *free_pages, *cursor, *shared; int32_t *mapped_out, *cursor_out, *cu; int64_t* slots;
  long max_tokens; int rows, width, n_free, group;
};
__device__ __forceinline__ int page_need(const PageArgs& a, int r, int& map) {
  const long len = (long)max(a.cached[r], 0) + max(a.fresh[r], 0), cov = a.cover ? max((long)a.cover[r], len) : len;
  map = min(max(a.mapped[r], 0), a.width);
  return (int)min((cov + KV4_PAGE - 1) / KV4_PAGE, (long)a.width);
}
__device__ __forceinline__ PageRow page_row(const PageArgs& a, int r, int& alias, int& map) {
  const int need = page_need(a, r, map);
  alias = 0;
  if (a.shared) {
    const int g = r / a.group, first = g * a.group;
    if (r != first) {
      int m0; const int n0 = page_need(a, first, m0);
      alias = min(min(max(a.shared[g], 0) / KV4_PAGE, need), max(m0, n0));
    }
  }
  return PageRow{need, max(map, alias)};
}
// sum over a wave's lanes: inside the rows of 16 by lane moves of the vector pipe, the four rows as scalars
__device__ __forceinline__ long wave_total(long x) {
  auto moved = [&](auto C) {
    constexpr int c = decltype(C)::value;
    return (long)(((uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(x >> 32), c, 0xf, 0xf, true) << 32) | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, c, 0xf, 0xf, true));
  };
  x += moved(std::integral_constant<int, 0xB1>()); x += moved(std::integral_constant<int, 0x4E>());      // lane ^ 1, ^ 2
  x += moved(std::integral_constant<int, 0x141>()); x += moved(std::integral_constant<int, 0x140>());    // mirrored inside 8 and inside 16 lanes
  long s = 0;
#pragma unroll
  for (int i = 0; i < 64; i += 16) s += (long)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)x, i));
  return s;
}
// RPB = 1: a workgroup per row; 8: a wave per row (the sum over the rows before is made once for eight)
template <int RPB>
__global__ __launch_bounds__(RPB == 1 ? 256 : 512) void page_tables_extend_kernel(PageArgs a) {
  constexpr int T = RPB == 1 ? 256 : 512, STEP = RPB == 1 ? T : 64;
  __shared__ long red[2][T / 64];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r0 = blockIdx.x * RPB;
  const int r = RPB == 1 ? r0 : min(r0 + wave, a.rows - 1);
  const int first = a.group > 1 ? r / a.group * a.group : r;
  // the row's own numbers and those of rows [r0, r) and [first, r): requested together with the sum over the rows before
  const int start = a.cursor[0];
  int alias, map; const PageRow p = page_row(a, r, alias, map);
  int al0 = 0, map0 = 0, begin0 = 0;
  if (first != r) begin0 = page_row(a, first, al0, map0).begin;
  long in_block = 0, in_block_tok = 0, in_group = 0;
  for (int i = min(r0, first) + lane; i < r; i += 64) {
    int al, m; const PageRow q = page_row(a, i, al, m);
    const int own = max(q.need - q.begin, 0);
    if (i >= r0) { in_block += own; in_block_tok += max(a.fresh[i], 0); }
    if (i >= first) in_group += own;
  }
  long before = 0, tok = 0;                                          // pages taken and tokens packed by the rows [0, r0)
  if (!a.shared) {                                                   // no groups: the loads of eight rows at once
#pragma unroll 8
    for (int i = tid; i < r0; i += T) { int m; const int need = page_need(a, i, m); before += max(need - m, 0); tok += max(a.fresh[i], 0); }
  } else {
    for (int i = tid; i < r0; i += T) { int al, m; const PageRow q = page_row(a, i, al, m); before += max(q.need - q.begin, 0); tok += max(a.fresh[i], 0); }
  }
  before = wave_total(before); tok = wave_total(tok);
  if (!lane) { red[0][wave] = before; red[1][wave] = tok; }
  if (r > min(r0, first)) { in_block = wave_total(in_block); in_block_tok = wave_total(in_block_tok); in_group = wave_total(in_group); }
  __syncthreads();
  if (RPB > 1 && r0 + wave >= a.rows) return;
  before = start + in_block; tok = in_block_tok;
#pragma unroll
  for (int i = 0; i < T / 64; ++i) { before += red[0][i]; tok += red[1][i]; }
  const long before_first = before - in_group;
  const int32_t* row0 = a.tables + (long)first * a.width;
  int32_t* row = a.tables + (long)r * a.width;
  auto from_free = [&](long i) { return i >= 0 && i < a.n_free ? a.free_pages[i] : -1; };
  auto lookup = [&](int c) {                                         // the row's page of column c < max(map, need) after the call
    if (c < map) return (int)row[c];
    if (c < alias) return c < map0 ? (int)row0[c] : from_free(before_first + c - begin0);
    return c < p.need ? from_free(before + c - p.begin) : -1;
  };
  const int n = max(a.fresh[r], 0), have = max(a.cached[r], 0), at = RPB == 1 ? tid : lane;
  // RPB = 1: gridDim.y workgroups share the row's tokens, the first of them writes the rest
  const long end = min((long)n, a.max_tokens - tok);
#pragma unroll 4
  for (long t = at + (long)blockIdx.y * STEP; t < end; t += (long)gridDim.y * STEP) {
    const long pos = (long)have + t, c = pos / KV4_PAGE;
    const long page = c < a.width ? (long)lookup((int)c) : -1;
    a.slots[tok + t] = page >= 0 ? page * KV4_PAGE + (pos & 31) : -1;
  }
  if (blockIdx.y) return;
  for (int c = map + at; c < p.need; c += STEP) row[c] = lookup(c);
  auto to32 = [](long x) { return (int)min(x, 0x7fffffffl); };       // sums of nonsense lengths stay above every limit
  if (at == 0) { a.mapped_out[r] = max(map, p.need); a.cu[r] = to32(tok); }
  if (r == a.rows - 1) {
    if (at == 0) { a.cu[a.rows] = to32(tok + n); a.cursor_out[0] = to32(before + max(p.need - p.begin, 0)); }
    for (long i = tok + n + at; i < a.max_tokens; i += STEP) a.slots[i] = -1;
  }
}

extern "C" int unimp_page_tables_extend(int32_t* tables, int rows, int width, const int32_t* mapped, const int32_t* cached, const int32_t* fresh, const int32_t* cover,
                                        const int32_t* free_pages, int n_free, const int32_t* cursor, int group, const int32_t* shared_len, int32_t* mapped_out,
                                        int32_t* cursor_out, int64_t* slots, int64_t max_tokens, int32_t* cu, void* stream) {
  if (!tables || !mapped || !cached || !fresh || (!free_pages && n_free > 0) || !cursor || !mapped_out || !cursor_out || !cu || (max_tokens > 0 && !slots))
    return unimp_set_error(UNIMP_ERR_ARG, "page_tables_extend: null pointer");
  if (rows <= 0 || rows > 65536 || width <= 0 || n_free < 0 || max_tokens < 0 || group < 1 || (rows % group))      // every workgroup sums over the rows before it
    return unimp_set_error(UNIMP_ERR_SHAPE, "page_tables_extend: rows a positive multiple of group, at most 65536; width positive");
  if (mapped == mapped_out || cursor == cursor_out) return unimp_set_error(UNIMP_ERR_ARG, "page_tables_extend: the blocks read mapped and cursor throughout; outputs of their own");
  PageArgs a{tables, mapped, cached, fresh, cover, free_pages, cursor, shared_len, mapped_out, cursor_out, cu, slots, (long)max_tokens, rows, width, n_free, group};
  // a workgroup per row below 1 024 rows (600 rows x 300 tokens: 4.8 us against 6.1 for a wave per row; 1 000 x 1: 5.0 both, 2 000 x 1: 9.4 against 5.7, 4 000 x 2: 17.9 | 9.6)
  const int64_t share = max_tokens / ((int64_t)rows * 2048);
  if (rows < 1024) hipLaunchKernelGGL((page_tables_extend_kernel<1>), dim3(rows, (unsigned)(share < 1 ? 1 : share > 64 ? 64 : share)), dim3(256), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL((page_tables_extend_kernel<8>), dim3((rows + 7) / 8), dim3(512), 0, (hipStream_t)stream, a);
  return unimp_check_launch("page_tables_extend");
}

// ------------------------------------------------------------------------------------------- beam reorder
// Row j of a group goes on with the hypothesis of row src[j].  Its whole columns (all 32 tokens written) never change again: the table rows take the
// page ids over, and several rows may name one page.  Only the column that the next token goes to holds a page per row that must be copied; the K pages of a
// column are enough for ever, since a column's pages stop changing when it is full.  Thread (layer, 16-byte chunk) moves its chunk of all K rows through
// registers: in place, whatever the permutation.  Bound by the pages that move (80 beams x 32 layers x 32 heads x 80, 0.22 GB: 49 us, 4.5 TB/s); 5 beams 6 us.
template <int KMAX>
__global__ __launch_bounds__(256) void kv4_reorder_beams_kernel(uint8_t* __restrict__ pages, long layer_stride, long n_pages, long page_stride, int32_t* __restrict__ tables,
                                                                int width, int K, const int64_t* __restrict__ src, const int64_t* __restrict__ pos) {
  const int grp = blockIdx.z, tid = threadIdx.x;
  const int64_t p = pos[(long)grp * K];
  if (p < 0) return;
  const long now = p >> 5;
  int32_t* tab = tables + (long)grp * K * width;
  int from[KMAX];
#pragma unroll
  for (int j = 0; j < KMAX; ++j) {
    const int64_t s = j < K ? src[(long)grp * K + j] : j;
    from[j] = s >= 0 && s < K ? (int)s : j;
  }
  if (blockIdx.x == gridDim.x - 1) {                                 // the table rows: one block per group
    if (blockIdx.y) return;
    for (long c = tid; c < min(now, (long)width); c += 256) {
      int32_t e[KMAX];
#pragma unroll
      for (int j = 0; j < KMAX; ++j) if (j < K) e[j] = tab[(long)from[j] * width + c];
#pragma unroll
      for (int j = 0; j < KMAX; ++j) if (j < K) tab[(long)j * width + c] = e[j];
    }
    return;
  }
  if (!(p & 31) || now >= width) return;                             // nothing in the current page yet
  const long chunk = ((long)blockIdx.x * 256 + tid) * 16;
  if (chunk >= page_stride) return;
  uint8_t* base = pages + (long)blockIdx.y * layer_stride + chunk;
  u32x4 x[KMAX];
#pragma unroll
  for (int j = 0; j < KMAX; ++j) {
    const int32_t pg = j < K && from[j] != j ? tab[(long)from[j] * width + now] : -1;
    if (pg >= 0 && pg < n_pages) x[j] = *(const u32x4*)(base + pg * page_stride);
  }
#pragma unroll
  for (int j = 0; j < KMAX; ++j) if (j < K && from[j] != j) {
    const int32_t pf = tab[(long)from[j] * width + now], pg = tab[(long)j * width + now];
    if (pf >= 0 && pf < n_pages && pg >= 0 && pg < n_pages) *(u32x4*)(base + pg * page_stride) = x[j];
  }
}

extern "C" int unimp_kv4_reorder_beams(void* pages, int64_t layer_stride, int layers, int64_t n_pages, int heads, int hd, int32_t* tables, int width, int group,
                                       int n_groups, const int64_t* src_local, const int64_t* pos, void* stream) {
  const int pb = unimp_kv4_page_bytes(hd);
  if (pb < 0) return unimp_set_error(UNIMP_ERR_SHAPE, "kv4: head dim 64, 80 or 128");
  if (layers <= 0 || n_groups <= 0 || group <= 1 || width <= 0) return UNIMP_OK;          // empty tensors have no pointers
  if ((!pages && n_pages > 0 && heads > 0) || !tables || !src_local || !pos) return unimp_set_error(UNIMP_ERR_ARG, "kv4_reorder_beams: null pointer");
  if (group > 16 || layers > 65535 || n_groups > 65535) return unimp_set_error(UNIMP_ERR_SHAPE, "kv4_reorder_beams: at most 16 beams, 65535 layers and groups");
  if (((uintptr_t)pages | layer_stride) & 15) return unimp_set_error(UNIMP_ERR_ALIGN, "kv4_reorder_beams: 16-byte aligned pages and layer stride");
  const long stride = (long)heads * pb;
  dim3 grid((unsigned)((stride / 16 + 255) / 256 + 1), layers, n_groups);
#define KV4_REORDER(KM) hipLaunchKernelGGL((kv4_reorder_beams_kernel<KM>), grid, dim3(256), 0, (hipStream_t)stream, (uint8_t*)pages, (long)layer_stride, (long)n_pages, \
                                           stride, tables, width, group, src_local, pos)
  if (group <= 4) KV4_REORDER(4);
  else if (group <= 8) KV4_REORDER(8);
  else KV4_REORDER(16);
#undef KV4_REORDER
  return unimp_check_launch("kv4_reorder_beams");
}
