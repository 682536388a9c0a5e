// Attention of one new token per row over the 4-bit pages (kv4.h): o = softmax(scale q k_j + slope j) v_j over the row's cached tokens j < len.
// (eval_rec.py:100-110 / eval_exp.py:103-113 / eval_img_gen.py:102-111: the cached decode step inside Flamingo.generate.)
#include "kv4.h"
#include "unimp_hip.h"

struct Kv4AttnArgs {
  const bf16* q; long q_rs, q_hs; const uint8_t* pages; long n_pages; int kv_heads; const int32_t* tables; long t_stride; int width; const int32_t* lens;
  int rows, heads; float scale; const float* alibi; bf16* o; long o_rs, o_hs; int group; const int32_t* shared;
};

// one block per (row, query head), a wave takes every fourth tile of 64 tokens: lane = token for the scores, lane = dim for the values
template <int D>
__global__ __launch_bounds__(256) void kv4_attn_kernel(Kv4AttnArgs a) {
  using P = Kv4<D>;
  __shared__ float qs[D], ps[4][64], part[4][D], pm[4], pl[4];
  __shared__ int pgs[4][2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.y, h = blockIdx.x, kvh = h / (a.heads / a.kv_heads);
  const int len = min(max(a.lens[row], 0), a.width * KV4_PAGE);
  for (int d = tid; d < D; d += 256) qs[d] = bf2f(a.q[row * a.q_rs + h * a.q_hs + d]) * a.scale * 1.4426950408889634f;
  __syncthreads();
  const float slope = a.alibi ? a.alibi[h] * 1.4426950408889634f : 0.f;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int base = w * 64; base < len; base += 256) {
    const int t = base + lane;
    int pg = t < len ? a.tables[row * a.t_stride + (t >> 5)] : -1;
    if (pg >= a.n_pages) pg = -1;
    if (!(lane & 31)) pgs[w][lane >> 5] = pg;
    float s = -INFINITY;
    if (pg >= 0) {
      const uint8_t* page = a.pages + ((long)pg * a.kv_heads + kvh) * P::BYTES;
      s = 0.f;
      for (int b = 0; b < P::NB; ++b) {
        const int nd = b == P::NB - 1 ? P::BLK_LAST : 32;
        float x = 0.f;
        for (int j = 0; j < nd; j += 8) {
          const uint32_t c = *(const uint32_t*)(page + P::k_byte(t & 31, b) + j / 2);
          for (int i = 0; i < 8; ++i) x = fmaf(kv4_value((c >> (4 * i)) & 15u), qs[32 * b + j + i], x);
        }
        s = fmaf(x, kv4_scale(page[P::ks_byte(t & 31, b)]), s);
      }
      s = fmaf(slope, (float)(t - len + 1), s);
    }
    const float mx = fmaxf(m, wave_max(s)), r = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
    const float p = pg < 0 ? 0.f : __builtin_amdgcn_exp2f(s - (mx == -INFINITY ? 0.f : mx));
    m = mx;
    l = fmaf(l, r, wave_sum(p));
    ps[w][lane] = p;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    o0 *= r; o1 *= r;
    for (int j = 0; j < 64; ++j) {
      const int pj = pgs[w][j >> 5];
      if (pj < 0 || base + j >= len) continue;
      const uint8_t* page = a.pages + ((long)pj * a.kv_heads + kvh) * P::BYTES;
      const int tt = j & 31, sh = 4 * kv4_nibble(tt);
      const float pp = ps[w][j];
      o0 = fmaf(pp, kv4_value((*(const uint32_t*)(page + P::v_dword(tt, lane)) >> sh) & 15u) * kv4_scale(page[P::vs_byte(tt, lane >> 5)]), o0);
      if (lane + 64 < D) o1 = fmaf(pp, kv4_value((*(const uint32_t*)(page + P::v_dword(tt, lane + 64)) >> sh) & 15u) * kv4_scale(page[P::vs_byte(tt, (lane + 64) >> 5)]), o1);
    }
    __builtin_amdgcn_wave_barrier();
  }
  part[w][lane] = o0;
  if (lane + 64 < D) part[w][lane + 64] = o1;
  if (!lane) { pm[w] = m; pl[w] = l; }
  __syncthreads();
  const float M = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]));
  for (int d = tid; d < D; d += 256) {
    float L = 0.f, x = 0.f;
    for (int i = 0; i < 4; ++i) {
      const float e = pm[i] == -INFINITY && pl[i] == 0.f ? 0.f : __builtin_amdgcn_exp2f(pm[i] - (M == -INFINITY ? 0.f : M));
      L = fmaf(pl[i], e, L); x = fmaf(part[i][d], e, x);
    }
    a.o[row * a.o_rs + h * a.o_hs + d] = f2bf(L == 0.f ? 0.f : x / L);
  }
}

extern "C" int64_t unimp_kv4_attn_workspace(const unimp_kv4_attn_desc*) { return 0; }

extern "C" int unimp_kv4_attn_decode(const unimp_kv4_attn_desc* d, float* workspace, void* stream) {
  (void)workspace;
  if (!d || !d->q || !d->pages || !d->tables || !d->lens || !d->out) return unimp_set_error(UNIMP_ERR_ARG, "kv4_attn_decode: null pointer");
  if (d->rows <= 0 || d->heads <= 0) return UNIMP_OK;
  if (d->kv_heads <= 0 || d->heads % d->kv_heads || d->heads / d->kv_heads > 16 || d->width < 0 || d->width > (1 << 26) || d->rows > 65535 || d->heads > 65535)
    return unimp_set_error(UNIMP_ERR_SHAPE, "kv4_attn_decode: query heads a multiple of the key heads, at most 16 to one; at most 65535 rows, 2^26 pages of a row");
  if (d->hd != 64 && d->hd != 80 && d->hd != 128) return unimp_set_error(UNIMP_ERR_SHAPE, "kv4: head dim 64, 80 or 128");
  if ((uintptr_t)d->pages & 15) return unimp_set_error(UNIMP_ERR_ALIGN, "kv4_attn_decode: 16-byte aligned pages");
  Kv4AttnArgs a{(const bf16*)d->q, d->q_row_stride, d->q_head_stride, (const uint8_t*)d->pages, d->n_pages, d->kv_heads, d->tables, d->table_stride, d->width, d->lens,
                d->rows, d->heads, d->scale, d->alibi_slopes, (bf16*)d->out, d->o_row_stride, d->o_head_stride, d->group, d->shared_len};
  dim3 grid(d->heads, d->rows);
  switch (d->hd) {
    case 64: hipLaunchKernelGGL((kv4_attn_kernel<64>), grid, dim3(256), 0, (hipStream_t)stream, a); break;
    case 80: hipLaunchKernelGGL((kv4_attn_kernel<80>), grid, dim3(256), 0, (hipStream_t)stream, a); break;
    case 128: hipLaunchKernelGGL((kv4_attn_kernel<128>), grid, dim3(256), 0, (hipStream_t)stream, a); break;
    default: return unimp_set_error(UNIMP_ERR_SHAPE, "kv4: head dim 64, 80 or 128");
  }
  return unimp_check_launch("kv4_attn_decode");
}
