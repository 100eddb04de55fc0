// Attention of the newest tokens of every sequence over a paged cache (sm_100a).
//
// Row i < counts[b] of q stands at position p = len_b - counts_b + i and sees the keys j <= p:
//   out_i = sum_j softmax_j(scale q'_i . k'_j) v_j,  q' = [a cos f_p | a sin f_p | rest], k'_j = [a cos(f_j + b) | a sin(f_j + b) | rest],
//   a = softplus of the first r features.
// One CTA per (row, head, sequence): its threads take one key each, 128 at a time, with a running maximum and sum.
#include "kernels.h"
#include "paged.cuh"

namespace pope {

struct PagedAttnP {
  PagedPtrs c;
  int H, Nq, Nk, r;
  float scale_log2;
  const int32_t* counts;
  const float *freqs, *bias;
  int64_t sfn, bias_sh;
  const void* q;
  void* out;
  Strides sq, so;
  float* lse;
};

template <typename T, int STORE, int D>
__global__ void __launch_bounds__(128) paged_attn_kernel(PagedAttnP p) {
  __shared__ float qc[D], qs[D], prob[128], red[8];
  __shared__ int64_t rows[128];
  const int tid = threadIdx.x, i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h % p.c.Hk, r = p.r;
  pdl_wait();
  const int len = max(0, min(p.c.seq_lens[b], p.Nk)), cnt = p.counts ? max(0, min(p.counts[b], p.Nq)) : p.Nq;
  const int pos = len - cnt + i;
  const int end = i < cnt ? max(pos + 1, 0) : 0;
  const T* qrow = static_cast<const T*>(p.q) + b * p.sq.b + h * p.sq.h + (int64_t)i * p.sq.n;
  if (tid < D && end > 0) {
    float x = to_f32<T>(qrow[tid]), s = 0.f, c = 1.f;
    if (tid < r) x = softplus_f(x), sincosf(p.freqs[(int64_t)pos * p.sfn + tid], &s, &c);
    qc[tid] = x * c, qs[tid] = x * s;
  }
  float m = -CUDART_INF_F, l = 0.f, o = 0.f;
  for (int key0 = 0; key0 < end; key0 += 128) {
    __syncthreads();
    const int j = key0 + tid;
    float s = -CUDART_INF_F;
    rows[tid] = j < end ? paged_row(p.c, b, hk, j) : -1;
    if (rows[tid] >= 0) {
      const uint8_t* krow = p.c.k + rows[tid] * p.c.row_bytes;
      const float ks = STORE == POPE_STORE_16 ? 1.f : p.c.k_scales[rows[tid]];
      s = 0.f;
      for (int c = 0; c < D; c += 4) {
        float x[4];
        if constexpr (STORE == POPE_STORE_16) {
          for (int e = 0; e < 4; ++e) x[e] = to_f32<T>(reinterpret_cast<const T*>(krow)[c + e]);
        } else {
          codes_to_f32<STORE>(*reinterpret_cast<const uint32_t*>(krow + c), x);
        }
        for (int e = 0; e < 4; ++e) {
          float y = x[e] * ks;
          if (c + e < r) {
            float sn, cs, sb, cb;
            sincosf(p.freqs[(int64_t)j * p.sfn + c + e], &sn, &cs);
            sincosf(p.bias[hk * p.bias_sh + c + e], &sb, &cb);
            y = softplus_f(y);
            s += y * (cs * cb - sn * sb) * qc[c + e] + y * (sn * cb + cs * sb) * qs[c + e];
          } else {
            s += y * qc[c + e];
          }
        }
      }
      s *= p.scale_log2;
    }
    const float wm = warp_max(s);
    if (tid % 32 == 0) red[tid / 32] = wm;
    __syncthreads();
    const float mn = fmaxf(fmaxf(m, fmaxf(red[0], red[1])), fmaxf(red[2], red[3]));
    const float mu = mn == -CUDART_INF_F ? 0.f : mn, alpha = ex2_approx(m - mu), e = ex2_approx(s - mu);
    prob[tid] = e;
    const float ws = warp_sum(e);
    if (tid % 32 == 0) red[4 + tid / 32] = ws;
    __syncthreads();
    l = l * alpha + red[4] + red[5] + red[6] + red[7], o *= alpha, m = mn;
    if (tid < D) {
      for (int t = 0; t < min(128, end - key0); ++t) {
        if (rows[t] < 0) continue;
        const uint8_t* vrow = p.c.v + rows[t] * p.c.row_bytes;
        float x;
        if constexpr (STORE == POPE_STORE_16) {
          x = to_f32<T>(reinterpret_cast<const T*>(vrow)[tid]);
        } else {
          float w[4];
          codes_to_f32<STORE>(*reinterpret_cast<const uint32_t*>(vrow + tid / 4 * 4), w);
          x = (tid % 4 == 0 ? w[0] : tid % 4 == 1 ? w[1] : tid % 4 == 2 ? w[2] : w[3]) * p.c.v_scales[rows[t]];
        }
        o = fmaf(prob[t], x, o);
      }
    }
  }
  if (tid < D) static_cast<T*>(p.out)[b * p.so.b + h * p.so.h + (int64_t)i * p.so.n + tid] = from_f32<T>(l > 0.f || l != l ? o / l : 0.f);
  if (p.lse && tid == 0) p.lse[((int64_t)b * p.H + h) * p.Nq + i] = l > 0.f || l != l ? m * LN2 + logf(l) : -CUDART_INF_F;
}

bool attn_paged_supported(const PopePagedAttnArgs& a) {
  const PopeShape& s = a.shape;
  if (s.dtype != POPE_BF16 && s.dtype != POPE_F16) return false;
  if (s.d != 64 && s.d != 96 && s.d != 128) return false;
  if (s.r % 8 != 0 || (s.r > 0 && (a.embed.sf.b != 0 || a.embed.sf.h != 0))) return false;
  return a.cache.kv.page_size % 64 == 0;
}

// Rows that share a key head, up to which one pass over the keys per block of 32 is taken
static bool few_rows(const PopeShape& s) { return (int64_t)s.Nq * (s.H / s.Hk) <= 64; }

size_t attn_paged_workspace(const PopePagedAttnArgs& a) { return few_rows(a.shape) ? paged_rows_workspace(a) : 0; }

template <typename T, int STORE, int D> static cudaError_t paged_attn_t(const PopePagedAttnArgs& a, cudaStream_t st) {
  PagedAttnP p;
  p.c = paged_ptrs(a.cache, a.shape.Hk, a.shape.d);
  if (!p.c.status) return cudaErrorInvalidSymbol;
  p.H = a.shape.H, p.Nq = a.shape.Nq, p.Nk = a.shape.Nk, p.r = a.shape.r, p.scale_log2 = a.softmax_scale * LOG2E;
  p.counts = a.counts, p.freqs = a.embed.freqs, p.bias = a.embed.bias, p.sfn = a.embed.sf.n, p.bias_sh = a.embed.bias_stride_h;
  p.q = a.q, p.out = a.out, p.sq = Strides(a.sq), p.so = Strides(a.so), p.lse = a.lse;
  return launch_dependent(paged_attn_kernel<T, STORE, D>, dim3(p.Nq, p.H, a.shape.B), dim3(128), 0, st, p);
}
template <typename T, int STORE> static cudaError_t paged_attn_d(const PopePagedAttnArgs& a, cudaStream_t st) {
  const int d = a.shape.d;
  return d == 64 ? paged_attn_t<T, STORE, 64>(a, st) : d == 96 ? paged_attn_t<T, STORE, 96>(a, st) : paged_attn_t<T, STORE, 128>(a, st);
}
template <typename T> static cudaError_t paged_attn_s(const PopePagedAttnArgs& a, cudaStream_t st) {
  switch (a.cache.store) {
    case POPE_STORE_INT8: return paged_attn_d<T, POPE_STORE_INT8>(a, st);
    case POPE_STORE_E4M3: return paged_attn_d<T, POPE_STORE_E4M3>(a, st);
    default: return paged_attn_d<T, POPE_STORE_16>(a, st);
  }
}
cudaError_t attn_paged(const PopePagedAttnArgs& a, cudaStream_t st) {
  if (few_rows(a.shape)) return paged_rows(a, st);
  return a.shape.dtype == POPE_BF16 ? paged_attn_s<__nv_bfloat16>(a, st) : paged_attn_s<__half>(a, st);
}

}  // namespace pope
