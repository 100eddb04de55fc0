// Attention of FEW new tokens per sequence over a paged cache (sm_100a): one decode token over a cache that holds 8 bits, drafted
// tokens, the last short piece of a prompt.
//
// The query rows that share a key head -- the newest tokens of a sequence times the heads of the group -- are packed into blocks of
// 16 or 32 (row = token * group + head).  A call then is one pass over K and V, each key transformed once for all rows of the block:
//
//   loader warp    : tiles of 64 keys (K rows, V rows, fp16 cos / sin rows, row scales) through a ring of shared-memory stages, by
//                    tensor-map copies in 128-byte-swizzled rows; the page of a tile comes from the page table
//   8 worker warps : two groups of four take turns with the tiles, a warp owns 16 keys of a tile.  K' never exists in memory: a lane
//                    reads 16 bytes of a key and turns them into the B fragments of mma.sync m16n8k16 in its registers.  (The order of the
//                    features inside a product is free as long as Q' uses the same one, so a lane's fragment is made of the
//                    features that sit next to each other in its key.)  The scores' accumulator fragments are, as they are, the A
//                    fragments of P V.  Every warp keeps its own running (max, sum, output); they meet at the end.
//
// The tensor cores are used through mma.sync because the operand is made in registers: writing it to shared memory for tcgen05 would
// cost as much as the products of a 16-row block, which are a small part of the time either way.
//
// With q' = (a_q cos fq, a_q sin fq), k' = (a_k cos(fk + b), a_k sin(fk + b)) a rotated feature adds a_k (Qc cos fk + Qs sin fk),
// Qc = a_q cos(fq - b), Qs = a_q sin(fq - b): the head's bias sits in the query.
//
// 8-bit codes: K' and Q' are fp16 whatever the compute type (11 bits instead of 8).  Rows beyond 2^15 are brought down by a factor that
// returns with the scores.  V enters the products as its codes, exact in fp16, and its scale s_j goes into the probability:
// p_j s_j = 2^(score + log2 s_j - m), with m the running maximum of that sum, so that it stays in fp16's range whatever the scales
// are, while the softmax's own sum adds 2^(score - m) in fp32.
#include <algorithm>

#include "kernels.h"
#include "paged.cuh"

namespace pope {

struct PagedRowsP {
  int B, H, Hk, G, Nq, Nk, r, nsplit, nstages, blocks;   // G: query heads per key head; blocks: row blocks per (sequence, key head)
  int page_size, max_pages, num_pages;
  float scale_log2;
  const int32_t *page_table, *seq_lens, *counts;
  const float *k_scales, *v_scales;
  const float *freqs, *bias;
  int64_t sfn, bias_sh;
  const void* q;
  void* out;
  Strides sq, so;
  float* lse;
  float *part_o, *part_ml;   // [unit][split][row][D] and [unit][split][row][max (log2 units), sum]
  unsigned int *done, *status;
};

constexpr int PR_TILE = 64, PR_NW = 8, PR_MAX_SPLIT = 64, PR_BLOCK = PR_TILE * 128;   // PR_BLOCK: 64 rows of 128 bytes

template <typename TM> __device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t saddr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(saddr)
               : "memory");
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 v = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}
// softplus(x) / ln 2 = max(y, 0) + log2(1 + 2^-|y|), y = x log2(e)
__device__ __forceinline__ float softplus_log2(float y) { return fmaxf(y, 0.f) + lg2_approx(1.f + ex2_approx(-fabsf(y))); }

// Four codes of each of two keys, first features first -> fp16 pairs (key 0, key 1) of the four features
template <int STORE> __device__ __forceinline__ void code_pairs(uint32_t a, uint32_t b, uint32_t (&h)[4]) {
  if constexpr (STORE == POPE_STORE_INT8) a ^= 0x80808080u, b ^= 0x80808080u;
  const uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);
  if constexpr (STORE == POPE_STORE_INT8) {
    // 1024 + (code + 128), exact, minus 1152
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const uint32_t m[4] = {__byte_perm(lo, 0x64646464u, 0x4140), __byte_perm(lo, 0x64646464u, 0x4342), __byte_perm(hi, 0x64646464u, 0x4140),
                           __byte_perm(hi, 0x64646464u, 0x4342)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&m[i]), off);
      h[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  } else {
    const uint32_t m[4] = {lo & 0xffffu, lo >> 16, hi & 0xffffu, hi >> 16};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw v = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)m[i], __NV_E4M3);
      h[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
}

constexpr float PR_BIG = 32768.f;   // magnitudes of fp16 operands stay below twice this

template <typename T, int STORE, int D, int MT>
__global__ void __launch_bounds__(32 * (PR_NW + 1), 1)
    paged_rows_kernel(PagedRowsP p, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                      const __grid_constant__ CUtensorMap tmap_t) {
  constexpr bool Q8 = STORE != POPE_STORE_16;
  using TM = std::conditional_t<Q8, __half, T>;            // operand type of the products
  constexpr bool HALF = std::is_same_v<TM, __half>;
  constexpr int RB = 16 * MT;
  constexpr int VL = Q8 ? 16 : 8;                          // features in a lane's 16 bytes of a key
  constexpr int FPI = 4 * VL;                              // features of a key that its four lanes read together
  constexpr int NI = (D + FPI - 1) / FPI, DP = NI * FPI;
  constexpr int NH = VL / 8;
  constexpr int KBLK = (D * (Q8 ? 1 : 2) + 127) / 128;     // 128-byte blocks of a row
  constexpr int EPB = Q8 ? 128 : 64;                       // elements of one
  constexpr int NT = D / 8;                                // output column tiles
  constexpr int FL = D / 8;                                // 8-bit V: neighbouring features of a lane

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int r = p.r, tblk = (r + 63) / 64, RP = (r + FPI - 1) / FPI * FPI;
  const int stage_bytes = (2 * KBLK + 2 * tblk) * PR_BLOCK + (Q8 ? 1024 : 0);
  const int pitch = (DP + RP) * 2 + ((DP + RP) % 64 == 0 ? 64 : 0);   // an odd multiple of 64 bytes: eight rows x 64 bytes on distinct banks
  const size_t ring = (size_t)p.nstages * stage_bytes, red_bytes = (size_t)PR_NW * RB * D * 4;
  uint8_t* qsm = smem + (ring > red_bytes ? ring : red_bytes);        // Q': [RB] rows of (cos or plain features, sin features)
  float* red_ml = reinterpret_cast<float*>(qsm + RB * pitch);         // [PR_NW][RB][2]
  float* row_scale = red_ml + PR_NW * RB * 2;                         // [RB] what was taken off a row of Q'
  int* row_pos = reinterpret_cast<int*>(row_scale + RB);              // [RB] position, -1 = no row
  float* bias_cs = reinterpret_cast<float*>(row_pos + RB);            // [2][r]
  uint64_t* full = reinterpret_cast<uint64_t*>(bias_cs + 2 * r);
  uint64_t* empty = full + p.nstages;
  unsigned int* last_s = reinterpret_cast<unsigned int*>(empty + p.nstages);

  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int split = blockIdx.x % p.nsplit, u = blockIdx.x / p.nsplit;
  const int rb = u % p.blocks, bk = u / p.blocks, hk = bk % p.Hk, b = bk / p.Hk;
  if (tid == 0) {
    for (int s = 0; s < p.nstages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], PR_NW / 2);
    mbar_init_fence();
  }
  pdl_wait();
  const int len = max(0, min(p.seq_lens[b], p.Nk)), cnt = p.counts ? max(0, min(p.counts[b], p.Nq)) : p.Nq;
  const int rows = min(RB, cnt * p.G - rb * RB);                                       // of this block that are queries (may be negative)
  const int first_pos = len - cnt + rb * RB / p.G;                                     // position of the first one
  const int kend = rows > 0 ? max(0, min(len, len - cnt + (rb * RB + rows - 1) / p.G + 1)) : 0;   // keys that the last one sees
  const int tiles_all = (kend + PR_TILE - 1) / PR_TILE;
  const int kb = (int)((int64_t)tiles_all * split / p.nsplit) * PR_TILE;
  const int ke = min(kend, (int)((int64_t)tiles_all * (split + 1) / p.nsplit) * PR_TILE);
  const int T_tiles = ke > kb ? (ke - kb + PR_TILE - 1) / PR_TILE : 0;
  __syncthreads();
  bool failed = false;

  if (w == PR_NW) {
    // =============================== loader =====================================================
    const uint32_t bytes = (uint32_t)(2 * KBLK + 2 * tblk) * PR_BLOCK + (Q8 ? 512 : 0);
    int page = 0;
    for (int jt = 0, s = 0, par = 0; jt < T_tiles; ++jt) {
      if ((jt & 31) == 0) {   // pages of the next 32 tiles; one outside the pool is never dereferenced (clamped, status bit 1)
        const int mine = jt + lane, lp = (kb + mine * PR_TILE) / p.page_size;
        page = 0;
        if (mine < T_tiles) {
          page = lp < p.max_pages ? p.page_table[(int64_t)b * p.max_pages + lp] : -1;
          if (page < 0 || page >= p.num_pages) page = 0, atomicOr(p.status, 2u);
        }
      }
      const int pg = __shfl_sync(0xffffffffu, page, jt & 31);
      if (lane == 0) {
        if (jt >= p.nstages) {
          failed = !mbar_wait(&empty[s], par ^ 1, WAIT_LIMIT);
          if (failed) drain_copies(full, p.nstages, jt - p.nstages, jt);
        }
        if (!failed) {
          const int key0 = kb + jt * PR_TILE, row = key0 % p.page_size;
          uint8_t* st = smem + (size_t)s * stage_bytes;
          mbar_expect_tx(&full[s], bytes);
#pragma unroll
          for (int c = 0; c < KBLK; ++c) tma_load_4d(st + c * PR_BLOCK, &tmap_k, &full[s], c * EPB, row, hk, pg);
          uint8_t* tt = st + 2 * KBLK * PR_BLOCK;
          for (int c = 0; c < tblk; ++c) {
            tma_load_4d(tt + c * PR_BLOCK, &tmap_t, &full[s], c * 64, key0, 0, 0);
            tma_load_4d(tt + (tblk + c) * PR_BLOCK, &tmap_t, &full[s], c * 64, key0, 1, 0);
          }
          if constexpr (Q8) {
            const int64_t at = ((int64_t)pg * p.Hk + hk) * p.page_size + row;
            uint8_t* sc = tt + 2 * tblk * PR_BLOCK;
            bulk_load(sc, p.k_scales + at, 256, &full[s]), bulk_load(sc + 256, p.v_scales + at, 256, &full[s]);
          }
#pragma unroll
          for (int c = 0; c < KBLK; ++c) tma_load_4d(st + (KBLK + c) * PR_BLOCK, &tmap_v, &full[s], c * EPB, row, hk, pg);
        }
      }
      failed = __shfl_sync(0xffffffffu, (int)failed, 0) != 0;
      if (failed) break;
      if (++s == p.nstages) s = 0, par ^= 1;
    }
    if (failed && lane == 0) atomicOr(p.status, 1u);
    return;   // nothing below is a block-wide barrier
  }

  // =============================== workers ======================================================
  auto worker_sync = []() { asm volatile("bar.sync 1, %0;" ::"n"(32 * PR_NW) : "memory"); };
  for (int c = tid; c < r; c += 32 * PR_NW) sincosf(p.bias[hk * p.bias_sh + c], &bias_cs[r + c], &bias_cs[c]);
  worker_sync();
  for (int row = w; row < RB; row += PR_NW) {   // a warp per row of Q'
    const int rho = rb * RB + row, i = rho / p.G, head = hk + (rho - i * p.G) * p.Hk, pos = len - cnt + i;
    const bool live = row < rows && pos >= 0;
    const T* qrow = static_cast<const T*>(p.q) + b * p.sq.b + head * p.sq.h + (int64_t)i * p.sq.n;
    float qc[DP / 32], qs[DP / 32], mx = 0.f;
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) {
      const int c = lane + 32 * j;
      qc[j] = live && c < D ? to_f32<T>(qrow[c]) : 0.f, qs[j] = 0.f;
      if (live && c < r) {
        float sn, cs;
        sincosf(p.freqs[(int64_t)pos * p.sfn + c], &sn, &cs);
        const float a = softplus_f(qc[j]) * (HALF ? 1.f : LN2);   // (the bf16 keys' magnitudes come in units of ln 2)
        qc[j] = a * (cs * bias_cs[c] + sn * bias_cs[r + c]), qs[j] = a * (sn * bias_cs[c] - cs * bias_cs[r + c]);
      }
      mx = fmaxf(mx, fmaxf(fabsf(qc[j]), fabsf(qs[j])));
    }
    float down = 1.f;
    if constexpr (Q8) {
      mx = warp_max(mx);
      if (mx > PR_BIG && mx < CUDART_INF_F) down = PR_BIG / mx;
    }
    TM* dst = reinterpret_cast<TM*>(qsm + row * pitch);
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) {
      const int c = lane + 32 * j;
      dst[c] = from_f32<TM>(qc[j] * down);
      if (c < RP) dst[DP + c] = from_f32<TM>(qs[j] * down);
    }
    if (lane == 0) row_scale[row] = p.scale_log2 / down, row_pos[row] = live ? pos : -1;
  }
  worker_sync();

  const int g = lane >> 2, t = lane & 3, sub = w & 3;
  const uint8_t* qlane = qsm + g * pitch + t * (VL * 2);
  constexpr bool QREG = MT == 1;
  uint4 qreg_c[QREG ? NI : 1][NH][2], qreg_s[QREG ? NI : 1][NH][2];   // the A fragments, eight features of rows g and g + 8 each
  if constexpr (QREG) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint8_t* a = qlane + e * 8 * pitch + (i * FPI + h * 8) * 2;
          qreg_c[i][h][e] = *reinterpret_cast<const uint4*>(a);
          qreg_s[i][h][e] = i * FPI < r ? *reinterpret_cast<const uint4*>(a + DP * 2) : make_uint4(0, 0, 0, 0);
        }
  }
  int pos_of[MT][2];
  float sc_of[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) pos_of[m][e] = row_pos[m * 16 + e * 8 + g], sc_of[m][e] = row_scale[m * 16 + e * 8 + g];
  float m_run[MT][2], l_run[MT][2], o[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    m_run[m][0] = m_run[m][1] = -CUDART_INF_F, l_run[m][0] = l_run[m][1] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[m][n][e] = 0.f;
  }

  int s = (w >> 2) % p.nstages;
  uint32_t par = 0;
  for (int jt = w >> 2; jt < T_tiles; jt += 2) {
    const int key0 = kb + jt * PR_TILE + sub * 16;   // first key of this warp
    uint8_t* st = smem + (size_t)s * stage_bytes;
    const uint8_t* tt = st + 2 * KBLK * PR_BLOCK;
    const float* scl = reinterpret_cast<const float*>(tt + 2 * tblk * PR_BLOCK);
    if (!mbar_wait(&full[s], par, WAIT_LIMIT)) {
      failed = true;
      break;
    }
    // ---- scores: two tiles of eight keys ------------------------------------------------------------
    float sco[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sco[m][n][e] = 0.f;
    float ks[2] = {1.f, 1.f}, kd[2] = {1.f, 1.f};   // 8-bit: a key's scale, and the factor that brings its operands down
    if constexpr (Q8) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        ks[n] = scl[sub * 16 + n * 8 + g];
        const float top = ks[n] * kCodeTop<STORE>;
        kd[n] = top > PR_BIG ? PR_BIG / top : 1.f;
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int ch = 4 * i + t;
      const bool rot_i = i * FPI < r;   // (the same for all lanes)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int row = sub * 16 + n * 8 + g;
        const uint4 raw = *reinterpret_cast<const uint4*>(st + (ch >> 3) * PR_BLOCK + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
        const uint32_t rw[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const int f0 = ch * VL + h * 8;   // first of the lane's eight features
          uint32_t kc[4], kn[4];            // fragments: features (f0, f0 + 1), ...
          if (!rot_i) {
            if constexpr (!Q8) {
#pragma unroll
              for (int e = 0; e < 4; ++e) kc[e] = rw[e];
            } else {
              const float f = ks[n] * kd[n];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float x[4];
                codes_to_f32<STORE>(rw[h * 2 + e], x);
                kc[2 * e] = pack2<__half>(x[0] * f, x[1] * f), kc[2 * e + 1] = pack2<__half>(x[2] * f, x[3] * f);
              }
            }
          } else {
            const bool rot = f0 < r;
            const uint8_t* trow = tt + (f0 >> 6) * PR_BLOCK + row * 128 + ((((f0 >> 3) & 7) ^ (row & 7)) << 4);
            uint4 cr = *reinterpret_cast<const uint4*>(trow);
            const uint4 sr = *reinterpret_cast<const uint4*>(trow + tblk * PR_BLOCK);   // (zeros where nothing is rotated)
            if (!rot) cr = make_uint4(0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u);
            const uint32_t cw[4] = {cr.x, cr.y, cr.z, cr.w}, sw[4] = {sr.x, sr.y, sr.z, sr.w};
            float x[8];
            if constexpr (!Q8) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 v = unpack2<T>(rw[e]);
                x[2 * e] = v.x, x[2 * e + 1] = v.y;
              }
            } else {
              codes_to_f32<STORE>(rw[h * 2], *reinterpret_cast<float(*)[4]>(x));
              codes_to_f32<STORE>(rw[h * 2 + 1], *reinterpret_cast<float(*)[4]>(x + 4));
            }
            const float unit = ks[n] * LOG2E, back = HALF ? LN2 * kd[n] : 1.f, plain = ks[n] * kd[n];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float a = softplus_log2(x[e] * unit) * back;
              x[e] = rot ? a : x[e] * plain;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (HALF) {
                const uint32_t a = pack2<__half>(x[2 * e], x[2 * e + 1]);
                kc[e] = hmul2(a, cw[e]), kn[e] = hmul2(a, sw[e]);
              } else {
                const float2 c = unpack2<__half>(cw[e]), v = unpack2<__half>(sw[e]);
                kc[e] = pack2<TM>(x[2 * e] * c.x, x[2 * e + 1] * c.y), kn[e] = pack2<TM>(x[2 * e] * v.x, x[2 * e + 1] * v.y);
              }
            }
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            uint4 a0, a1;
            const uint8_t* qa = qlane + m * 16 * pitch + (i * FPI + h * 8) * 2;
            if constexpr (QREG) a0 = qreg_c[i][h][0], a1 = qreg_c[i][h][1];
            else a0 = *reinterpret_cast<const uint4*>(qa), a1 = *reinterpret_cast<const uint4*>(qa + 8 * pitch);
            mma16816<TM>(sco[m][n], a0.x, a1.x, a0.y, a1.y, kc[0], kc[1]);
            mma16816<TM>(sco[m][n], a0.z, a1.z, a0.w, a1.w, kc[2], kc[3]);
            if (rot_i) {
              if constexpr (QREG) a0 = qreg_s[i][h][0], a1 = qreg_s[i][h][1];
              else a0 = *reinterpret_cast<const uint4*>(qa + DP * 2), a1 = *reinterpret_cast<const uint4*>(qa + DP * 2 + 8 * pitch);
              mma16816<TM>(sco[m][n], a0.x, a1.x, a0.y, a1.y, kn[0], kn[1]);
              mma16816<TM>(sco[m][n], a0.z, a1.z, a0.w, a1.w, kn[2], kn[3]);
            }
          }
        }
      }
    }
    // ---- softmax: rows g and g + 8, keys 2 t, 2 t + 1 of both tiles -----------------------------------
    float kup[2][2], vs[2][2], lvs[2][2];
    if constexpr (Q8) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float2 k2 = *reinterpret_cast<const float2*>(scl + sub * 16 + n * 8 + 2 * t);
        const float2 v2 = *reinterpret_cast<const float2*>(scl + 64 + sub * 16 + n * 8 + 2 * t);
        kup[n][0] = fmaxf(1.f, k2.x * (kCodeTop<STORE> / PR_BIG)), kup[n][1] = fmaxf(1.f, k2.y * (kCodeTop<STORE> / PR_BIG));
        vs[n][0] = v2.x, vs[n][1] = v2.y;
        lvs[n][0] = fmaxf(lg2_approx(v2.x), -100.f), lvs[n][1] = fmaxf(lg2_approx(v2.y), -100.f);
      }
    }
    const bool clean = key0 + 16 <= min(ke, first_pos + 1);   // every row sees every key of this warp
    uint32_t pa[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float mx[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = sco[m][n][e] * sc_of[m][e >> 1];
          if constexpr (Q8) v *= kup[n][e & 1];
          if (!clean && key0 + n * 8 + 2 * t + (e & 1) > min(ke - 1, pos_of[m][e >> 1])) v = -CUDART_INF_F;
          sco[m][n][e] = v;
          mx[e >> 1] = fmaxf(mx[e >> 1], Q8 ? v + lvs[n][e & 1] : v);
        }
      // the maximum may lag by 2^8: most tiles then need neither a reduction nor a rescale
      if (__any_sync(0xffffffffu, mx[0] > m_run[m][0] + 8.f || mx[1] > m_run[m][1] + 8.f)) {
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
          mx[e] = fmaxf(mx[e], m_run[m][e]);
          alpha[e] = mx[e] == -CUDART_INF_F ? 1.f : ex2_approx(m_run[m][e] - mx[e]);
          m_run[m][e] = mx[e], l_run[m][e] *= alpha[e];
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[m][n][e] *= alpha[e >> 1];
      }
      float pr[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float mu = m_run[m][e >> 1];
          const float x = ex2_approx(sco[m][n][e] - (mu == -CUDART_INF_F ? 0.f : mu));
          l_run[m][e >> 1] += x;
          pr[n][e] = x;
          if constexpr (Q8) pr[n][e] = sco[m][n][e] == -CUDART_INF_F ? 0.f : x * vs[n][e & 1];   // (unused rows may have any scale)
        }
      pa[m][0] = pack2<TM>(pr[0][0], pr[0][1]), pa[m][1] = pack2<TM>(pr[0][2], pr[0][3]);
      pa[m][2] = pack2<TM>(pr[1][0], pr[1][1]), pa[m][3] = pack2<TM>(pr[1][2], pr[1][3]);
    }
    // ---- O += P V --------------------------------------------------------------------------------------
    uint8_t* vt = st + KBLK * PR_BLOCK;
    if constexpr (!Q8) {
      if (key0 + 16 > ke) {   // rows behind the last key may hold anything, and 0 * NaN is NaN
        const int dead = min(16, key0 + 16 - ke);
        for (int i = lane; i < dead * KBLK * 8; i += 32)
          *reinterpret_cast<uint4*>(vt + (i / 8 / dead) * PR_BLOCK + (sub * 16 + 16 - dead + i / 8 % dead) * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      const int row = sub * 16 + (lane & 15);
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t bf[4];
        const int ch = n + (lane >> 4);
        ldmatrix_x4_trans(bf, smem_u32(vt + (ch >> 3) * PR_BLOCK + row * 128 + (((ch & 7) ^ (row & 7)) << 4)));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          mma16816<TM>(o[m][n], pa[m][0], pa[m][1], pa[m][2], pa[m][3], bf[0], bf[1]);
          mma16816<TM>(o[m][n + 1], pa[m][0], pa[m][1], pa[m][2], pa[m][3], bf[2], bf[3]);
        }
      }
    } else {
      uint32_t vw[4][FL / 4];   // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9: features FL g ...
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = sub * 16 + 2 * t + (i & 1) + (i >> 1) * 8;
        const uint8_t* vrow = vt + row * 128;
        if constexpr (FL == 16) {
          const uint4 x = *reinterpret_cast<const uint4*>(vrow + ((g ^ (row & 7)) << 4));
          vw[i][0] = x.x, vw[i][1] = x.y, vw[i][2] = x.z, vw[i][3] = x.w;
        } else if constexpr (FL == 8) {
          const uint2 x = *reinterpret_cast<const uint2*>(vrow + (((g >> 1) ^ (row & 7)) << 4) + (g & 1) * 8);
          vw[i][0] = x.x, vw[i][1] = x.y;
        } else {
#pragma unroll
          for (int c = 0; c < FL / 4; ++c) {
            const int off = g * FL + 4 * c;
            vw[i][c] = *reinterpret_cast<const uint32_t*>(vrow + (((off >> 4) ^ (row & 7)) << 4) + (off & 15));
          }
        }
      }
#pragma unroll
      for (int c = 0; c < FL / 4; ++c) {
        uint32_t lo[4], hi[4];
        code_pairs<STORE>(vw[0][c], vw[1][c], lo), code_pairs<STORE>(vw[2][c], vw[3][c], hi);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int m = 0; m < MT; ++m) mma16816<TM>(o[m][4 * c + e], pa[m][0], pa[m][1], pa[m][2], pa[m][3], lo[e], hi[e]);
      }
    }
    fence_async_smem();   // the tile has been read: the loader's next copy may write over it
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
    if ((s += 2) >= p.nstages) s -= p.nstages, par ^= 1;
  }
  if (failed && lane == 0) atomicOr(p.status, 1u);

  // ---- the warps' results meet ---------------------------------------------------------------------
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l_run[m][e] += __shfl_xor_sync(0xffffffffu, l_run[m][e], 1);
      l_run[m][e] += __shfl_xor_sync(0xffffffffu, l_run[m][e], 2);
      // (a lane's maximum is its row's: it changes for all four lanes of the row together)
      if (t == 0) red_ml[(w * RB + m * 16 + e * 8 + g) * 2] = m_run[m][e], red_ml[(w * RB + m * 16 + e * 8 + g) * 2 + 1] = l_run[m][e];
    }
  worker_sync();   // every tile has been read: the ring takes the warps' outputs
  float* red_o = reinterpret_cast<float*>(smem) + (size_t)w * RB * D;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = Q8 ? (2 * t + (e & 1)) * FL + n : n * 8 + 2 * t + (e & 1);
        red_o[(m * 16 + (e >> 1) * 8 + g) * D + c] = o[m][n][e];
      }
  worker_sync();
  auto write_out = [&](int row, int c, float x) {
    const int rho = rb * RB + row, i = rho / p.G, head = hk + (rho - i * p.G) * p.Hk;
    static_cast<T*>(p.out)[b * p.so.b + head * p.so.h + (int64_t)i * p.so.n + c] = from_f32<T>(x);
  };
  auto write_lse = [&](int row, float M, float L) {
    const int rho = rb * RB + row, i = rho / p.G, head = hk + (rho - i * p.G) * p.Hk;
    if (p.lse) p.lse[((int64_t)b * p.H + head) * p.Nq + i] = L != 0.f ? M * LN2 + logf(L) : -CUDART_INF_F;
  };
  const int out_rows = min(RB, p.Nq * p.G - rb * RB);   // (padding is written too)
  const int64_t slot = ((int64_t)u * p.nsplit + split) * RB;
  for (int i = tid; i < out_rows * D; i += 32 * PR_NW) {
    const int row = i / D, c = i - row * D;
    float M = -CUDART_INF_F, L = 0.f, acc = 0.f;
#pragma unroll
    for (int ww = 0; ww < PR_NW; ++ww) M = fmaxf(M, red_ml[(ww * RB + row) * 2]);
    const float mu = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
    for (int ww = 0; ww < PR_NW; ++ww) {
      const float f = ex2_approx(red_ml[(ww * RB + row) * 2] - mu);   // 0 for a warp without visible keys
      L = fmaf(red_ml[(ww * RB + row) * 2 + 1], f, L), acc = fmaf(reinterpret_cast<const float*>(smem)[(size_t)(ww * RB + row) * D + c], f, acc);
    }
    if (row_pos[row] < 0) M = -CUDART_INF_F, L = acc = 0.f;   // (where every query sees every key the other rows of the block were not told apart)
    if (p.nsplit == 1) {
      write_out(row, c, L != 0.f ? acc / L : 0.f);
      if (c == 0) write_lse(row, M, L);
    } else {
      p.part_o[(slot + row) * D + c] = acc;
      if (c == 0) p.part_ml[(slot + row) * 2] = M, p.part_ml[(slot + row) * 2 + 1] = L;
    }
  }
  if (p.nsplit == 1) return;
  // The CTA that finishes last merges the splits of its unit.
  __threadfence();
  worker_sync();
  if (tid == 0) *last_s = atomicAdd(p.done + u, 1u) == (unsigned)p.nsplit - 1u;
  worker_sync();
  if (!*last_s) return;
  __threadfence();
  float* wgt = reinterpret_cast<float*>(smem);   // [RB][nsplit] weights of the splits
  const int64_t slot0 = (int64_t)u * p.nsplit * RB;
  for (int row = w; row < out_rows; row += PR_NW) {
    float m2[PR_MAX_SPLIT / 32], l2[PR_MAX_SPLIT / 32], M = -CUDART_INF_F, L = 0.f;
#pragma unroll
    for (int i = 0; i < PR_MAX_SPLIT / 32; ++i) {
      const int sp = lane + 32 * i;
      const float2 ml = sp < p.nsplit ? __ldcg(reinterpret_cast<const float2*>(p.part_ml + (slot0 + (int64_t)sp * RB + row) * 2))
                                      : make_float2(-CUDART_INF_F, 0.f);
      m2[i] = ml.x, l2[i] = ml.y, M = fmaxf(M, ml.x);
    }
    M = warp_max(M);
    const float mu = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
    for (int i = 0; i < PR_MAX_SPLIT / 32; ++i) {
      m2[i] = ex2_approx(m2[i] - mu);
      L += m2[i] * l2[i];
    }
    L = warp_sum(L);
#pragma unroll
    for (int i = 0; i < PR_MAX_SPLIT / 32; ++i)
      if (lane + 32 * i < p.nsplit) wgt[row * p.nsplit + lane + 32 * i] = m2[i];
    if (lane == 0) red_ml[row] = L, write_lse(row, M, L);
  }
  worker_sync();
  for (int i = tid; i < out_rows * D; i += 32 * PR_NW) {
    const int row = i / D, c = i - row * D;
    float acc = 0.f;
#pragma unroll 8
    for (int sp = 0; sp < p.nsplit; ++sp) acc = fmaf(wgt[row * p.nsplit + sp], __ldcg(p.part_o + (slot0 + (int64_t)sp * RB + row) * D + c), acc);
    write_out(row, c, red_ml[row] != 0.f ? acc / red_ml[row] : 0.f);
  }
}

// ---- host side ---------------------------------------------------------------------------------------
static int rows_mt(const PopeShape& s) { return (int64_t)s.Nq * (s.H / s.Hk) > 16 ? 2 : 1; }
static int rows_blocks(const PopeShape& s) {
  const int64_t rows = (int64_t)s.Nq * (s.H / s.Hk);
  return (int)((rows + 16 * rows_mt(s) - 1) / (16 * rows_mt(s)));
}

// Key ranges per unit: whole waves of one CTA per SM times a CTA's tiles plus what it costs beside them (about four tiles' time).
static int rows_split(const PopeShape& s) {
  const int tiles = (s.Nk + PR_TILE - 1) / PR_TILE;
  const int64_t units = (int64_t)s.B * s.Hk * rows_blocks(s);
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int n = 1; n <= std::min(tiles, PR_MAX_SPLIT); ++n) {
    const int64_t cost = (units * n + 147) / 148 * ((tiles + n - 1) / n + 4);
    if (cost < best_cost) best = n, best_cost = cost;
  }
  return best;
}

// workspace: [counters][partial outputs][partial max, sum][fp16 cos / sin tables]
struct RowsWs {
  size_t part_o, part_ml, table, total;
};
static RowsWs rows_ws(const PopeShape& s) {
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t units = (size_t)s.B * s.Hk * rows_blocks(s), slots = units * rows_split(s) * 16 * rows_mt(s);
  RowsWs w;
  w.part_o = up(units * sizeof(unsigned int));
  w.part_ml = w.part_o + up(slots * s.d * sizeof(float));
  w.table = w.part_ml + up(slots * 2 * sizeof(float));
  w.total = w.table + up((size_t)s.Nk * s.r * 4);
  return w;
}
size_t paged_rows_workspace(const PopePagedAttnArgs& a) { return rows_ws(a.shape).total; }

template <typename T, int STORE, int D, int MT> static cudaError_t paged_rows_t(const PopePagedAttnArgs& a, cudaStream_t st) {
  constexpr bool Q8 = STORE != POPE_STORE_16;
  const PopeShape& s = a.shape;
  const PopePagedKV& kv = a.cache.kv;
  const RowsWs ws = rows_ws(s);
  uint8_t* base = static_cast<uint8_t*>(a.workspace);
  __half* table = reinterpret_cast<__half*>(base + ws.table);
  PagedRowsP p = {};
  p.B = s.B, p.H = s.H, p.Hk = s.Hk, p.G = s.H / s.Hk, p.Nq = s.Nq, p.Nk = s.Nk, p.r = s.r, p.nsplit = rows_split(s), p.blocks = rows_blocks(s);
  p.page_size = kv.page_size, p.max_pages = kv.max_pages_per_seq, p.num_pages = kv.num_pages;
  p.scale_log2 = a.softmax_scale * LOG2E;
  p.page_table = kv.page_table, p.seq_lens = kv.seq_lens, p.counts = a.counts;
  p.k_scales = a.cache.k_scales, p.v_scales = a.cache.v_scales;
  p.freqs = a.embed.freqs, p.bias = a.embed.bias, p.sfn = a.embed.sf.n, p.bias_sh = a.embed.bias_stride_h;
  p.q = a.q, p.out = a.out, p.sq = Strides(a.sq), p.so = Strides(a.so), p.lse = a.lse;
  p.done = reinterpret_cast<unsigned int*>(base);
  p.part_o = reinterpret_cast<float*>(base + ws.part_o), p.part_ml = reinterpret_cast<float*>(base + ws.part_ml);
  p.status = tc_status_ptr();
  if (!p.status) return cudaErrorInvalidSymbol;

  CUtensorMap mk, mv, mt;
  const bool bf16 = s.dtype == POPE_BF16;
  const int64_t row = s.d, head = row * kv.page_size, page = head * s.Hk;
  bool ok;
  if constexpr (Q8) {
    ok = make_code_tmap(&mk, kv.k_pages, s.d, kv.page_size, s.Hk, kv.num_pages, row, head, page, PR_TILE) &&
         make_code_tmap(&mv, kv.v_pages, s.d, kv.page_size, s.Hk, kv.num_pages, row, head, page, PR_TILE);
  } else {
    ok = make_wide_tmap(&mk, kv.k_pages, bf16, s.d, kv.page_size, s.Hk, kv.num_pages, row, head, page, PR_TILE) &&
         make_wide_tmap(&mv, kv.v_pages, bf16, s.d, kv.page_size, s.Hk, kv.num_pages, row, head, page, PR_TILE);
  }
  // (without rotated features nothing is copied through the third map)
  ok = ok && (s.r > 0 ? make_wide_tmap(&mt, table, false, s.r, s.Nk, 2, 1, s.r, (int64_t)s.Nk * s.r, 0, PR_TILE) : (mt = mk, true));
  if (!ok) return cudaErrorNotSupported;

  constexpr int RB = 16 * MT, FPI = Q8 ? 64 : 32, DP = (D + FPI - 1) / FPI * FPI, KBLK = (D * (Q8 ? 1 : 2) + 127) / 128;
  const int tblk = (s.r + 63) / 64, RP = (s.r + FPI - 1) / FPI * FPI;
  const size_t stage = (size_t)(2 * KBLK + 2 * tblk) * PR_BLOCK + (Q8 ? 1024 : 0), red = (size_t)PR_NW * RB * D * 4;
  const size_t pitch = (DP + RP) * 2 + ((DP + RP) % 64 == 0 ? 64 : 0);
  const size_t fixed = 1024 + RB * pitch + (size_t)PR_NW * RB * 8 + RB * 8 + 2 * (size_t)s.r * 4 + 2 * 8 * 8 + 64;
  int nst = (int)((kMaxDynamicSmem - fixed) / stage);
  p.nstages = nst > 8 ? 8 : nst;
  if (p.nstages < 2) return cudaErrorInvalidValue;
  const size_t smem = fixed + std::max(p.nstages * stage, red);
  if (smem > (size_t)kMaxDynamicSmem) return cudaErrorInvalidValue;
  const auto kernel = paged_rows_kernel<T, STORE, D, MT>;
  cudaError_t e;
  if ((e = ensure_max_smem<paged_rows_kernel<T, STORE, D, MT>>()) != cudaSuccess) return e;
  const unsigned units = (unsigned)(s.B * s.Hk * p.blocks);
  const dim3 grid(units * (unsigned)p.nsplit), block(32 * (PR_NW + 1));
  // behind the table kernel, which also zeroes the counters
  if (s.r > 0) {
    if ((e = launch_trig_tables(a.embed, s.Nk, s.r, nullptr, nullptr, table, table + (size_t)s.Nk * s.r, st, 1, 1, p.done, (int)units)) != cudaSuccess) return e;
    return launch_dependent(kernel, grid, block, smem, st, p, mk, mv, mt);
  }
  if (p.nsplit > 1 && (e = cudaMemsetAsync(p.done, 0, units * sizeof(unsigned int), st)) != cudaSuccess) return e;
  kernel<<<grid, block, smem, st>>>(p, mk, mv, mt);
  return cudaGetLastError();
}
template <typename T, int STORE, int D> static cudaError_t paged_rows_m(const PopePagedAttnArgs& a, cudaStream_t st) {
  return rows_mt(a.shape) == 1 ? paged_rows_t<T, STORE, D, 1>(a, st) : paged_rows_t<T, STORE, D, 2>(a, st);
}
template <typename T, int STORE> static cudaError_t paged_rows_d(const PopePagedAttnArgs& a, cudaStream_t st) {
  const int d = a.shape.d;
  return d == 64 ? paged_rows_m<T, STORE, 64>(a, st) : d == 96 ? paged_rows_m<T, STORE, 96>(a, st) : paged_rows_m<T, STORE, 128>(a, st);
}
template <typename T> static cudaError_t paged_rows_s(const PopePagedAttnArgs& a, cudaStream_t st) {
  switch (a.cache.store) {
    case POPE_STORE_INT8: return paged_rows_d<T, POPE_STORE_INT8>(a, st);
    case POPE_STORE_E4M3: return paged_rows_d<T, POPE_STORE_E4M3>(a, st);
    default: return paged_rows_d<T, POPE_STORE_16>(a, st);
  }
}
cudaError_t paged_rows(const PopePagedAttnArgs& a, cudaStream_t st) {
  return a.shape.dtype == POPE_BF16 ? paged_rows_s<__nv_bfloat16>(a, st) : paged_rows_s<__half>(a, st);
}

}  // namespace pope
