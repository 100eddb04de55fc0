// What the two tcgen05 kernels of the paged attention share (sm_100a): 128 packed query rows of a key head (row = token * group + head) whose
// unnormalised outputs sit in tensor memory leave the CTA, whole or as the part of a key range; a small kernel behind them merges the parts.
// (Merged by the CTA that finished its row block last, 18 parts of a block took 50 us: one SM does not have the loads in flight.)
#pragma once
#include "paged.cuh"

namespace pope {

constexpr int PAGED_ROWS = 128;        // rows of a CTA
constexpr int PAGED_SM_WARPS = 8;      // softmax warps: two threads per row, warp & 3 picks the rows, warp >> 2 the half of the columns
constexpr int PAGED_MAX_SPLIT = 32;    // key ranges of a row block: a lane each in the merge

struct PagedOut {
  int H, Hk, G, Nq, nsplit;
  void* o;
  Strides so;
  float* lse;                // may be null
  float *part_o, *part_ml;   // [row block][split][128][D], [row block][split][128][max (log2 units), sum]
};
inline PagedOut paged_out(const PopePagedAttnArgs& a, int nsplit, float* part_o, float* part_ml) {
  PagedOut e;
  e.H = a.shape.H, e.Hk = a.shape.Hk, e.G = a.shape.H / a.shape.Hk, e.Nq = a.shape.Nq, e.nsplit = nsplit;
  e.o = a.out, e.so = Strides(a.so), e.lse = a.lse, e.part_o = part_o, e.part_ml = part_ml;
  return e;
}
inline bool rows_wide(const void* ptr, const PopeStride3& t) {   // rows on 16-byte boundaries
  return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && t.b % 8 == 0 && t.h % 8 == 0 && t.n % 8 == 0;
}

// The softmax warps (threads 0 .. 255), all products of the CTA completed: row tid & 127, half tid >> 7 of its D columns from `tmem_o` on.  TWO: the halves
// of a row's keys have accumulators of their own, 128 columns apart, and maxima of their own.  `l_half`: the row's sum over this thread's
// keys, 0 for a row that is no query; m: its maximum.  xch: 512 floats of shared memory that nobody reads any more.
template <typename T, int D, bool TWO>
__device__ __forceinline__ void paged_epilogue(const PagedOut& e, uint32_t tmem_o, float* xch, int ub, int split, int b, int hk, int rb, float l_half, float m_half) {
  const int tid = threadIdx.x, rloc = tid & 127, part = tid >> 7;
  auto all_sync = []() { asm volatile("bar.sync 5, %0;" ::"n"(32 * PAGED_SM_WARPS) : "memory"); };
  all_sync();   // (every thread is past its last look at xch)
  xch[part * PAGED_ROWS + rloc] = m_half, xch[(2 + part) * PAGED_ROWS + rloc] = l_half;
  all_sync();
  const float m0 = xch[rloc], m1 = xch[PAGED_ROWS + rloc], m = fmaxf(m0, m1), mu = m == -CUDART_INF_F ? 0.f : m;
  const float f0 = TWO ? ex2_approx(m0 - mu) : 1.f, f1 = TWO ? ex2_approx(m1 - mu) : 1.f;   // 0 for a half without visible keys
  const float l = xch[2 * PAGED_ROWS + rloc] * f0 + xch[3 * PAGED_ROWS + rloc] * f1;
  fence_after_sync();
  const int rho = rb * PAGED_ROWS + rloc, tok = rho / e.G, head = hk + (rho - tok * e.G) * e.Hk;
  const bool whole = e.nsplit == 1, out_row = rho < e.Nq * e.G;   // (padding is written too)
  const float inv = l != 0.f && whole ? 1.f / l : 1.f;
  const uint32_t o_addr = tmem_o + ((uint32_t)(((tid >> 5) & 3) * 32) << 16) + part * (D / 2);
  T* orow = static_cast<T*>(e.o) + b * e.so.b + head * e.so.h + (int64_t)tok * e.so.n + part * (D / 2);
  const int64_t slot = (int64_t)ub * e.nsplit + split;
  float* prow = e.part_o + (slot * PAGED_ROWS + rloc) * D + part * (D / 2);
#pragma unroll
  for (int c0 = 0; c0 < D / 2; c0 += 16) {
    uint32_t ov[16], ov1[16];
    tmem_ld16(o_addr + c0, ov);
    if constexpr (TWO) tmem_ld16(o_addr + 128 + c0, ov1);
    tmem_ld_wait();
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = l != 0.f ? __uint_as_float(ov[i]) * inv : 0.f;   // (without a visible key O may hold anything)
      // (NaN factors stay NaN)
      if constexpr (TWO)
        x[i] = l != 0.f ? ((f0 != 0.f ? __uint_as_float(ov[i]) * f0 : 0.f) + (f1 != 0.f ? __uint_as_float(ov1[i]) * f1 : 0.f)) * inv : 0.f;
    }
    if (out_row && whole) {
#pragma unroll
      for (int i = 0; i < 16; i += 8)
        *reinterpret_cast<uint4*>(orow + c0 + i) =
            make_uint4(pack2<T>(x[i], x[i + 1]), pack2<T>(x[i + 2], x[i + 3]), pack2<T>(x[i + 4], x[i + 5]), pack2<T>(x[i + 6], x[i + 7]));
    } else if (out_row) {
#pragma unroll
      for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(prow + c0 + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
  }
  if (part == 0 && out_row) {
    if (!whole) e.part_ml[(slot * PAGED_ROWS + rloc) * 2] = l != 0.f ? m : -CUDART_INF_F, e.part_ml[(slot * PAGED_ROWS + rloc) * 2 + 1] = l;
    else if (e.lse) e.lse[((int64_t)b * e.H + head) * e.Nq + tok] = l != 0.f ? m * LN2 + logf(l) : -CUDART_INF_F;
  }
}

// out and lse from the parts of `blocks` row blocks, behind the kernel that wrote them
cudaError_t launch_paged_merge(const PagedOut& e, int dtype, int d, int blocks, int blocks_per_unit, cudaStream_t st);

}  // namespace pope
