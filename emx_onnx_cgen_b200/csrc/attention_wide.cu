// Attention over many query rows: the 256-row tile pass of K_ATTENTION_FLASH
// (attention_flash.cu has the operator, its mathematics and the 128-row pass).
//
// Per key tile a query row costs as much tensor-pipe time (2 x D x 128 flops at
// 8192 flops a clock and SM) as exponential time (128 at 16 a clock and SM) at
// D = 128, and half of it at D = 64: both units have to stay busy.  One CTA per
// SM therefore keeps two 128-row tiles in flight, so that one tile's products
// run while the other's softmax does, on key tiles of 128:
//   warps 0-3 / 4-7: softmax of tile A / B, one thread per query row;
//   warp 8: TMA producer of the K and V tiles both row tiles read;
//   warp 9: all products, in the order S_A, S_B, then per key tile
//           O_A += P_A V, next S_A, O_B += P_B V, next S_B;
//   warp 10: zeroes V rows past the last visible key in the last tile.
// TMEM: S_A, S_B, O_A, O_B, 128 columns each.  The weights P (fp16) go back
// into the first half of their score columns and are the A operand of the second
// product from there: no shared-memory round trip, and since the products of one
// thread complete in order, "S_j is ready" also says that O holds tile j - 1, so
// neither rescaling O nor overwriting S needs a wait of its own.
// The row's scores live in registers (setmaxnreg moves the producers' share to
// the softmax warps); pairs of scores are scaled and summed by two-wide fp32
// instructions.  Every wait is bounded (tc100.cuh).
#include <cuda_fp16.h>

#include "attention_flash.cuh"
#include "f32x2.cuh"
#include "host_util.h"
#include "kernels.h"
#include "tc100.cuh"
#include "tmem32.cuh"

namespace emx {

constexpr int AW_M = 128;  // rows of one row tile; a work item has two
constexpr int AW_N = 128;  // keys per tile
constexpr int AW_THREADS = 384;
constexpr uint32_t AW_SLAB = 128u * 128u;  // 64 fp16 columns of 128 rows: 16 KB
constexpr uint32_t AW_S_COL = 0, AW_O_COL = 256;  // + 128 for tile B
constexpr int AW_REGS_SOFTMAX = 208, AW_REGS_OTHER = 80;
constexpr int AW_REGS_LAUNCH = (2 * AW_REGS_SOFTMAX + AW_REGS_OTHER) / 3 + 1;  // per thread at launch, at least

// D += A B with A in TMEM (lane = row, 16 fp16 in 8 columns)
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int NS, int MASK>
__global__ void __launch_bounds__(AW_THREADS, 1) attention_wide_kernel(const __grid_constant__ TileParams p) {
  constexpr uint32_t TILE = NS * AW_SLAB;
  constexpr int ST = NS == 1 ? 4 : 2;  // K and V stages
  extern __shared__ __align__(1024) uint8_t aw_raw[];
  if (smem_u32(aw_raw) & 1023u) {  // the swizzled operands need a 1 KB aligned window
    if (threadIdx.x == 0) record_error(p.err, DEV_BAD_CONFIG);
    return;
  }
  uint8_t* s_q = aw_raw;  // tile A, tile B
  uint8_t* s_k = s_q + 2 * TILE;
  uint8_t* s_v = s_k + ST * TILE;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(s_v + ST * TILE);
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_empty = v_full + ST;
  uint64_t* s_full = v_empty + ST;  // [2] scores of tile A / B ready (and O up to the key tile before)
  uint64_t* p_full = s_full + 2;    // [2] weights written, O rescaled
  uint64_t* o_done = p_full + 2;    // [2] the last product of tile A / B is complete
  uint64_t* v_last = o_done + 2;    // the last V tile has arrived ...
  uint64_t* v_clean = v_last + 1;   // ... and its hidden rows are zero
  uint64_t* drain = v_clean + 1;
  uint32_t* holder = reinterpret_cast<uint32_t*>(drain + 1);
  int* span = reinterpret_cast<int*>(holder + 1);  // [2]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* const err = p.err;

  // ---------------- work item
  const bool shared = (int)blockIdx.x < p.first1;  // rows of every sequence
  const ItemClass& cl = p.cls[shared ? 1 : 0];
  int id = (int)blockIdx.x - (shared ? 0 : p.first1);
  const int split = id % cl.splits;
  id /= cl.splits;
  const int tile = cl.tiles - 1 - id % cl.tiles;  // later tokens, which see more keys, first
  id /= cl.tiles;
  const int kvh = id % p.HKV;
  const int b = id / p.HKV;  // 0 for rows of every sequence
  const int rows_all = (int)(p.TQ.d * p.group.d) * (shared ? p.B : 1);
  const int row0 = tile * 2 * AW_M;
  const int rows = min(2 * AW_M, rows_all - row0);
  const bool has_b = rows > AW_M;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&o_done[s], 1);
    }
    mbar_init(v_last, 1);
    mbar_init(v_clean, 1);
    mbar_init(drain, 1);
    fence_barrier_init();
    span[0] = 0x7fffffff;
    span[1] = 0;
  }
  if (warp == 9) {
    tmem_alloc(holder, 512);
    tmem_relinquish();
  }
  pdl_wait();  // Q, K, V, masks and counts may come from the preceding kernel
  pdl_launch_dependents();

  // ---------------- Q tiles, zero past the head size and the rows
  for (int i = threadIdx.x; i < 2 * AW_M * NS * 8; i += AW_THREADS) {
    const int c = i % (NS * 8), r = i / (NS * 8);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < rows && c * 8 < p.D) {
      const RowId w = row_of(row0 + r, p.group, p.TQ, kvh, b, shared);
      v = *reinterpret_cast<const uint4*>(p.q + (int64_t)w.b * p.q_sb + (int64_t)w.h * p.q_sh + (int64_t)w.t * p.q_st +
                                          c * 8);
    }
    const int rt = r & (AW_M - 1);
    *reinterpret_cast<uint4*>(s_q + (r >> 7) * TILE + (c >> 3) * AW_SLAB + rt * 128 + (((c & 7) ^ (rt & 7)) << 4)) = v;
  }
  fence_async_shared();

  // ---------------- key tiles that some row sees, as in attention_flash.cu: the past's first, positions count
  // through the tiles
  const int np = cl.past ? (p.tp + AW_N - 1) / AW_N : 0;
  int keys = shared ? 0 : p.tk;
  if (!shared) {
    if (p.causal) keys = min(keys, p.group.div(row0 + rows - 1) + 1);
    if (p.counts) {
      const long long n = p.counts[b];
      if (n < 0 || n > p.tk) record_error(err, DEV_BAD_INDEX);
      keys = min(keys, (int)max(0ll, min(n, (long long)p.tk)));
    }
  }
  int pbeg = 0, pend = keys > 0 ? np * AW_N + keys : (cl.past ? p.tp : 0);
  __syncthreads();  // span initialised
  if (MASK == MASK_BITS) {
    if (threadIdx.x < rows) {
      const RowId w = row_of(row0 + threadIdx.x, p.group, p.TQ, kvh, b, shared);
      const int4 v = p.spans[w.b * p.mask_sb + w.h * p.mask_sh + w.t * p.mask_st];
      if (cl.past && v.z < v.w) {
        atomicMin(&span[0], v.z);
        atomicMax(&span[1], v.w);
      }
      if (!shared && v.x < v.y) {
        atomicMin(&span[0], np * AW_N + v.x);
        atomicMax(&span[1], np * AW_N + v.y);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *holder;
  if (MASK == MASK_BITS) {
    pbeg = span[0];
    pend = min(pend, span[1]);
  }
  const int j_lo = pbeg < pend ? pbeg / AW_N : 0, j_hi = pbeg < pend ? (pend + AW_N - 1) / AW_N : 0;
  const int per = j_hi - j_lo;
  const int j0 = j_lo + (int)((long long)per * split / cl.splits);
  const int J = j_lo + (int)((long long)per * (split + 1) / cl.splits) - j0;
  const int nv = pend - (j0 + J - 1) * AW_N;  // visible keys of the last tile, when fewer than all
  const bool clean = J > 0 && nv < AW_N;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AW_REGS_OTHER));
    if (warp == 8 && lane == 0) {
      // ---------------- producer
      bool ok = true;
      int issued = 0;
      for (int j = 0; j < J && ok; ++j) {
        const int s = j % ST, jj = j0 + j;
        const int in_past = jj < np ? 1 : 0, key0 = (in_past ? jj : jj - np) * AW_N;
        const int kb = in_past && p.past_shared ? 0 : b;
        const uint32_t ph = (uint32_t)(j / ST - 1) & 1u;
        if (j >= ST && !mbar_wait(&k_empty[s], ph, err, DEV_TIMEOUT_PRODUCER)) ok = false;
        if (!ok) break;
        mbar_arrive_expect_tx(&k_full[s], TILE);
#pragma unroll
        for (int c = 0; c < NS; ++c)
          tma_load_4d(s_k + s * TILE + c * AW_SLAB, &p.map_k[in_past], &k_full[s], 64 * c, key0, kvh, kb);
        issued = 2 * j + 1;
        if (j >= ST && !mbar_wait(&v_empty[s], ph, err, DEV_TIMEOUT_PRODUCER)) ok = false;
        if (!ok) break;
        mbar_arrive_expect_tx(&v_full[s], TILE);
#pragma unroll
        for (int c = 0; c < NS; ++c)
          tma_load_4d(s_v + s * TILE + c * AW_SLAB, &p.map_v[in_past], &v_full[s], 64 * c, key0, kvh, kb);
        issued = 2 * j + 2;
      }
      if (!ok) {  // error path: let the copies in flight land before the CTA exits
        for (int i = max(0, issued - 2 * ST); i < issued; ++i) {
          const int j = i >> 1;
          (void)mbar_wait((i & 1) ? &v_full[j % ST] : &k_full[j % ST], (uint32_t)(j / ST) & 1u, nullptr, 0);
        }
      }
    } else if (warp == 9 && lane == 0 && J > 0) {
      // ---------------- products
      const uint32_t idesc_s = make_idesc(1u, 0u, 0u, AW_M, AW_N);
      const uint32_t idesc_o = make_idesc(1u, 0u, 0u, AW_M, (uint32_t)((p.DV + 15) & ~15)) | (1u << 16);
      const int nks = (p.D + 15) / 16;
      const uint32_t qa = smem_u32(s_q), ka = smem_u32(s_k), va = smem_u32(s_v);
      auto scores = [&](int x, int j) {  // S_x = Q_x K_j^T
        const uint32_t q = qa + x * TILE, k = ka + (j % ST) * TILE;
        for (int ks = 0; ks < nks; ++ks) {
          const uint32_t off = (uint32_t)(ks >> 2) * AW_SLAB + (uint32_t)(ks & 3) * 32u;
          mma_f16(tmem + AW_S_COL + 128u * x, smem_desc_k_sw128(q + off, 1024), smem_desc_k_sw128(k + off, 1024), idesc_s,
                  ks > 0 ? 1u : 0u);
        }
        tc_commit(&s_full[x]);
      };
      auto values = [&](int x, int j) {  // O_x += P_x V_j
        const uint32_t v = va + (j % ST) * TILE;
#pragma unroll
        for (int kk = 0; kk < AW_N / 16; ++kk)
          mma_f16_ts(tmem + AW_O_COL + 128u * x, tmem + AW_S_COL + 128u * x + 8u * kk,
                     smem_desc_mn_sw128(v + (uint32_t)kk * 16u * 128u, AW_SLAB, 1024u), idesc_o, (j | kk) ? 1u : 0u);
      };
      bool ok = mbar_wait(&k_full[0], 0, err, DEV_TIMEOUT_MMA);
      if (ok) {
        tc_fence_after();
        scores(0, 0);
        if (has_b) scores(1, 0);
        tc_commit(&k_empty[0]);
      }
      for (int j = 0; j < J && ok; ++j) {
        const uint32_t ph = (uint32_t)(j / ST) & 1u;
        ok = mbar_wait(&v_full[j % ST], ph, err, DEV_TIMEOUT_MMA);
        if (ok && clean && j == J - 1) {
          mbar_arrive(v_last);
          ok = mbar_wait(v_clean, 0, err, DEV_TIMEOUT_MMA);
        }
        const bool more = j + 1 < J;
        for (int x = 0; x < (has_b ? 2 : 1) && ok; ++x) {
          ok = mbar_wait(&p_full[x], (uint32_t)j & 1u, err, DEV_TIMEOUT_MMA);
          if (!ok) break;
          tc_fence_after();
          values(x, j);
          if (x == (has_b ? 1 : 0)) tc_commit(&v_empty[j % ST]);
          if (more) {
            if (x == 0) ok = mbar_wait(&k_full[(j + 1) % ST], (uint32_t)((j + 1) / ST) & 1u, err, DEV_TIMEOUT_MMA);
            if (!ok) break;
            tc_fence_after();
            scores(x, j + 1);
            if (x == (has_b ? 1 : 0)) tc_commit(&k_empty[(j + 1) % ST]);
          } else {
            tc_commit(&o_done[x]);
          }
        }
      }
      // every MMA completes before TMEM is released
      tc_commit(drain);
      (void)mbar_wait(drain, 0, nullptr, 0);
    } else if (warp == 10 && clean) {
      // ---------------- values past the last visible key take no part
      const int s = (J - 1) % ST;
      const bool ok = mbar_wait(v_last, 0, err, DEV_TIMEOUT_MMA);
      if (__all_sync(0xffffffffu, ok)) {
        for (int i = lane; i < (AW_N - nv) * 8 * NS; i += 32) {
          const int c = i % (8 * NS), r = nv + i / (8 * NS);
          *reinterpret_cast<uint4*>(s_v + s * TILE + (c >> 3) * AW_SLAB + r * 128 + (c & 7) * 16) =
              make_uint4(0u, 0u, 0u, 0u);
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_clean);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AW_REGS_SOFTMAX));
    // ---------------- softmax and epilogue: thread = query row (warp % 4 = TMEM lane quarter)
    const int x = warp >> 2, quarter = warp & 3;
    const int r = x * AW_M + quarter * 32 + lane;
    if (x == 0 || has_b) {
      const bool live = r < rows;
      const RowId w = row_of(row0 + (live ? r : 0), p.group, p.TQ, kvh, b, shared);
      const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
      const uint32_t s_col = lane_base + AW_S_COL + 128u * x, o_col = lane_base + AW_O_COL + 128u * x;
      const int row_end = p.causal ? min(keys, w.t + 1) : keys;
      const unsigned long long* words = nullptr;
      unsigned long long word[2] = {0ull, 0ull};  // the next tile's, loaded a tile ahead
      if (MASK == MASK_BITS) {
        words = p.bits + (w.b * p.mask_sb + w.h * p.mask_sh + w.t * p.mask_st) * p.words +
                (cl.past ? 0 : p.words_past) + 2 * j0;
        if (J > 0) word[0] = words[0], word[1] = words[1];
      }
      float m_used = -INFINITY;  // reference of the exponentials, log2 units
      float l = 0.0f;
      const float sc = p.scale_log2;
      const bool pos = sc > 0.0f;
      const float mul = pos ? sc : 1.0f;
      const F2 mul2v(mul, mul);
      bool ok = true;
      for (int j = 0; j < J && ok; ++j) {
        const int jj = j0 + j;
        const bool in_past = jj < np;
        const int end = (in_past ? p.tp : row_end) - (in_past ? jj : jj - np) * AW_N;
        unsigned long long vis[2] = {~0ull, ~0ull};
        if (end < 128) {
          vis[0] = end >= 64 ? ~0ull : end > 0 ? (1ull << end) - 1 : 0ull;
          vis[1] = end > 64 ? (1ull << (end - 64)) - 1 : 0ull;
        }
        if (MASK == MASK_BITS) {
          vis[0] &= word[0], vis[1] &= word[1];
          if (j + 1 < J) word[0] = words[2 * j + 2], word[1] = words[2 * j + 3];
        }
        ok = mbar_wait(&s_full[x], (uint32_t)j & 1u, err, DEV_TIMEOUT_EPILOGUE);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sv[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_col + 32u * c, sv[c]);
        tmem_wait_ld();
        if (!pos) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) sv[c][i] = __float_as_uint(__uint_as_float(sv[c][i]) * sc);
        }
        // keys the row does not see become -inf; tiles every row of the warp sees whole skip the test
        if (!__all_sync(0xffffffffu, (vis[0] & vis[1]) == ~0ull)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t half = (uint32_t)(vis[c >> 1] >> (32 * (c & 1)));
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(half & (1u << i))) sv[c][i] = 0xff800000u;
          }
        }
        float mxp[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mxp[c] = __uint_as_float(sv[c][0]);
#pragma unroll
          for (int i = 1; i < 31; i += 2)
            mxp[c] = fmaxf(mxp[c], fmaxf(__uint_as_float(sv[c][i]), __uint_as_float(sv[c][i + 1])));
          mxp[c] = fmaxf(mxp[c], __uint_as_float(sv[c][31]));
        }
        const float mx = fmaxf(fmaxf(mxp[0], mxp[1]), fmaxf(mxp[2], mxp[3])) * mul;
        bool rescale = false;
        float alpha = 1.0f;
        if (mx > m_used + AFK_RESCALE || m_used == -INFINITY) {
          rescale = j > 0 && m_used != -INFINITY;
          if (rescale) alpha = ex2_approx(m_used - mx);
          m_used = mx;
        }
        const float neg_m = m_used == -INFINITY ? 0.0f : -m_used;
        const F2 neg2(neg_m, neg_m);
        F2 sum[2] = {F2(0.0f, 0.0f), F2(0.0f, 0.0f)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pw[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const uint32_t* s2 = &sv[2 * h + (i >> 4)][2 * (i & 15)];
            const F2 e = fma2(F2(__uint_as_float(s2[0]), __uint_as_float(s2[1])), mul2v, neg2);
            const F2 w2(ex2_approx(e.lo()), ex2_approx(e.hi()));
            sum[i & 1] = add2(sum[i & 1], w2);
            pw[i] = pack_f16x2(w2.lo(), w2.hi());
          }
          tmem_st32(s_col + 32u * h, pw);
        }
        l = fmaf(l, alpha, (sum[0].lo() + sum[0].hi()) + (sum[1].lo() + sum[1].hi()));
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
          for (int c = 0; c < 4 * NS; ++c) {
            uint32_t o[16];
            tmem_ld16(o_col + 16u * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st16(o_col + 16u * c, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
      }
      // ---------------- epilogue
      if (ok && J > 0) {
        ok = mbar_wait(&o_done[x], 0, err, DEV_TIMEOUT_EPILOGUE);
        ok = __all_sync(0xffffffffu, ok);
      }
      if (ok) {
        tc_fence_after();
        const bool part = p.part_o != nullptr;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int64_t row = ((int64_t)w.b * (int)p.TQ.d + w.t) * p.HQ + w.h;
        const int64_t slot_row = (int64_t)(cl.part0 + split) * ((int64_t)p.B * (int)p.TQ.d * p.HQ) + row;
        uint16_t* orow = p.o + (int64_t)w.b * p.o_sb + (int64_t)w.h * p.o_sh + (int64_t)w.t * p.o_st;
        float* prow = part ? p.part_o + slot_row * p.DV : nullptr;
        if (part && live) p.part_ml[slot_row] = make_float2(m_used, l);
        if (!(part && J == 0)) {  // the merge does not read the output of an item with l = 0
#pragma unroll
          for (int c = 0; c < 2 * NS; ++c) {
            uint32_t o[32];
            if (J > 0) {
              tmem_ld32(o_col + 32u * c, o);
              tmem_wait_ld();
            }
            if (l == 0.0f) {  // a row that sees no key gives 0 whatever the values hold
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = 0u;
            }
            if (live) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                if (32 * c + i >= p.DV) continue;
                if (part) {
                  *reinterpret_cast<uint4*>(prow + 32 * c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                  *reinterpret_cast<uint4*>(prow + 32 * c + i + 4) = make_uint4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]);
                } else {
                  uint4 v;
                  v.x = pack_f16x2(__uint_as_float(o[i + 0]) * inv, __uint_as_float(o[i + 1]) * inv);
                  v.y = pack_f16x2(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                  v.z = pack_f16x2(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
                  v.w = pack_f16x2(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
                  *reinterpret_cast<uint4*>(orow + 32 * c + i) = v;
                }
              }
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ host side
static size_t wide_smem(int ns) {
  const int st = ns == 1 ? 4 : 2;
  return (size_t)(2 + 2 * st) * ns * AW_SLAB + 256;
}

typedef void (*WideKernel)(const TileParams);

static WideKernel wide_kernel(int ns, int mask) {
  static const WideKernel table[2][2] = {{attention_wide_kernel<1, MASK_NONE>, attention_wide_kernel<1, MASK_BITS>},
                                         {attention_wide_kernel<2, MASK_NONE>, attention_wide_kernel<2, MASK_BITS>}};
  return table[ns - 1][mask];
}

cudaError_t prepare_attention_wide() {
  for (int ns = 1; ns <= 2; ++ns)
    for (int m = 0; m < 2; ++m) {
      cudaFuncAttributes a;
      cudaError_t e = cudaFuncGetAttributes(&a, wide_kernel(ns, m));
      if (e != cudaSuccess) return e;
      // the softmax warps' larger share comes out of the registers the launch holds: with fewer, they would wait for ever
      if (a.numRegs < AW_REGS_LAUNCH) return cudaErrorInvalidKernelImage;
      e = cudaFuncSetAttribute(wide_kernel(ns, m), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)wide_smem(ns));
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

cudaError_t launch_attention_wide(const TileParams& p, int slabs, int mask, unsigned items, cudaStream_t stream) {
  return launch_pdl(wide_kernel(slabs, mask), dim3(items), dim3(AW_THREADS), wide_smem(slabs), stream, p);
}

}  // namespace emx
