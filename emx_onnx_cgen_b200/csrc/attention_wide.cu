// Attention over many query rows: the 256-row tile pass of K_ATTENTION_FLASH
// (attention_flash.cu has the operator, its mathematics and the 128-row pass).
//
// Per key tile a query row costs as much tensor-pipe time (2 x D x 64 fused
// multiply-adds at 4096 a clock and SM) as exponential time (64 at 16 a clock
// and SM) at D = 128, and half of it at D = 64: both units have to stay busy.
// One persistent CTA per SM keeps two 128-row tiles in flight, each with two
// score buffers, so the softmax of one key tile runs beside the products of
// others and waits for none of them in the steady state:
//   warps 0-3 / 4-7: softmax of row tile A / B, one thread per query row; they
//           also bring in the next work item's query rows;
//   warp 8: TMA producer of the 64-key K and V tiles that both row tiles read;
//   warp 9: all products: S_A(0), S_B(0), S_A(1), S_B(1), then per key tile j
//           O_A += P_A(j) V_j, S_A(j + 2), O_B += P_B(j) V_j, S_B(j + 2);
//   warp 10: zeroes V rows past the last visible key in an item's last tile;
//   warp 11: works out the items' key ranges, two items ahead.
// TMEM: 2 x 64 score columns and 128 output columns for each row tile.  The
// weights P (fp16) go back into the first half of their scores' columns and are
// the A operand of the second product from there: no shared-memory round trip.
// The products of one thread complete in order, so "S(j) is ready" also says
// that P(j - 2), whose place it takes, has been used.  The output is rescaled
// only when a row's maximum has grown by 2^8, after P(j - 1) V is complete.
// Pairs of scores are scaled and summed by two-wide fp32 instructions.  Every
// wait is bounded (tc100.cuh).
#include <cuda_fp16.h>

#include "attention_flash.cuh"
#include "f32x2.cuh"
#include "host_util.h"
#include "kernels.h"
#include "tc100.cuh"
#include "tmem32.cuh"

namespace emx {

constexpr int AW_M = 128;  // rows of one row tile; a work item has two
constexpr int AW_N = 64;   // keys per tile
constexpr int AW_ST = 4;   // K and V stages
constexpr int AW_THREADS = 384;
constexpr uint32_t AW_QSLAB = AW_M * 128u;  // 64 fp16 columns of 128 rows: 16 KB
constexpr uint32_t AW_KSLAB = AW_N * 128u;  // of 64 keys: 8 KB
constexpr uint32_t AW_O_COL = 256;          // outputs; scores of tile x, buffer i at 128 x + 64 i

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

// A work item: which rows, and which of its key tiles.
struct WideItem {
  int row0, rows, kvh, b, split;
  bool shared;
};

__device__ __forceinline__ WideItem wide_item(const TileParams& p, int id) {
  WideItem w;
  w.shared = id < p.first1;  // rows of every sequence
  const ItemClass& cl = p.cls[w.shared ? 1 : 0];
  if (!w.shared) id -= p.first1;
  w.split = id % cl.splits;
  id /= cl.splits;
  const int tile = cl.tiles - 1 - id % cl.tiles;  // later tokens, which see more keys, first
  id /= cl.tiles;
  w.kvh = id % p.HKV;
  w.b = id / p.HKV;  // 0 for rows of every sequence
  w.row0 = tile * 2 * AW_M;
  w.rows = min(2 * AW_M, (int)(p.TQ.d * p.group.d) * (w.shared ? p.B : 1) - w.row0);
  return w;
}

// Key tiles [j0, j0 + J) of an item, keys of the current ones that some row may see, and visible keys of the last tile.
struct WideKeys {
  int j0, J, keys, last;
};

constexpr int AW_BARS = 4 * AW_ST + 3 * 4 + 2 + 2 + 4 + 1;
constexpr uint32_t AW_TAIL = AW_BARS * 8 + 2 * sizeof(WideKeys) + 16;

template <int NS, int MASK>
__global__ void __launch_bounds__(AW_THREADS, 1) attention_wide_kernel(const __grid_constant__ TileParams p) {
  constexpr uint32_t QTILE = NS * AW_QSLAB, KTILE = NS * AW_KSLAB;
  extern __shared__ __align__(1024) uint8_t aw_raw[];
  if (smem_u32(aw_raw) & 1023u) {  // the swizzled operands need a 1 KB aligned window
    if (threadIdx.x == 0) record_error(p.err, DEV_BAD_CONFIG);
    return;
  }
  uint8_t* s_q = aw_raw;  // tile A, tile B
  uint8_t* s_k = s_q + 2 * QTILE;
  uint8_t* s_v = s_k + AW_ST * KTILE;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(s_v + AW_ST * KTILE);
  uint64_t* k_empty = k_full + AW_ST;
  uint64_t* v_full = k_empty + AW_ST;
  uint64_t* v_empty = v_full + AW_ST;
  uint64_t* s_full = v_empty + AW_ST;  // [tile][buffer] scores ready
  uint64_t* p_full = s_full + 4;       // [tile][buffer] weights written, output rescaled
  uint64_t* pv_done = p_full + 4;      // [tile][buffer] the key tile is in the output
  uint64_t* q_full = pv_done + 4;      // [tile] the item's query rows are in shared memory
  uint64_t* v_last = q_full + 2;       // an item's last V tile has arrived ...
  uint64_t* v_clean = v_last + 1;      // ... and its hidden rows are zero
  uint64_t* info_full = v_clean + 1;   // [2] an item's key range is known
  uint64_t* info_empty = info_full + 2;
  uint64_t* drain = info_empty + 2;
  WideKeys* s_info = reinterpret_cast<WideKeys*>(drain + 1);  // [2]
  uint32_t* holder = reinterpret_cast<uint32_t*>(s_info + 2);

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  int* const err = p.err;
  if (threadIdx.x == 0) {
    for (int s = 0; s < AW_ST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&pv_done[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 4);
      mbar_init(&info_full[s], 1);
      mbar_init(&info_empty[s], 11);  // producer, products, cleaner, 8 softmax warps
    }
    mbar_init(v_last, 1);
    mbar_init(v_clean, 1);
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *holder, 0);
  pdl_wait();  // Q, K, V, masks and counts may come from the preceding kernel
  pdl_launch_dependents();

  // the item's key range, read by every role (whole warps)
  auto item_keys = [&](int n, WideKeys& k) -> bool {
    const bool ok = mbar_wait(&info_full[n & 1], (uint32_t)(n >> 1) & 1u, err, DEV_TIMEOUT_PRODUCER);
    if (!__all_sync(0xffffffffu, ok)) return false;
    k = s_info[n & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&info_empty[n & 1]);
    return true;
  };

  if (warp == 11) {
    // ---------------- key ranges: tiles of the past first, positions count through the tiles (attention_flash.cu)
    for (int n = 0, id = blockIdx.x; id < p.items; ++n, id += gridDim.x) {
      const WideItem w = wide_item(p, id);
      const ItemClass& cl = p.cls[w.shared ? 1 : 0];
      const int np = cl.past ? (p.tp + AW_N - 1) / AW_N : 0;
      int keys = w.shared ? 0 : p.tk;
      if (!w.shared) {
        if (p.causal) keys = min(keys, p.group.div(w.row0 + w.rows - 1) + 1);
        if (p.counts) {
          const long long c = p.counts[w.b];
          if (c < 0 || c > p.tk) record_error(err, DEV_BAD_INDEX);
          keys = min(keys, (int)max(0ll, min(c, (long long)p.tk)));
        }
      }
      int pbeg = 0, pend = keys > 0 ? np * AW_N + keys : (cl.past ? p.tp : 0);
      if (MASK == MASK_BITS) {
        int lo = 0x7fffffff, hi = 0;
#pragma unroll
        for (int i = 0; i < 2 * AW_M; i += 32) {
          if (i + lane >= w.rows) continue;
          const RowId r = row_of(w.row0 + i + lane, p.group, p.TQ, w.kvh, w.b, w.shared);
          const int4 v = p.spans[r.b * p.mask_sb + r.h * p.mask_sh + r.t * p.mask_st];
          if (cl.past && v.z < v.w) lo = min(lo, v.z), hi = max(hi, v.w);
          if (!w.shared && v.x < v.y) lo = min(lo, np * AW_N + v.x), hi = max(hi, np * AW_N + v.y);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        pbeg = lo, pend = min(pend, hi);
      }
      const int j_lo = pbeg < pend ? pbeg / AW_N : 0, j_hi = pbeg < pend ? (pend + AW_N - 1) / AW_N : 0;
      WideKeys k;
      k.j0 = j_lo + (int)((long long)(j_hi - j_lo) * w.split / cl.splits);
      k.J = j_lo + (int)((long long)(j_hi - j_lo) * (w.split + 1) / cl.splits) - k.j0;
      k.keys = keys;
      k.last = pend - (k.j0 + k.J - 1) * AW_N;
      if (n >= 2 && !__all_sync(0xffffffffu, mbar_wait(&info_empty[n & 1], (uint32_t)((n >> 1) - 1) & 1u, err,
                                                       DEV_TIMEOUT_PRODUCER)))
        break;
      if (lane == 0) {
        s_info[n & 1] = k;
        mbar_arrive(&info_full[n & 1]);
      }
      __syncwarp();
    }
  } else if (warp == 8) {
    // ---------------- producer (lane 0 issues)
    int nkv = 0, issued = 0;  // key tiles so far; copies so far (K and V of a tile count one each)
    bool ok = true;
    for (int n = 0, id = blockIdx.x; id < p.items && ok; ++n, id += gridDim.x) {
      WideKeys k;
      if (!item_keys(n, k)) {
        ok = false;
        break;
      }
      const WideItem w = wide_item(p, id);
      const int np = p.cls[w.shared ? 1 : 0].past ? (p.tp + AW_N - 1) / AW_N : 0;
      if (lane == 0) {
        for (int j = 0; j < k.J; ++j, ++nkv) {
          const int s = nkv % AW_ST, jj = k.j0 + j;
          const int in_past = jj < np ? 1 : 0, key0 = (in_past ? jj : jj - np) * AW_N;
          const int kb = in_past && p.past_shared ? 0 : w.b;
          const uint32_t ph = (uint32_t)(nkv / AW_ST - 1) & 1u;
          if (nkv >= AW_ST && !mbar_wait(&k_empty[s], ph, err, DEV_TIMEOUT_PRODUCER)) ok = false;
          if (!ok) break;
          mbar_arrive_expect_tx(&k_full[s], KTILE);
#pragma unroll
          for (int c = 0; c < NS; ++c)
            tma_load_4d(s_k + s * KTILE + c * AW_KSLAB, &p.map_k[in_past], &k_full[s], 64 * c, key0, w.kvh, kb);
          issued = 2 * nkv + 1;
          if (nkv >= AW_ST && !mbar_wait(&v_empty[s], ph, err, DEV_TIMEOUT_PRODUCER)) ok = false;
          if (!ok) break;
          mbar_arrive_expect_tx(&v_full[s], KTILE);
#pragma unroll
          for (int c = 0; c < NS; ++c)
            tma_load_4d(s_v + s * KTILE + c * AW_KSLAB, &p.map_v[in_past], &v_full[s], 64 * c, key0, w.kvh, kb);
          issued = 2 * nkv + 2;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    }
    if (!ok && lane == 0) {  // error path: let the copies in flight land before the CTA exits
      for (int i = max(0, issued - 2 * AW_ST); i < issued; ++i) {
        const int j = i >> 1;
        (void)mbar_wait((i & 1) ? &v_full[j % AW_ST] : &k_full[j % AW_ST], (uint32_t)(j / AW_ST) & 1u, nullptr, 0);
      }
    }
  } else if (warp == 9) {
    // ---------------- products.  The whole warp goes through the waits and one elected thread issues: its operands
    // are then known to be uniform, and a product costs the tensor pipe's time instead of its issue (about 100
    // clocks an instruction from a thread picked by its lane number).
    const uint32_t idesc_s = make_idesc(1u, 0u, 0u, AW_M, AW_N);
    const uint32_t idesc_o = make_idesc(1u, 0u, 0u, AW_M, (uint32_t)((p.DV + 15) & ~15)) | (1u << 16);
    const int nks = (p.D + 15) / 16;
    const uint64_t q_desc = smem_desc_k_sw128(smem_u32(s_q), 1024), k_desc = smem_desc_k_sw128(smem_u32(s_k), 1024);
    const uint64_t v_desc = smem_desc_mn_sw128(smem_u32(s_v), AW_KSLAB, 1024u);
    auto wait = [&](uint64_t* bar, int phase) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, (uint32_t)phase & 1u, err, DEV_TIMEOUT_MMA));
    };
    int nkv = 0;            // key tiles of the items before
    int nt[2] = {0, 0};     // the same of each row tile (an item may have only tile A)
    int nq[2] = {0, 0};     // items of each row tile
    int nclean = 0;         // items whose last V tile was cleaned
    bool ok = true;
    for (int n = 0, id = blockIdx.x; id < p.items && ok; ++n, id += gridDim.x) {
      WideKeys k;
      if (!item_keys(n, k)) break;
      if (k.J == 0) continue;
      const WideItem w = wide_item(p, id);
      const int tiles = w.rows > AW_M ? 2 : 1;
      auto scores = [&](int x, int j) -> bool {  // S_x(j) = Q_x K_j^T, after the K tile's arrival
        const int kv = nkv + j, s = kv % AW_ST, buf = (nt[x] + j) & 1;
        if (x == 0 && !wait(&k_full[s], kv / AW_ST)) return false;
        tc_fence_after();
        if (elect_one()) {
          // descriptors hold addresses in 16-byte units in their low bits: a step along d is an addition
          const uint64_t q = q_desc + x * (QTILE >> 4), kt = k_desc + s * (KTILE >> 4);
          const uint32_t d = tmem + 128u * x + 64u * buf;
#pragma unroll
          for (int ks = 0; ks < 4 * NS; ++ks)
            if (ks < nks)
              mma_f16(d, q + ((ks >> 2) * AW_QSLAB + (ks & 3) * 32u) / 16u, kt + ((ks >> 2) * AW_KSLAB + (ks & 3) * 32u) / 16u,
                      idesc_s, ks > 0 ? 1u : 0u);
          tc_commit(&s_full[2 * x + buf]);
          if (x == tiles - 1) tc_commit(&k_empty[s]);
        }
        __syncwarp();
        return true;
      };
      for (int x = 0; x < tiles && ok; ++x) {
        ok = wait(&q_full[x], nq[x]);
        if (ok) ok = scores(x, 0);
      }
      for (int x = 0; x < tiles && ok && k.J > 1; ++x) ok = scores(x, 1);
      for (int j = 0; j < k.J && ok; ++j) {
        const int kv = nkv + j, s = kv % AW_ST;
        ok = wait(&v_full[s], kv / AW_ST);
        if (ok && j == k.J - 1 && k.last < AW_N) {
          if (lane == 0) mbar_arrive(v_last);
          ok = wait(v_clean, nclean);
          ++nclean;
        }
        for (int x = 0; x < tiles && ok; ++x) {
          const int c = nt[x] + j, buf = c & 1;
          ok = wait(&p_full[2 * x + buf], c >> 1);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t v = v_desc + s * (KTILE >> 4);
#pragma unroll
            for (int kk = 0; kk < AW_N / 16; ++kk)  // O_x += P_x(j) V_j
              mma_f16_ts(tmem + AW_O_COL + 128u * x, tmem + 128u * x + 64u * buf + 8u * kk, v + kk * (16u * 128u / 16u),
                         idesc_o, (j | kk) ? 1u : 0u);
            tc_commit(&pv_done[2 * x + buf]);
            if (x == tiles - 1) tc_commit(&v_empty[s]);
          }
          __syncwarp();
          if (j + 2 < k.J) ok = scores(x, j + 2);
        }
      }
      nkv += k.J;
      for (int x = 0; x < tiles; ++x) nt[x] += k.J, ++nq[x];
    }
    // every MMA completes before TMEM is released
    if (elect_one()) {
      tc_commit(drain);
      (void)mbar_wait(drain, 0, nullptr, 0);
    }
    __syncwarp();
  } else if (warp == 10) {
    // ---------------- values past the last visible key take no part
    int nkv = 0, nclean = 0;
    for (int n = 0, id = blockIdx.x; id < p.items; ++n, id += gridDim.x) {
      WideKeys k;
      if (!item_keys(n, k)) break;
      nkv += k.J;
      if (k.J == 0 || k.last >= AW_N) continue;
      const int s = (nkv - 1) % AW_ST;
      const bool ok = mbar_wait(v_last, (uint32_t)nclean & 1u, err, DEV_TIMEOUT_MMA);
      if (!__all_sync(0xffffffffu, ok)) break;
      for (int i = lane; i < (AW_N - k.last) * 8 * NS; i += 32) {
        const int c = i % (8 * NS), r = k.last + i / (8 * NS);
        *reinterpret_cast<uint4*>(s_v + s * KTILE + (c >> 3) * AW_KSLAB + r * 128 + (c & 7) * 16) =
            make_uint4(0u, 0u, 0u, 0u);
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(v_clean);
      ++nclean;
    }
  } else {
    // ---------------- softmax and epilogue: thread = query row (warp % 4 = TMEM lane quarter)
    const int x = warp >> 2, quarter = warp & 3;
    const int rt = quarter * 32 + lane;  // row within the tile
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_col = lane_base + AW_O_COL + 128u * x;
    const float sc = p.scale_log2;
    const bool pos = sc > 0.0f;
    const float mul = pos ? sc : 1.0f;
    const F2 mul2v(mul, mul);
    int nt = 0;  // key tiles of this row tile so far
    // query rows of tile x, zero past the head size and the rows: this warp's 32 rows, 32 lanes over the pieces
    auto load_q = [&](const WideItem& w) {
      constexpr int PIECES = NS * 8;
#pragma unroll
      for (int part = 0; part < PIECES; part += 8) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = (part + i) * 32 + lane, c = e % PIECES, r = quarter * 32 + e / PIECES, rr = x * AW_M + r;
          v[i] = make_uint4(0u, 0u, 0u, 0u);
          if (rr < w.rows && c * 8 < p.D) {
            const RowId q = row_of(w.row0 + rr, p.group, p.TQ, w.kvh, w.b, w.shared);
            v[i] = *reinterpret_cast<const uint4*>(p.q + (int64_t)q.b * p.q_sb + (int64_t)q.h * p.q_sh +
                                                   (int64_t)q.t * p.q_st + c * 8);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int e = (part + i) * 32 + lane, c = e % PIECES, r = quarter * 32 + e / PIECES;
          *reinterpret_cast<uint4*>(s_q + x * QTILE + (c >> 3) * AW_QSLAB + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[i];
        }
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[x]);
    };
    int id = blockIdx.x;
    WideItem w = {};
    WideKeys k = {};
    bool ok = id < p.items && item_keys(0, k);
    if (ok) {
      w = wide_item(p, id);
      if (k.J > 0 && x * AW_M < w.rows) load_q(w);
    }
    for (int n = 0; ok; ++n) {
      const int r = x * AW_M + rt;
      const bool mine = x * AW_M < w.rows, live = r < w.rows;  // whether the tile, the row exists
      const ItemClass& cl = p.cls[w.shared ? 1 : 0];
      const RowId row = row_of(w.row0 + (live ? r : 0), p.group, p.TQ, w.kvh, w.b, w.shared);
      float m_used = -INFINITY;  // reference of the exponentials, log2 units
      float l = 0.0f;
      const int J = mine ? k.J : 0;
      if (J > 0) {
        const int np = cl.past ? (p.tp + AW_N - 1) / AW_N : 0;
        const int row_end = p.causal ? min(k.keys, row.t + 1) : k.keys;
        const unsigned long long* words = nullptr;
        unsigned long long word = 0ull;  // the next tile's, loaded a tile ahead
        if (MASK == MASK_BITS) {
          words = p.bits + (row.b * p.mask_sb + row.h * p.mask_sh + row.t * p.mask_st) * p.words +
                  (cl.past ? 0 : p.words_past) + k.j0;
          word = words[0];
        }
        for (int j = 0; j < J; ++j) {
          const int jj = k.j0 + j, c = nt + j, buf = c & 1;
          const bool in_past = jj < np;
          const int end = (in_past ? p.tp : row_end) - (in_past ? jj : jj - np) * AW_N;
          unsigned long long vis = ~0ull;  // visible keys of the tile, one bit each
          if (end < AW_N) vis = end > 0 ? (1ull << end) - 1 : 0ull;
          if (MASK == MASK_BITS) {
            vis &= word;
            if (j + 1 < J) word = words[j + 1];
          }
          const uint32_t s_col = lane_base + 128u * x + 64u * buf;
          ok = mbar_wait(&s_full[2 * x + buf], (uint32_t)(c >> 1) & 1u, err, DEV_TIMEOUT_EPILOGUE);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t sv[2][32];
          tmem_ld32(s_col, sv[0]);
          tmem_ld32(s_col + 32u, sv[1]);
          tmem_wait_ld();
          if (!pos) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 32; ++i) sv[h][i] = __float_as_uint(__uint_as_float(sv[h][i]) * sc);
          }
          // keys the row does not see become -inf; tiles every row of the warp sees whole skip the test
          if (!__all_sync(0xffffffffu, vis == ~0ull)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t half = (uint32_t)(vis >> (32 * h));
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(half & (1u << i))) sv[h][i] = 0xff800000u;
            }
          }
          float mxp[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t* v = &sv[q >> 1][16 * (q & 1)];
            mxp[q] = __uint_as_float(v[0]);
#pragma unroll
            for (int i = 1; i < 15; i += 2) mxp[q] = fmaxf(mxp[q], fmaxf(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
            mxp[q] = fmaxf(mxp[q], __uint_as_float(v[15]));
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
          uint32_t pw[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const uint32_t* s2 = &sv[i >> 4][2 * (i & 15)];
            const F2 e = fma2(F2(__uint_as_float(s2[0]), __uint_as_float(s2[1])), mul2v, neg2);
            const F2 w2(ex2_approx(e.lo()), ex2_approx(e.hi()));
            sum[i & 1] = add2(sum[i & 1], w2);
            pw[i] = pack_f16x2(w2.lo(), w2.hi());
          }
          tmem_st32(s_col, pw);
          l = fmaf(l, alpha, (sum[0].lo() + sum[0].hi()) + (sum[1].lo() + sum[1].hi()));
          if (__any_sync(0xffffffffu, rescale)) {
            // P(j - 1) V has to be in the output before it is rescaled (P(j - 3) V is: S(j - 1) was issued after it, so
            // the barrier is at most one phase behind)
            ok = mbar_wait(&pv_done[2 * x + (buf ^ 1)], (uint32_t)((c - 1) >> 1) & 1u, err, DEV_TIMEOUT_EPILOGUE);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < 4 * NS; ++q) {
              uint32_t o[16];
              tmem_ld16(o_col + 16u * q, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(o_col + 16u * q, o);
            }
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * x + buf]);
        }
        if (!ok) break;
        nt += J;
      }
      // ---------------- the next item's query rows: this item's products have read theirs (its last scores are here)
      const int done_J = J, done_split = w.split, part0 = cl.part0;
      id += gridDim.x;
      bool next = id < p.items;
      if (next) {
        ok = item_keys(n + 1, k);
        if (ok) {
          w = wide_item(p, id);
          if (k.J > 0 && x * AW_M < w.rows) load_q(w);
        }
      }
      // ---------------- epilogue
      if (mine) {
        if (ok && done_J > 0) {
          ok = mbar_wait(&pv_done[2 * x + ((nt - 1) & 1)], (uint32_t)((nt - 1) >> 1) & 1u, err, DEV_TIMEOUT_EPILOGUE);
          ok = __all_sync(0xffffffffu, ok);
        }
        if (ok) {
          tc_fence_after();
          const bool part = p.part_o != nullptr;
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
          const int64_t at = ((int64_t)row.b * (int)p.TQ.d + row.t) * p.HQ + row.h;
          const int64_t slot_row = (int64_t)(part0 + done_split) * ((int64_t)p.B * (int)p.TQ.d * p.HQ) + at;
          uint16_t* orow = p.o + (int64_t)row.b * p.o_sb + (int64_t)row.h * p.o_sh + (int64_t)row.t * p.o_st;
          float* prow = part ? p.part_o + slot_row * p.DV : nullptr;
          if (part && live) p.part_ml[slot_row] = make_float2(m_used, l);
          if (!(part && done_J == 0)) {  // the merge does not read the output of an item with l = 0
#pragma unroll
            for (int q = 0; q < 2 * NS; ++q) {
              uint32_t o[32];
              if (done_J > 0) {
                tmem_ld32(o_col + 32u * q, o);
                tmem_wait_ld();
              }
              if (l == 0.0f) {  // a row that sees no key gives 0 whatever the values hold
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0u;
              }
              if (live) {
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                  if (32 * q + i >= p.DV) continue;
                  if (part) {
                    *reinterpret_cast<uint4*>(prow + 32 * q + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    *reinterpret_cast<uint4*>(prow + 32 * q + i + 4) = make_uint4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]);
                  } else {
                    uint4 v;
                    v.x = pack_f16x2(__uint_as_float(o[i + 0]) * inv, __uint_as_float(o[i + 1]) * inv);
                    v.y = pack_f16x2(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                    v.z = pack_f16x2(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
                    v.w = pack_f16x2(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
                    *reinterpret_cast<uint4*>(orow + 32 * q + i) = v;
                  }
                }
              }
            }
          }
          tc_fence_before();  // the output is read before this tile's next weights are announced
        }
      }
      if (!next) break;
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
  return (size_t)ns * (2 * AW_QSLAB + 2 * AW_ST * AW_KSLAB) + AW_TAIL;
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
      cudaError_t e =
          cudaFuncSetAttribute(wide_kernel(ns, m), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)wide_smem(ns));
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

cudaError_t launch_attention_wide(const TileParams& p, int slabs, int mask, int num_sms, cudaStream_t stream) {
  const int grid = p.items < num_sms ? p.items : num_sms;
  return launch_pdl(wide_kernel(slabs, mask), dim3((unsigned)grid), dim3(AW_THREADS), wide_smem(slabs), stream, p);
}

}  // namespace emx
