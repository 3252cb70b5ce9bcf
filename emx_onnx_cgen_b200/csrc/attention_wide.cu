// Attention over many query rows: the 256-row tile pass of K_ATTENTION_FLASH
// (attention_flash.cu has the operator, its mathematics and the 128-row pass).
//
// Per key tile a query row costs as much tensor-pipe time (2 x D x 128 fused
// multiply-adds at 4096 a clock and SM) as exponential time (128 at 16 a clock
// and SM) at D = 128, and half of it at D = 64: both units have to stay busy.
// One persistent CTA per SM keeps two 128-row tiles in flight, so that one
// tile's products run while the other's softmax does, on key tiles of 128 (a
// warp's step costs some 400 clocks beside its exponentials, and products of
// 64 keys are bound by their operand reads):
//   warps 0-3 / 4-7: softmax of row tile A / B, one thread per query row;
//   warp 8: TMA producer of the K and V tiles that both row tiles read;
//   warp 9: all products: S_A(0), S_B(0), then per key tile j
//           O_A += P_A(j) V_j, S_A(j + 1), O_B += P_B(j) V_j, S_B(j + 1);
//   warp 10: query rows of tile A, as soon as the item before has its last scores;
//           zeroes V rows past the last visible key in an item's last tile;
//   warp 11: works out the items' key ranges, an item ahead; query rows of tile B.
// TMEM: S_A, S_B, O_A, O_B, 128 columns each.  The weights P (fp16) go back
// into the first half of their scores' columns and are the A operand of the
// second product from there (no shared-memory round trip), in two halves, so
// that the first 64 keys' product runs beside the other 64 keys' exponentials.
// The products of one thread complete in order, so "S(j + 1) is ready" also says
// that O holds tile j: neither rescaling O nor overwriting S needs a wait of its
// own.  A row's 128 scores live in registers (setmaxnreg moves the other warps'
// share to the softmax warps); pairs of scores are scaled and summed by two-wide
// fp32 instructions.  Every wait is bounded (tc100.cuh).
//
// Measured: 4 x 32 heads of 128, 2048 rows, 2048-4096 of 4096 keys (8 key/value
// heads): 418 to 459 us over several boards, 0.90 to 0.99 PFLOP/s, 64 to 71 % of
// what a library product sustains at the board's power limit.  Two row tiles' step takes 3000 clocks, of which the
// products need 2050; a tile's own chain (products, TMEM load 120, maximum 350,
// exponentials 1150) is 2100, and the other tile's softmax shares its issue
// slots.  At D = 64 (8 x 16 heads, 448 x up to 1500) the step is as long: 49.3 to
// 52.3 us.
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
constexpr uint32_t AW_SLAB = 128u * 128u;  // 64 fp16 columns of 128 rows or keys: 16 KB
constexpr uint32_t AW_O_COL = 256;         // outputs; scores and weights of tile x at 128 x
constexpr int AW_REGS_SOFTMAX = 208, AW_REGS_OTHER = 88;  // two warpgroups and one: 3 x 168, what the launch holds

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

// 2^x of a pair on the fp32 units: x = n + f with n the nearest integer (added to 1.5 * 2^23 it lands in the low
// bits), 2^f by a degree-4 polynomial on [-1/2, 1/2] (least maximum relative error, 2.7e-6 as evaluated: 1/180 of
// the fp16 rounding that follows), n into the exponent.  Below -126 the result is 2^-126; x <= 127.
__device__ __forceinline__ F2 ex2_poly(F2 x) {
  x = F2(fmaxf(x.lo(), -126.0f), fmaxf(x.hi(), -126.0f));
  const F2 magic(12582912.0f, 12582912.0f), minus(-12582912.0f, -12582912.0f);
  const F2 t = add2(x, magic), n = add2(t, minus);
  const F2 f = fma2(n, F2(-1.0f, -1.0f), x);
  F2 y = fma2(F2(0.009570102207362652f, 0.009570102207362652f), f, F2(0.05591785907745361f, 0.05591785907745361f));
  y = fma2(y, f, F2(0.240247443318367f, 0.240247443318367f));
  y = fma2(y, f, F2(0.6931217908859253f, 0.6931217908859253f));
  y = fma2(y, f, F2(0.9999992847442627f, 0.9999992847442627f));
  return F2(__uint_as_float(__float_as_uint(y.lo()) + (__float_as_uint(t.lo()) << 23)),
            __uint_as_float(__float_as_uint(y.hi()) + (__float_as_uint(t.hi()) << 23)));
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
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

constexpr int wide_stages(int ns) { return ns == 1 ? 4 : 2; }  // K and V tiles in shared memory, of each
constexpr int AW_BARS = 4 * 4 + 2 + 4 + 2 + 2 + 2 + 2 + 4 + 1;
constexpr uint32_t AW_STAGE = 8 * 32 * 128;  // output staging: 32 rows of 128 bytes for each softmax warp
constexpr uint32_t AW_TAIL = AW_BARS * 8 + 2 * sizeof(WideKeys) + 16;

template <int NS, int MASK>
__global__ void __launch_bounds__(AW_THREADS, 1) attention_wide_kernel(const __grid_constant__ TileParams p) {
  constexpr uint32_t TILE = NS * AW_SLAB;
  constexpr int ST = wide_stages(NS);
  extern __shared__ __align__(1024) uint8_t aw_raw[];
  if (smem_u32(aw_raw) & 1023u) {  // the swizzled operands need a 1 KB aligned window
    if (threadIdx.x == 0) record_error(p.err, DEV_BAD_CONFIG);
    return;
  }
  uint8_t* s_q = aw_raw;  // tile A, tile B
  uint8_t* s_k = s_q + 2 * TILE;
  uint8_t* s_v = s_k + ST * TILE;
  uint8_t* s_stage = s_v + ST * TILE;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(s_stage + AW_STAGE);
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_empty = v_full + ST;
  uint64_t* s_full = v_empty + ST;  // [tile] scores ready, the key tiles before are in the output
  uint64_t* p_full = s_full + 2;    // [tile][half] weights of 64 keys written, output rescaled
  uint64_t* o_done = p_full + 4;    // [tile] an item's last key tile is in the output
  uint64_t* q_full = o_done + 2;    // [tile] the item's query rows are in shared memory
  uint64_t* q_empty = q_full + 2;   // [tile] ... and have been read
  uint64_t* v_last = q_empty + 2;       // an item's last V tile has arrived ...
  uint64_t* v_clean = v_last + 1;      // ... and its hidden rows are zero
  uint64_t* info_full = v_clean + 1;   // [2] an item's key range is known
  uint64_t* info_empty = info_full + 2;
  uint64_t* drain = info_empty + 2;
  WideKeys* s_info = reinterpret_cast<WideKeys*>(drain + 1);  // [2]
  uint32_t* holder = reinterpret_cast<uint32_t*>(s_info + 2);

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  int* const err = p.err;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 4; ++s) mbar_init(&p_full[s], 4);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&o_done[s], 1);
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
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

  // the item's key range, read by every role (whole warps)
  auto item_keys = [&](int n, WideKeys& k) -> bool {
    const bool ok = mbar_wait(&info_full[n & 1], (uint32_t)(n >> 1) & 1u, err, DEV_TIMEOUT_PRODUCER);
    if (!__all_sync(0xffffffffu, ok)) return false;
    k = s_info[n & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&info_empty[n & 1]);
    return true;
  };

  // Query rows of tile x of an item, zero past the head size and the rows, once the products have read the rows
  // before: TMA tiles of (head of the group, token), or, where a tile is no such box, this warp's 16-byte copies.
  auto load_q = [&](const WideItem& w, int x, int nth) -> bool {
    if (nth > 0 && !__all_sync(0xffffffffu, mbar_wait(&q_empty[x], (uint32_t)(nth - 1) & 1u, err, DEV_TIMEOUT_PRODUCER)))
      return false;
    if (p.q_boxes[w.shared ? 1 : 0]) {
      if (lane == 0) {
        const int t0 = p.group.div(w.row0 + x * AW_M);
        mbar_arrive_expect_tx(&q_full[x], TILE);
#pragma unroll
        for (int c = 0; c < NS; ++c)
          tma_load_5d(s_q + x * TILE + c * AW_SLAB, &p.map_q[w.shared ? 1 : 0], &q_full[x], 64 * c, 0, t0, w.kvh, w.b);
      }
      __syncwarp();
      return true;
    }
    constexpr int PIECES = NS * 8;
    const int c = lane % PIECES;
#pragma unroll 1
    for (int r = lane / PIECES; r < AW_M; r += 32 / PIECES) {
      const int rr = x * AW_M + r;
      uint8_t* dst = s_q + x * TILE + (c >> 3) * AW_SLAB + r * 128 + (((c & 7) ^ (r & 7)) << 4);
      if (rr < w.rows && c * 8 < p.D) {
        const RowId q = row_of(w.row0 + rr, p.group, p.TQ, w.kvh, w.b, w.shared);
        cp_async16(dst, p.q + (int64_t)q.b * p.q_sb + (int64_t)q.h * p.q_sh + (int64_t)q.t * p.q_st + c * 8);
      } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    cp_async_commit();
    cp_async_wait_group<0>();
    fence_async_shared();
    __syncwarp();
    if (lane == 0) mbar_arrive(&q_full[x]);
    return true;
  };

  // On the way out of a loader of query rows: its last copies (those before them have been read) have landed.
  auto q_landed = [&](int x, int loads) {
    if (loads > 0) (void)mbar_wait(&q_full[x], (uint32_t)(loads - 1) & 1u, nullptr, 0);
  };

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AW_REGS_OTHER));
  if (warp == 11) {
    // ---------------- key ranges: tiles of the past first, positions count through the tiles (attention_flash.cu)
    // (not beside the wait above, where it costs registers in the softmax)
    if (p.publish && blockIdx.x == 0) publish_waited(err, 1);
    pdl_launch_dependents();
    int nq = 0;  // items of tile B
    for (int n = 0, id = blockIdx.x; id < p.items; ++n, id += gridDim.x) {
      const WideItem w = wide_item(p, id);
      const ItemClass& cl = p.cls[w.shared ? 1 : 0];
      const int np = cl.past ? (p.tp + AW_N - 1) / AW_N : 0;
      int keys = w.shared ? 0 : p.tk;
      if (!w.shared) {
        if (p.causal) keys = min(keys, p.group.div(w.row0 + w.rows - 1) + 1);
        if (p.counts) {
          const long long c = p.counts[w.b];
          if (c < 0 || c > p.tk) record_bad_index(err);
          keys = min(keys, (int)max(0ll, min(c, (long long)p.tk)));
        }
      }
      int pbeg = 0, pend = keys > 0 ? np * AW_N + keys : (cl.past ? p.tp : 0);
      if (MASK == MASK_BITS) {
        int lo = 0x7fffffff, hi = 0;
        int4 v[8];  // (lanes past the last row read that row's again: no branch between the loads)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const RowId r = row_of(w.row0 + min(32 * i + lane, w.rows - 1), p.group, p.TQ, w.kvh, w.b, w.shared);
          v[i] = p.spans[r.b * p.mask_sb + r.h * p.mask_sh + r.t * p.mask_st];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (cl.past && v[i].z < v[i].w) lo = min(lo, v[i].z), hi = max(hi, v[i].w);
          if (!w.shared && v[i].x < v[i].y) lo = min(lo, np * AW_N + v[i].x), hi = max(hi, np * AW_N + v[i].y);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        pbeg = lo, pend = min(pend, hi);
      }
      const int j_lo = pbeg < pend ? pbeg / AW_N : 0, j_hi = pbeg < pend ? (pend + AW_N - 1) / AW_N : 0;
      WideKeys k;
      k.j0 = j_lo + split_start(j_hi - j_lo, w.split, cl.splits);
      k.J = j_lo + split_start(j_hi - j_lo, w.split + 1, cl.splits) - k.j0;
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
      if (k.J > 0 && w.rows > AW_M) {
        if (!load_q(w, 1, nq)) break;
        ++nq;
      }
    }
    q_landed(1, nq);
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
          const int s = nkv % ST, jj = k.j0 + j;
          const int in_past = jj < np ? 1 : 0, key0 = (in_past ? jj : jj - np) * AW_N;
          const int kb = in_past && p.past_shared ? 0 : w.b;
          const uint32_t ph = (uint32_t)(nkv / ST - 1) & 1u;
          if (p.drop_keys && nkv > 0) ok = false;
          if (ok && nkv >= ST && !mbar_wait(&k_empty[s], ph, err, DEV_TIMEOUT_PRODUCER)) ok = false;
          if (!ok) break;
          mbar_arrive_expect_tx(&k_full[s], TILE);
#pragma unroll
          for (int c = 0; c < NS; ++c)
            tma_load_4d(s_k + s * TILE + c * AW_SLAB, &p.map_k[in_past], &k_full[s], 64 * c, key0, w.kvh, kb);
          issued = 2 * nkv + 1;
          if (nkv >= ST && !mbar_wait(&v_empty[s], ph, err, DEV_TIMEOUT_PRODUCER)) ok = false;
          if (!ok) break;
          mbar_arrive_expect_tx(&v_full[s], TILE);
#pragma unroll
          for (int c = 0; c < NS; ++c)
            tma_load_4d(s_v + s * TILE + c * AW_SLAB, &p.map_v[in_past], &v_full[s], 64 * c, key0, w.kvh, kb);
          issued = 2 * nkv + 2;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    }
    if (!ok && lane == 0) {  // error path: let the copies in flight land before the CTA exits
      for (int i = max(0, issued - 2 * ST); i < issued; ++i) {
        const int j = i >> 1;
        (void)mbar_wait((i & 1) ? &v_full[j % ST] : &k_full[j % ST], (uint32_t)(j / ST) & 1u, nullptr, 0);
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
    const uint64_t v_desc = smem_desc_mn_sw128(smem_u32(s_v), AW_SLAB, 1024u);
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
        const int kv = nkv + j, s = kv % ST;
        if (x == 0 && !wait(&k_full[s], kv / ST)) return false;
        tc_fence_after();
        if (elect_one()) {
          // descriptors hold addresses in 16-byte units in their low bits: a step along d is an addition
          const uint64_t q = q_desc + x * (TILE >> 4), kt = k_desc + s * (TILE >> 4);
#pragma unroll
          for (int ks = 0; ks < 4 * NS; ++ks) {
            const uint32_t off = ((ks >> 2) * AW_SLAB + (ks & 3) * 32u) / 16u;
            if (ks < nks) mma_f16(tmem + 128u * x, q + off, kt + off, idesc_s, ks > 0 ? 1u : 0u);
          }
          tc_commit(&s_full[x]);
          if (x == tiles - 1) tc_commit(&k_empty[s]);
          if (j == k.J - 1) tc_commit(&q_empty[x]);
        }
        __syncwarp();
        return true;
      };
      for (int x = 0; x < tiles && ok; ++x) {
        ok = wait(&q_full[x], nq[x]);
        if (ok) ok = scores(x, 0);
      }
      for (int j = 0; j < k.J && ok; ++j) {
        const int kv = nkv + j, s = kv % ST;
        ok = wait(&v_full[s], kv / ST);
        if (ok && j == k.J - 1 && k.last < AW_N) {
          if (lane == 0) mbar_arrive(v_last);
          ok = wait(v_clean, nclean);
          ++nclean;
        }
        for (int x = 0; x < tiles && ok; ++x) {
          const uint64_t v = v_desc + s * (TILE >> 4);
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // O_x += P_x(j) V_j, 64 keys at a time
            if (!ok) break;
            ok = wait(&p_full[2 * x + h], nt[x] + j);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
                mma_f16_ts(tmem + AW_O_COL + 128u * x, tmem + 128u * x + 8u * kk, v + kk * (16u * 128u / 16u), idesc_o,
                           (j | kk) ? 1u : 0u);
              if (h == 1 && x == tiles - 1) tc_commit(&v_empty[s]);
              if (h == 1 && j == k.J - 1) tc_commit(&o_done[x]);
            }
            __syncwarp();
          }
          if (ok && j + 1 < k.J) ok = scores(x, j + 1);
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
    // ---------------- query rows of tile A; values past the last visible key take no part
    int nkv = 0, nclean = 0, nq = 0;
    for (int n = 0, id = blockIdx.x; id < p.items; ++n, id += gridDim.x) {
      WideKeys k;
      if (!item_keys(n, k)) break;
      if (k.J > 0) {
        if (!load_q(wide_item(p, id), 0, nq)) break;
        ++nq;
      }
      nkv += k.J;
      if (k.J == 0 || k.last >= AW_N) continue;
      const int s = (nkv - 1) % ST;
      const bool ok = mbar_wait(v_last, (uint32_t)nclean & 1u, err, DEV_TIMEOUT_MMA);
      if (!__all_sync(0xffffffffu, ok)) break;
      for (int i = lane; i < (AW_N - k.last) * 8 * NS; i += 32) {
        const int c = i % (8 * NS), r = k.last + i / (8 * NS);
        *reinterpret_cast<uint4*>(s_v + s * TILE + (c >> 3) * AW_SLAB + r * 128 + (c & 7) * 16) =
            make_uint4(0u, 0u, 0u, 0u);
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(v_clean);
      ++nclean;
    }
    q_landed(0, nq);
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AW_REGS_SOFTMAX));
    // ---------------- softmax and epilogue: thread = query row (warp % 4 = TMEM lane quarter)
    const int x = warp >> 2, quarter = warp & 3;
    const int rt = quarter * 32 + lane;  // row within the tile
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_col = lane_base + AW_O_COL + 128u * x;
    const float sc = p.scale_log2;
    const bool pos = sc > 0.0f;
    const float mul = pos ? sc : 1.0f;
    int nt = 0, nitems = 0;  // key tiles, items of this row tile so far
    int id = blockIdx.x;
    WideItem w = {};
    WideKeys k = {};
    bool ok = id < p.items && item_keys(0, k);
    if (ok) w = wide_item(p, id);
    for (int n = 0; ok; ++n) {
      const int r = x * AW_M + rt;
      const bool mine = x * AW_M < w.rows, live = r < w.rows;  // whether the tile, the row exists
      const ItemClass& cl = p.cls[w.shared ? 1 : 0];
      const RowId row = row_of(w.row0 + (live ? r : 0), p.group, p.TQ, w.kvh, w.b, w.shared);
      float m_used = -INFINITY;  // reference of the exponentials, log2 units
      float l = 0.0f;
      F2 mul2v(mul, mul);
      const int J = mine ? k.J : 0;
      if (J > 0) {
        const int np = cl.past ? (p.tp + AW_N - 1) / AW_N : 0;
        const int row_end = p.causal ? min(k.keys, row.t + 1) : k.keys;
        const unsigned long long* words = nullptr;
        unsigned long long word[2] = {0ull, 0ull};  // the next tile's, loaded a tile ahead
        if (MASK == MASK_BITS) {
          words = p.bits + (row.b * p.mask_sb + row.h * p.mask_sh + row.t * p.mask_st) * p.words +
                  (cl.past ? 0 : p.words_past) + 2 * k.j0;
          word[0] = words[0], word[1] = words[1];
        }
        for (int j = 0; j < J; ++j) {
          const int jj = k.j0 + j;
          const bool in_past = jj < np;
          const int end = (in_past ? p.tp : row_end) - (in_past ? jj : jj - np) * AW_N;
          unsigned long long vis[2] = {~0ull, ~0ull};  // visible keys of the tile, one bit each
          if (end < AW_N) {
            vis[0] = end >= 64 ? ~0ull : end > 0 ? (1ull << end) - 1 : 0ull;
            vis[1] = end > 64 ? (1ull << (end - 64)) - 1 : 0ull;
          }
          if (MASK == MASK_BITS) {
            vis[0] &= word[0], vis[1] &= word[1];
            if (j + 1 < J) word[0] = words[2 * j + 2], word[1] = words[2 * j + 3];
          }
          const uint32_t s_col = lane_base + 128u * x;
          ok = mbar_wait(&s_full[x], (uint32_t)(nt + j) & 1u, err, DEV_TIMEOUT_EPILOGUE);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t sv[4][32];
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld32(s_col + 32u * q, sv[q]);
          tmem_wait_ld();
          if (!pos) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int i = 0; i < 32; ++i) sv[q][i] = __float_as_uint(__uint_as_float(sv[q][i]) * sc);
          }
          // keys the row does not see become -inf; tiles every row of the warp sees whole skip the test
          if (!__all_sync(0xffffffffu, (vis[0] & vis[1]) == ~0ull)) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t half = (uint32_t)(vis[q >> 1] >> (32 * (q & 1)));
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(half & (1u << i))) sv[q][i] = 0xff800000u;
            }
          }
          // NaN scores make the maximum NaN, an infinite one is made to: either makes the whole row NaN, as exp does
          float mxp[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const uint32_t* v = &sv[q >> 1][16 * (q & 1)];
            mxp[q] = __uint_as_float(v[0]);
#pragma unroll
            for (int i = 1; i < 15; i += 2)
              mxp[q] = max3_nan(mxp[q], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
            mxp[q] = max_nan(mxp[q], __uint_as_float(v[15]));
          }
          const float mx = max_nan(max_nan(max_nan(mxp[0], mxp[1]), max_nan(mxp[2], mxp[3])),
                                   max_nan(max_nan(mxp[4], mxp[5]), max_nan(mxp[6], mxp[7]))) * mul;
          bool rescale = false;
          float alpha = 1.0f;
          // (rows of large scores come through here every time)
          const bool stop = !(mx - m_used <= AFK_RESCALE) || large_scores(m_used);
          if (!(mx - m_used <= AFK_RESCALE)) {  // (also where there was none before)
            rescale = j > 0 && m_used != -INFINITY;
            if (rescale) alpha = ex2_approx(m_used - mx);
            m_used = mx == INFINITY ? NAN : mx;
          }
          if (__any_sync(0xffffffffu, stop)) {
            const bool large = __any_sync(0xffffffffu, large_scores(m_used));
            mul2v = large ? F2(1.0f, 1.0f) : F2(mul, mul);
            if (large && pos) {
#pragma unroll
              for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 32; ++i) sv[q][i] = __float_as_uint(__uint_as_float(sv[q][i]) * sc);
            }
            if (__any_sync(0xffffffffu, rescale)) {
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
          }
          const float neg_m = m_used == -INFINITY ? 0.0f : -m_used;
          const F2 neg2(neg_m, neg_m);
          F2 sum[2] = {F2(0.0f, 0.0f), F2(0.0f, 0.0f)};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int q = 2 * h; q < 2 * h + 2; ++q) {
              uint32_t pw[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const F2 e = fma2(F2(__uint_as_float(sv[q][2 * i]), __uint_as_float(sv[q][2 * i + 1])), mul2v, neg2);
                // At D > 64 an eighth of the exponentials runs on the fp32 units, beside the exponential unit's:
                // [4, 32, 2048 x 4096, 128] takes 412 us so, 423 us with none and with a quarter.  At D <= 64 issue
                // slots are what is short: [8, 16, 448 x 1500, 64] takes 50.6 us with none, 51.2 and 52.6 us with
                // an eighth and a quarter.
                const F2 w2 = NS == 2 && i % 8 == 7 ? ex2_poly(e) : F2(ex2_approx(e.lo()), ex2_approx(e.hi()));
                sum[i & 1] = add2(sum[i & 1], w2);  // (before the rounding)
                pw[i] = pack_f16x2(w2.lo(), w2.hi());
              }
              tmem_st16(s_col + 16u * q, pw);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * x + h]);
          }
          l = fmaf(l, alpha, (sum[0].lo() + sum[0].hi()) + (sum[1].lo() + sum[1].hi()));
        }
        if (!ok) break;
        if (m_used == -INFINITY) l = 0.0f;  // no visible key: what is there are 2^-126 of ex2_poly
        nt += J, ++nitems;
      }
      // ---------------- the next item
      const int done_J = J, done_split = w.split, part0 = cl.part0;
      id += gridDim.x;
      bool next = id < p.items;
      if (next) {
        ok = item_keys(n + 1, k);
        if (ok) w = wide_item(p, id);
      }
      // ---------------- epilogue
      if (mine) {
        if (ok && done_J > 0) {
          ok = mbar_wait(&o_done[x], (uint32_t)(nitems - 1) & 1u, err, DEV_TIMEOUT_EPILOGUE);
          ok = __all_sync(0xffffffffu, ok);
        }
        if (ok) {
          tc_fence_after();
          const bool part = p.part_o != nullptr;
          const float inv = part ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
          const int64_t at = ((int64_t)row.b * (int)p.TQ.d + row.t) * p.HQ + row.h;
          const int64_t slot0 = (int64_t)(part0 + done_split) * ((int64_t)p.B * (int)p.TQ.d * p.HQ);
          // where this row's results start; rows past the last have none
          const long long mine_at = !live ? -1 : part ? (slot0 + at) * p.DV
                                              : row.b * p.o_sb + row.h * p.o_sh + row.t * p.o_st;
          if (part && live) p.part_ml[slot0 + at] = make_float2(m_used, l);
          if (!(part && done_J == 0)) {  // the merge does not read the output of an item with l = 0
            // 128 bytes of a row at a time through shared memory (swizzled by the row), so that eight lanes write a
            // row's 128 bytes together
            uint8_t* const stage = s_stage + warp * 32 * 128;
            const int bytes = p.DV * (part ? 4 : 2), cols = part ? 32 : 64;
#pragma unroll 1
            for (int c0 = 0; c0 < p.DV; c0 += cols) {
#pragma unroll 1
              for (int h = 0; h < cols; h += 32) {
                uint32_t o[32];
                if (done_J > 0) {
                  tmem_ld32(o_col + (uint32_t)(c0 + h), o);
                  tmem_wait_ld();
                }
                if (l == 0.0f) {  // a row that sees no key gives 0 whatever the values hold
#pragma unroll
                  for (int i = 0; i < 32; ++i) o[i] = 0u;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  if (part) {
                    *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) =
                        make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                  } else if (i < 4) {
                    uint4 v;
                    v.x = pack_f16x2(__uint_as_float(o[8 * i + 0]) * inv, __uint_as_float(o[8 * i + 1]) * inv);
                    v.y = pack_f16x2(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv);
                    v.z = pack_f16x2(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv);
                    v.w = pack_f16x2(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv);
                    *reinterpret_cast<uint4*>(stage + lane * 128 + (((h / 8 + i) ^ (lane & 7)) << 4)) = v;
                  }
                }
              }
              __syncwarp();
              uint8_t* const out = part ? reinterpret_cast<uint8_t*>(p.part_o) : reinterpret_cast<uint8_t*>(p.o);
              const int piece = lane & 7, byte = c0 * (part ? 4 : 2) + piece * 16;
#pragma unroll
              for (int r0 = 0; r0 < 32; r0 += 4) {
                const int rr = r0 + (lane >> 3);
                const long long to = __shfl_sync(0xffffffffu, mine_at, rr);
                const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 128 + ((piece ^ (rr & 7)) << 4));
                if (to >= 0 && byte < bytes) *reinterpret_cast<uint4*>(out + to * (part ? 4 : 2) + byte) = v;
              }
              __syncwarp();
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
  return (size_t)ns * (2 + 2 * wide_stages(ns)) * AW_SLAB + AW_STAGE + AW_TAIL;
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
      if (3 * a.numRegs < 2 * AW_REGS_SOFTMAX + AW_REGS_OTHER) return cudaErrorInvalidKernelImage;
      e = cudaFuncSetAttribute(wide_kernel(ns, m), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)wide_smem(ns));
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

cudaError_t launch_attention_wide(const TileParams& p, int slabs, int mask, int num_sms, cudaStream_t stream) {
  const int grid = p.items < num_sms ? p.items : num_sms;
  return launch_pdl(wide_kernel(slabs, mask), dim3((unsigned)grid), dim3(AW_THREADS), wide_smem(slabs), stream, p);
}

}  // namespace emx
