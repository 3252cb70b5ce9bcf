// ONNX Attention (opsets 23/24), fp16 in and out, for the forms a decoder
// layer uses beside plain self-attention: queries and keys of different
// lengths (cross attention), boolean and additive masks, valid key counts,
// grouped key/value heads, head sizes up to 128, and a past that is one prefix
// shared by the whole batch.  (attention.cu repeats the reference's fp16
// rounding, attention_tc.cu is the unmasked 128-wide fast mode.)
//
// Mathematics: per query row, over its visible keys,
//   o = sum_k 2^(x_k - m) v_k / sum_k 2^(x_k - m),   x_k = (scale q.k + mask_k) log2 e
// evaluated online tile by tile: running reference m, sum l and output
// accumulator are fp32 (TMEM for the latter); the weights are rounded to fp16
// for the second matrix product (half an fp16 step each, 2^-11 relative: the
// output type's own step; 2^-25 of the reference's weight below 2^-14 of it).
// This pass's sum adds the rounded weights; the 256-row and the few-row pass
// add them as they are, which keeps the conversions out of the sum's chain.
// Either way numerator and sum are within half a step per weight of exact.  A
// row that sees no key gives 0.  Additive entries are taken relative to a mask
// reference of the row (attention_flash.cuh) before the score is added, so
// scores keep their digits beside masks as large as the type's lowest value.
//
// Rows: the query rows that read the same keys are packed into tiles of 128
// whatever (token, head, sequence) they come from -- the group of query heads
// of one key/value head, all tokens, and, against a shared prefix, all
// sequences of the batch.  Against a shared prefix the prefix's K and V are so
// read once for the batch instead of once per sequence.
//
// Key ranges: the past ("segment 1") and the current keys ("segment 0") are
// separate work items, and each may be split further along the keys when there
// are too few row tiles for the SMs.  With more than one item per row every
// item writes its (m, l, o) in fp32 and attention_combine_kernel merges them:
//   M = max m_s,  o = sum 2^(m_s - M) o_s / sum 2^(m_s - M) l_s
// in a fixed order, so results do not depend on timing.
//
// One CTA per work item, two per SM.  Warp 0: TMA producer of K and V tiles of
// 64 keys.  Warp 1: S_j = Q K_j^T (tcgen05 kind::f16) into one of two TMEM
// score buffers.  Warp 2: O += P_j V_j.  Warps 4-7: one thread per query row,
// softmax and epilogue; a warp without rows leaves at once.  Every wait is
// bounded (tc100.cuh).  Operand layouts in shared memory are the 128-byte
// swizzle the TMA writes: Q and K as 64-wide slabs (K-major), P one such slab,
// V as 64-wide slabs read MN-major.
//
// What bounds it: at two CTAs an SM the softmax warps' issue slots (64 scores a
// row and tile in registers, an exponential each), then, for short keys, the
// set-up of a work item (TMEM, barriers, Q: some 5 us).  [57, 16, 45 x 2952, 96]
// with an fp16 additive mask: 211 us, 221 TFLOP/s; [3, 12, 77 x 333, 80]: 16.4
// to 17.1 us, three launches.
//
// Boolean masks are first packed by mask_pack_kernel to one 64-bit word per
// (mask row, 64 keys) plus each row's first and last visible key, so a row's
// thread reads 8 aligned bytes per tile whatever the mask's alignment, and
// tiles outside the rows' span (padding) are not read at all.  Additive masks are
// first laid out by tiles (mask_tiles_kernel).  Keys past a
// work item's last visible key inside its last tile have their V rows zeroed
// in shared memory: what padding holds, NaN included, reaches no result.
#include <cuda_fp16.h>

#include "attention_flash.cuh"
#include <algorithm>

#include "host_util.h"
#include "kernels.h"
#include "tc100.cuh"
#include "tmem32.cuh"

namespace emx {

constexpr int AFK_M = 128;  // packed query rows per work item
constexpr int AFK_N = 64;   // keys per tile
constexpr int AFK_THREADS = 256;
constexpr uint32_t AFK_QSLAB = AFK_M * 128u;  // 64 fp16 columns of the Q tile (and the P tile): 16 KB
constexpr uint32_t AFK_KSLAB = AFK_N * 128u;  // 64 fp16 columns of a K or V tile: 8 KB
constexpr uint32_t AFK_TMEM_COLS = 256;       // scores at columns 0 and 64, output at 128
constexpr uint32_t AFK_O_COL = 128;

// Eight entries of an additive mask from 16 bytes of fp16, or 32 of fp32.
__device__ __forceinline__ void mask_entries(const uint4& v, float (&mk)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
    mk[2 * e] = f.x;
    mk[2 * e + 1] = f.y;
  }
}
__device__ __forceinline__ void mask_entries(const uint4& a, const uint4& b, float (&mk)[8]) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) mk[e] = __uint_as_float(w[e]);
}

// Eight fp16 entries with -inf for keys whose bit is not set.
__device__ __forceinline__ uint4 hide_entries(uint4 v, uint32_t see) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (!(see & (1u << (2 * e)))) w[e] = (w[e] & 0xffff0000u) | 0xfc00u;
    if (!(see & (2u << (2 * e)))) w[e] = (w[e] & 0xffffu) | 0xfc000000u;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The largest of a tile's fp16 entries (NaN left out).
template <int N>
__device__ __forceinline__ float largest_entry(const uint4 (&raw)[N]) {
  __half2 m[4];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __half2 v = *reinterpret_cast<const __half2*>(&w[e]);
      m[e] = i == 0 ? v : __hmax2(m[e], v);
    }
  }
  const float2 f = __half22float2(__hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3])));
  return fmaxf(f.x, f.y);
}

template <int NS, int MASK>
__global__ void __launch_bounds__(AFK_THREADS, 2) attention_flash_kernel(const __grid_constant__ TileParams p) {
  constexpr bool ADD32 = MASK == MASK_ADD32, ADD = MASK == MASK_ADD || ADD32;
  using Ref = MaskReference<ADD32>;
  constexpr uint32_t QTILE = NS * AFK_QSLAB, KTILE = NS * AFK_KSLAB;
  constexpr int ST = NS == 1 ? 4 : 2;  // K and V stages: 64 KB of loads in flight per CTA at either head size
  extern __shared__ __align__(1024) uint8_t afk_raw[];
  if (smem_u32(afk_raw) & 1023u) {  // the swizzled operands need a 1 KB aligned window
    if (threadIdx.x == 0) record_error(p.err, DEV_BAD_CONFIG);
    return;
  }
  uint8_t* s_q = afk_raw;
  uint8_t* s_k = s_q + QTILE;
  uint8_t* s_v = s_k + ST * KTILE;
  uint8_t* s_p = s_v + ST * KTILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_p + AFK_QSLAB);
  uint64_t* k_full = bars;
  uint64_t* k_empty = bars + ST;
  uint64_t* v_full = bars + 2 * ST;
  uint64_t* v_empty = bars + 3 * ST;
  uint64_t* s_full = bars + 4 * ST;
  uint64_t* s_empty = s_full + 2;
  uint64_t* p_full = s_full + 4;
  uint64_t* o_done = s_full + 5;
  uint64_t* drain = s_full + 6;  // [2]
  uint32_t* holder = reinterpret_cast<uint32_t*>(s_full + 8);
  int* span = reinterpret_cast<int*>(holder + 1);  // [2] first and end key of the work item's rows

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
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
  const int row0 = tile * AFK_M;
  const int rows = min(AFK_M, rows_all - row0);
  const int nact = (rows + 31) >> 5;  // softmax warps with rows

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], (uint32_t)nact);
      mbar_init(&drain[s], 1);
    }
    mbar_init(p_full, (uint32_t)nact);
    mbar_init(o_done, 1);
    fence_barrier_init();
    span[0] = 0x7fffffff;
    span[1] = 0;
  }
  if (warp == 1) {
    tmem_alloc(holder, AFK_TMEM_COLS);
    tmem_relinquish();
  }
  pdl_wait();  // Q, K, V, masks and counts may come from the preceding kernel
  if (p.publish && blockIdx.x == 0 && threadIdx.x == 0) publish_waited(p.err, 1);
  pdl_launch_dependents();

  // ---------------- Q tile, zero past the head size and the rows
  for (int i = threadIdx.x; i < AFK_M * NS * 8; i += AFK_THREADS) {
    const int c = i % (NS * 8), r = i / (NS * 8);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < rows && c * 8 < p.D) {
      const RowId w = row_of(row0 + r, p.group, p.TQ, kvh, b, shared);
      v = *reinterpret_cast<const uint4*>(p.q + (int64_t)w.b * p.q_sb + (int64_t)w.h * p.q_sh + (int64_t)w.t * p.q_st +
                                          c * 8);
    }
    *reinterpret_cast<uint4*>(s_q + (c >> 3) * AFK_QSLAB + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
  }
  fence_async_shared();

  // ---------------- keys that some row of the work item sees: key tiles, the past's first.  Positions count
  // through the tiles: past key k is position k, current key k is position np * AFK_N + k.
  const int np = cl.past ? (p.tp + AFK_N - 1) / AFK_N : 0;
  int keys = shared ? 0 : p.tk;
  if (!shared) {
    if (p.causal) keys = min(keys, p.group.div(row0 + rows - 1) + 1);
    if (p.counts) {
      const long long n = p.counts[b];
      if (n < 0 || n > p.tk) record_bad_index(err);
      keys = min(keys, (int)max(0ll, min(n, (long long)p.tk)));
    }
  }
  int pbeg = 0, pend = keys > 0 ? np * AFK_N + keys : (cl.past ? p.tp : 0);
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
        atomicMin(&span[0], np * AFK_N + v.x);
        atomicMax(&span[1], np * AFK_N + v.y);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *holder, 0);
  if (MASK == MASK_BITS) {
    pbeg = span[0];
    pend = min(pend, span[1]);
  }
  // this split's share of the tiles
  const int j_lo = pbeg < pend ? pbeg / AFK_N : 0, j_hi = pbeg < pend ? (pend + AFK_N - 1) / AFK_N : 0;
  const int j0 = j_lo + split_start(j_hi - j_lo, split, cl.splits);
  const int J = j_lo + split_start(j_hi - j_lo, split + 1, cl.splits) - j0;

  if (warp == 0) {
    if (lane == 0 && J > 0) {
      // ---------------- producer
      bool ok = true;
      int issued = 0;
      for (int j = 0; j < J && ok; ++j) {
        const int s = j % ST, jj = j0 + j;
        const int in_past = jj < np ? 1 : 0, key0 = (in_past ? jj : jj - np) * AFK_N;
        const int kb = in_past && p.past_shared ? 0 : b;
        const uint32_t ph = (uint32_t)(j / ST - 1) & 1u;
        if (p.drop_keys && j > 0) ok = false;
        if (ok && j >= ST && !mbar_wait(&k_empty[s], ph, err, DEV_TIMEOUT_PRODUCER)) ok = false;
        if (!ok) break;
        mbar_arrive_expect_tx(&k_full[s], KTILE);
#pragma unroll
        for (int c = 0; c < NS; ++c)
          tma_load_4d(s_k + s * KTILE + c * AFK_KSLAB, &p.map_k[in_past], &k_full[s], 64 * c, key0, kvh, kb);
        issued = 2 * j + 1;
        if (j >= ST && !mbar_wait(&v_empty[s], ph, err, DEV_TIMEOUT_PRODUCER)) ok = false;
        if (!ok) break;
        mbar_arrive_expect_tx(&v_full[s], KTILE);
#pragma unroll
        for (int c = 0; c < NS; ++c)
          tma_load_4d(s_v + s * KTILE + c * AFK_KSLAB, &p.map_v[in_past], &v_full[s], 64 * c, key0, kvh, kb);
        issued = 2 * j + 2;
      }
      if (!ok) {  // error path: let the copies in flight land before the CTA exits
        for (int i = max(0, issued - 2 * ST); i < issued; ++i) {
          const int j = i >> 1;
          (void)mbar_wait((i & 1) ? &v_full[j % ST] : &k_full[j % ST], (uint32_t)(j / ST) & 1u, nullptr, 0);
        }
      }
    }
  } else if (warp == 1) {
    if (J > 0) {
      // ---------------- S issuer.  The warp goes through the waits together and an elected thread issues: operands
      // known to be uniform cost a product the tensor pipe's time, not some 100 clocks of issue an instruction.
      const uint32_t idesc = make_idesc(1u, 0u, 0u, AFK_M, AFK_N);
      const int nks = (p.D + 15) / 16;
      const uint64_t q = smem_desc_k_sw128(smem_u32(s_q), 1024), k = smem_desc_k_sw128(smem_u32(s_k), 1024);
      for (int j = 0; j < J; ++j) {
        const int s = j % ST, sb = j & 1;
        bool ok = mbar_wait(&k_full[s], (uint32_t)(j / ST) & 1u, err, DEV_TIMEOUT_MMA);
        if (ok && j >= 2) ok = mbar_wait(&s_empty[sb], (uint32_t)((j >> 1) - 1) & 1u, err, DEV_TIMEOUT_MMA);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        if (elect_one()) {
          // descriptors hold addresses in 16-byte units in their low bits: a step along d is an addition
          const uint64_t kt = k + s * (KTILE >> 4);
#pragma unroll
          for (int ks = 0; ks < 4 * NS; ++ks)
            if (ks < nks)
              mma_f16(tmem + (uint32_t)(sb * AFK_N), q + ((ks >> 2) * AFK_QSLAB + (ks & 3) * 32u) / 16u,
                      kt + ((ks >> 2) * AFK_KSLAB + (ks & 3) * 32u) / 16u, idesc, ks > 0 ? 1u : 0u);
          tc_commit(&s_full[sb]);
          tc_commit(&k_empty[s]);
        }
        __syncwarp();
      }
      // every MMA this thread issued completes before TMEM is released
      if (elect_one()) {
        tc_commit(&drain[0]);
        (void)mbar_wait(&drain[0], 0, nullptr, 0);
      }
      __syncwarp();
    }
  } else if (warp == 2) {
    if (J > 0) {
      // ---------------- P.V issuer (as the S issuer)
      const uint64_t pd = smem_desc_k_sw128(smem_u32(s_p), 1024), v = smem_desc_mn_sw128(smem_u32(s_v), AFK_KSLAB, 1024u);
      const uint32_t idesc = make_idesc(1u, 0u, 0u, AFK_M, (uint32_t)((p.DV + 15) & ~15)) | (1u << 16);
      for (int j = 0; j < J; ++j) {
        const int s = j % ST;
        bool ok = mbar_wait(&v_full[s], (uint32_t)(j / ST) & 1u, err, DEV_TIMEOUT_MMA);
        if (!__all_sync(0xffffffffu, ok)) break;
        const int nv = pend - (j0 + j) * AFK_N;
        if (nv < AFK_N) {  // keys past the last visible one: their values take no part
          for (int i = lane; i < (AFK_N - nv) * 8 * NS; i += 32) {
            const int c = i % (8 * NS), r = nv + i / (8 * NS);
            *reinterpret_cast<uint4*>(s_v + s * KTILE + (c >> 3) * AFK_KSLAB + r * 128 + (c & 7) * 16) =
                make_uint4(0u, 0u, 0u, 0u);
          }
          fence_async_shared();
          __syncwarp();
        }
        ok = mbar_wait(p_full, (uint32_t)j & 1u, err, DEV_TIMEOUT_MMA);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vt = v + s * (KTILE >> 4);
#pragma unroll
          for (int kk = 0; kk < AFK_N / 16; ++kk)
            mma_f16(tmem + AFK_O_COL, pd + kk * 2u, vt + kk * (16u * 128u / 16u), idesc, (j > 0 || kk > 0) ? 1u : 0u);
          tc_commit(o_done);
          tc_commit(&v_empty[s]);
        }
        __syncwarp();
      }
      if (elect_one()) {
        tc_commit(&drain[1]);
        (void)mbar_wait(&drain[1], 0, nullptr, 0);
      }
      __syncwarp();
    }
  } else if (warp >= 4 && warp - 4 < nact) {
    // ---------------- softmax and epilogue: thread = query row (warp % 4 = TMEM lane quarter)
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const bool live = r < rows;
    const RowId w = row_of(row0 + (live ? r : 0), p.group, p.TQ, kvh, b, shared);
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const int row_end = p.causal ? min(keys, w.t + 1) : keys;  // end of the current keys this row may see
    const int64_t mrow = MASK == MASK_NONE ? 0 : w.b * p.mask_sb + w.h * p.mask_sh + w.t * p.mask_st;
    float m_used = -INFINITY;  // reference of the exponentials, log2 units
    float l = 0.0f;            // sum of the fp16-rounded weights
    const float sc = p.scale_log2;
    const bool pos = sc > 0.0f;
    const unsigned long long* words = MASK == MASK_BITS ? p.bits + mrow * p.words + (cl.past ? 0 : p.words_past) + j0 : nullptr;
    unsigned long long word = MASK == MASK_BITS && J > 0 ? words[0] : 0ull;  // the next tile's, loaded a tile ahead
    const uint4* entries = p.add;  // this row's piece 0 of the tile
    if (ADD) entries += mrow + (int64_t)((cl.past ? 0 : p.words_past) + j0) * (ADD32 ? 16 : 8) * p.mask_rows;
    float ref = 0.0f;  // mask reference
    bool ok = true;
    for (int j = 0; j < J && ok; ++j) {
      const int sb = j & 1, jj = j0 + j;
      const bool in_past = jj < np;
      const int key0 = (in_past ? jj : jj - np) * AFK_N;
      // visible keys of the tile, one bit each
      unsigned long long vis = ~0ull;
      const int end = (in_past ? p.tp : row_end) - key0;
      if (end < AFK_N) vis = end > 0 ? (1ull << end) - 1 : 0ull;
      if (MASK == MASK_BITS) {
        vis &= word;
        if (j + 1 < J) word = words[j + 1];
      }
      // the tile's mask entries: fp16, held from here on; fp32, loaded where they are used (twice the registers)
      uint4 raw[MASK == MASK_ADD ? 8 : 1];
      if (MASK == MASK_ADD) {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = __ldg(entries + i * p.mask_rows);
      }
      // tiles every row of the warp sees whole skip the test of its keys
      const bool cut = !__all_sync(0xffffffffu, vis == ~0ull);
      auto load_entries = [&](int i, float (&mk)[8]) {  // of keys 8i .. 8i + 7
        if (MASK == MASK_ADD) mask_entries(raw[i], mk);
        else mask_entries(__ldg(entries + 2 * i * p.mask_rows), __ldg(entries + (2 * i + 1) * p.mask_rows), mk);
      };
      ok = mbar_wait(&s_full[sb], (uint32_t)(j >> 1) & 1u, err, DEV_TIMEOUT_EPILOGUE);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t sv[2][32];
      tmem_ld32(tmem + lane_base + (uint32_t)(sb * AFK_N), sv[0]);
      tmem_ld32(tmem + lane_base + (uint32_t)(sb * AFK_N + 32), sv[1]);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[sb]);
      if (!pos) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) sv[c][i] = __float_as_uint(__uint_as_float(sv[c][i]) * sc);
      }
      float mul = pos ? sc : 1.0f;
      // keys the row does not see become -inf, and so do their fp16 entries, whatever they are
      auto hide = [&]() {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t half = c ? (uint32_t)(vis >> 32) : (uint32_t)vis;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(half & (1u << i))) sv[c][i] = 0xff800000u;
        }
      };
      if (cut && !ADD32) {
        if (MASK == MASK_ADD) {
#pragma unroll
          for (int i = 0; i < 8; ++i) raw[i] = hide_entries(raw[i], (uint32_t)(vis >> (8 * i)));
        }
        hide();
      }
      if (ADD) {
        // the largest entry of a key that the row sees; does it move the reference?
        float top = -INFINITY;
        if (MASK == MASK_ADD) {
          top = largest_entry(raw);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float mk[8];
            load_entries(i, mk);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (!cut || ((vis >> (8 * i + e)) & 1u)) top = fmaxf(top, mk[e]);
          }
        }
        if (Ref::moves(top, ref, m_used)) {
          m_used = Ref::moved(m_used, ref, Ref::of(top));
          ref = Ref::of(top);
        }
        // scores with their entries (-inf hides the key); from here on as without a mask
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float mk[8];
            load_entries(4 * c + i / 8, mk);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              sv[c][i + e] = __float_as_uint(Ref::score(mk[e], ref, __uint_as_float(sv[c][i + e]) * mul));
          }
        if (cut && ADD32) hide();
        mul = 1.0f;
      }
      float mxp[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i) mxp[i & 3] = fmaxf(mxp[i & 3], __uint_as_float(sv[c][i]));
      const float mx = fmaxf(fmaxf(mxp[0], mxp[1]), fmaxf(mxp[2], mxp[3])) * mul;
      float m_new = m_used;
      bool rescale = false;
      // (rows of large scores come through here every time)
      bool stop = !(mx - m_used <= AFK_RESCALE) || large_scores(m_used);
      if (!(mx - m_used <= AFK_RESCALE) && mx > -INFINITY) {  // (also where there was none before)
        m_new = mx;
        rescale = j > 0 && m_used != -INFINITY;
      }
      if (!ADD) stop = __any_sync(0xffffffffu, stop);
      if (!ADD && stop && __any_sync(0xffffffffu, large_scores(m_new))) {
        if (pos) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) sv[c][i] = __float_as_uint(__uint_as_float(sv[c][i]) * sc);
        }
        mul = 1.0f;
      }
      const float alpha = rescale ? ex2_approx(m_used - m_new) : 1.0f;
      const float neg_m = m_new == -INFINITY ? 0.0f : -m_new;
      uint32_t pw[2][16];
      float lp[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e0 = ex2_approx(fmaf(__uint_as_float(sv[c][2 * i]), mul, neg_m));
          const float e1 = ex2_approx(fmaf(__uint_as_float(sv[c][2 * i + 1]), mul, neg_m));
          pw[c][i] = pack_f16x2(e0, e1);
          lp[i & 3] = add_f16((uint16_t)(pw[c][i] >> 16), add_f16((uint16_t)pw[c][i], lp[i & 3]));
        }
      l = l * alpha + ((lp[0] + lp[1]) + (lp[2] + lp[3]));
      m_used = m_new;
      // P_{j-1} V_{j-1} must be done before P is overwritten and O rescaled
      if (j > 0) {
        ok = mbar_wait(o_done, (uint32_t)(j - 1) & 1u, err, DEV_TIMEOUT_EPILOGUE);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
          for (int c = 0; c < 2 * NS; ++c) {
            uint32_t o[32];
            tmem_ld32(tmem + lane_base + AFK_O_COL + 32u * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tmem + lane_base + AFK_O_COL + 32u * c, o);
          }
          tmem_wait_st();
        }
      }
      // P row r: keys 8g .. 8g+7 are 16-byte chunk g of the row, swizzled by the row
#pragma unroll
      for (int g = 0; g < AFK_N / 8; ++g) {
        const int c = g >> 2, i = (g & 3) * 4;
        *reinterpret_cast<uint4*>(s_p + r * 128 + ((g ^ (r & 7)) << 4)) =
            make_uint4(pw[c][i], pw[c][i + 1], pw[c][i + 2], pw[c][i + 3]);
      }
      if (ADD) entries += (ADD32 ? 16 : 8) * p.mask_rows;
      fence_async_shared();  // the generic writes of P become visible to the tensor cores
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    // ---------------- epilogue
    if (ok && J > 0) {
      ok = mbar_wait(o_done, (uint32_t)(J - 1) & 1u, err, DEV_TIMEOUT_EPILOGUE);
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
      if (ADD && part && live) p.part_ref[slot_row] = ref;
      if (!(part && J == 0)) {  // the merge does not read the output of an item with l = 0
#pragma unroll
        for (int c = 0; c < 2 * NS; ++c) {
          uint32_t o[32];
          if (J > 0) {
            tmem_ld32(tmem + lane_base + AFK_O_COL + 32u * c, o);
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
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, AFK_TMEM_COLS);
  }
}

// ------------------------------------------------------------------ merging split key ranges
// One warp per query row, DV / 4 lanes with four columns each; slots in order.
// MASK: of additive masks, maxima are relative to mask references; they are taken to the slots' largest one first.
template <int MASK>
__global__ void __launch_bounds__(256) attention_combine_kernel(const float* __restrict__ part_o,
                                                                const float2* __restrict__ part_ml,
                                                                const float* __restrict__ part_ref, int slots,
                                                                int64_t rows, int TQ, int HQ, int DV,
                                                                uint16_t* __restrict__ o, int64_t o_sb, int64_t o_sh,
                                                                int64_t o_st, int* published /*or null*/) {
  pdl_wait();
  if (published && blockIdx.x == 0 && threadIdx.x == 0) publish_waited(published, 0);
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  // lane s: slot s0 + s; the first 32 slots' (m, l) are loaded once
  const float2 none = make_float2(-INFINITY, 0.0f);
  constexpr bool REF = MASK == MASK_ADD || MASK == MASK_ADD32;
  using Ref = MaskReference<MASK == MASK_ADD32>;
  float ref = -INFINITY;
  if (REF) {
    for (int s = lane; s < slots; s += 32)
      if (part_ml[(int64_t)s * rows + row].y != 0.0f) ref = fmaxf(ref, part_ref[(int64_t)s * rows + row]);
#pragma unroll
    for (int d = 16; d; d >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, d));
  }
  auto slot_ml = [&](int s) {
    float2 ml = part_ml[(int64_t)s * rows + row];
    if (REF && ml.y != 0.0f) ml.x += Ref::from(ref, part_ref[(int64_t)s * rows + row]);
    return ml;
  };
  float2 ml = lane < slots ? slot_ml(lane) : none;
  const float2 first = ml;
  float m = ml.y != 0.0f ? ml.x : -INFINITY;
  for (int s = lane + 32; s < slots; s += 32) {
    ml = slot_ml(s);
    if (ml.y != 0.0f) m = fmaxf(m, ml.x);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float l = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < slots; s0 += 32) {
    ml = s0 == 0 ? first : s0 + lane < slots ? slot_ml(s0 + lane) : none;
    const float wgt = ml.y != 0.0f ? ex2_approx(ml.x - m) : 0.0f;
    const uint32_t seen = __ballot_sync(0xffffffffu, ml.y != 0.0f);  // the others saw no key: their output is not written
    float part_l = ml.y != 0.0f ? wgt * ml.y : 0.0f;
#pragma unroll
    for (int d = 16; d; d >>= 1) part_l += __shfl_xor_sync(0xffffffffu, part_l, d);
    l += part_l;
    // four slots' loads at once
    for (int s = 0; s < 32 && s0 + s < slots; s += 4) {
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = (seen >> (s + i)) & 1u && lane * 4 < DV
                   ? *reinterpret_cast<const float4*>(part_o + ((int64_t)(s0 + s + i) * rows + row) * DV + lane * 4)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ws = __shfl_sync(0xffffffffu, wgt, s + i);
        acc.x += ws * v[i].x;
        acc.y += ws * v[i].y;
        acc.z += ws * v[i].z;
        acc.w += ws * v[i].w;
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (lane * 4 < DV) {
    const int h = (int)(row % HQ);
    const int64_t bt = row / HQ;
    uint16_t* y = o + (bt / TQ) * o_sb + h * o_sh + (bt % TQ) * o_st + lane * 4;
    *reinterpret_cast<uint2*>(y) = make_uint2(pack_f16x2(acc.x * inv, acc.y * inv), pack_f16x2(acc.z * inv, acc.w * inv));
  }
}

// ------------------------------------------------------------------ packing boolean masks
// One CTA per mask row of `len` bytes (key k: past keys first); words of segment
// 1 (the past) come first, then those of segment 0, each segment from a fresh
// word.  A thread makes 16 bits (2 bytes of a word) from 16 mask bytes: one load
// where they lie on 16 bytes and within the row, else one by one.
__global__ void __launch_bounds__(256) mask_pack_kernel(const uint8_t* __restrict__ mask, int len, int past, int keys,
                                                        int words1, int words, int vec,
                                                        unsigned long long* __restrict__ bits, int4* __restrict__ spans) {
  __shared__ int s_span[4];  // first and end of segment 0, first and end of segment 1
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x < 4) s_span[threadIdx.x] = threadIdx.x & 1 ? 0 : 0x7fffffff;
  __syncthreads();
  const int64_t row = blockIdx.x;
  const uint8_t* src = mask + row * len;
  uint16_t* dst = reinterpret_cast<uint16_t*>(bits + row * words);
  int lo[2] = {0x7fffffff, 0x7fffffff}, hi[2] = {0, 0};
#pragma unroll 2
  for (int i = threadIdx.x; i < words * 4; i += 256) {
    const int seg = i < words1 * 4 ? 1 : 0;
    const int k0 = (seg ? i : i - words1 * 4) * 16, at = (seg ? 0 : past) + k0;  // key of the segment, of the row
    const int n = min((seg ? past : keys) - k0, len - at);                       // keys of these 16 that exist
    uint32_t m = 0;
    if (vec && n >= 16) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + at));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      // bytes that are not 0 -> bits 0, 8, 16, 24 -> the top nibble in order
#pragma unroll
      for (int e = 0; e < 4; ++e) m |= (((__vcmpne4(w[e], 0u) & 0x01010101u) * 0x10204080u) >> 28) << (4 * e);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e < n && src[at + e] != 0) m |= 1u << e;
    }
    dst[i] = (uint16_t)m;
    if (m) {
      if (seg) lo[1] = min(lo[1], k0 + __ffs(m) - 1), hi[1] = max(hi[1], k0 + 32 - __clz(m));
      else lo[0] = min(lo[0], k0 + __ffs(m) - 1), hi[0] = max(hi[0], k0 + 32 - __clz(m));
    }
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int l = __reduce_min_sync(0xffffffffu, lo[s]), h = __reduce_max_sync(0xffffffffu, hi[s]);
    if ((threadIdx.x & 31) == 0 && h) {
      atomicMin(&s_span[2 * s], l);
      atomicMax(&s_span[2 * s + 1], h);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) spans[row] = make_int4(s_span[0], s_span[1], s_span[2], s_span[3]);
}

// ------------------------------------------------------------------ whole tiles of additive masks
// y[tile][16-byte piece][row]: the past's tiles, then the current keys', -inf past the mask's length and each part's
// keys.  A row's thread reads its row of a tile 16 bytes at a time: straight from the mask, 32 rows' pieces are 32
// sectors of 32 rows ([57, 16, 45 x 2952, 96] with a mask row per query took 810 us so); from here they are 512 bytes in
// line.  A CTA copies 32 rows of a tile through shared memory.
template <typename T>
__global__ void __launch_bounds__(256) mask_tiles_kernel(const T* __restrict__ mask, int len, int past, int keys, int words1,
                                                         int words, int64_t rows, uint4* __restrict__ y) {
  constexpr int E = 16 / sizeof(T), PIECES = 64 / E;
  __shared__ uint4 s_tile[32][PIECES + 1];  // (the padding spreads a piece's rows over the banks)
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row0 = (int64_t)blockIdx.x * 32;
  const int here = (int)min((int64_t)32, rows - row0);
  for (int w = blockIdx.y; w < words; w += gridDim.y) {
    const bool in_past = w < words1;
    const int k0 = (in_past ? w : w - words1) * 64, at = (in_past ? 0 : past) + k0;
    const int n = min((in_past ? past : keys) - k0, len - at);  // entries of the tile that exist
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int x = threadIdx.x + 256 * i, r = x >> 6, k = x & 63;
      T v = (T)-INFINITY;
      if (r < here && k < n) v = mask[(row0 + r) * len + at + k];
      reinterpret_cast<T*>(s_tile[r])[k] = v;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < 32 * PIECES; x += 256) {
      const int r = x & 31, piece = x >> 5;
      if (r < here) y[((int64_t)w * PIECES + piece) * rows + row0 + r] = s_tile[r][piece];
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ host side
static size_t flash_smem(int ns) {
  const int st = ns == 1 ? 4 : 2;
  return (size_t)ns * AFK_QSLAB + 2 * (size_t)st * ns * AFK_KSLAB + AFK_QSLAB + 256;
}

typedef void (*FlashKernel)(const TileParams);

static FlashKernel flash_kernel(int ns, int mask) {
  static const FlashKernel table[2][4] = {
      {attention_flash_kernel<1, MASK_NONE>, attention_flash_kernel<1, MASK_BITS>, attention_flash_kernel<1, MASK_ADD>,
       attention_flash_kernel<1, MASK_ADD32>},
      {attention_flash_kernel<2, MASK_NONE>, attention_flash_kernel<2, MASK_BITS>, attention_flash_kernel<2, MASK_ADD>,
       attention_flash_kernel<2, MASK_ADD32>}};
  return table[ns - 1][mask];
}

static int flash_slabs(const PlanOp& op) {
  return (op.ip[AF_D] > op.ip[AF_DV] ? op.ip[AF_D] : op.ip[AF_DV]) > 64 ? 2 : 1;
}

int prepare_attention_flash(const PlanOp& op, void* const*, OpState*, int, char* msg, size_t n) {
  const int64_t d = op.ip[AF_D], dv = op.ip[AF_DV];
  if (d < 8 || d > 128 || d % 8 || dv < 8 || dv > 128 || dv % 8)
    return fail(msg, n, 5, "Attention: head sizes %lld/%lld, needs multiples of 8 up to 128", (long long)d, (long long)dv);
  if (op.ip[AF_K_ST] > 0x7fffffff || op.ip[AF_V_ST] > 0x7fffffff)
    return fail(msg, n, 5, "Attention: key stride of more than 2^31 elements");
  // (plans from before the references were kept have no room for them)
  if (op.ip[AF_MASK_KIND] >= AF_MASK_F16 && op.ip[AF_SPLITS_K] + op.ip[AF_SPLITS_P] > 1 && op.ip[AF_PART_WIDTH] < dv + 3)
    return fail(msg, n, 5, "Attention: split keys under an additive mask, planned for another version of this library; plan it again");
  cudaError_t re = prepare_attention_rows();
  if (re == cudaSuccess) re = prepare_attention_wide();
  if (re != cudaSuccess) return fail(msg, n, 4, "cudaFuncSetAttribute: %s", cudaGetErrorString(re));
  for (int s = AF_Q_SB; s <= AF_O_ST; ++s)
    if (op.ip[s] % 8) return fail(msg, n, 5, "Attention: strides must be 16-byte multiples");
  for (int ns = 1; ns <= 2; ++ns)
    for (int m = 0; m < 4; ++m) {
      cudaError_t e =
          cudaFuncSetAttribute(flash_kernel(ns, m), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)flash_smem(ns));
      if (e != cudaSuccess) return fail(msg, n, 4, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    }
  return 0;
}

// 4-D map (d, t, h, b) over an fp16 tensor with element strides (1, st, sh, sb),
// boxes of 64 d x `tile_keys` tokens.
static int make_tmap_kv(CUtensorMap* map, const void* base, int64_t d, int64_t t, int64_t heads, int64_t batch,
                        int64_t st, int64_t sh, int64_t sb, int tile_keys) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return 4;
  cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)t, (cuuint64_t)heads, (cuuint64_t)batch};
  cuuint64_t strides[3] = {(cuuint64_t)st * 2, (cuuint64_t)sh * 2, (cuuint64_t)sb * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)tile_keys, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 4;
}

// Query rows as 5-D tiles of 64 d x 128 rows (token, head of the group), for the
// class whose rows run over one sequence, or over all of them: possible where a
// group divides 128 and tokens (and sequences) lie evenly.  Returns whether.
static int make_tmap_q(CUtensorMap* map, const RowsParams& r, int64_t tokens, int64_t st, int64_t sequences, int64_t sb) {
  EncodeTiledFn enc = encode_tiled_fn();
  const int64_t group = r.group.d;
  if (!enc || 128 % group) return 0;
  cuuint64_t dims[5] = {(cuuint64_t)r.D, (cuuint64_t)group, (cuuint64_t)tokens, (cuuint64_t)r.HKV, (cuuint64_t)sequences};
  cuuint64_t strides[4] = {(cuuint64_t)r.q_sh * 2, (cuuint64_t)st * 2, (cuuint64_t)(group * r.q_sh) * 2, (cuuint64_t)sb * 2};
  cuuint32_t box[5] = {64, (cuuint32_t)group, (cuuint32_t)(128 / group), 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<uint16_t*>(r.q), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Fills what the tile pass needs beside the rows' parameters.
static int tile_params(TileParams& p, const RowsParams& r, const ItemClass* cls, int first1, int items,
                       bool wide) {
  const int tile_keys = wide ? 128 : AFK_N;
  p.cls[0] = cls[0], p.cls[1] = cls[1], p.first1 = first1, p.items = items;
  p.q = r.q, p.o = r.o, p.part_o = r.part_o, p.part_ml = r.part_ml, p.part_ref = r.part_ref;
  p.q_sb = r.q_sb, p.q_sh = r.q_sh, p.q_st = r.q_st, p.o_sb = r.o_sb, p.o_sh = r.o_sh, p.o_st = r.o_st;
  p.B = r.B, p.HQ = r.HQ, p.HKV = r.HKV, p.group = r.group, p.TQ = r.TQ, p.D = r.D, p.DV = r.DV;
  p.causal = r.causal, p.tk = r.tk, p.tp = r.tp, p.past_shared = r.past_shared;
  p.counts = r.counts;
  p.mask_sb = r.mask_sb, p.mask_sh = r.mask_sh, p.mask_st = r.mask_st;
  p.mask_len = r.mask_len;
  p.scale_log2 = r.scale_log2;
  p.err = r.err;
  const int64_t tq = r.TQ.d;
  if (wide) {  // (the 128-row pass copies its query rows)
    p.q_boxes[0] = make_tmap_q(&p.map_q[0], r, tq, r.q_st, r.B, r.q_sb);
    if (tq == 1 || r.q_sb == tq * r.q_st)
      p.q_boxes[1] = make_tmap_q(&p.map_q[1], r, r.B * tq, tq == 1 ? r.q_sb : r.q_st, 1, (int64_t)r.B * r.q_sb);
  }
  int rc = make_tmap_kv(&p.map_k[0], r.k, p.D, p.tk, p.HKV, p.B, r.k_st, r.k_sh, r.k_sb, tile_keys);
  if (!rc) rc = make_tmap_kv(&p.map_v[0], r.v, p.DV, p.tk, p.HKV, p.B, r.v_st, r.v_sh, r.v_sb, tile_keys);
  if (p.tp > 0) {
    const int copies = p.past_shared ? 1 : p.B;
    if (!rc)
      rc = make_tmap_kv(&p.map_k[1], r.past_k, p.D, p.tp, p.HKV, copies, p.D, (int64_t)p.tp * p.D,
                        (int64_t)p.HKV * p.tp * p.D, tile_keys);
    if (!rc)
      rc = make_tmap_kv(&p.map_v[1], r.past_v, p.DV, p.tp, p.HKV, copies, p.DV, (int64_t)p.tp * p.DV,
                        (int64_t)p.HKV * p.tp * p.DV, tile_keys);
  }
  return rc;
}

int launch_attention_flash(const PlanOp& op, void* const* ptrs, const OpState*, const LaunchCtx& ctx, int* launches) {
  RowsParams r{};
  const int64_t* s = &op.ip[AF_Q_SB];
  auto ptr = [&](int i) -> void* { return op.t[i] >= 0 ? ptrs[op.t[i]] : nullptr; };
  r.B = (int)eff_batch(ctx, op, op.ip[AF_B]);
  r.HQ = (int)op.ip[AF_HQ];
  r.HKV = (int)op.ip[AF_HKV];
  const int64_t group = r.HQ / r.HKV, tq = op.ip[AF_TQ];
  r.group = SmallDiv::of((uint32_t)group);
  r.TQ = SmallDiv::of((uint32_t)tq);
  r.D = (int)op.ip[AF_D];
  r.DV = (int)op.ip[AF_DV];
  r.causal = (int)op.ip[AF_CAUSAL];
  r.tk = (int)op.ip[AF_TK];
  r.tp = (int)op.ip[AF_TP];
  r.past_shared = (int)op.ip[AF_PAST_SHARED];
  r.scale_log2 = (float)(op.fp[AFF_SCALE] * 1.4426950408889634);
  r.q = (const uint16_t*)ptr(0), r.k = (const uint16_t*)ptr(1), r.v = (const uint16_t*)ptr(2);
  r.past_k = (const uint16_t*)ptr(5), r.past_v = (const uint16_t*)ptr(6);
  r.o = (uint16_t*)ptr(3);
  r.q_sb = s[0], r.q_sh = s[1], r.q_st = s[2], r.k_sb = s[3], r.k_sh = s[4], r.k_st = s[5];
  r.v_sb = s[6], r.v_sh = s[7], r.v_st = s[8], r.o_sb = s[9], r.o_sh = s[10], r.o_st = s[11];
  r.counts = (const long long*)ptr(7);
  r.err = ctx.d_error;
  if (r.B <= 0 || tq <= 0) return 0;
  for (int i : {0, 1, 2, 3, 5, 6})
    if ((uintptr_t)ptr(i) & 15u) return REFUSED_ALIGNMENT;
  if ((uintptr_t)r.counts & 7u) return REFUSED_ALIGNMENT;
  const int kind = (int)op.ip[AF_MASK_KIND];
  const int variant = kind == AF_MASK_NONE ? MASK_NONE : kind == AF_MASK_BOOL ? MASK_BITS : kind == AF_MASK_F16 ? MASK_ADD : MASK_ADD32;
  const bool additive = variant == MASK_ADD || variant == MASK_ADD32;
  r.mask_sb = op.ip[AF_MASK_SB], r.mask_sh = op.ip[AF_MASK_SH], r.mask_st = op.ip[AF_MASK_ST];
  r.mask_len = (int)op.ip[AF_MASK_LEN];
  r.mask_bool = variant == MASK_BITS ? (const uint8_t*)ptr(4) : nullptr;
  r.mask_add = additive ? ptr(4) : nullptr;
  if (additive && ((uintptr_t)r.mask_add & (variant == MASK_ADD32 ? 3u : 1u))) return REFUSED_ALIGNMENT;

  // ---------------- work items of the two classes
  const int64_t rows = (int64_t)r.B * tq * r.HQ;
  const int pass_own = (int)op.ip[AF_PASS_OWN], pass_past = (int)op.ip[AF_PASS_PAST];
  const bool apart = r.tp > 0 && pass_past != AF_PASS_NONE;  // a shared past in items of its own
  auto tiles_of = [](int64_t n, int pass) {
    const int m = pass == AF_PASS_ROWS8 ? 8 : pass == AF_PASS_ROWS16 ? 16 : pass == AF_PASS_WIDE ? 2 * AFK_M : AFK_M;
    return (int)((n + m - 1) / m);
  };
  ItemClass cls[2] = {};
  cls[0].splits = (int)op.ip[AF_SPLITS_K];
  cls[0].tiles = tiles_of(tq * group, pass_own);
  cls[0].past = r.tp > 0 && !apart;
  int64_t items[2] = {(int64_t)r.B * r.HKV * cls[0].tiles * cls[0].splits, 0};
  int slots = cls[0].splits;
  if (apart) {
    cls[1].splits = (int)op.ip[AF_SPLITS_P];
    cls[1].tiles = tiles_of(r.B * tq * group, pass_past);
    cls[1].part0 = slots;
    cls[1].past = 1;
    items[1] = (int64_t)r.HKV * cls[1].tiles * cls[1].splits;
    slots += cls[1].splits;
  }
  // (SmallDiv: rows divided by the group, and, against a shared past, by the tokens)
  if (items[0] + items[1] > 0x7fffffff || (apart ? r.B : 1) * tq * group * group > 0xffffffffll ||
      (apart && r.B * tq * tq > 0xffffffffll))
    return REFUSED_SIZE;
  if (slots > 1) {
    // (m, l) pairs behind the outputs, mask references behind them, all sized for the compiled batch
    r.part_o = (float*)ptr(8);
    r.part_ml = (float2*)(r.part_o + (int64_t)slots * rows * r.DV);
    if (additive) r.part_ref = (float*)(r.part_ml + (int64_t)slots * rows);
  }

  // ---------------- passes: one kernel for both classes, or the past's first and the own keys' beside it
  auto is_rows = [](int pass) { return pass == AF_PASS_ROWS8 || pass == AF_PASS_ROWS16; };
  const bool together = !apart || pass_own == pass_past;
  cudaError_t e = cudaSuccess;
  for (int step = together ? 1 : 0; step < 2 && e == cudaSuccess; ++step) {
    const int pass = together ? pass_own : (step == 0 ? pass_past : pass_own);
    const int64_t n1 = together ? items[1] : (step == 0 ? items[1] : 0);
    const int64_t n0 = together || step == 1 ? items[0] : 0;
    if (is_rows(pass)) {
      // a work item's boolean mask has to fit the kernel's bits
      auto most_keys = [](int64_t tp, int64_t tk, int splits) {
        const int64_t blocks = (tp + 15) / 16 + (tk + 15) / 16;
        return (blocks + splits - 1) / splits * 16;
      };
      if (variant == MASK_BITS &&
          ((n0 && most_keys(cls[0].past ? r.tp : 0, r.tk, cls[0].splits) > AF_ROWS_MASK_KEYS) ||
           (n1 && most_keys(r.tp, 0, cls[1].splits) > AF_ROWS_MASK_KEYS)))
        return 5;
      r.cls[0] = cls[0], r.cls[1] = cls[1], r.first1 = (int)n1;
      for (int c = 0; c < 2; ++c) {
        // (an absent class divides by 1)
        r.by[c][0] = SmallDiv::of(cls[c].splits ? cls[c].splits : 1), r.by[c][1] = SmallDiv::of(cls[c].tiles ? cls[c].tiles : 1);
        const int64_t largest = std::max<int64_t>(std::max(cls[c].splits, cls[c].tiles), r.HKV);
        if (std::max<int64_t>(n0 + n1, most_keys(r.tp, r.tk, 1)) * largest > 0xffffffffll) return REFUSED_SIZE;
      }
      r.by_hkv = SmallDiv::of(r.HKV);
      r.late_wait = !together && step == 1;
      e = launch_attention_rows(r, pass == AF_PASS_ROWS8 ? 1 : 2, variant, (int)op.ip[AF_WARPS], (unsigned)(n0 + n1), ctx.stream);
    } else {
      TileParams p{};
      const int tile_keys = pass == AF_PASS_WIDE ? 128 : AFK_N;
      if (pass == AF_PASS_WIDE && additive) return 5;  // (never planned)
      int rc = tile_params(p, r, cls, (int)n1, (int)(n0 + n1), pass == AF_PASS_WIDE);
      p.publish = !together;
      p.drop_keys = (ctx.fault & FAULT_DROP_KEY_TILES) != 0;
      if (rc) return rc;
      const int64_t mrows = p.mask_sb ? p.mask_sb * p.B : op.ip[AF_MASK_ROWS];
      p.words_past = (p.tp + tile_keys - 1) / tile_keys * (tile_keys / 64);
      p.words = p.words_past + (p.tk + tile_keys - 1) / tile_keys * (tile_keys / 64);
      if (variant == MASK_BITS) {
        p.spans = (const int4*)ptr(9);
        p.bits = (const unsigned long long*)(p.spans + mrows);
        e = launch_pdl(mask_pack_kernel, dim3((unsigned)mrows), dim3(256), 0, ctx.stream, r.mask_bool, p.mask_len, p.tp,
                       p.tk, p.words_past, p.words,
                       (int)(p.mask_len % 16 == 0 && p.tp % 16 == 0 && ((uintptr_t)r.mask_bool & 15u) == 0),
                       (unsigned long long*)p.bits, (int4*)p.spans);
        ++*launches;
      } else if (additive) {
        p.add = (const uint4*)ptr(9);
        p.mask_rows = mrows;
        const dim3 grid((unsigned)((mrows + 31) / 32), (unsigned)std::min(p.words, 65535));
        if (variant == MASK_ADD32)
          e = launch_pdl(mask_tiles_kernel<float>, grid, dim3(256), 0, ctx.stream, (const float*)r.mask_add, p.mask_len, p.tp,
                         p.tk, p.words_past, p.words, mrows, (uint4*)ptr(9));
        else
          e = launch_pdl(mask_tiles_kernel<__half>, grid, dim3(256), 0, ctx.stream, (const __half*)r.mask_add, p.mask_len,
                         p.tp, p.tk, p.words_past, p.words, mrows, (uint4*)ptr(9));
        ++*launches;
      }
      if (e != cudaSuccess) return 4;
      const int ns = flash_slabs(op);
      e = pass == AF_PASS_WIDE ? launch_attention_wide(p, ns, variant, ctx.num_sms, ctx.stream)
                               : launch_pdl(flash_kernel(ns, variant), dim3((unsigned)(n0 + n1)), dim3(AFK_THREADS),
                                            flash_smem(ns), ctx.stream, p);
    }
    ++*launches;
  }
  if (e == cudaSuccess && slots > 1) {
    e = launch_pdl(variant == MASK_ADD     ? attention_combine_kernel<MASK_ADD>
                   : variant == MASK_ADD32 ? attention_combine_kernel<MASK_ADD32>
                                           : attention_combine_kernel<MASK_NONE>,
                   dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, ctx.stream, (const float*)r.part_o,
                   (const float2*)r.part_ml, (const float*)r.part_ref, slots, rows, (int)tq, r.HQ, r.DV, r.o, r.o_sb, r.o_sh,
                   r.o_st, together ? nullptr : r.err);
    ++*launches;
  }
  return e == cudaSuccess ? 0 : 4;
}

}  // namespace emx
