// Attention for few query rows per key/value head: decoding steps, drafted
// tokens, single tokens over encoder states (see attention_flash.cu for the
// operator and its mathematics; this kernel is one of its passes).
//
// What bounds it is the read of K and V: up to 16 query rows share every key,
// 4 flops a byte and row at most, so nothing is staged -- a warp loads the
// K and V of its key block from global memory straight into the operand
// registers of mma.sync.m16n8k16, 16 bytes a thread and load, and hides the
// latency behind the other warps of the SM.  (The tcgen05 form needs a 128-row
// tile, tensor maps, barriers and TMEM set up per work item; at these sizes a
// work item is over before that has paid off.)  Both products run transposed,
//   S^T [16 keys x 8 rows] = K Q^T,   O^T [16 d x 8 rows] += V^T P^T,
// so the row tiles are 8 wide and the big operands are the A side:
//   * the contraction over d may take d in any order, so thread t of a quad
//     takes the 16-byte pieces t, t + 4, ... of a key's row, which serve two
//     k-steps each, and the same pieces of the query rows;
//   * the rows of O^T (d) may be in any order as well: thread group g loads
//     16-byte piece g of four keys' V rows and pairs up the keys' halves;
//   * P^T reaches its operand layout through two 8 x 8 register transposes.
//
// One work item is (sequence, key/value head, range of 16-key blocks); its 2 to
// 8 warps take the blocks in turn and merge through shared memory.  The past and
// the current keys of a sequence are one list of blocks, or, when the past is
// shared by the batch, two kinds of items: rows of several sequences against
// the past, each sequence's rows against its own keys.  Blocks whose keys a
// boolean mask hides from every row are not loaded.
#include <cuda_fp16.h>

#include "attention_flash.cuh"
#include "host_util.h"
#include "kernels.h"
#include "tc100.cuh"
#include "tmem32.cuh"

namespace emx {

constexpr int AR_WARPS = 8;  // most warps of a work item

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// NS: 64-wide slabs of the head size; NT: tiles of 8 query rows; MASK: AF_MASK_* folded to none / boolean / additive
template <int NS, int NT, int MASK>
__global__ void __launch_bounds__(32 * AR_WARPS, NS == 2 && NT == 2 ? 1 : 2)
    attention_rows_kernel(const __grid_constant__ RowsParams p) {
  constexpr int KM = NS == 2 ? 1 : 2;  // 16-key groups per block: 8 KB of K and V per warp at either head size
  constexpr int KB = 16 * KM;
  constexpr int NC = 2 * NS;           // 16-byte pieces of a key row per thread
  constexpr int OW = 64 * NS + 4;      // padded row of the merge buffer
  extern __shared__ __align__(16) float s_all[];  // rows_smem() bytes
  const int warps = blockDim.x >> 5;
  float(*s_o)[8 * NT][OW] = reinterpret_cast<float(*)[8 * NT][OW]>(s_all);
  float(*s_m)[8 * NT] = reinterpret_cast<float(*)[8 * NT]>(s_all + warps * 8 * NT * OW);
  float(*s_l)[8 * NT] = s_m + warps;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (!p.late_wait) pdl_wait();
  pdl_launch_dependents();

  // ---------------- work item
  const bool past_item = (int)blockIdx.x < p.first1;
  const ItemClass& cl = p.cls[past_item ? 1 : 0];
  int id = (int)blockIdx.x - (past_item ? 0 : p.first1);
  const int split = id % cl.splits;
  id /= cl.splits;
  const int tile = id % cl.tiles;
  id /= cl.tiles;
  const int kvh = id % p.HKV, b = id / p.HKV;
  const int rows_all = (int)(p.TQ.d * p.group.d) * (past_item ? p.B : 1);
  const int row0 = tile * 8 * NT, rows = min(8 * NT, rows_all - row0);
  const bool two = NT == 2 && rows > 8;
  int keys = past_item ? 0 : p.tk;  // current keys that some row sees
  if (!past_item) {
    if (p.causal) keys = min(keys, p.group.div(row0 + rows - 1) + 1);
    if (p.counts) {
      const long long n = p.counts[b];
      if ((n < 0 || n > p.tk) && threadIdx.x == 0) record_error(p.err, DEV_BAD_INDEX);
      keys = min(keys, (int)max(0ll, min(n, (long long)p.tk)));
    }
  }
  const int past = cl.past ? p.tp : 0;
  const int pblocks = (past + KB - 1) / KB, blocks = pblocks + (keys + KB - 1) / KB;
  const int blk0 = (int)((long long)blocks * split / cl.splits), blk1 = (int)((long long)blocks * (split + 1) / cl.splits);

  const uint16_t* kc = p.k + (int64_t)b * p.k_sb + (int64_t)kvh * p.k_sh;
  const uint16_t* vc = p.v + (int64_t)b * p.v_sb + (int64_t)kvh * p.v_sh;
  const int64_t ph = ((int64_t)(p.past_shared ? 0 : b) * p.HKV + kvh) * p.tp;
  const uint16_t* kp = p.past_k + ph * p.D;
  const uint16_t* vp = p.past_v + ph * p.DV;
  // this thread's first piece: K of key g, V of key 2t
  kc += (int64_t)g * p.k_st + 8 * t, kp += g * p.D + 8 * t;
  vc += (int64_t)(2 * t) * p.v_st + 8 * g, vp += 2 * t * p.DV + 8 * g;

  // ---------------- the rows whose scores this thread holds (2t, 2t + 1 of each tile): mask row and key limit
  int64_t mrow[NT][2];
  int lim[NT][2];
  int lim_all = 0x7fffffff;  // keys below it are within every row's limit (rows past the last have none)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * n + 2 * t + e;
      const RowId w = row_of(row0 + min(r, rows - 1), p.group, p.TQ, kvh, b, past_item);
      mrow[n][e] = MASK == MASK_NONE ? 0 : (w.b * p.mask_sb + w.h * p.mask_sh + w.t * p.mask_st) * (int64_t)p.mask_len;
      lim[n][e] = r >= rows || past_item ? 0x7fffffff : p.tp + (p.causal ? min(keys, w.t + 1) : keys);
      lim_all = min(lim_all, lim[n][e]);
    }
  if (!past_item && p.causal) {
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) lim_all = min(lim_all, __shfl_xor_sync(0xffffffffu, lim_all, d));
  }
  // ---------------- query rows as the B operand: row g of each tile, this thread's pieces
  uint4 q[NT][NC];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + g;
    const RowId w = row_of(row0 + min(r, rows - 1), p.group, p.TQ, kvh, b, past_item);
    const uint16_t* src = p.q + (int64_t)w.b * p.q_sb + (int64_t)w.h * p.q_sh + (int64_t)w.t * p.q_st;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = 8 * (t + 4 * c);
      q[n][c] = r < rows && d < p.D ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0u, 0u, 0u, 0u);
    }
  }

  uint4 k[KM][2][NC], v[KM][4][NS];
  // pieces past the head size stay zero; a whole block's loads have no other condition
  bool k_in[NC], v_in[NS];
#pragma unroll
  for (int c = 0; c < NC; ++c) k_in[c] = 8 * (t + 4 * c) < p.D;
#pragma unroll
  for (int s = 0; s < NS; ++s) v_in[s] = 64 * s + 8 * g < p.DV;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  auto load_k = [&](int blk) {
    const bool is_past = blk < pblocks;
    const int k0 = (is_past ? blk : blk - pblocks) * KB, n = (is_past ? past : keys) - k0;
    const int ks = is_past ? p.D : (int)p.k_st;
    const uint16_t* src = (is_past ? kp : kc) + (int64_t)k0 * ks;
    const int64_t step = (int64_t)ks * 8;
    const bool whole = n >= KB;
#pragma unroll
    for (int m = 0; m < KM; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = whole || 16 * m + 8 * h + g < n;
#pragma unroll
        for (int c = 0; c < NC; ++c) k[m][h][c] = in && k_in[c] ? ld_stream(src + (2 * m + h) * step + 32 * c) : zero;
      }
  };
  auto load_v = [&](int blk) {
    const bool is_past = blk < pblocks;
    const int k0 = (is_past ? blk : blk - pblocks) * KB, n = (is_past ? past : keys) - k0;
    const int vs = is_past ? p.DV : (int)p.v_st;
    const uint16_t* src = (is_past ? vp : vc) + (int64_t)k0 * vs;
    const int64_t step = (int64_t)vs * 8;
    const bool whole = n >= KB;
#pragma unroll
    for (int m = 0; m < KM; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = whole || 16 * m + 8 * (e >> 1) + 2 * t + (e & 1) < n;
#pragma unroll
        for (int s = 0; s < NS; ++s)
          v[m][e][s] = in && v_in[s] ? ld_stream(src + (2 * m + (e >> 1)) * step + (e & 1) * vs + 64 * s) : zero;
      }
  };
  // mask entries of a block at this thread's scores: [m][half][n][e]; returns whether any lane sees any key
  float mk[MASK == MASK_ADD ? KM * 4 * NT : 1];
  auto load_mask = [&](int blk) -> uint32_t {
    const bool is_past = blk < pblocks;
    const int k0 = (is_past ? blk : blk - pblocks) * KB, pos0 = (is_past ? 0 : p.tp) + k0;
    const int seg_end = is_past ? past : p.tp + keys;
    if (MASK == MASK_NONE && pos0 + KB <= min(lim_all, seg_end)) return ~0u;
    uint32_t see = 0;
#pragma unroll
    for (int m = 0; m < KM; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int pos = pos0 + 16 * m + 8 * h + g;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i = ((m * 2 + h) * NT + n) * 2 + e;
            bool ok = pos < min(lim[n][e], seg_end);
            if (MASK != MASK_NONE) ok = ok && pos < p.mask_len;
            if (MASK == MASK_BITS) ok = ok && __ldg(p.mask_bool + mrow[n][e] + pos) != 0;
            if (MASK == MASK_ADD) {
              mk[i] = ok ? additive_entry(p.mask_add, p.add_f32, mrow[n][e] + pos) : 0.0f;
              ok = ok && mk[i] != -INFINITY;
              if (!ok) mk[i] = 0.0f;
            }
            see |= (ok ? 1u : 0u) << i;
          }
      }
    return see;
  };

  float o[NT][NS][4][4];  // O^T: [row tile][slab][d pair][(d, row), (d, row + 1), (d + 1, row), (d + 1, row + 1)]
  float m_ref[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) m_ref[n][e] = -INFINITY, l[n][e] = 0.0f;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][s][j][e] = 0.0f;
  }
  const float sc = p.scale_log2;

  int blk = blk0 + warp;
  uint32_t see = 0;
  bool need = false;
  const bool any_block = blk < blk1;
  if (any_block) {  // the first block is loaded beside its mask
    load_k(blk);
    load_v(blk);
    see = load_mask(blk);
    need = MASK == MASK_NONE || __any_sync(0xffffffffu, see != 0);
  }
  for (; blk < blk1; blk += warps) {
    const int next = blk + warps;
    uint32_t see_next = 0;
    bool need_next = false;
    // ---------------- S^T
    float s[KM][NT][4];
    if (need) {
#pragma unroll
      for (int m = 0; m < KM; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][n][e] = 0.0f;
          if (n == 1 && !two) continue;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            mma_16816(s[m][n], k[m][0][c].x, k[m][1][c].x, k[m][0][c].y, k[m][1][c].y, q[n][c].x, q[n][c].y);
            mma_16816(s[m][n], k[m][0][c].z, k[m][1][c].z, k[m][0][c].w, k[m][1][c].w, q[n][c].z, q[n][c].w);
          }
        }
      // scores in log2 units; entries the row does not see are -inf
#pragma unroll
      for (int m = 0; m < KM; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][n][e] *= sc;
      if (MASK != MASK_NONE || see != ~0u) {
#pragma unroll
        for (int m = 0; m < KM; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = ((m * 2 + (e >> 1)) * NT + n) * 2 + (e & 1);
              if (!((see >> i) & 1u)) s[m][n][e] = -INFINITY;
            }
      }
      bool grow = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (n == 1 && !two) continue;
          float x = -INFINITY;
#pragma unroll
          for (int m = 0; m < KM; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float y = s[m][n][2 * h + e];
              if (MASK == MASK_ADD) y = fmaf(mk[((m * 2 + h) * NT + n) * 2 + e], AFK_LOG2E, y);
              x = fmaxf(x, y);
            }
          top[n][e] = x;
          grow = grow || x > m_ref[n][e] + AFK_RESCALE || (m_ref[n][e] == -INFINITY && x > -INFINITY);
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (n == 1 && !two) continue;
            float x = top[n][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            const float old = m_ref[n][e];
            if (x > old + AFK_RESCALE || old == -INFINITY) {
              m_ref[n][e] = x;
              const float alpha = old == -INFINITY ? 0.0f : ex2_approx(old - x);
              l[n][e] *= alpha;
#pragma unroll
              for (int sl = 0; sl < NS; ++sl)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  o[n][sl][j][e] *= alpha;
                  o[n][sl][j][e + 2] *= alpha;
                }
            }
          }
      }
      // weights
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (n == 1 && !two) continue;
          const float neg = m_ref[n][e] == -INFINITY ? 0.0f : -m_ref[n][e];
#pragma unroll
          for (int m = 0; m < KM; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float off = neg;
              if (MASK == MASK_ADD) off = fmaf(mk[((m * 2 + h) * NT + n) * 2 + e], AFK_LOG2E, neg);
              s[m][n][2 * h + e] = ex2_approx(s[m][n][2 * h + e] + off);
              l[n][e] += s[m][n][2 * h + e];
            }
        }
    }
    // ---------------- the next block's mask and K, then O^T += V^T P^T
    if (next < blk1) {
      see_next = load_mask(next);
      need_next = MASK == MASK_NONE || __any_sync(0xffffffffu, see_next != 0);
      if (need_next) load_k(next);
    }
    if (need) {
#pragma unroll
      for (int m = 0; m < KM; ++m) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (n == 0 || two) pb[n][h] = transpose_8x8(pack_f16x2(s[m][n][2 * h], s[m][n][2 * h + 1]));
#pragma unroll
        for (int sl = 0; sl < NS; ++sl)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w0 = word_of(v[m][0][sl], j), w1 = word_of(v[m][1][sl], j);
            const uint32_t w2 = word_of(v[m][2][sl], j), w3 = word_of(v[m][3][sl], j);
            const uint32_t a0 = __byte_perm(w0, w1, 0x5410), a1 = __byte_perm(w0, w1, 0x7632);
            const uint32_t a2 = __byte_perm(w2, w3, 0x5410), a3 = __byte_perm(w2, w3, 0x7632);
            mma_16816(o[0][sl][j], a0, a1, a2, a3, pb[0][0], pb[0][1]);
            if (NT == 2 && two) mma_16816(o[NT - 1][sl][j], a0, a1, a2, a3, pb[NT - 1][0], pb[NT - 1][1]);
          }
      }
    }
    if (need_next) load_v(next);
    see = see_next;
    need = need_next;
  }

  // ---------------- merge the warps, write the rows
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (n == 1 && !two) continue;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
      const int r = 8 * n + 2 * t + e;
      if (g == 0) {
        s_m[warp][r] = m_ref[n][e];
        s_l[warp][r] = l[n][e];
      }
      if (!any_block) continue;  // l = 0: nothing reads this warp's output
#pragma unroll
      for (int sl = 0; sl < NS; ++sl)
#pragma unroll
        for (int j = 0; j < 4; j += 2)
          *reinterpret_cast<float4*>(&s_o[warp][r][64 * sl + 8 * g + 2 * j]) =
              make_float4(o[n][sl][j][e], o[n][sl][j][e + 2], o[n][sl][j + 1][e], o[n][sl][j + 1][e + 2]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * 16 * NS; i += blockDim.x) {
    const int r = i / (16 * NS), d = (i % (16 * NS)) * 4;
    float m = -INFINITY, sum = 0.0f;
    for (int w = 0; w < warps; ++w)
      if (s_l[w][r] != 0.0f) m = fmaxf(m, s_m[w][r]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < warps; ++w) {
      if (s_l[w][r] == 0.0f) continue;
      const float f = ex2_approx(s_m[w][r] - m);
      const float4 x = *reinterpret_cast<const float4*>(&s_o[w][r][d]);
      sum += f * s_l[w][r];
      acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
    }
    if (d >= p.DV) continue;
    const RowId w = row_of(row0 + r, p.group, p.TQ, kvh, b, past_item);
    if (p.part_o) {
      const int64_t at = (int64_t)(cl.part0 + split) * ((int64_t)p.B * (int)p.TQ.d * p.HQ) + ((int64_t)w.b * (int)p.TQ.d + w.t) * p.HQ + w.h;
      if (d == 0) p.part_ml[at] = make_float2(m, sum);
      *reinterpret_cast<float4*>(p.part_o + at * p.DV + d) = acc;
    } else {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      *reinterpret_cast<uint2*>(p.o + (int64_t)w.b * p.o_sb + (int64_t)w.h * p.o_sh + (int64_t)w.t * p.o_st + d) =
          make_uint2(pack_f16x2(acc.x * inv, acc.y * inv), pack_f16x2(acc.z * inv, acc.w * inv));
    }
  }
  // This grid may run beside the pass before it, which has passed its own wait (so all that came before both is
  // complete) and whose results it neither reads nor writes.  One CTA ends after that pass, so this grid does,
  // and the merge kernel's wait for this grid covers both.
  if (p.late_wait && blockIdx.x == gridDim.x - 1) pdl_wait();
}

// ------------------------------------------------------------------ host side
static size_t rows_smem(int ns, int nt, int warps) {
  return (size_t)warps * 8 * nt * (64 * ns + 4 + 2) * sizeof(float);
}

template <int NS, int NT>
static cudaError_t launch_variant(const RowsParams& p, int mask, int warps, unsigned items, cudaStream_t stream) {
  auto kernel = mask == MASK_NONE ? attention_rows_kernel<NS, NT, MASK_NONE>
                : mask == MASK_BITS ? attention_rows_kernel<NS, NT, MASK_BITS>
                                    : attention_rows_kernel<NS, NT, MASK_ADD>;
  return launch_pdl(kernel, dim3(items), dim3(32 * warps), rows_smem(NS, NT, warps), stream, p);
}

cudaError_t prepare_attention_rows() {
  // only the widest form needs more than a launch's default shared memory
  cudaError_t e = cudaSuccess;
  for (auto kernel : {attention_rows_kernel<2, 2, MASK_NONE>, attention_rows_kernel<2, 2, MASK_BITS>,
                      attention_rows_kernel<2, 2, MASK_ADD>})
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rows_smem(2, 2, AR_WARPS));
  return e;
}

cudaError_t launch_attention_rows(const RowsParams& p, int row_tiles, int mask, int warps, unsigned items,
                                  cudaStream_t stream) {
  if (warps < 1 || warps > AR_WARPS) return cudaErrorInvalidValue;
  const bool wide = p.D > 64 || p.DV > 64;
  if (row_tiles == 1)
    return wide ? launch_variant<2, 1>(p, mask, warps, items, stream) : launch_variant<1, 1>(p, mask, warps, items, stream);
  return wide ? launch_variant<2, 2>(p, mask, warps, items, stream) : launch_variant<1, 2>(p, mask, warps, items, stream);
}

}  // namespace emx
