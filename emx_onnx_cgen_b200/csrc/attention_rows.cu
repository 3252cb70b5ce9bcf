// Attention for few query rows per key/value head: decoding steps, drafted
// tokens, single tokens over encoder states (see attention_flash.cu for the
// operator and its mathematics; this kernel is one of its passes).
//
// What bounds it is the read of K and V: up to 16 query rows share every key,
// 4 flops a byte and row at most.  Each warp copies its 16-key blocks of K and V
// into a ring of its own in shared memory (cp.async, 24 KB a warp), two to five
// blocks ahead of the one it works on: with the blocks in registers, one ahead,
// a block cost a memory latency (1.2 us).  At D <= 64 and up to 8 rows a step
// takes two blocks: the chain of a step (scores, maximum, exponentials,
// transposes, output) is 1500 clocks long and two warps a scheduler do not cover
// it (16 sequences x 16 heads, up to 1500 keys, D = 64: 16.4 to 17.8 us over
// several boards, 4.2 to 4.5 TB/s of valid keys; 4 us more with one block).  128
// sequences x 8 heads of 4 rows, 150 keys on average, D = 128: 29 us alone, 3.5
// TB/s, a third of the stalls at the CTA's barriers.  The products are
// mma.sync.m16n8k16: a tcgen05 form needs a 128-row tile, tensor maps, barriers
// and TMEM set up per work item, and at these sizes a work item is over before
// that has paid off.
// Both products run transposed,
//   S^T [16 keys x 8 rows] = K Q^T,   O^T [16 d x 8 rows] += V^T P^T,
// so the row tiles are 8 wide and the big operands are the A side:
//   * the contraction over d may take d in any order, so thread t of a quad
//     takes the 16-byte pieces t, t + 4, ... of a key's row, which serve two
//     k-steps each, and the same pieces of the query rows;
//   * the rows of O^T (d) may be in any order as well: thread group g reads
//     16-byte piece g of four keys' V rows and pairs up the keys' halves;
//   * P^T reaches its operand layout through two 8 x 8 register transposes.
// Piece c of key row r lies at place c ^ (r & 6) ^ 4 (r & 1) of the row, which
// keeps both operands' reads free of bank conflicts.
//
// One work item is (sequence, key/value head, range of 16-key blocks); its
// warps take the blocks in turn and merge through shared memory.  The past and
// the current keys of a sequence are one list of blocks, or, when the past is
// shared by the batch, two kinds of items: rows of several sequences against
// the past, each sequence's rows against its own keys.  The item's part of a
// boolean mask is first turned into bits in shared memory, beside the first
// blocks' copies, once for the rows that share a mask row; blocks after its last
// visible key are not read (but for the first copies, which are on their way by
// then), and values behind that key take no part.
#include <cuda_fp16.h>

#include "attention_flash.cuh"
#include "host_util.h"
#include "kernels.h"
#include "tc100.cuh"
#include "tmem32.cuh"

namespace emx {

constexpr int AR_WARPS = 8;        // most warps of a work item
constexpr int AR_KB = 16;          // keys per block
constexpr int AR_RING = 24 * 1024; // bytes of a warp's ring

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

// 16 bytes global -> shared, or 16 zero bytes
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// Where piece c of key row r lies in its row.
__device__ __forceinline__ int rows_place(int r, int c) { return c ^ (r & 6) ^ ((r & 1) << 2); }

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <bool F32>
__device__ __forceinline__ float additive_entry(const void* mask, int64_t at) {
  return F32 ? __ldg(static_cast<const float*>(mask) + at) : __half2float(__ldg(static_cast<const __half*>(mask) + at));
}

// NS: 64-wide slabs of the head size; NT: tiles of 8 query rows; MASK: MASK_*
template <int NS, int NT, int MASK>
__global__ void __launch_bounds__(32 * AR_WARPS, 1) attention_rows_kernel(const __grid_constant__ RowsParams p) {
  constexpr int NC = 2 * NS;                      // 16-byte pieces of a key row per thread
  constexpr int ROW = 128 * NS;                   // bytes of a key row in the ring
  constexpr int U = NS == 1 && NT == 1 ? 2 : 1;   // blocks of a step
  constexpr int BLOCK = 2 * AR_KB * ROW;          // K and V of a block
  constexpr int STAGE = U * BLOCK;
  constexpr int ST = AR_RING / STAGE;             // 3 steps, or 6 at NS = 1, NT = 2
  constexpr int OW = 64 * NS + 4;                 // padded row of the merge buffer
  constexpr bool ADD = MASK == MASK_ADD || MASK == MASK_ADD32, ADD32 = MASK == MASK_ADD32;
  using Ref = MaskReference<ADD32>;
  extern __shared__ __align__(128) uint8_t s_all[];  // rows_smem() bytes
  __shared__ uint32_t s_bits[MASK == MASK_BITS ? 8 * NT * AF_ROWS_MASK_KEYS / 32 : 1];  // [row][32 keys]
  __shared__ int s_range[2];
  __shared__ float2 s_row[8 * NT];
  __shared__ float s_ref[ADD ? 8 * NT : 1];
  const int warps = blockDim.x >> 5;
  float(*s_o)[8 * NT][OW] = reinterpret_cast<float(*)[8 * NT][OW]>(s_all);  // once the ring is done with
  float(*s_m)[8 * NT] = reinterpret_cast<float(*)[8 * NT]>(s_all + (size_t)warps * 8 * NT * OW * 4);
  float(*s_l)[8 * NT] = s_m + warps, (*s_r)[8 * NT] = s_l + warps;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // Launched beside a tile pass, this grid starts when that one's CTAs have all passed their wait, which the acquire
  // confirms; whatever came before both is then visible here.  If it does not, this grid waits for the tile pass.
  if (!p.late_wait || !others_waited(p.err)) pdl_wait();
  pdl_launch_dependents();

  // ---------------- work item
  const bool past_item = (int)blockIdx.x < p.first1;
  const ItemClass& cl = p.cls[past_item ? 1 : 0];
  int id = (int)blockIdx.x - (past_item ? 0 : p.first1);
  const SmallDiv *by = p.by[past_item ? 1 : 0];  // splits, tiles
  const int id1 = by[0].div(id), split = id - id1 * cl.splits, id2 = by[1].div(id1), tile = id1 - id2 * cl.tiles;
  const int b = p.by_hkv.div(id2), kvh = id2 - b * p.HKV;
  const int rows_all = (int)(p.TQ.d * p.group.d) * (past_item ? p.B : 1);
  const int row0 = tile * 8 * NT, rows = min(8 * NT, rows_all - row0);
  const bool two = NT == 2 && rows > 8;
  int keys = past_item ? 0 : p.tk;  // current keys that some row sees
  if (!past_item) {
    if (p.causal) keys = min(keys, p.group.div(row0 + rows - 1) + 1);
    if (p.counts) {
      const long long n = p.counts[b];
      if ((n < 0 || n > p.tk) && threadIdx.x == 0) record_bad_index(p.err);
      keys = min(keys, (int)max(0ll, min(n, (long long)p.tk)));
    }
  }
  const int past = cl.past ? p.tp : 0;
  const int pblocks = (past + AR_KB - 1) / AR_KB, blocks = pblocks + (keys + AR_KB - 1) / AR_KB;
  const int share = by[0].div(blocks + cl.splits - 1);  // (blocks * splits < 2^32 as well)
  const int blk0 = min(blocks, share * split);
  int blk1 = min(blocks, share * (split + 1));

  const uint16_t* kc = p.k + (int64_t)b * p.k_sb + (int64_t)kvh * p.k_sh;
  const uint16_t* vc = p.v + (int64_t)b * p.v_sb + (int64_t)kvh * p.v_sh;
  const int64_t ph = ((int64_t)(p.past_shared ? 0 : b) * p.HKV + kvh) * p.tp;
  const uint16_t* kp = p.past_k + ph * p.D;
  const uint16_t* vp = p.past_v + ph * p.DV;

  // ---------------- copies: this warp's n-th step takes the U blocks from blk0 + U (warp + n warps), in stage n % ST
  const uint32_t ring = smem_u32(s_all) + warp * AR_RING;
  auto issue = [&](int blk, int stage) {
#pragma unroll
    for (int u = 0; u < U; ++u, ++blk) {
      if (blk >= blk1) break;
      const bool is_past = blk < pblocks;
      const int k0 = (is_past ? blk : blk - pblocks) * AR_KB, n = (is_past ? past : keys) - k0;
      const int ks = is_past ? p.D : (int)p.k_st, vs = is_past ? p.DV : (int)p.v_st;
      constexpr int PIECES = 8 * NS, STEP = 32 / PIECES;
      const int c = lane % PIECES, r0 = lane / PIECES;
      const uint16_t* ksrc = (is_past ? kp : kc) + (int64_t)(k0 + r0) * ks + 8 * c;
      const uint16_t* vsrc = (is_past ? vp : vc) + (int64_t)(k0 + r0) * vs + 8 * c;
      const int64_t k_step = (int64_t)STEP * ks, v_step = (int64_t)STEP * vs;
      const uint32_t dst = ring + stage * STAGE + u * BLOCK;
      const bool k_in = 8 * c < p.D, v_in = 8 * c < p.DV;
#pragma unroll
      for (int i = 0; i < AR_KB; i += STEP) {
        const int r = r0 + i;
        const bool in = r < n;
        const uint32_t at = dst + r * ROW + rows_place(r, c) * 16;
        // rows past the keys and pieces past the head size are zero (what is not taken is not read either)
        cp_async16_or_zero(at, in && k_in ? ksrc : p.k, in && k_in);
        cp_async16_or_zero(at + AR_KB * ROW, in && v_in ? vsrc : p.v, in && v_in);
        ksrc += k_step, vsrc += v_step;
      }
    }
    cp_async_commit();  // (an empty group keeps the count)
  };
#pragma unroll 1  // (straight-line copies cost more in instruction fetches than they gain)
  for (int n = 0; n < ST - 1; ++n) issue(blk0 + U * (warp + n * warps), n);

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
      mrow[n][e] = !ADD ? 0 : (w.b * p.mask_sb + w.h * p.mask_sh + w.t * p.mask_st) * (int64_t)p.mask_len;
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

  // ---------------- boolean mask: bits of the item's keys, counted through its blocks; the blocks worth reading
  // Rows with one mask row share its bits: all rows of a sequence's item where neither heads nor tokens have their
  // own, a token's group of heads where heads have not, else none.
  const bool one_row = p.mask_sh == 0 && p.mask_st == 0 && !past_item;
  const int token0 = p.group.div(row0);
  auto bits_of = [&](int r) { return one_row ? 0 : p.mask_sh == 0 ? p.group.div(row0 + r) - token0 : r; };
  const uint32_t* bit_row[NT][2];  // this thread's rows
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) bit_row[n][e] = s_bits + bits_of(min(8 * n + 2 * t + e, rows - 1)) * (AF_ROWS_MASK_KEYS / 32);
  int first = blk0;  // bits of block i start at bit (i - blk0) * AR_KB
  int key_end = (blk1 - blk0) * AR_KB;  // end of the visible keys, counted the same way (the copies zero keys past `keys`)
  if (MASK == MASK_BITS) {
    if (threadIdx.x < 2) s_range[threadIdx.x] = threadIdx.x ? 0 : 0x7fffffff;
    __syncthreads();
    const int words = ((blk1 - blk0) * AR_KB + 31) / 32, mask_rows = bits_of(rows - 1) + 1;
    int lo = 0x7fffffff, hi = 0;
    // a warp takes 256 keys of a row at a time, eight loads in flight
    constexpr int LOADS = 8;
    const int groups = (words + LOADS - 1) / LOADS;
#pragma unroll 1
    for (int i = warp; i < groups * mask_rows; i += warps) {
      const int r = i / groups, w4 = (i - r * groups) * LOADS;
      // (a row with these bits: the first of the token's, if the tile has it)
      const int row = one_row || p.mask_sh != 0 ? row0 + r : max(row0, (token0 + r) * (int)p.group.d);
      const RowId w = row_of(row, p.group, p.TQ, kvh, b, past_item);
      const uint8_t* src = p.mask_bool + (w.b * p.mask_sb + w.h * p.mask_sh + w.t * p.mask_st) * (int64_t)p.mask_len;
      uint8_t v[LOADS];
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int blk = blk0 + ((w4 + u) * 32 + lane) / AR_KB, in_blk = lane % AR_KB;
        const bool is_past = blk < pblocks;
        const int k = (is_past ? blk : blk - pblocks) * AR_KB + in_blk, pos = (is_past ? 0 : p.tp) + k;
        v[u] = blk < blk1 && k < (is_past ? past : keys) && pos < p.mask_len ? __ldg(src + pos) : (uint8_t)0;
      }
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const uint32_t bits = __ballot_sync(0xffffffffu, v[u] != 0);
        if (w4 + u >= words) break;
        if (lane == 0) s_bits[r * (AF_ROWS_MASK_KEYS / 32) + w4 + u] = bits;
        if (bits) {
          lo = min(lo, (w4 + u) * 32 + __ffs(bits) - 1);
          hi = max(hi, (w4 + u) * 32 + 32 - __clz(bits));
        }
      }
    }
    if (lane == 0 && hi) {
      atomicMin(&s_range[0], lo);
      atomicMax(&s_range[1], hi);
    }
    __syncthreads();
    const int lo_blk = s_range[1] ? blk0 + s_range[0] / AR_KB : blk1;
    const int hi_blk = s_range[1] ? blk0 + (s_range[1] + AR_KB - 1) / AR_KB : blk0;
    // later copies stop at the last block with a visible key; the blocks before the first are passed over below
    blk1 = min(blk1, hi_blk);
    first = lo_blk;
    key_end = s_range[1];
  }

  // additive mask entries of a step at this thread's scores, loaded a step ahead
  float mk[U][ADD ? 4 * NT : 1], mk_next[U][ADD ? 4 * NT : 1];
  auto load_add = [&](int blk) {
#pragma unroll
    for (int u = 0; u < (ADD ? U : 0); ++u, ++blk) {
      const bool is_past = blk < pblocks;
      const int k0 = (is_past ? blk : blk - pblocks) * AR_KB, pos0 = (is_past ? 0 : p.tp) + k0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int pos = pos0 + 8 * h + g;
        const bool in = blk < blk1 && k0 + 8 * h + g < (is_past ? past : keys);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            mk_next[u][(h * NT + n) * 2 + e] =
                in && pos < p.mask_len ? additive_entry<ADD32>(p.mask_add, mrow[n][e] + pos) : -INFINITY;
      }
    }
  };

  float o[NT][NS][4][4];  // O^T: [row tile][slab][d pair][(d, row), (d, row + 1), (d + 1, row), (d + 1, row + 1)]
  float m_ref[NT][2], l[NT][2], ref[NT][2];  // ref: mask references
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) m_ref[n][e] = -INFINITY, l[n][e] = 0.0f, ref[n][e] = 0.0f;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][s][j][e] = 0.0f;
  }
  const float sc = p.scale_log2;
  bool any_block = false;
  // operand addresses within a stage: K row g (and g + 8), V rows 2t, 2t + 1 (and + 8)
  const uint32_t k_row = ring + g * ROW, v_row = ring + AR_KB * ROW + 2 * t * ROW;
  const int k_swz = rows_place(g, 0), v_swz0 = rows_place(2 * t, 0), v_swz1 = rows_place(2 * t + 1, 0);

  load_add(blk0 + U * warp);
  for (int n = 0, blk = blk0 + U * warp; blk < blk1; ++n, blk += U * warps) {
    cp_async_wait_group<ST - 2>();  // this step's copies (one group a step) are done, for every lane
    __syncwarp();
    issue(blk + (ST - 1) * U * warps, (n + ST - 1) % ST);  // into the stage of the step before this one
    if (ADD) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4 * NT; ++i) mk[u][i] = mk_next[u][i];
      load_add(blk + U * warps);
    }
    if (MASK == MASK_BITS && blk + U - 1 < first) continue;
    any_block = true;
    const uint32_t stage = (uint32_t)(n % ST) * STAGE;
    // ---------------- which of this thread's scores count: [block][half][tile][row]
    uint32_t see = ~0u;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool is_past = blk + u < pblocks;
      const int k0 = (is_past ? blk + u : blk + u - pblocks) * AR_KB, pos0 = (is_past ? 0 : p.tp) + k0;
      const int seg_end = blk + u >= blk1 ? 0 : is_past ? past : p.tp + keys;
      if (MASK == MASK_NONE && pos0 + AR_KB <= min(lim_all, seg_end)) continue;
      const int bit = (blk + u - blk0) * AR_KB;
#pragma unroll
      for (int n2 = 0; n2 < NT; ++n2)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t bits = 0xffffu;
          if (MASK == MASK_BITS && blk + u < blk1)
            bits = bit_row[n2][e][bit >> 5] >> (bit & 31);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int pos = pos0 + 8 * h + g, i = (h * NT + n2) * 2 + e;
            bool ok = pos < min(lim[n2][e], seg_end) && ((bits >> (8 * h + g)) & 1u);
            if (ADD) {
              ok = ok && mk[u][i] != -INFINITY;
              if (!ok) mk[u][i] = -INFINITY;
            }
            if (!ok) see &= ~(1u << (4 * NT * u + i));
          }
        }
    }
    // ---------------- S^T
    uint4 k[U][2][NC];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint32_t at = k_row + stage + u * BLOCK + (((t + 4 * c) ^ k_swz) << 4);
        k[u][0][c] = lds128(at);
        k[u][1][c] = lds128(at + 8 * ROW);
      }
    float s[U][NT][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int n2 = 0; n2 < NT; ++n2) {
        float s2[4];  // two chains of products
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][n2][e] = s2[e] = 0.0f;
        if (n2 == 1 && !two) continue;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          mma_16816(s[u][n2], k[u][0][c].x, k[u][1][c].x, k[u][0][c].y, k[u][1][c].y, q[n2][c].x, q[n2][c].y);
          mma_16816(s2, k[u][0][c].z, k[u][1][c].z, k[u][0][c].w, k[u][1][c].w, q[n2][c].z, q[n2][c].w);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][n2][e] = (s[u][n2][e] + s2[e]) * sc;
      }
    // V in K's registers, on its way during the softmax
    uint4 v[U][NS][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int sl = 0; sl < NS; ++sl) {
        const uint32_t at = v_row + stage + u * BLOCK;
        v[u][sl][0] = lds128(at + (((8 * sl + g) ^ v_swz0) << 4));
        v[u][sl][1] = lds128(at + ROW + (((8 * sl + g) ^ v_swz1) << 4));
        v[u][sl][2] = lds128(at + 8 * ROW + (((8 * sl + g) ^ v_swz0) << 4));
        v[u][sl][3] = lds128(at + 9 * ROW + (((8 * sl + g) ^ v_swz1) << 4));
      }
    // keys behind the item's last visible one, and blocks before its first, take no part whatever their values hold
    if ((blk + U - blk0) * AR_KB > key_end) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((blk + u - blk0) * AR_KB + 2 * t + (i & 1) + 8 * (i >> 1) >= key_end) {
#pragma unroll
            for (int sl = 0; sl < NS; ++sl) v[u][sl][i] = make_uint4(0u, 0u, 0u, 0u);
          }
    }
    if (MASK == MASK_BITS && U == 2 && blk < first) {
#pragma unroll
      for (int i = 0; i < 4 * NS; ++i) v[0][i >> 2][i & 3] = make_uint4(0u, 0u, 0u, 0u);
    }
    // scores in log2 units; entries the row does not see are -inf
    if (see != ~0u) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n2 = 0; n2 < NT; ++n2)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!((see >> (4 * NT * u + ((e >> 1) * NT + n2) * 2 + (e & 1))) & 1u)) s[u][n2][e] = -INFINITY;
    }
    // the largest entry of a row's visible keys may move its mask reference; then the entries join the scores
    if (ADD) {
      float most[NT][2];
      bool move = false;
#pragma unroll
      for (int n2 = 0; n2 < NT; ++n2)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          most[n2][e] = -INFINITY;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) most[n2][e] = fmaxf(most[n2][e], mk[u][(h * NT + n2) * 2 + e]);
          move = move || Ref::moves(most[n2][e], ref[n2][e], m_ref[n2][e]);
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int n2 = 0; n2 < NT; ++n2)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = most[n2][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            if (Ref::moves(x, ref[n2][e], m_ref[n2][e])) {
              m_ref[n2][e] = Ref::moved(m_ref[n2][e], ref[n2][e], Ref::of(x));
              ref[n2][e] = Ref::of(x);
            }
          }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n2 = 0; n2 < NT; ++n2)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[u][n2][e] = Ref::score(mk[u][((e >> 1) * NT + n2) * 2 + (e & 1)], ref[n2][e & 1], s[u][n2][e]);
    }
    bool grow = false;
    float top[NT][2];
#pragma unroll
    for (int n2 = 0; n2 < NT; ++n2)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (n2 == 1 && !two) continue;
        float x = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
          x = fmaxf(x, fmaxf(s[u][n2][e], s[u][n2][2 + e]));
        top[n2][e] = x;
        grow = grow || x - m_ref[n2][e] > AFK_RESCALE;  // (or the first one: inf > 8)
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n2 = 0; n2 < NT; ++n2)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (n2 == 1 && !two) continue;
          float x = top[n2][e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
          const float old = m_ref[n2][e];
          if (x - old > AFK_RESCALE || old == -INFINITY) {
            m_ref[n2][e] = x;
            const float alpha = old == -INFINITY ? 0.0f : ex2_approx(old - x);
            l[n2][e] *= alpha;
#pragma unroll
            for (int sl = 0; sl < NS; ++sl)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                o[n2][sl][j][e] *= alpha;
                o[n2][sl][j][e + 2] *= alpha;
              }
          }
        }
    }
    // ---------------- weights, as the B operand of the second product
    uint32_t pb[U][NT][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int n2 = 0; n2 < NT; ++n2) {
        if (n2 == 1 && !two) continue;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float neg = m_ref[n2][e] == -INFINITY ? 0.0f : -m_ref[n2][e];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            s[u][n2][2 * h + e] = ex2_approx(s[u][n2][2 * h + e] + neg);
            l[n2][e] += s[u][n2][2 * h + e];  // (before the rounding)
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) pb[u][n2][h] = transpose_8x8(pack_f16x2(s[u][n2][2 * h], s[u][n2][2 * h + 1]));
      }
    // ---------------- O^T += V^T P^T
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int sl = 0; sl < NS; ++sl) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w0 = word_of(v[u][sl][0], j), w1 = word_of(v[u][sl][1], j);
          const uint32_t w2 = word_of(v[u][sl][2], j), w3 = word_of(v[u][sl][3], j);
          const uint32_t a0 = __byte_perm(w0, w1, 0x5410), a1 = __byte_perm(w0, w1, 0x7632);
          const uint32_t a2 = __byte_perm(w2, w3, 0x5410), a3 = __byte_perm(w2, w3, 0x7632);
          mma_16816(o[0][sl][j], a0, a1, a2, a3, pb[u][0][0], pb[u][0][1]);
          if (NT == 2 && two) mma_16816(o[NT - 1][sl][j], a0, a1, a2, a3, pb[u][NT - 1][0], pb[u][NT - 1][1]);
        }
      }
    __syncwarp();  // the stage's readers are done before its next copies
  }
  cp_async_wait_group<0>();

  // ---------------- merge the warps (over the rings), write the rows
  __syncthreads();
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
        if (ADD) s_r[warp][r] = ref[n][e];
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
  // thread (row, warp): that warp's factor 2^(m - M) in place of its m, the row's M and sum beside them
  {
    const int r = threadIdx.x >> 3, w = threadIdx.x & 7;
    if (r < 8 * NT) {  // whole groups of eight lanes; CTAs of fewer threads than rows x 8 go around below
      for (int rr = r; rr < 8 * NT; rr += blockDim.x >> 3) {
        const bool in = w < warps && rr < rows;
        const float lw = in ? s_l[w][rr] : 0.0f;
        float mw = in && lw != 0.0f ? s_m[w][rr] : -INFINITY;
        if (ADD) {  // maxima relative to the warps' largest reference
          const float rw = in && lw != 0.0f ? s_r[w][rr] : -INFINITY;
          float most = rw;
#pragma unroll
          for (int d = 4; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d, 8));
          if (in && lw != 0.0f) mw += Ref::from(most, rw);
          if (w == 0 && rr < rows) s_ref[rr] = most;
        }
        float m = mw, sum;
#pragma unroll
        for (int d = 4; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d, 8));
        const float f = lw != 0.0f ? ex2_approx(mw - m) : 0.0f;
        sum = f * lw;
#pragma unroll
        for (int d = 4; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d, 8);
        if (in) s_m[w][rr] = f;
        if (w == 0 && rr < rows) s_row[rr] = make_float2(m, sum);
      }
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < rows * 16 * NS; i += blockDim.x) {
    const int r = i / (16 * NS), d = (i % (16 * NS)) * 4;
    if (d >= p.DV) continue;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < AR_WARPS; ++w) {
      const float f = w < warps ? s_m[w][r] : 0.0f;
      if (f == 0.0f) continue;  // a warp without keys has written no output
      const float4 x = *reinterpret_cast<const float4*>(&s_o[w][r][d]);
      acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
    }
    const float2 ms = s_row[r];
    const RowId w = row_of(row0 + r, p.group, p.TQ, kvh, b, past_item);
    if (p.part_o) {
      const int64_t at = (int64_t)(cl.part0 + split) * ((int64_t)p.B * (int)p.TQ.d * p.HQ) + ((int64_t)w.b * (int)p.TQ.d + w.t) * p.HQ + w.h;
      if (d == 0) p.part_ml[at] = ms;
      if (ADD && d == 0) p.part_ref[at] = s_ref[r];
      *reinterpret_cast<float4*>(p.part_o + at * p.DV + d) = acc;
    } else {
      const float inv = ms.y == 0.0f ? 0.0f : 1.0f / ms.y;
      *reinterpret_cast<uint2*>(p.o + (int64_t)w.b * p.o_sb + (int64_t)w.h * p.o_sh + (int64_t)w.t * p.o_st + d) =
          make_uint2(pack_f16x2(acc.x * inv, acc.y * inv), pack_f16x2(acc.z * inv, acc.w * inv));
    }
  }
  // This grid neither reads nor writes the results of the tile pass beside it.  One CTA ends after that pass, so this
  // grid does, and the merge kernel's wait for this grid covers both.
  if (p.late_wait && blockIdx.x == gridDim.x - 1) pdl_wait();
}

// ------------------------------------------------------------------ host side
static size_t rows_smem(int ns, int nt, int warps) {
  const size_t merge = (size_t)warps * 8 * nt * (64 * ns + 4 + 3) * sizeof(float), ring = (size_t)warps * AR_RING;
  return merge > ring ? merge : ring;
}

template <int NS, int NT>
static const void* rows_kernel(int mask) {
  return mask == MASK_NONE ? (const void*)attention_rows_kernel<NS, NT, MASK_NONE>
         : mask == MASK_BITS ? (const void*)attention_rows_kernel<NS, NT, MASK_BITS>
         : mask == MASK_ADD  ? (const void*)attention_rows_kernel<NS, NT, MASK_ADD>
                             : (const void*)attention_rows_kernel<NS, NT, MASK_ADD32>;
}

static const void* rows_kernel(bool wide, int row_tiles, int mask) {
  if (row_tiles == 1) return wide ? rows_kernel<2, 1>(mask) : rows_kernel<1, 1>(mask);
  return wide ? rows_kernel<2, 2>(mask) : rows_kernel<1, 2>(mask);
}

cudaError_t prepare_attention_rows() {
  for (int i = 0; i < 16; ++i) {
    cudaError_t e = cudaFuncSetAttribute(rows_kernel(i & 1, 1 + ((i >> 1) & 1), i >> 2),
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, AR_WARPS * AR_RING);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t launch_attention_rows(const RowsParams& p, int row_tiles, int mask, int warps, unsigned items,
                                  cudaStream_t stream) {
  if (warps < 1 || warps > AR_WARPS) return cudaErrorInvalidValue;
  const bool wide = p.D > 64 || p.DV > 64;
  auto kernel = reinterpret_cast<void (*)(const RowsParams)>(const_cast<void*>(rows_kernel(wide, row_tiles, mask)));
  return launch_pdl(kernel, dim3(items), dim3(32 * warps), rows_smem(wide ? 2 : 1, row_tiles, warps), stream, p);
}

}  // namespace emx
