// What the passes of K_ATTENTION_FLASH share: how query rows are packed, the
// additive mask's entries, and the few-row pass (attention_rows.cu).
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

namespace emx {

constexpr float AFK_RESCALE = 8.0f;  // the output is rescaled when a row's maximum grows by more (log2 units)
constexpr float AFK_LOG2E = 1.4426950408889634f;

// Exponents are score * scale - m in one fused step, m the rounded product of the largest score, so they are off by half
// a step of m at most, by the same in numerator and sum.  From 2^24 on (a step of 2) a row's scores are scaled, and
// rounded like m, first: from 2^27 on its largest weight could leave fp16's range either way.
constexpr float AFK_LARGE = 0x1p24f;
__device__ __forceinline__ bool large_scores(float m) { return fabsf(m) >= AFK_LARGE && m > -INFINITY; }

enum { MASK_NONE = 0, MASK_BITS = 1, MASK_ADD = 2 /*fp16 entries*/, MASK_ADD32 = 3 };  // kernel variants

struct RowId {
  int b, h, t;
};

// Division of the rows' small numbers by a launch's constant: n / d = (n * magic) >> 32 with magic = 2^32 / d + 1 is
// exact while n * d < 2^32 (checked by the host; d = 1 has no 32-bit magic and is its own case).
struct SmallDiv {
  uint32_t d, magic;
  __host__ static SmallDiv of(uint32_t d) { return {d, d > 1 ? (uint32_t)((1ull << 32) / d + 1) : 0u}; }
  __host__ __device__ __forceinline__ int div(int n) const {
#ifdef __CUDA_ARCH__
    return d == 1 ? n : (int)__umulhi((uint32_t)n, magic);
#else
    return d == 1 ? n : (int)(((unsigned long long)(uint32_t)n * magic) >> 32);
#endif
  }
};

// Row r of a work item's rows: (token, head of the group), tokens slowest, of
// sequence b, or of every sequence one after the other.
__host__ __device__ __forceinline__ RowId row_of(int r, const SmallDiv& group, const SmallDiv& TQ, int kvh, int b,
                                                 bool all_sequences) {
  const int bt = group.div(r), g = r - bt * (int)group.d;
  RowId id;
  id.h = kvh * (int)group.d + g;
  id.b = b, id.t = bt;
  if (all_sequences) {
    id.b = TQ.div(bt);
    id.t = bt - id.b * (int)TQ.d;
  }
  return id;
}

// An entry of an additive mask may be so large that a score added to it loses its digits, and entries so far apart that
// their difference decides alone.  The passes therefore hold a row's running maximum as a pair (mask reference R,
// maximum m of score + (entry - R)): R is the largest visible entry of some key tile, and moves when a later one is
// more than AFK_REFERENCE above it, so keys that matter have small differences to it, formed before the score is added.
// Partial results carry R beside (m, l).  fp32 entries from 2^56 on leave no digit of a score in 64 bits either: their
// keys count without it (those at the type's lowest value weigh the same among themselves).
constexpr float AFK_ALONE = 0x1p56f;
constexpr float AFK_REFERENCE = 16.0f;

// R is held in log2 units for fp16 entries, as the entry itself for fp32 ones (whose product may leave the range).
template <bool F32>
struct MaskReference {
  static __device__ __forceinline__ float of(float entry) { return F32 ? entry : entry * AFK_LOG2E; }
  // log2 units from reference r to reference (or entry) to
  static __device__ __forceinline__ float from(float r, float to) { return F32 ? (to - r) * AFK_LOG2E : to - r; }
  // score (log2 units) with its key's entry; -inf hides the key whatever its score is
  static __device__ __forceinline__ float score(float entry, float r, float s) {
    if (F32) return fmaf(entry - r, AFK_LOG2E, fabsf(entry) >= AFK_ALONE ? 0.0f : s);
    return entry == -INFINITY ? -INFINITY : s + fmaf(entry, AFK_LOG2E, -r);
  }
  // whether a largest visible entry moves the reference of a row with maximum m (-inf: it has none yet)
  static __device__ __forceinline__ bool moves(float entry, float r, float m) {
    return entry > -INFINITY && (m == -INFINITY || from(r, of(entry)) > AFK_REFERENCE);
  }
  // the maximum m under the new reference (a difference beyond fp32 leaves the keys before no weight, but -inf stands
  // for none seen)
  static __device__ __forceinline__ float moved(float m, float r, float to) {
    return m == -INFINITY ? m : fmaxf(m - from(r, to), -FLT_MAX);
  }
};

// The work items of a pass come in two classes: 0, the rows of one sequence
// against its own keys (behind its past where `past` is set: one list of key
// tiles, the past's first), and 1, the rows of every sequence against a past
// that they share.  Items of class 1 have the lower block indices.
struct ItemClass {
  int splits;  // items along the keys
  int tiles;   // row tiles per key/value head (and sequence)
  int part0;   // first slot of partial results
  int past;
};

// Item `split` of `splits` takes floor(n split / splits) up to the next item's first of n tiles (32-bit: n may be
// 2^25, splits some hundreds).
__host__ __device__ __forceinline__ int split_start(int n, int split, int splits) {
  const int whole = n / splits;
  return whole * split + (n - whole * splits) * split / splits;
}

struct TileParams {
  CUtensorMap map_k[2], map_v[2];  // current keys, past: 4-D (d, key, head, batch), box (64, tile keys, 1, 1), 128-byte swizzle
  CUtensorMap map_q[2];  // per class: 5-D (d, head of the group, token, key/value head, sequence), 128 rows a box
  int q_boxes[2];        // whether 128 consecutive rows of the class are such a box
  ItemClass cls[2];
  int first1, items;  // items of class 1, of both
  const uint16_t* q;
  uint16_t* o;
  float* part_o;    // [slot][row][DV], null: one item per row, written to o
  float2* part_ml;  // [slot][row] (m, l)
  float* part_ref;  // [slot][row] mask references, additive masks only
  int64_t q_sb, q_sh, q_st, o_sb, o_sh, o_st;
  int B, HQ, HKV, D, DV, causal, tk, tp, past_shared;
  SmallDiv group, TQ;
  const long long* counts;  // valid current keys of each sequence, or null
  int64_t mask_sb, mask_sh, mask_st;  // mask row of (b, h, t): b * sb + h * sh + t * st
  const unsigned long long* bits;     // packed boolean mask [row][words], the past's words first
  const int4* spans;                  // per mask row: first and end visible current key, first and end visible past key
  // additive mask in whole 64-key tiles, the past's first, -inf past the mask's length and past each part's keys:
  // [tile][16-byte piece of its keys][mask row], so that neighbouring rows' loads of a piece are neighbours
  const uint4* add;
  int64_t mask_rows;
  int words, words_past, mask_len;
  float scale_log2;
  int publish;    // the own keys' few-row pass runs beside this one: tell it when this one has waited (publish_waited)
  int drop_keys;  // failure-detection test hook (FAULT_DROP_KEY_TILES)
  int* err;
};

struct RowsParams {
  ItemClass cls[2];
  SmallDiv by[2][2], by_hkv;  // by a class's splits and tiles, by the key/value heads
  int first1;
  const uint16_t *q, *k, *v, *past_k, *past_v;
  uint16_t* o;
  float* part_o;
  float2* part_ml;
  float* part_ref;
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st, o_sb, o_sh, o_st;
  int B, HQ, HKV, D, DV, causal, tp, tk, past_shared;
  SmallDiv group, TQ;
  const long long* counts;
  int64_t mask_sb, mask_sh, mask_st;
  const uint8_t* mask_bool;
  const void* mask_add;
  int mask_len;
  float scale_log2;
  int late_wait;  // launched beside a tile pass (publish) whose results it does not read
  int* err;
};

cudaError_t prepare_attention_wide();
cudaError_t launch_attention_wide(const TileParams& p, int slabs, int mask, int num_sms, cudaStream_t stream);
cudaError_t prepare_attention_rows();
cudaError_t launch_attention_rows(const RowsParams& p, int row_tiles, int mask, int warps, unsigned items,
                                  cudaStream_t stream);

}  // namespace emx
