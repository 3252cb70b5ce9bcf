// RMSNormalization and RotaryEmbedding (opset 23), fp16 and fp32.
//
// K_NORM_ROPE: per head row x of D elements of token (b, t)
//   y = x / sqrt(mean(x^2) + eps) * scale          (when a norm feeds the rotation)
//   (y_a, y_b) -> (y_a c - y_b s, y_a s + y_b c)   over the first ROT elements
// with pairs (i, i + ROT/2), or (2i, 2i+1) interleaved, and c, s the token's
// row of the tables.  Everything between the load and the store is fp32 and
// rounded once at the end (the separate operators would round in between).
// The element orders of x and y are strides, so the exchange of the token and
// head axes that stands between the two operators in a graph costs nothing,
// and Q and K of a layer go in one launch.
//
// The bound is memory: every element is read and written once.  A row is
// spread over LPR lanes, each holding the two 16-byte pieces that pair up, so
// a rotation needs no exchange and the row sum log2(LPR) shuffles; a lane
// group takes HPG head rows of its token and loads the token's table entries
// once for them.  8 x 4096 tokens of 32 + 8 fp16 heads of 128 (671 MB moved)
// take 134 us, 5.0 TB/s; back to back 125 us, and as long with the arithmetic
// taken out.  4 x 2048 tokens: 37 us.  One token of 32 sequences: 7.7 us, of
// which 7 are the host's call.
//
// K_RMS_NORM: rows of any length, a warp per row up to 1024 elements, else a
// CTA per row; the second pass over the row hits L1 / L2.  8192 fp16 rows of
// 8192 elements: 47 us, 5.7 TB/s; of 4096: 35 us, 3.9 TB/s.
#include <cuda_fp16.h>
#include <stdint.h>

#include "f32x2.cuh"
#include "host_util.h"
#include "kernels.h"
#include "tc100.cuh"

namespace emx {

struct RopeItem {
  const void* x;
  const void* scale;  // null: no norm
  void* y;
  int64_t x_sb, x_st, x_sh, y_sb, y_st, y_sh;
  int heads;
  float eps;
};

struct RopeParams {
  RopeItem item[2];
  const void *cos, *sin;
  const long long* pos;
  int64_t tokens;
  int T, D, rot, interleaved, heads /*of both items*/;
  int groups[2];  // lane groups per token of each item
  float inv_d;
  int64_t positions;
  int* err;
};

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }

// 16 bytes as fp32 values
template <typename T>
struct Chunk;
template <>
struct Chunk<__half> {
  static constexpr int N = 8;
  __device__ static __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  __device__ static __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Chunk<float> {
  static constexpr int N = 4;
  __device__ static __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  __device__ static __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// Row of the tables that token (b, t) = `token` uses, or -1 (error recorded) for an id out of range.
__device__ __forceinline__ int64_t table_row(const RopeParams& p, int64_t token) {
  if (!p.positions) return token;
  const long long at = p.pos[token];
  if (at >= 0 && at < p.positions) return at;
  record_bad_index(p.err);
  return -1;
}

// 1 / sqrt(v), 0 of an infinite v: rsqrtf (2 steps of fp32 at most) for fp16 results, one Newton step more for fp32's.
template <typename T>
__device__ __forceinline__ float inv_sqrt(float v) {
  const float y = rsqrtf(v);
  return sizeof(T) == 2 || v == INFINITY ? y : fmaf(y * 0.5f, fmaf(-v * y, y, 1.0f), y);
}

// A row's norm factor 1 / sqrt(mean(x^2) + eps) is taken in two parts, x * pre * inv, where the squares leave fp32's
// range: above it, v = mean + eps is infinite (or NaN); below it, squares under 2^-126 lose their digits, which counts
// where v < 2^-90.  The row's squares are then summed again with pre = 2^-96 or 2^96, a power of two:
//   inv = 1 / sqrt(mean((pre x)^2) + pre^2 eps),
// all of it in range, and what underflows now is below the sum's last digit.  An infinite element keeps inv at 0, so
// the row's finite elements are 0 and it is NaN, as in x / sqrt(inf).  (fp16 rows: 2^-48 / N <= mean < 2^33, or infinite
// with an infinite element: nothing to sum again.)
__device__ __forceinline__ bool squares_in_range(float v) { return v >= 0x1p-90f && v < INFINITY; }
__device__ __forceinline__ float norm_pre(float v) { return v < 1.0f ? 0x1p96f : 0x1p-96f; }
__device__ __forceinline__ float norm_inv_pre(float mean, float eps, float pre) {
  return inv_sqrt<float>(mean + eps * pre * pre);  // (pre^2 alone is beyond fp32)
}

// Vector form: D and the rotated halves are whole 16-byte pieces, every row starts on 16 bytes.
// A lane's two pieces hold V pairs (f, s): (piece 0, piece 1) element by element, or neighbours of one piece
// (INTER).  Norm scale and rotation make one 2 x 2 matrix per pair, formed once for the group's rows:
//   f' = inv (f wf cos - s ws sin),  s' = inv (f wf sin + s ws cos).
// RING > 0: lane groups stay and go from token to token; every lane copies its own pieces asynchronously to
// shared memory, RING - 1 groups ahead, so that loads are under way all the time whatever the registers hold.
template <typename T, int LPR, int HPG, int RING, bool INTER>
__global__ void __launch_bounds__(256, RING ? 2 : 3) norm_rope_kernel(const __grid_constant__ RopeParams p) {
  constexpr int V = Chunk<T>::N;
  constexpr int SLOTS = 2 * HPG;  // pieces of a lane per group
  extern __shared__ uint4 s_ring[];  // [RING][SLOTS][256]
  pdl_wait();
  pdl_launch_dependents();
  const int u = threadIdx.x % LPR;
  // lanes of one group take the same path throughout and shuffle among themselves only
  const uint32_t group_mask = LPR == 32 ? 0xffffffffu : ((1u << (LPR & 31)) - 1u) << (threadIdx.x & 31 & ~(LPR - 1));
  const uint32_t per_token = (uint32_t)(p.groups[0] + p.groups[1]), total = (uint32_t)p.tokens * per_token;
  const uint32_t stride = gridDim.x * (256u / LPR);
  uint32_t gi = blockIdx.x * (256u / LPR) + threadIdx.x / LPR;  // lane group (their count fits 32 bits)
  const int nc = p.D / V, rc = p.rot / V;
  // this lane's two pieces and whether they rotate
  int c0 = 2 * u, c1 = 2 * u + 1;
  bool turn = c0 < rc;
  if (!INTER) {
    turn = u < rc / 2;
    c0 = turn ? u : rc + 2 * (u - rc / 2);
    c1 = turn ? u + rc / 2 : c0 + 1;
  }
  const bool has0 = c0 < nc, has1 = c1 < nc;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  // a group's token, tensor and first row
  struct Place {
    uint32_t token;
    int sel, j, b, t;
  };
  auto place = [&](uint32_t at) {
    Place w;
    w.token = at / per_token;
    w.j = (int)(at - w.token * per_token);
    w.sel = w.j >= p.groups[0] ? 1 : 0;  // a group's rows are of one tensor
    if (w.sel) w.j -= p.groups[0];
    w.b = (int)(w.token / (uint32_t)p.T);
    w.t = (int)(w.token - (uint32_t)w.b * (uint32_t)p.T);
    return w;
  };
  auto fetch = [&](uint32_t at, int slot) {
    if (at < total) {
      const Place w = place(at);
      const RopeItem& it = p.item[w.sel];
      const int step = p.groups[w.sel];
      const T* x = static_cast<const T*>(it.x) + w.b * it.x_sb + w.t * it.x_st + w.j * it.x_sh;
      uint4* dst = s_ring + slot * SLOTS * 256 + threadIdx.x;
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        if (w.j + i * step < it.heads) {
          if (has0) cp_async16(dst + (2 * i) * 256, x + c0 * V);
          if (has1) cp_async16(dst + (2 * i + 1) * 256, x + c1 * V);
        }
        x += step * it.x_sh;
      }
    }
    cp_async_commit();  // (an empty group keeps the count)
  };
  auto load_tables = [&](int64_t row, uint4& c4, uint4& s4) {
    const int64_t at = row * (p.rot / 2) + u * V;
    c4 = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.cos) + at);
    s4 = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.sin) + at);
  };
  auto row_of_group = [&](uint32_t at) {
    return turn && at < total ? table_row(p, at / per_token) : 0;
  };
  // The ring's table entries are read one group ahead, their row's number two (it may be a position to load).
  int64_t row_now = 0, row_next = 0;
  uint4 cos_next = zero, sin_next = zero;
  if (RING) {
#pragma unroll
    for (int n = 0; n < RING - 1; ++n) fetch(gi + n * stride, n);
    row_now = row_of_group(gi);
    row_next = row_of_group(gi + stride);
    if (turn && row_now >= 0) load_tables(row_now, cos_next, sin_next);
  }
  int slot = 0;
#pragma unroll 1
  for (; gi < total; gi += stride) {
    const Place w = place(gi);
    const RopeItem& it = p.item[w.sel];
    const int step = p.groups[w.sel];
    uint4 xv[RING ? 1 : HPG][2];
    if (!RING) {
      const T* x = static_cast<const T*>(it.x) + w.b * it.x_sb + w.t * it.x_st + w.j * it.x_sh;
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        const bool in = w.j + i * step < it.heads;
        xv[RING ? 0 : i][0] = in && has0 ? __ldcs(reinterpret_cast<const uint4*>(x + c0 * V)) : zero;
        xv[RING ? 0 : i][1] = in && has1 ? __ldcs(reinterpret_cast<const uint4*>(x + c1 * V)) : zero;
        x += step * it.x_sh;
      }
    }
    const bool norm = it.scale != nullptr;
    F2 ff[V / 2], fs[V / 2], sf[V / 2], ss[V / 2];  // f' = inv (ff f - fs s), s' = inv (sf f + ss s), two pairs each
    {
      float w0[V], w1[V], cs[V], sn[V];
      if (norm) {
        const T* sc = static_cast<const T*>(it.scale);
        Chunk<T>::unpack(has0 ? *reinterpret_cast<const uint4*>(sc + c0 * V) : zero, w0);
        Chunk<T>::unpack(has1 ? *reinterpret_cast<const uint4*>(sc + c1 * V) : zero, w1);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) w0[e] = w1[e] = 1.0f;
      }
      // cosines and sines of the V pairs: entries uV .. uV + V - 1 of the token's rows
      const uint4 tc = RING ? cos_next : zero, ts = RING ? sin_next : zero;
      if (RING) {
        cos_next = sin_next = zero;
        if (turn && row_next >= 0) load_tables(row_next, cos_next, sin_next);
        const bool bad = row_now < 0;
        row_now = row_next;
        row_next = row_of_group(gi + 2 * stride);
        Chunk<T>::unpack(tc, cs);
        Chunk<T>::unpack(ts, sn);
        if (!turn || bad) {
#pragma unroll
          for (int e = 0; e < V; ++e) cs[e] = turn ? __int_as_float(0x7fc00000) : 1.0f, sn[e] = turn ? cs[e] : 0.0f;
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) cs[e] = 1.0f, sn[e] = 0.0f;
        if (turn) {
          const int64_t row = table_row(p, w.token);
          uint4 c4 = zero, s4 = zero;
          if (row >= 0) load_tables(row, c4, s4);
          Chunk<T>::unpack(c4, cs);
          Chunk<T>::unpack(s4, sn);
          if (row < 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) cs[e] = sn[e] = __int_as_float(0x7fc00000);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float(&wv)[V] = 2 * e < V ? w0 : w1;  // INTER: pairs e, e + 1 are four neighbours of one piece
        const int at = (2 * e) % V;
        const F2 wf = INTER ? F2(wv[at], wv[at + 2]) : F2(w0[e], w0[e + 1]);
        const F2 ws = INTER ? F2(wv[at + 1], wv[at + 3]) : F2(w1[e], w1[e + 1]);
        const F2 c2(cs[e], cs[e + 1]), s2(sn[e], sn[e + 1]), m2(-sn[e], -sn[e + 1]);
        ff[e / 2] = mul2(wf, c2), fs[e / 2] = mul2(ws, m2), sf[e / 2] = mul2(wf, s2), ss[e / 2] = mul2(ws, c2);
      }
    }
    if constexpr (RING > 0) {
      cp_async_wait_group<RING - 2>();  // own copies of this group
      fetch(gi + (RING - 1) * stride, (slot + RING - 1) % RING);
    }
    T* y = static_cast<T*>(it.y) + w.b * it.y_sb + w.t * it.y_st + w.j * it.y_sh;
    const int64_t hop = step * it.y_sh;
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      if (w.j + i * step >= it.heads) break;
      if (RING) {
        const uint4* src = s_ring + slot * SLOTS * 256 + threadIdx.x;
        xv[0][0] = has0 ? src[(2 * i) * 256] : zero;
        xv[0][1] = has1 ? src[(2 * i + 1) * 256] : zero;
      }
      float a[V], c[V];
      Chunk<T>::unpack(xv[RING ? 0 : i][0], a);
      Chunk<T>::unpack(xv[RING ? 0 : i][1], c);
      F2 f[V / 2], s[V / 2];
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float(&x)[V] = 2 * e < V ? a : c;
        const int at = (2 * e) % V;
        f[e / 2] = INTER ? F2(x[at], x[at + 2]) : F2(a[e], a[e + 1]);
        s[e / 2] = INTER ? F2(x[at + 1], x[at + 3]) : F2(c[e], c[e + 1]);
      }
      float inv = 1.0f;
      if (norm) {
        F2 q0 = mul2(f[0], f[0]), q1 = mul2(s[0], s[0]);
#pragma unroll
        for (int e = 1; e < V / 2; ++e) q0 = fma2(f[e], f[e], q0), q1 = fma2(s[e], s[e], q1);
        float sum = (q0.lo() + q0.hi()) + (q1.lo() + q1.hi());
#pragma unroll
        for (int d = LPR / 2; d; d >>= 1) sum += __shfl_xor_sync(group_mask, sum, d, LPR);
        const float v = fmaf(sum, p.inv_d, it.eps);
        inv = inv_sqrt<T>(v);
        if (sizeof(T) == 4 && !squares_in_range(v)) {  // (the group's lanes share v)
          const float pre = norm_pre(v);
          const F2 pre2(pre, pre);
#pragma unroll
          for (int e = 0; e < V / 2; ++e) f[e] = mul2(f[e], pre2), s[e] = mul2(s[e], pre2);
          q0 = mul2(f[0], f[0]), q1 = mul2(s[0], s[0]);
#pragma unroll
          for (int e = 1; e < V / 2; ++e) q0 = fma2(f[e], f[e], q0), q1 = fma2(s[e], s[e], q1);
          sum = (q0.lo() + q0.hi()) + (q1.lo() + q1.hi());
#pragma unroll
          for (int d = LPR / 2; d; d >>= 1) sum += __shfl_xor_sync(group_mask, sum, d, LPR);
          inv = norm_inv_pre(sum * p.inv_d, it.eps, pre);
        }
      }
      const F2 inv2(inv, inv);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        F2 f1 = mul2(ff[e], f[e]), s1 = mul2(ss[e], s[e]);
        if (turn) {  // elements behind the rotation stay apart, whatever they hold
          f1 = fma2(fs[e], s[e], f1);
          s1 = fma2(sf[e], f[e], s1);
        }
        f1 = mul2(f1, inv2), s1 = mul2(s1, inv2);
        float(&x)[V] = 4 * e < V ? a : c;
        const int at = (4 * e) % V;
        (INTER ? x[at] : a[2 * e]) = f1.lo(), (INTER ? x[at + 2] : a[2 * e + 1]) = f1.hi();
        (INTER ? x[at + 1] : c[2 * e]) = s1.lo(), (INTER ? x[at + 3] : c[2 * e + 1]) = s1.hi();
      }
      if (has0) *reinterpret_cast<uint4*>(y + c0 * V) = Chunk<T>::pack(a);
      if (has1) *reinterpret_cast<uint4*>(y + c1 * V) = Chunk<T>::pack(c);
      y += hop;
    }
    if (RING) slot = slot + 1 == RING ? 0 : slot + 1;
  }
}

// Any head size, rotation width and alignment: a warp per head row, a pair of elements per lane and step.
template <typename T>
__global__ void __launch_bounds__(256) norm_rope_any_kernel(const __grid_constant__ RopeParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int64_t token = row / p.heads;
  if (token >= p.tokens) return;
  int h = (int)(row - token * p.heads);
  const bool second = h >= p.item[0].heads;
  const RopeItem& it = p.item[second ? 1 : 0];
  if (second) h -= p.item[0].heads;
  const int b = (int)(token / p.T), t = (int)(token - (int64_t)b * p.T);
  const T* x = static_cast<const T*>(it.x) + b * it.x_sb + t * it.x_st + h * it.x_sh;
  T* y = static_cast<T*>(it.y) + b * it.y_sb + t * it.y_st + h * it.y_sh;
  const T* sc = static_cast<const T*>(it.scale);
  float inv = 1.0f, pre = 1.0f;
  if (sc) {
    auto sum = [&]() {
      float ss = 0.0f;
      for (int e = lane; e < p.D; e += 32) {
        const float v = to_f32(x[e]) * pre;
        ss = fmaf(v, v, ss);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
      return ss;
    };
    const float v = fmaf(sum(), p.inv_d, it.eps);
    inv = inv_sqrt<T>(v);
    if (sizeof(T) == 4 && !squares_in_range(v)) {
      pre = norm_pre(v);
      inv = norm_inv_pre(sum() * p.inv_d, it.eps, pre);
    }
  }
  const int64_t at = table_row(p, token);
  const int half = p.rot / 2;
  const T* ct = static_cast<const T*>(p.cos) + at * half;
  const T* st = static_cast<const T*>(p.sin) + at * half;
  for (int i = lane; i < half; i += 32) {
    const int ea = p.interleaved ? 2 * i : i, eb = p.interleaved ? 2 * i + 1 : i + half;
    const float c = at >= 0 ? to_f32(ct[i]) : __int_as_float(0x7fc00000);
    const float s = at >= 0 ? to_f32(st[i]) : __int_as_float(0x7fc00000);
    const float va = to_f32(x[ea]) * pre * inv * (sc ? to_f32(sc[ea]) : 1.0f);
    const float vb = to_f32(x[eb]) * pre * inv * (sc ? to_f32(sc[eb]) : 1.0f);
    from_f32(va * c - vb * s, y[ea]);
    from_f32(va * s + vb * c, y[eb]);
  }
  for (int e = p.rot + lane; e < p.D; e += 32) from_f32(to_f32(x[e]) * pre * inv * (sc ? to_f32(sc[e]) : 1.0f), y[e]);
}

constexpr int NR_RING = 3;  // groups of four rows a lane holds at once in shared memory: 96 KB a CTA, two CTAs an SM

template <typename T, int LPR, int HPG, int RING>
static cudaError_t launch_vec_rows(RopeParams p, int num_sms, cudaStream_t stream) {
  for (int i = 0; i < 2; ++i) p.groups[i] = (p.item[i].heads + HPG - 1) / HPG;
  const int64_t groups = p.tokens * (p.groups[0] + p.groups[1]);
  int64_t blocks = (groups * LPR + 255) / 256;
  // (the ring runs past the last group by less than a grid's worth)
  if (groups > 0x7fff0000ll || blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  if (RING && blocks > 2 * num_sms) blocks = 2 * num_sms;
  auto kernel = p.interleaved ? norm_rope_kernel<T, LPR, HPG, RING, true> : norm_rope_kernel<T, LPR, HPG, RING, false>;
  const size_t smem = (size_t)RING * 2 * HPG * 256 * 16;
  if (RING) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(kernel, dim3((unsigned)blocks), dim3(256), smem, stream, p);
}

template <typename T, int LPR>
static cudaError_t launch_vec(const RopeParams& p, const LaunchCtx& ctx) {
  // One row per lane group at once, or, for more, four rows per group in lane groups that stay: 1024 / 3000 / 8192
  // tokens of 40 fp16 heads of 128 take 13.4 / 21.4 / 41.0 us so and 14.3 / 28.6 / 63.5 us with a row each, 512 tokens
  // 10.2 us both, 256 tokens 10.2 and 8.2 us.  An fp32 lane has half the pairs, whose matrices are what the four rows
  // share: 2048 / 4096 / 8192 tokens of 16 fp32 heads of 80 take 16.4 / 22.5 / 32.8 us and 15.2 / 22.5 / 38.9 us.
  return p.tokens * p.heads * LPR > (int64_t)ctx.num_sms * (sizeof(T) == 2 ? 1536 : 6144)
             ? launch_vec_rows<T, LPR, 4, NR_RING>(p, ctx.num_sms, ctx.stream)
             : launch_vec_rows<T, LPR, 1, 0>(p, ctx.num_sms, ctx.stream);
}

template <typename T>
static int launch_rope_t(const RopeParams& p, int items, const LaunchCtx& ctx, int* launches) {
  constexpr int V = Chunk<T>::N;
  const int nc = p.D / V;
  // whole pieces of every row, of its rotated halves and of the tables' rows
  bool vec = p.D % V == 0 && (p.rot / 2) % V == 0 && nc <= 64;
  uintptr_t bases = (uintptr_t)p.cos | (uintptr_t)p.sin;
  for (int i = 0; i < items; ++i) {
    const RopeItem& it = p.item[i];
    bases |= (uintptr_t)it.x | (uintptr_t)it.y | (uintptr_t)it.scale;
    vec = vec && (it.x_sb % V | it.x_st % V | it.x_sh % V | it.y_sb % V | it.y_st % V | it.y_sh % V) == 0;
  }
  if ((bases & (sizeof(T) - 1)) != 0 || ((uintptr_t)p.pos & 7u) != 0) return REFUSED_ALIGNMENT;
  vec = vec && (bases & 15u) == 0;
  cudaError_t e;
  if (vec) {
    const int pairs = (nc + 1) / 2;
    if (pairs <= 4) e = launch_vec<T, 4>(p, ctx);
    else if (pairs <= 8) e = launch_vec<T, 8>(p, ctx);
    else if (pairs <= 16) e = launch_vec<T, 16>(p, ctx);
    else e = launch_vec<T, 32>(p, ctx);
  } else {
    const int64_t blocks = (p.tokens * p.heads + 7) / 8;
    if (blocks > 0x7fffffff) return REFUSED_SIZE;
    e = launch_pdl(norm_rope_any_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, ctx.stream, p);
  }
  if (e == cudaErrorInvalidConfiguration) return REFUSED_SIZE;  // (launch_vec_rows)
  ++*launches;
  return e == cudaSuccess ? 0 : 4;
}

int launch_norm_rope(const PlanOp& op, void* const* ptrs, const OpState*, const LaunchCtx& ctx, int* launches) {
  RopeParams p{};
  auto ptr = [&](int i) -> void* { return op.t[i] >= 0 ? ptrs[op.t[i]] : nullptr; };
  p.cos = ptr(0);
  p.sin = ptr(1);
  p.pos = (const long long*)ptr(2);
  p.T = (int)op.ip[NR_T];
  p.tokens = eff_batch(ctx, op, op.ip[NR_B]) * p.T;
  p.D = (int)op.ip[NR_D];
  p.inv_d = 1.0f / (float)p.D;
  p.rot = (int)op.ip[NR_ROT];
  p.interleaved = (int)op.ip[NR_INTERLEAVED];
  p.positions = op.ip[NR_POSITIONS];
  p.err = ctx.d_error;
  const int items = (int)op.ip[NR_ITEMS];
  for (int i = 0; i < items; ++i) {
    RopeItem& it = p.item[i];
    const int64_t* s = &op.ip[i ? NR_H1 : NR_H0];
    it.x = ptr(3 + 3 * i);
    it.scale = ptr(4 + 3 * i);
    it.y = ptr(5 + 3 * i);
    it.heads = (int)s[0];
    it.x_sb = s[1], it.x_st = s[2], it.x_sh = s[3], it.y_sb = s[4], it.y_st = s[5], it.y_sh = s[6];
    it.eps = (float)op.fp[NRF_EPS0 + i];
    p.heads += it.heads;
  }
  if (p.tokens <= 0 || p.heads <= 0) return 0;
  return op.ip[NR_F32] ? launch_rope_t<float>(p, items, ctx, launches)
                       : launch_rope_t<__half>(p, items, ctx, launches);
}

// ------------------------------------------------------------------ RMSNormalization
// WARPS warps per row; VEC: 16-byte accesses (N a multiple of the piece, 16-byte bases).
template <typename T, int WARPS, bool VEC>
__global__ void __launch_bounds__(256) rms_norm_kernel(const T* __restrict__ x, const T* __restrict__ scale,
                                                       T* __restrict__ y, int64_t rows, int64_t n, float eps) {
  constexpr int V = VEC ? Chunk<T>::N : 1;
  __shared__ float s_sum[8];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x * (int64_t)(8 / WARPS) + (threadIdx.x >> 5) / WARPS;
  const int tid = threadIdx.x % (32 * WARPS);
  if (WARPS == 1 && row >= rows) return;  // a CTA per row has no rows past the end
  const T* xr = x + row * n;
  T* yr = y + row * n;
  float pre = 1.0f;
  auto sum = [&]() {
    float ss = 0.0f;
    for (int64_t e = (int64_t)tid * V; e < n; e += 32 * WARPS * V) {
      if (VEC) {
        float f[Chunk<T>::N];
        Chunk<T>::unpack(*reinterpret_cast<const uint4*>(xr + e), f);
#pragma unroll
        for (int i = 0; i < Chunk<T>::N; ++i) ss = fmaf(f[i] * pre, f[i] * pre, ss);
      } else {
        const float f = to_f32(xr[e]) * pre;
        ss = fmaf(f, f, ss);
      }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    if (WARPS > 1) {
      if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = ss;
      __syncthreads();
      ss = 0.0f;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) ss += s_sum[i];
    }
    return ss;
  };
  const float v = sum() / (float)n + eps;
  float inv = inv_sqrt<T>(v);
  if (sizeof(T) == 4 && !squares_in_range(v)) {  // (all of a row's threads)
    pre = norm_pre(v);
    if (WARPS > 1) __syncthreads();  // the first sum's parts have been read
    inv = norm_inv_pre(sum() / (float)n, eps, pre);
  }
  for (int64_t e = (int64_t)tid * V; e < n; e += 32 * WARPS * V) {
    if (VEC) {
      float f[Chunk<T>::N], w[Chunk<T>::N];
      Chunk<T>::unpack(*reinterpret_cast<const uint4*>(xr + e), f);
      Chunk<T>::unpack(*reinterpret_cast<const uint4*>(scale + e), w);
#pragma unroll
      for (int i = 0; i < Chunk<T>::N; ++i) f[i] = f[i] * pre * inv * w[i];
      *reinterpret_cast<uint4*>(yr + e) = Chunk<T>::pack(f);
    } else {
      from_f32(to_f32(xr[e]) * pre * inv * to_f32(scale[e]), yr[e]);
    }
  }
}

template <typename T>
static int launch_rms_t(const void* x, const void* scale, void* y, int64_t rows, int64_t n, float eps,
                        const LaunchCtx& ctx, int* launches) {
  if (((uintptr_t)x | (uintptr_t)scale | (uintptr_t)y) & (sizeof(T) - 1)) return REFUSED_ALIGNMENT;
  const bool vec = n % Chunk<T>::N == 0 && (((uintptr_t)x | (uintptr_t)scale | (uintptr_t)y) & 15u) == 0;
  const bool wide = n > 1024;
  const int64_t blocks = wide ? rows : (rows + 7) / 8;
  if (blocks > 0x7fffffff) return REFUSED_SIZE;
  auto kernel = wide ? (vec ? rms_norm_kernel<T, 8, true> : rms_norm_kernel<T, 8, false>)
                     : (vec ? rms_norm_kernel<T, 1, true> : rms_norm_kernel<T, 1, false>);
  cudaError_t e = launch_pdl(kernel, dim3((unsigned)blocks), dim3(256), 0, ctx.stream, (const T*)x, (const T*)scale,
                             (T*)y, rows, n, eps);
  ++*launches;
  return e == cudaSuccess ? 0 : 4;
}

int launch_rms_norm(const PlanOp& op, void* const* ptrs, const OpState*, const LaunchCtx& ctx, int* launches) {
  const int64_t rpb = op.ip[RN_ROWS_PER_BATCH];
  const int64_t rows = op.ip[IP_BATCHED] && ctx.batch > 0 ? ctx.batch * rpb : op.ip[RN_ROWS];
  if (rows <= 0) return 0;
  const void *x = ptrs[op.t[0]], *scale = ptrs[op.t[1]];
  void* y = ptrs[op.t[2]];
  return op.ip[RN_F32] ? launch_rms_t<float>(x, scale, y, rows, op.ip[RN_N], (float)op.fp[RNF_EPS], ctx, launches)
                       : launch_rms_t<__half>(x, scale, y, rows, op.ip[RN_N], (float)op.fp[RNF_EPS], ctx, launches);
}

}  // namespace emx
