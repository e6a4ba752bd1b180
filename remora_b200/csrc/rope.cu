// rope.cu -- rotary positions, on their own (forward and gradient) and fused
// with the append of keys and values to a paged cache.  The reference has no
// counterpart (README.md:12 lists attention as in progress); these sit before
// the attention entry points.
//
// Pair i of a head turns by the angle pos[axis(i)] * freq[i]:
//   a' = a cos - b sin,   b' = a sin + b cos
// and its gradient is the same with the angle negated (a rotation's transpose
// is its inverse).  Several position rows (time, height, width) are one: each
// frequency names the row it follows.
//
// The angle is never formed.  A frequency is kept as a fixed-point fraction of
// a turn, F = freq / (2 pi) * 2^64, so that pos * F modulo 2^64 is the phase in
// turns with the whole turns already gone: integer arithmetic, exact for every
// 32-bit position up to the 2^-64 rounding of F.  The nearest quarter turn
// comes off as an integer too, which leaves at most pi/4 for sincospif and an
// error of 2^-25 of that, however far the position (and whatever the frequency:
// below a turn per position it is a long double product, above by words).
//
// Bound: HBM (each element read once and written once).  A block takes a few
// tokens at a time, puts their cosines and sines into shared memory (one
// sincos per pair and token, whatever the number of heads), and then moves
// whole heads in vectors of up to 8 pairs, the loads issued before the angles.
//
// B200, device time: 268.6 MB of bf16 [4,4096,32,128] (heads first, three
// axes) 45.8 us = 5.86 TB/s, where a copy of the same bytes takes 42.6; 8192
// tokens of 32 + 2 x 8 heads into an e4m3 cache (184.7 MB) 36.6 us = 5.05
// TB/s.  What it took: a thread keeping its unit of the head and walking over
// heads (65 -> 51 us with the angles read without bank conflicts), one
// multiply-add per stride and paired conversions (-> 47), streaming stores.
// Blocks of 128 threads, 64 registers, 8 to an SM: 256 threads 50 us, 9 and 10
// blocks (spills) 56 and 61, 7 blocks 52, 3 units a thread in 6 blocks 54.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "runtime.cuh"

namespace rb {
namespace rope {

constexpr int kThreads = 128;
constexpr int kMaxHalf = 128;     // pairs of a head: rot <= 256
constexpr int kMaxAxes = 8;
constexpr int kTileAngles = 1024;  // pairs of one tile of tokens in shared memory
constexpr int kTileTokens = 128;
constexpr int64_t kNone = INT64_MIN;
constexpr int kUnits = 2;          // units a thread holds in registers

struct Turns {
  uint64_t f[kMaxHalf];  // freq / (2 pi), fraction of a turn in 2^-64
  uint8_t axis[kMaxHalf];
};

// One tensor of heads: rows [token][head][D], strides in elements (of tokens and
// heads in 32 bits, so that an address is one multiply-add each).  A token is
// b * S + s.
struct Heads {
  const void* in;
  void* out;
  int64_t in_b, out_b;
  int32_t in_s, in_h, out_s, out_h;
  int32_t H;
};

struct Args {
  Heads q, k, v;  // k and v: out is the cache, addressed by slot
  const int32_t* pos;
  int64_t ld_pos;
  const int32_t* slots;
  int64_t c_blk_k, c_tok_k, c_head_k, c_blk_v, c_tok_v, c_head_v;
  int32_t tokens, S;
  Divisor batch;      // S
  int32_t num_blocks, bs;
  int32_t D, half;
  int32_t tile;       // tokens of a block's iteration
  int32_t rot_units;  // units of V pairs in a head
  int32_t units;      // those and the units of 2V plain elements behind them
  int32_t pass;       // heads side by side: kThreads / units
  Divisor heads;      // of a token
  float k_scale, v_scale, k_inverse, v_inverse;
  float sign;
  Turns turns;
};

// Two neighbouring elements at a time (one for V = 1): the conversions of a pair are one
// instruction each way.
__device__ __forceinline__ float2 widen2(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 widen2(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t narrow2(float x, float y, __nv_bfloat16) {
  return pack_bf16x2(x, y);
}
__device__ __forceinline__ uint32_t narrow2(float x, float y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint16_t narrow2(float x, float y, __nv_fp8_e4m3) {
  return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
}

// V elements in accesses of up to 16 bytes (V * sizeof(T) is a power of two;
// the host checked that every address is a multiple of it, up to 16).
template <typename T, int V>
struct Raw {
  static constexpr int kBytes = V * (int)sizeof(T);
  static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {  // read once: not kept in the caches
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = v.x;
        w[4 * i + 1] = v.y;
        w[4 * i + 2] = v.z;
        w[4 * i + 3] = v.w;
      }
    } else if constexpr (kBytes == 8) {
      const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
      w[0] = v.x;
      w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
    } else {
      w[0] = __ldcs(reinterpret_cast<const uint16_t*>(p));
    }
  }
  // Streaming stores: first to leave L2 when room is short (46.8 -> 45.6 us for 268 MB), and
  // still there for the next kernel when it is not.
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        __stcs(reinterpret_cast<uint4*>(p) + i,
               make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
    } else if constexpr (kBytes == 8) {
      __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(p) = w[0];
    } else if constexpr (kBytes == 2) {
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
    } else {
      *reinterpret_cast<uint8_t*>(p) = (uint8_t)w[0];
    }
  }
  __device__ __forceinline__ void widen(float (&x)[V]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < (V + 1) / 2; ++i) {
        const float2 f = widen2(w[i], T());
        x[2 * i] = f.x;
        if constexpr (V > 1) x[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void narrow(const float (&x)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(x[i]);
    } else if constexpr (V == 1) {
      w[0] = narrow2(x[0], 0.0f, T());
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) w[i] = narrow2(x[2 * i], x[2 * i + 1], T());
    } else {
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        w[i] = narrow2(x[4 * i], x[4 * i + 1], T()) |
               (uint32_t)narrow2(x[4 * i + 2], x[4 * i + 3], T()) << 16;
    }
  }
};
template <typename T, int V>
__device__ __forceinline__ void store_raw(T* p, const float (&x)[V]) {
  Raw<T, V> r;
  r.narrow(x);
  r.store(p);
}

// cos and sin of pos turns of F, with the sine's sign.
__device__ __forceinline__ float2 phase(int32_t pos, uint64_t F, float sign) {
  const uint64_t turn = (uint64_t)(int64_t)pos * F;
  const uint32_t hi = (uint32_t)((turn + 0x80000000ull) >> 32);
  const uint32_t quarter = (hi + 0x20000000u) >> 30;
  const int32_t rest = (int32_t)(hi - (quarter << 30));  // [-2^29, 2^29): an eighth of a turn
  float s, c;
  sincospif((float)rest * 4.656612873077393e-10f, &s, &c);  // 2^-31: half turns
  float cs = quarter & 1 ? -s : c, sn = quarter & 1 ? c : s;
  if (quarter & 2) { cs = -cs; sn = -sn; }
  return make_float2(cs, sn * sign);
}

// x / scale, rounded to nearest, from the rounded inverse of scale: a residual in one fused
// step corrects the product (Markstein, "Computation of elementary functions on the IBM RISC
// System/6000 processor", 1990).  So a value next to a border of the 8-bit type falls as the
// division says.  Beyond 512 the 8-bit type is saturated and the plain product does (the
// residual of an infinite one would be NaN).
__device__ __forceinline__ float divided(float x, float scale, float inverse) {
  const float q = x * inverse;
  const float r = fmaf(fmaf(-q, scale, x), inverse, q);
  return fabsf(q) < 512.0f ? r : q;
}

// What a thread holds of one head: two vectors of V elements, at lo and hi: V pairs to turn,
// or up to 2V elements to copy.
template <typename T, int V>
struct Unit {
  Raw<T, V> x, y;
  T* out;     // q: where its head goes
  int32_t t;  // token of the tile, -1: none
  int32_t h;  // head: q's, then k's, then v's
};

// Every head, of q, k or v, is cut into the same units, so a thread keeps its unit (lo, hi and
// the pairs in between) and walks over heads; 128 / units heads go side by side.
template <typename T, typename C, int V, bool kInter, bool kAppend>
__global__ void __launch_bounds__(kThreads, 8) k_rope(const __grid_constant__ Args a) {
  __shared__ __align__(16) float2 cs[2][kTileAngles];
  // append: a token's rows in the two caches, or kNone
  __shared__ int64_t krow[2][kAppend ? kTileTokens : 1], vrow[2][kAppend ? kTileTokens : 1];
  const int tid = threadIdx.x;
  const int mine = tid / a.units, unit = tid - mine * a.units;  // head of the pass, unit
  const int lo = unit < a.rot_units ? (kInter ? 2 * V * unit : V * unit)
                                    : 2 * a.half + 2 * V * (unit - a.rot_units);
  const int hi = unit < a.rot_units && !kInter ? a.half + lo : lo + V;
  const bool turns_ = unit < a.rot_units, two = hi < a.D, any = mine < a.pass;
  // through a pointer that the compiler cannot see into: the lanes read different frequencies,
  // which the constant cache would serve one at a time
  const Turns* turns = &a.turns;
  asm volatile("" : "+l"(turns));
  Unit<T, V> u[kUnits];

  auto load = [&](Unit<T, V>& w, int t0, int all, int r0) {
    const int row = r0 + mine;
    w.t = -1;
    if (!any || row >= all) return;
    w.t = a.heads.div(row);
    w.h = row - w.t * (int)a.heads.d;
    const int tok = t0 + w.t;
    const T* in;
    if (!kAppend || w.h < a.q.H) {
      in = (const T*)a.q.in + (int64_t)w.h * a.q.in_h;
      w.out = (T*)a.q.out + (int64_t)w.h * a.q.out_h;
      if (kAppend || a.S == a.tokens) {
        in += (int64_t)tok * a.q.in_s;
        w.out += (int64_t)tok * a.q.out_s;
      } else {
        const int b = a.batch.div(tok), s = tok - b * a.S;
        in += b * a.q.in_b + (int64_t)s * a.q.in_s;
        w.out += b * a.q.out_b + (int64_t)s * a.q.out_s;
      }
    } else {
      const int h = w.h - a.q.H;
      in = h < a.k.H
               ? (const T*)a.k.in + (int64_t)tok * a.k.in_s + (int64_t)h * a.k.in_h
               : (const T*)a.v.in + (int64_t)tok * a.v.in_s + (int64_t)(h - a.k.H) * a.v.in_h;
    }
    w.x.load(in + lo);
    if (two) w.y.load(in + hi);
  };
  auto finish = [&](const Unit<T, V>& w, int buf) {
    if (w.t < 0) return;
    float x[V], y[V];
    w.x.widen(x);
    w.y.widen(y);
    if (turns_ && (!kAppend || w.h < a.q.H + a.k.H)) {
      float2 turn[V];
      if constexpr (V == 1) {
        turn[0] = cs[buf][w.t * a.half + unit];
      } else {
        // pairs 2j and 2j+1 of a unit lie together, those of all units after one another: the
        // lanes of a warp read neighbouring 16 bytes
        const float4* p =
            reinterpret_cast<const float4*>(cs[buf]) + w.t * (V / 2) * a.rot_units + unit;
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
          const float4 r = p[j * a.rot_units];
          turn[2 * j] = make_float2(r.x, r.y);
          turn[(2 * j + 1) % V] = make_float2(r.z, r.w);
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 r = turn[i];
        // interleaved: the pairs are neighbours of the 2V elements x | y
        float& p = kInter ? (2 * i < V ? x[2 * i % V] : y[2 * i % V]) : x[i];
        float& q = kInter ? (2 * i + 1 < V ? x[(2 * i + 1) % V] : y[(2 * i + 1) % V]) : y[i];
        const float b = p;
        p = b * r.x - q * r.y;
        q = b * r.y + q * r.x;
      }
    }
    if (!kAppend || w.h < a.q.H) {
      store_raw<T, V>(w.out + lo, x);
      if (two) store_raw<T, V>(w.out + hi, y);
      return;
    }
    const bool is_v = w.h >= a.q.H + a.k.H;
    const int64_t row = is_v ? vrow[buf][w.t] : krow[buf][w.t];
    if (row == kNone) return;
    if constexpr (sizeof(C) == 1) {
      const float scale = is_v ? a.v_scale : a.k_scale;
      const float inverse = is_v ? a.v_inverse : a.k_inverse;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[i] = divided(x[i], scale, inverse);
        y[i] = divided(y[i], scale, inverse);
      }
    }
    C* out = is_v ? (C*)a.v.out + row + (w.h - a.q.H - a.k.H) * a.c_head_v
                  : (C*)a.k.out + row + (w.h - a.q.H) * a.c_head_k;
    store_raw<C, V>(out + lo, x);
    if (two) store_raw<C, V>(out + hi, y);
  };

  int buf = 0;
  const int step = gridDim.x * a.tile;
  for (int t0 = blockIdx.x * a.tile; t0 < a.tokens; t0 += step, buf ^= 1) {
    const int n = min(a.tile, a.tokens - t0), all = n * (int)a.heads.d;
#pragma unroll
    for (int e = 0; e < kUnits; ++e) load(u[e], t0, all, e * a.pass);
    // the angles, while the loads are under way
    for (int i = tid; i < n * a.half; i += kThreads) {
      const int t = i / a.half, f = i - t * a.half;
      const float2 r = phase(a.pos[turns->axis[f] * a.ld_pos + t0 + t], turns->f[f], a.sign);
      const int k = f / V, in = f % V;
      cs[buf][V == 1 ? i : 2 * ((t * (V / 2) + in / 2) * a.rot_units + k) + in % 2] = r;
    }
    if (kAppend && tid < n) {
      const int32_t s = a.slots[t0 + tid];
      const int32_t page = s / a.bs, off = s - page * a.bs;
      const bool in = s >= 0 && page < a.num_blocks;
      if (!in && s != -1) atomicExch(&g_device_error, 3);
      krow[buf][tid] = in ? page * a.c_blk_k + off * a.c_tok_k : kNone;
      vrow[buf][tid] = in ? page * a.c_blk_v + off * a.c_tok_v : kNone;
    }
    // one barrier a tile: its buffers are written again two tiles on, behind the next barrier
    __syncthreads();
    for (int r0 = 0;;) {
#pragma unroll
      for (int e = 0; e < kUnits; ++e) finish(u[e], buf);
      r0 += kUnits * a.pass;
      if (r0 >= all) break;
#pragma unroll
      for (int e = 0; e < kUnits; ++e) load(u[e], t0, all, r0 + e * a.pass);
    }
  }
}

inline bool fits32(int64_t stride) { return stride < (1ll << 31) && stride > -(1ll << 31); }
inline bool scale_ok(float s) { return s >= 1e-30f && s <= 1e30f; }

inline int dtype_bytes(int dt) {
  return dt == REMORA_B200_F32 ? 4 : dt == REMORA_B200_E4M3 ? 1 : 2;
}

// The widest V in {8 (16-bit types only), 4, 1} that keeps every vector access
// aligned: the pairs' halves, the plain tail, the strides and the bases.  bf16
// [4,4096,32,128]: 44 us at 8, 59 at 4, 157 at 1.
struct Fit {
  int v;
  explicit Fit(int bytes) : v(bytes == 2 ? 8 : 4) {}
  void elems(int64_t n) { while (v > 1 && n % v) v = v == 8 ? 4 : 1; }
  void base(const void* p, int bytes) {
    while (v > 1 && reinterpret_cast<uintptr_t>(p) % (v * bytes < 16 ? v * bytes : 16))
      v = v == 8 ? 4 : 1;
  }
  bool whole = true;  // every base at a multiple of its elements' size
  void rows(const void* p, int bytes, int64_t s0, int64_t s1, int64_t s2) {
    whole = whole && reinterpret_cast<uintptr_t>(p) % bytes == 0;
    elems(s0);
    elems(s1);
    elems(s2);
    base(p, bytes);
  }
};

// How a launch is cut, for heads of D elements of which 2 * half turn, v pairs at a time: units of
// a head (at most kThreads, which the caller checks), heads side by side, tokens of a tile, blocks.
struct Tiling {
  int units, pass, tile, grid;
};
inline Tiling tiling(int D, int half, int v, int heads, int64_t tokens) {
  Tiling t;
  t.units = (D / v + 1) / 2;  // half / v, and ceil of half the rest
  t.pass = std::max(kThreads / t.units, 1);
  // The tokens whose heads fill a block's units once, within the angles' room, and no more than
  // leave every SM a tile.  (Several rounds of units per tile measured slower: 8 tokens of 32 heads
  // 55 us against 47, 8 of 48 into e4m3 39.4 against 37.5; one token of 12 heads 5.9 against 5.6.)
  const int64_t room = std::min<int64_t>(kTileAngles / std::max(half, 1), kTileTokens);
  const int64_t most = std::min<int64_t>(room, tokens / num_sms());
  t.tile = (int)std::max<int64_t>(std::min<int64_t>(most, kUnits * t.pass / heads), 1);
  t.grid = (int)std::min<int64_t>((tokens + t.tile - 1) / t.tile, (int64_t)num_sms() * 16);
  return t;
}

template <typename T, typename C, bool kAppend>
int launch(Args& a, int v, int interleaved, cudaStream_t st) {
  const int heads = a.q.H + (kAppend ? a.k.H + a.v.H : 0);
  const Tiling t = tiling(a.D, a.half, v, heads, a.tokens);
  RB_CHECK_ARG(t.units <= kThreads,
               "rope: head_dim above %d needs sizes, strides and bases of whole 4 elements",
               2 * kThreads);
  a.rot_units = a.half / v;
  a.units = t.units;
  a.pass = t.pass;
  a.tile = t.tile;
  a.heads = Divisor((uint32_t)heads);
  const int grid = t.grid;
#define RB_ROPE(VV, I) k_rope<T, C, VV, I, kAppend><<<grid, kThreads, 0, st>>>(a)
#define RB_ROPE_V(I)                          \
  do {                                        \
    if constexpr (sizeof(T) == 2) {           \
      if (v == 8) RB_ROPE(8, I);              \
    }                                         \
    if (v == 4) RB_ROPE(4, I);                \
    else if (v == 1) RB_ROPE(1, I);           \
  } while (0)
  if (interleaved) RB_ROPE_V(true);
  else RB_ROPE_V(false);
#undef RB_ROPE_V
#undef RB_ROPE
  RB_LAUNCH_CHECK();
  return REMORA_B200_OK;
}

// freq / (2 pi) modulo one turn, in 2^-64 of a turn, for 1 <= |freq| < 2^64: the mantissa times
// floor(2^192 / (2 pi)) by words, of which the 64 bits behind the point are taken.  What the
// constant lacks is below 2^-128 turns; a product in long double would lose the bits behind the
// point to those in front of it.
inline uint64_t turns_of(double freq) {
  constexpr uint64_t c[3] = {0x36d8a5664f10e410ull, 0x7f09d5f47d4d3770ull, 0x28be60db9391054aull};
  int e;
  const uint64_t m = (uint64_t)std::ldexp(std::frexp(std::fabs(freq), &e), 53);
  uint64_t p[4];  // m * 2^192 / (2 pi)
  unsigned __int128 carry = 0;
  for (int i = 0; i < 3; ++i) {
    carry += (unsigned __int128)m * c[i];
    p[i] = (uint64_t)carry;
    carry >>= 64;
  }
  p[3] = (uint64_t)carry;
  const int down = 128 - (e - 53), word = down / 64, bit = down % 64;  // down in [117, 180]
  const uint64_t f = p[word] >> bit | (bit ? p[word + 1] << (64 - bit) : 0);
  return freq < 0 ? 0 - f : f;
}

// Checks and converts what both entry points share.
inline int angles(const char* who, Args& a, const int32_t* positions, int64_t ld_pos, int n_axes,
                  const double* freq, const int32_t* axis_of, int64_t rot, int64_t D,
                  int64_t tokens) {
  RB_CHECK_ARG(D >= 1 && D <= 512, "%s: head_dim must be in [1, 512], got %lld", who,
               (long long)D);
  RB_CHECK_ARG(rot >= 0 && rot % 2 == 0 && rot <= 2 * kMaxHalf && rot <= D,
               "%s: rot must be even, at most head_dim and at most %d, got %lld", who,
               2 * kMaxHalf, (long long)rot);
  RB_CHECK_ARG(n_axes >= 1 && n_axes <= kMaxAxes, "%s: n_axes must be in [1, %d], got %d", who,
               kMaxAxes, n_axes);
  RB_CHECK_ARG(tokens >= 0 && tokens <= (1ll << 30), "%s: at most 2^30 tokens, got %lld", who,
               (long long)tokens);
  RB_CHECK_ARG(rot == 0 || freq, "%s: freq is null", who);
  RB_CHECK_ARG(rot == 0 || tokens == 0 || positions, "%s: positions is null", who);
  RB_CHECK_ARG(n_axes == 1 || ld_pos >= tokens, "%s: ld_pos must be at least the tokens", who);
  a.half = (int)(rot / 2);
  a.D = (int)D;
  a.pos = positions;
  a.ld_pos = ld_pos;
  a.tokens = (int32_t)tokens;
  for (int i = 0; i < a.half; ++i) {
    RB_CHECK_ARG(std::fabs(freq[i]) < 18446744073709551616.0,
                 "%s: freq[%d] is not finite or not below 2^64", who, i);
    const int ax = axis_of ? axis_of[i] : 0;
    RB_CHECK_ARG(ax >= 0 && ax < n_axes, "%s: axis_of[%d] = %d is not in [0, %d)", who, i, ax,
                 n_axes);
    const long double t = (long double)freq[i] * 0.159154943091895335768883763373L;  // / (2 pi)
    if (t <= -1 || t >= 1) {
      a.turns.f[i] = turns_of(freq[i]);
    } else {
      const long double f = (t < 0 ? t + 1 : t) * 18446744073709551616.0L;
      a.turns.f[i] = f >= 18446744073709551615.0L ? 0 : (uint64_t)f;
    }
    a.turns.axis[i] = (uint8_t)ax;
  }
  return REMORA_B200_OK;
}

}  // namespace rope
}  // namespace rb

extern "C" int remora_b200_rope(const remora_b200_rope_args* args, void* stream) {
  using namespace rb;
  using namespace rb::rope;
  clear_error();
  RB_CHECK_ARG(args, "rope: args is null");
  const remora_b200_rope_args& p = *args;
  const int64_t B = p.B, S = p.S, H = p.H, D = p.D;
  RB_CHECK_ARG(p.dtype == REMORA_B200_BF16 || p.dtype == REMORA_B200_F16 || p.dtype == REMORA_B200_F32,
               "rope: dtype must be BF16, F16 or F32");
  RB_CHECK_ARG(B >= 0 && S >= 0 && H >= 0 && H <= 65536, "rope: bad shape");
  RB_CHECK_ARG(B <= (1ll << 30) && S <= (1ll << 30), "rope: bad shape");
  Args a = {};
  int rc = angles("rope", a, p.positions, p.ld_pos, p.n_axes, p.freq, p.axis_of, p.rot, D, B * S);
  if (rc) return rc;
  if (B * S * H == 0) return REMORA_B200_OK;
  RB_CHECK_ARG(p.x && p.out, "rope: null pointer");
  RB_CHECK_ARG(fits32(p.x_s) && fits32(p.x_h) && fits32(p.out_s) && fits32(p.out_h),
               "rope: strides of tokens and heads must be below 2^31 elements");
  RB_CHECK_ARG(!rows_overlap(B, p.out_b, D) && !rows_overlap(S, p.out_s, D) &&
                   !rows_overlap(H, p.out_h, D),
               "rope: the rows of out overlap");
  a.S = (int32_t)S;
  a.batch = Divisor((uint32_t)S);
  a.q = Heads{p.x, p.out, p.x_b, p.out_b, (int32_t)p.x_s, (int32_t)p.x_h, (int32_t)p.out_s,
              (int32_t)p.out_h, (int32_t)H};
  a.sign = p.inverse ? -1.0f : 1.0f;
  const int e = dtype_bytes(p.dtype);
  Fit f(e);
  f.elems(a.half);
  f.elems(D);
  f.rows(p.x, e, B > 1 ? p.x_b : 0, p.x_s, p.x_h);
  f.rows(p.out, e, B > 1 ? p.out_b : 0, p.out_s, p.out_h);
  RB_CHECK_ARG(f.whole && aligned4(p.positions), "rope: a pointer is not aligned to its elements");
  cudaStream_t st = as_stream(stream);
  if (p.dtype == REMORA_B200_BF16)
    return launch<__nv_bfloat16, __nv_bfloat16, false>(a, f.v, p.interleaved, st);
  if (p.dtype == REMORA_B200_F16) return launch<__half, __half, false>(a, f.v, p.interleaved, st);
  return launch<float, float, false>(a, f.v, p.interleaved, st);
}

extern "C" int remora_b200_rope_kv_append(const remora_b200_rope_kv_append_args* args,
                                          void* stream) {
  using namespace rb;
  using namespace rb::rope;
  clear_error();
  RB_CHECK_ARG(args, "rope_kv_append: args is null");
  const remora_b200_rope_kv_append_args& p = *args;
  const int64_t T = p.T, Hq = p.Hq, Hkv = p.Hkv, D = p.D;
  RB_CHECK_ARG(p.dtype == REMORA_B200_BF16 || p.dtype == REMORA_B200_F16,
               "rope_kv_append: dtype must be BF16 or F16");
  RB_CHECK_ARG(p.cache_dtype == p.dtype || p.cache_dtype == REMORA_B200_E4M3,
               "rope_kv_append: cache_dtype must be dtype or E4M3");
  RB_CHECK_ARG(T >= 0 && Hq >= 0 && Hkv >= 1 && Hq <= 65536 && Hkv <= 65536,
               "rope_kv_append: bad shape");
  RB_CHECK_ARG(p.block_size >= 1 && p.num_blocks >= 1 && p.block_size <= 0x7fffffff &&
                   p.num_blocks <= 0x7fffffff / p.block_size,
               "rope_kv_append: num_blocks * block_size must be in [1, 2^31)");
  RB_CHECK_ARG(scale_ok(p.k_scale) && scale_ok(p.v_scale),
               "rope_kv_append: the scales must lie in [1e-30, 1e30]");
  RB_CHECK_ARG(p.cache_dtype == REMORA_B200_E4M3 || (p.k_scale == 1.0f && p.v_scale == 1.0f),
               "rope_kv_append: the scales must be 1 unless the cache is E4M3");
  Args a = {};
  int rc = angles("rope_kv_append", a, p.positions, p.ld_pos, p.n_axes, p.freq, p.axis_of, p.rot, D, T);
  if (rc) return rc;
  if (T == 0) return REMORA_B200_OK;
  RB_CHECK_ARG((Hq == 0 || (p.q && p.q_out)) && p.k && p.v && p.slots && p.k_cache && p.v_cache,
               "rope_kv_append: null pointer");
  RB_CHECK_ARG(fits32(p.q_t) && fits32(p.q_h) && fits32(p.k_t) && fits32(p.k_h) &&
                   fits32(p.v_t) && fits32(p.v_h) && fits32(p.q_out_t) && fits32(p.q_out_h),
               "rope_kv_append: strides of tokens and heads must be below 2^31 elements");
  RB_CHECK_ARG(Hq == 0 || (!rows_overlap(T, p.q_out_t, D) && !rows_overlap(Hq, p.q_out_h, D)),
               "rope_kv_append: the rows of q_out overlap");
  RB_CHECK_ARG(!rows_overlap(p.num_blocks, p.kc_block, D) &&
                   !rows_overlap(p.block_size, p.kc_token, D) &&
                   !rows_overlap(Hkv, p.kc_head, D) && !rows_overlap(p.num_blocks, p.vc_block, D) &&
                   !rows_overlap(p.block_size, p.vc_token, D) && !rows_overlap(Hkv, p.vc_head, D),
               "rope_kv_append: the rows of a cache overlap");
  a.S = (int32_t)T;
  a.q = Heads{p.q, p.q_out, 0, 0, (int32_t)p.q_t, (int32_t)p.q_h, (int32_t)p.q_out_t,
              (int32_t)p.q_out_h, (int32_t)Hq};
  a.k = Heads{p.k, p.k_cache, 0, 0, (int32_t)p.k_t, (int32_t)p.k_h, 0, 0, (int32_t)Hkv};
  a.v = Heads{p.v, p.v_cache, 0, 0, (int32_t)p.v_t, (int32_t)p.v_h, 0, 0, (int32_t)Hkv};
  a.slots = p.slots;
  a.num_blocks = (int32_t)p.num_blocks;
  a.bs = (int32_t)p.block_size;
  a.c_blk_k = p.kc_block;
  a.c_tok_k = p.kc_token;
  a.c_head_k = p.kc_head;
  a.c_blk_v = p.vc_block;
  a.c_tok_v = p.vc_token;
  a.c_head_v = p.vc_head;
  a.k_scale = p.k_scale;
  a.v_scale = p.v_scale;
  a.k_inverse = 1.0f / p.k_scale;
  a.v_inverse = 1.0f / p.v_scale;
  a.sign = 1.0f;
  const int c = dtype_bytes(p.cache_dtype);
  Fit f(2);
  f.elems(a.half);
  f.elems(D);
  if (Hq) {
    f.rows(p.q, 2, p.q_t, p.q_h, 0);
    f.rows(p.q_out, 2, p.q_out_t, p.q_out_h, 0);
  }
  f.rows(p.k, 2, p.k_t, p.k_h, 0);
  f.rows(p.v, 2, p.v_t, p.v_h, 0);
  f.rows(p.k_cache, c, p.kc_block, p.kc_token, p.kc_head);
  f.rows(p.v_cache, c, p.vc_block, p.vc_token, p.vc_head);
  RB_CHECK_ARG(f.whole && aligned4(p.positions, p.slots),
               "rope_kv_append: a pointer is not aligned to its elements");
  cudaStream_t st = as_stream(stream);
  if (p.dtype == REMORA_B200_BF16)
    return p.cache_dtype == REMORA_B200_E4M3
               ? launch<__nv_bfloat16, __nv_fp8_e4m3, true>(a, f.v, p.interleaved, st)
               : launch<__nv_bfloat16, __nv_bfloat16, true>(a, f.v, p.interleaved, st);
  return p.cache_dtype == REMORA_B200_E4M3
             ? launch<__half, __nv_fp8_e4m3, true>(a, f.v, p.interleaved, st)
             : launch<__half, __half, true>(a, f.v, p.interleaved, st);
}
