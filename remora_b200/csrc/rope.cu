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
// error of 2^-25 of that, however far the position.
//
// Bound: HBM (each element read once and written once).  A block takes a few
// tokens at a time, puts their cosines and sines into shared memory (one
// sincos per pair and token, whatever the number of heads), and then moves
// whole heads in vectors of up to 8 pairs.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "runtime.cuh"

namespace rb {
namespace rope {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;     // pairs of a head: rot <= 256
constexpr int kMaxAxes = 8;
constexpr int kTileAngles = 2048;  // shared-memory pairs of one tile of tokens

struct Turns {
  uint64_t f[kMaxHalf];  // freq / (2 pi), fraction of a turn in 2^-64
  uint8_t axis[kMaxHalf];
};

// One tensor of heads: rows [token][head][D], strides in elements.  A token is
// b * S + s; a plain [token] stride has S = all tokens.
struct Heads {
  const void* in;
  void* out;
  int64_t in_b, in_s, in_h, out_b, out_s, out_h;
  int32_t H;
};

struct Args {
  Heads q, k, v;  // k and v: out is the cache, addressed by slot
  const int32_t* pos;
  int64_t ld_pos;
  const int32_t* slots;
  int64_t tokens, S;
  int64_t c_blk_k, c_tok_k, c_head_k, c_blk_v, c_tok_v, c_head_v;
  int32_t num_blocks, bs;
  int32_t D, half, n_axes;
  int32_t tile;         // tokens of a block's iteration
  int32_t rot_units;    // units of V pairs in a head
  int32_t units;        // those and the units of V plain elements behind them
  float k_scale, v_scale;
  float sign;
  Turns turns;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_fp8_e4m3 from_f(float v) {
  __nv_fp8_e4m3 r;
  r.__x = __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  return r;
}

// V elements in accesses of up to 16 bytes (V * sizeof(T) is a power of two;
// the host checked that every address is a multiple of it, up to 16).
template <typename T, int V>
struct Vec {
  static constexpr int kBytes = V * (int)sizeof(T);
  union U {
    T e[V];
    uint4 w16[kBytes >= 16 ? kBytes / 16 : 1];
    uint2 w8;
    uint32_t w4;
    uint16_t w2;
    uint8_t w1;
    __device__ U() {}
  };
  static __device__ __forceinline__ void load(const T* p, float (&x)[V]) {
    U u;
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) u.w16[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    } else if constexpr (kBytes == 8) {
      u.w8 = __ldcs(reinterpret_cast<const uint2*>(p));
    } else if constexpr (kBytes == 4) {
      u.w4 = __ldcs(reinterpret_cast<const uint32_t*>(p));
    } else {
      u.w2 = __ldcs(reinterpret_cast<const uint16_t*>(p));
    }
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = to_f<T>(u.e[i]);
  }
  static __device__ __forceinline__ void store(T* p, const float (&x)[V]) {
    U u;
#pragma unroll
    for (int i = 0; i < V; ++i) u.e[i] = from_f<T>(x[i]);
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = u.w16[i];
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(p) = u.w8;
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(p) = u.w4;
    } else if constexpr (kBytes == 2) {
      *reinterpret_cast<uint16_t*>(p) = u.w2;
    } else {
      *reinterpret_cast<uint8_t*>(p) = u.w1;
    }
  }
};

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

// The same division for every element: IEEE, so that a value next to a border
// of the 8-bit type falls as x / scale says.
template <typename C>
__device__ __forceinline__ float stored(float x, float scale) {
  if constexpr (sizeof(C) == 1) return __fdiv_rn(x, scale);
  return x;
}

template <typename T, typename C, int V, bool kInter>
__device__ __forceinline__ void turn_unit(const T* in, C* out, int half, int unit,
                                          const float2* cs, float scale) {
  float a[V], b[V], x[V], y[V];
  const int lo = kInter ? 2 * V * unit : V * unit;
  const int hi = kInter ? lo + V : half + lo;
  Vec<T, V>::load(in + lo, x);
  Vec<T, V>::load(in + hi, y);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    // interleaved: pairs are neighbours of the 2V elements x | y
    a[i] = kInter ? (2 * i < V ? x[2 * i < V ? 2 * i : 0] : y[2 * i < V ? 0 : 2 * i - V]) : x[i];
    b[i] = kInter ? (2 * i + 1 < V ? x[2 * i + 1 < V ? 2 * i + 1 : 0]
                                   : y[2 * i + 1 < V ? 0 : 2 * i + 1 - V])
                  : y[i];
  }
  float p[V], r[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 w = cs[V * unit + i];
    p[i] = stored<C>(a[i] * w.x - b[i] * w.y, scale);
    r[i] = stored<C>(a[i] * w.y + b[i] * w.x, scale);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (kInter) {
      if (2 * i < V) x[2 * i < V ? 2 * i : 0] = p[i];
      else y[2 * i < V ? 0 : 2 * i - V] = p[i];
      if (2 * i + 1 < V) x[2 * i + 1 < V ? 2 * i + 1 : 0] = r[i];
      else y[2 * i + 1 < V ? 0 : 2 * i + 1 - V] = r[i];
    } else {
      x[i] = p[i];
      y[i] = r[i];
    }
  }
  Vec<C, V>::store(out + lo, x);
  Vec<C, V>::store(out + hi, y);
}

template <typename T, typename C, int V>
__device__ __forceinline__ void copy_unit(const T* in, C* out, int at, float scale) {
  float x[V];
  Vec<T, V>::load(in + at, x);
  if constexpr (sizeof(C) == 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = stored<C>(x[i], scale);
  }
  Vec<C, V>::store(out + at, x);
}

template <typename T, typename C, int V, bool kInter, bool kAppend>
__global__ void __launch_bounds__(kThreads) k_rope(const __grid_constant__ Args a) {
  __shared__ float2 cs[kTileAngles];
  // a token's offsets: rope: its row in x and in out; append: its slot's rows in
  // the two caches, and whether it has a slot
  __shared__ int64_t first[kThreads], second[kThreads];
  __shared__ bool slot[kThreads];
  const int tid = threadIdx.x;
  const int plain = a.D / V;  // units of a head of v
  const int per_q = a.q.H * a.units;
  const int per_k = kAppend ? a.k.H * a.units : 0;
  const int per_tok = per_q + per_k + (kAppend ? a.v.H * plain : 0);
  for (int64_t t0 = (int64_t)blockIdx.x * a.tile; t0 < a.tokens;
       t0 += (int64_t)gridDim.x * a.tile) {
    const int n = (int)min((int64_t)a.tile, a.tokens - t0);
    __syncthreads();  // the tile before is read
    for (int i = tid; i < n * a.half; i += kThreads) {
      const int t = i / a.half, f = i - t * a.half;
      const int32_t pos = a.pos[a.turns.axis[f] * a.ld_pos + t0 + t];
      cs[i] = phase(pos, a.turns.f[f], a.sign);
    }
    if (kAppend && tid < n) {
      const int32_t s = a.slots[t0 + tid];
      const int32_t page = s / a.bs, off = s - page * a.bs;
      const bool there = s >= 0 && page < a.num_blocks;
      if (!there && s != -1) atomicExch(&g_device_error, 3);
      slot[tid] = there;
      first[tid] = page * a.c_blk_k + off * a.c_tok_k;
      second[tid] = page * a.c_blk_v + off * a.c_tok_v;
    } else if (!kAppend && tid < n) {
      const int64_t b = (t0 + tid) / a.S, s = t0 + tid - b * a.S;
      first[tid] = b * a.q.in_b + s * a.q.in_s;
      second[tid] = b * a.q.out_b + s * a.q.out_s;
    }
    __syncthreads();
    for (int i = tid; i < n * per_tok; i += kThreads) {
      const int t = i / per_tok;
      int u = i - t * per_tok;
      const int64_t tok = t0 + t;
      const float2* w = cs + t * a.half;
      if (u < per_q) {
        const int h = u / a.units;
        u -= h * a.units;
        const T* in = (const T*)a.q.in + (kAppend ? tok * a.q.in_s : first[t]) + h * a.q.in_h;
        T* out = (T*)a.q.out + (kAppend ? tok * a.q.out_s : second[t]) + h * a.q.out_h;
        if (u < a.rot_units) turn_unit<T, T, V, kInter>(in, out, a.half, u, w, 1.0f);
        else copy_unit<T, T, V>(in, out, 2 * a.half + (u - a.rot_units) * V, 1.0f);
      } else if (kAppend && slot[t]) {
        u -= per_q;
        if (u < per_k) {
          const int h = u / a.units;
          u -= h * a.units;
          const T* in = (const T*)a.k.in + tok * a.k.in_s + h * a.k.in_h;
          C* out = (C*)a.k.out + first[t] + h * a.c_head_k;
          if (u < a.rot_units) turn_unit<T, C, V, kInter>(in, out, a.half, u, w, a.k_scale);
          else copy_unit<T, C, V>(in, out, 2 * a.half + (u - a.rot_units) * V, a.k_scale);
        } else {
          u -= per_k;
          const int h = u / plain;
          u -= h * plain;
          const T* in = (const T*)a.v.in + tok * a.v.in_s + h * a.v.in_h;
          C* out = (C*)a.v.out + second[t] + h * a.c_head_v;
          copy_unit<T, C, V>(in, out, u * V, a.v_scale);
        }
      }
    }
  }
}

inline int dtype_bytes(int dt) {
  return dt == REMORA_B200_F32 ? 4 : dt == REMORA_B200_E4M3 ? 1 : 2;
}

// The widest V in {8, 4, 1} that keeps every vector access aligned: the pairs'
// halves, the plain tail, the strides and the bases.
struct Fit {
  int v = 8;
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

template <typename T, typename C, bool kAppend>
int launch(Args& a, int v, int interleaved, cudaStream_t st) {
  const int plain = a.D / v;
  a.rot_units = a.half / v;
  a.units = a.rot_units + (a.D - 2 * a.half) / v;
  const int64_t per_tok = (int64_t)a.q.H * a.units +
                          (kAppend ? (int64_t)a.k.H * a.units + (int64_t)a.v.H * plain : 0);
  // enough tokens for two units a thread, but no more than the angles' room
  int64_t tile = (2 * kThreads + per_tok - 1) / per_tok;
  tile = std::min<int64_t>({tile, kTileAngles / std::max(a.half, 8), kThreads});
  a.tile = (int)std::max<int64_t>(tile, 1);
  const int64_t tiles = (a.tokens + a.tile - 1) / a.tile;
  const int grid = (int)std::min<int64_t>(tiles, (int64_t)num_sms() * 8);
#define RB_ROPE(VV, I) k_rope<T, C, VV, I, kAppend><<<grid, kThreads, 0, st>>>(a)
  if (interleaved) {
    if (v == 8) RB_ROPE(8, true);
    else if (v == 4) RB_ROPE(4, true);
    else RB_ROPE(1, true);
  } else {
    if (v == 8) RB_ROPE(8, false);
    else if (v == 4) RB_ROPE(4, false);
    else RB_ROPE(1, false);
  }
#undef RB_ROPE
  RB_LAUNCH_CHECK();
  return REMORA_B200_OK;
}

// Checks and converts what both entry points share.
inline int angles(const char* who, Args& a, const int32_t* positions, int64_t ld_pos, int n_axes,
                  const double* freq, const int32_t* axis_of, int64_t rot, int64_t D,
                  int64_t tokens) {
  RB_CHECK_ARG(D >= 1 && D <= 1024, "%s: head_dim must be in [1, 1024], got %lld", who,
               (long long)D);
  RB_CHECK_ARG(rot >= 0 && rot % 2 == 0 && rot <= 2 * kMaxHalf && rot <= D,
               "%s: rot must be even, at most head_dim and at most %d, got %lld", who,
               2 * kMaxHalf, (long long)rot);
  RB_CHECK_ARG(n_axes >= 1 && n_axes <= kMaxAxes, "%s: n_axes must be in [1, %d], got %d", who,
               kMaxAxes, n_axes);
  RB_CHECK_ARG(tokens >= 0 && tokens <= (1ll << 40), "%s: bad number of tokens", who);
  RB_CHECK_ARG(rot == 0 || freq, "%s: freq is null", who);
  RB_CHECK_ARG(rot == 0 || tokens == 0 || positions, "%s: positions is null", who);
  RB_CHECK_ARG(n_axes == 1 || ld_pos >= tokens, "%s: ld_pos must be at least the tokens", who);
  a.half = (int)(rot / 2);
  a.D = (int)D;
  a.n_axes = n_axes;
  a.pos = positions;
  a.ld_pos = ld_pos;
  a.tokens = tokens;
  for (int i = 0; i < a.half; ++i) {
    RB_CHECK_ARG(std::isfinite(freq[i]), "%s: freq[%d] is not finite", who, i);
    const int ax = axis_of ? axis_of[i] : 0;
    RB_CHECK_ARG(ax >= 0 && ax < n_axes, "%s: axis_of[%d] = %d is not in [0, %d)", who, i, ax,
                 n_axes);
    long double t = (long double)freq[i] / 6.283185307179586476925286766559L;
    t -= floorl(t);
    const long double f = t * 18446744073709551616.0L;
    a.turns.f[i] = f >= 18446744073709551615.0L ? 0 : (uint64_t)f;
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
  RB_CHECK_ARG(B <= (1ll << 31) && S <= (1ll << 31), "rope: bad shape");
  Args a = {};
  int rc = angles("rope", a, p.positions, p.ld_pos, p.n_axes, p.freq, p.axis_of, p.rot, D, B * S);
  if (rc) return rc;
  if (B * S * H == 0) return REMORA_B200_OK;
  RB_CHECK_ARG(p.x && p.out, "rope: null pointer");
  a.S = S;
  a.q = Heads{p.x, p.out, p.x_b, p.x_s, p.x_h, p.out_b, p.out_s, p.out_h, (int32_t)H};
  a.sign = p.inverse ? -1.0f : 1.0f;
  const int e = dtype_bytes(p.dtype);
  Fit f;
  f.elems(a.half);
  f.elems(D);
  f.rows(p.x, e, B > 1 ? p.x_b : 0, p.x_s, p.x_h);
  f.rows(p.out, e, B > 1 ? p.out_b : 0, p.out_s, p.out_h);
  RB_CHECK_ARG(f.whole, "rope: a pointer is not aligned to its elements");
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
  RB_CHECK_ARG(std::isfinite(p.k_scale) && p.k_scale > 0 && std::isfinite(p.v_scale) && p.v_scale > 0,
               "rope_kv_append: the scales must be positive and finite");
  RB_CHECK_ARG(p.cache_dtype == REMORA_B200_E4M3 || (p.k_scale == 1.0f && p.v_scale == 1.0f),
               "rope_kv_append: the scales must be 1 unless the cache is E4M3");
  Args a = {};
  int rc = angles("rope_kv_append", a, p.positions, p.ld_pos, p.n_axes, p.freq, p.axis_of, p.rot, D, T);
  if (rc) return rc;
  if (T == 0) return REMORA_B200_OK;
  RB_CHECK_ARG((Hq == 0 || (p.q && p.q_out)) && p.k && p.v && p.slots && p.k_cache && p.v_cache,
               "rope_kv_append: null pointer");
  a.S = T;
  a.q = Heads{p.q, p.q_out, 0, p.q_t, p.q_h, 0, p.q_out_t, p.q_out_h, (int32_t)Hq};
  a.k = Heads{p.k, p.k_cache, 0, p.k_t, p.k_h, 0, 0, 0, (int32_t)Hkv};
  a.v = Heads{p.v, p.v_cache, 0, p.v_t, p.v_h, 0, 0, 0, (int32_t)Hkv};
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
  a.sign = 1.0f;
  const int c = dtype_bytes(p.cache_dtype);
  Fit f;
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
  RB_CHECK_ARG(f.whole, "rope_kv_append: a pointer is not aligned to its elements");
  cudaStream_t st = as_stream(stream);
  if (p.dtype == REMORA_B200_BF16)
    return p.cache_dtype == REMORA_B200_E4M3
               ? launch<__nv_bfloat16, __nv_fp8_e4m3, true>(a, f.v, p.interleaved, st)
               : launch<__nv_bfloat16, __nv_bfloat16, true>(a, f.v, p.interleaved, st);
  return p.cache_dtype == REMORA_B200_E4M3
             ? launch<__half, __nv_fp8_e4m3, true>(a, f.v, p.interleaved, st)
             : launch<__half, __half, true>(a, f.v, p.interleaved, st);
}
