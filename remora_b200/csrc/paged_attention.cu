// paged_attention.cu -- attention of one new token per request over a paged
// key-value cache (no counterpart in the reference, which lists attention as
// in progress, README.md:12; it stands beside the prefill form).
//
// For request r, query head h and the keys j of r:
//   s_j = scale q . k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),
// over the keys in parts, each with its own m, l = sum exp(s_j - m) and
// unnormalised o; parts join by weights exp(m_part - max m).
//
// Bound: HBM.  Each key and value is read once for the Hq / Hkv query heads
// that share it (at 4 heads of bf16, 4 flop a byte), so what matters is that
// every SM has enough copies in flight all the time, whatever the lengths:
//   - The lengths are on the device, so the split is made there.  All requests'
//     tiles (16 or 32 keys of one kv head) form one line; every warp takes the
//     same length of it, counting kItemCost tiles for each item that it starts
//     (128 requests of 8 to 16001 keys: 62.7 us without that cost, 51.0 with).
//     A warp walks its tiles alone, through items and requests, with no barrier
//     to the others.
//   - Tiles come by cp.async into a ring per warp, 128 KB in flight per SM (12
//     warps: 96, or 144 in tiles of 4 KB): the rows of a page are short (64 to
//     512 bytes) and lie where the block table says, so a copy is 16 bytes per
//     lane with one address per 16 keys, the table entry fetched a tile ahead.
//   - Products by mma.sync: one new token is 1 to 16 rows, far too few for a
//     128-row tile in tensor memory, and for up to 8 heads per kv head 15 to
//     27 % of this pipe is enough.  Scores have the keys as rows and the heads
//     as columns, so that no half of the instruction idles; the weights turn by
//     movmatrix into the second product's operand.  8-bit values become f16 in
//     registers, exactly.
//   - What crosses a warp's end joins in shared memory when the CTA is done,
//     what crosses a CTA's end in the second launch, at most two parts a CTA.
//     No atomics: the same inputs give the same bits.
//
// B200 (device time; the copy rate is 6462 GB/s): 64 requests of 7900 to 8190
// keys, 8 kv heads of 128 bf16 elements, 2.11 GB: 321 to 338 us, 6.2 to 6.6
// TB/s.  3 requests of 90 to 131 thousand keys over e4m3, 675 MB: 119 to 130 us
// (the SM clock under power decides).  128 ragged requests, 272 MB: 51 us, of
// which 7 are before the first and after the last tile.  700 keys: 9.2 us, two
// launches of cold code.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "runtime.cuh"

namespace rb {
namespace paged {

constexpr int kMaxRequests = 8192;
constexpr int kRingBytes = 196608;  // shared memory of a CTA's rings
// What starting and ending an item costs a warp, in tiles.  128 ragged requests: 62.7 us at 0,
// 51.0 at 2, 51.4 at 4.  A warp's share has no lower bound: 700 keys take 9.0 us at one share and
// 10.1, 12.3 and 14.7 us where a warp takes at least 2, 4 and 6.
constexpr int kItemCost = 2;
constexpr int kMostWarps = 12;

struct Args {
  const void *q, *kc, *vc;
  const int32_t *table, *lens;
  void* out;
  float* lse;
  int64_t q_t, q_h, o_t, o_h;
  int64_t kc_b, kc_t, kc_h, vc_b, vc_t, vc_h;
  int64_t ld_table, window;
  int64_t k_step, v_step;  // bytes between the rows of a warp's consecutive copies
  int32_t R, Hq, Hkv, D, num_blocks, bs, max_blocks;
  int32_t gq;        // query heads of a kv head
  Divisor page;      // bs
  int32_t whole16;   // 16 keys from a multiple of 16 on share a block
  float scale2, v_scale;  // scale2 = scale * log2(e) * the keys' scale
};

// ------------------------------------------------------------- fragments
__device__ __forceinline__ void ldm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// c += a (16 x 16) . b (16 x 8), M the 16-bit type of both.
template <typename M>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<M, __half>::value)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two values of the 8-bit type (the low or high half of x) as two of f16: exact.
__device__ __forceinline__ uint32_t f16x2_lo(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}"
      : "=r"(r)
      : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t f16x2_hi(uint32_t x) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}"
      : "=r"(r)
      : "r"(x));
  return r;
}
template <typename M>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<M, __half>::value) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  } else {
    return pack_bf16x2(lo, hi);
  }
}

template <typename M>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if constexpr (std::is_same<M, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
  } else {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
}

// ------------------------------------------------------------------ shapes
// By the bytes of a row (head_dim elements of the cache) and of an element: the keys of a tile, a
// tile's keys and values in bytes, the warps of a CTA and the tiles of a warp's ring.  8 KB tiles
// and rings of 3 for 8 warps keep 16 KB in flight per warp while it computes.  8-bit rows take the
// most instructions per byte (every element is widened), and 8 warps do not hide their latencies:
// 12 with shorter rings take 65 us where 8 take 94 (32 x 8k, 64 elements) and 124 where 8 take 124
// too (3 requests of 90 to 131 thousand keys, 128 elements), but 102 where 8 take 75 if two groups
// of heads fill the registers (16 heads per kv head: they spill).  For 16-bit rows of 128 bytes 12
// warps measured alike (53.2 and 52.6 us, 128 ragged requests), and 12 or 16 warps of half the keys
// slower (60 and 67 us against 56: more instructions per key).
__host__ __device__ constexpr int tile_keys(int rb) { return rb <= 128 ? 32 : 16; }
__host__ __device__ constexpr int tile_bytes(int rb) { return 2 * tile_keys(rb) * rb; }
__host__ __device__ constexpr int split_warps(int rb, int elem, int nt) {
  return tile_bytes(rb) > 8192 ? 4 : elem == 1 && rb <= 128 && nt == 1 ? kMostWarps : 8;
}
__host__ __device__ constexpr int ring_tiles(int rb, int elem, int nt) {
  return kRingBytes / (split_warps(rb, elem, nt) * tile_bytes(rb)) > 6
             ? 6
             : kRingBytes / (split_warps(rb, elem, nt) * tile_bytes(rb));
}

template <typename C, int D, int NT>
struct Shape {
  static constexpr int RB = D * (int)sizeof(C);  // bytes of a row
  static constexpr int CH = RB / 16;             // 16-byte pieces of a row
  static constexpr int KT = tile_keys(RB);
  static constexpr int SB = tile_bytes(RB);
  static constexpr int W = split_warps(RB, sizeof(C), NT);
  static constexpr int S = ring_tiles(RB, sizeof(C), NT);
  // a warp's ring; its two parts, in 32 bits, lie there in the end
  static constexpr int kRing = S * SB > 2 * NT * 8 * (D + 2) * 4 ? S * SB : 2 * NT * 8 * (D + 2) * 4;
  static constexpr size_t kSmem = (size_t)W * kRing;
  static_assert(S >= 2 && kSmem <= 200 * 1024, "ring");
};

// Piece c of row `row` lies at piece c ^ swz(row): the eight rows of an ldmatrix
// fall into eight different banks' groups (two rows to a 128-byte line if RB is 64).
template <int RB>
__device__ __forceinline__ int swz(int row) {
  return RB >= 128 ? (row & 7) : ((row >> 1) & 3);
}

// The tiles [first, end) of request length `len`: whole tiles of the keys it uses.
__device__ __forceinline__ void tiles_of(const Args& a, int32_t len, int KT, int& t0, int& t1) {
  const int64_t room = (int64_t)a.max_blocks * a.bs;
  const int32_t n = (int32_t)min((int64_t)max(len, 0), room);
  const int32_t start = a.window > 0 && n > a.window ? n - (int32_t)a.window : 0;
  t0 = start / KT;
  t1 = (int)(((int64_t)n + KT - 1) / KT);
}

// 16 bytes into shared memory at `dst`; zeros, and nothing read, if there is nothing.
__device__ __forceinline__ void copy16(uint32_t dst, const char* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const char* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}

// 2^x; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Stage {  // what the reader of a tile needs to know
  uint32_t mask;   // keys that count
  int32_t r, h;    // the item; r < 0: no tile, the walk is over
  uint32_t flags;  // 1: first tile of this worker's part, 2: first of the item, 4: last of the
                   // item, 8: last of the worker
};

// Shares of this lane's request: its tiles and an item's cost, or 0.  For one item.
__device__ __forceinline__ int32_t shares_of(const Args& a, int32_t len, int KT) {
  int t0, t1;
  tiles_of(a, len, KT, t0, t1);
  return t0 < t1 ? t1 - t0 + kItemCost : 0;
}
// The sum over a warp of values below 2^28.
__device__ __forceinline__ int64_t warp_sum(int32_t v) {
  return (int64_t)__reduce_add_sync(~0u, (unsigned)v & 0xffffu) +
         ((int64_t)__reduce_add_sync(~0u, (unsigned)v >> 16) << 16);
}

// A warp's walk over its tiles, as it fetches them.
template <typename T, typename C, int D, int kHeads>
struct Walk {
  using X = Shape<C, D, kHeads / 8>;
  int64_t at, end;     // the tile to come and the end of the walk, in shares
  int32_t g, r, h;     // group of 32 requests, request, item of the request
  int32_t t, t0, t1;   // tile, and the request's
  int32_t n, start;    // the request's keys [start, n)
  int32_t glen;        // this lane's request of the group: its length
  int32_t id;          // this lane's key of the tile to come: its block, and its place there
  int32_t off;
  bool ok, fresh;

  __device__ __forceinline__ void load_group(const Args& a, int lane) {
    const int i = g * 32 + lane;
    glen = i < a.R ? a.lens[i] : 0;
  }
  __device__ __forceinline__ void set_request(const Args& a) {
    const int32_t len = __shfl_sync(~0u, glen, r & 31);
    tiles_of(a, len, X::KT, t0, t1);
    n = (int32_t)min((int64_t)max(len, 0), (int64_t)a.max_blocks * a.bs);
    start = a.window > 0 && n > a.window ? n - (int32_t)a.window : 0;
  }
  // The block of this lane's key of tile t: fetched a tile ahead of its use.
  __device__ __forceinline__ void look_up(const Args& a, int lane) {
    const int32_t key = t * X::KT + (lane & (X::KT - 1));
    ok = key >= start && key < n;
    id = -1;
    off = 0;
    if (key < n) {  // (a key in front of the window may share its block with one that counts)
      const int32_t page = a.page.div(key);
      off = key - page * a.bs;
      // (an ordinary load: the table may be written after this kernel was set up)
      id = a.table[(int64_t)r * a.ld_table + page];
    }
  }
  __device__ __forceinline__ void next(const Args& a, int Hg, int lane) {
    ++t;
    ++at;
    fresh = false;
    if (t == t1) {
      fresh = true;
      at += kItemCost;
      if (++h == Hg) {
        h = 0;
        do {
          if (++r >= a.R) {  // the last item is done
            at = end;
            return;
          }
          if ((r & 31) == 0) {
            ++g;
            load_group(a, lane);
          }
          set_request(a);
        } while (t0 >= t1);
      }
      t = t0;
    }
    if (at < end) look_up(a, lane);
  }
  // Starts the copies of the next tile into `ring` (a stage), or commits nothing.  With the
  // walk's last tile, *item_end = the share of its item's last tile.
  __device__ __forceinline__ void fetch(const Args& a, int Hg, int ngr, char* ring, Stage* st,
                                        int64_t* item_end, int lane) {
    if (at < end) {
      const bool in = ok && id >= 0 && id < a.num_blocks;
      if (ok && !in) atomicExch(&g_device_error, 3);
      constexpr uint32_t kAll = X::KT == 32 ? ~0u : 0xffffu;
      const uint32_t mask = __ballot_sync(~0u, in) & kAll;
      const int hk = ngr == 1 ? h : h / ngr;
      const Stage about{mask, r, h,
                        (fresh ? 1u : 0u) | (t == t0 ? 2u : 0u) | (t == t1 - 1 ? 4u : 0u)};
      const int64_t ends_at = at + (t1 - 1 - t);
      if (fresh) {  // the item's queries are read when its first tile has come
        constexpr int kLines = D * 2 / 128;
        const T* qp = (const T*)a.q + r * a.q_t + (hk * a.gq + (h - hk * ngr) * kHeads) * a.q_h;
        for (int i = lane; i < kHeads * kLines; i += 32)
          if ((h - hk * ngr) * kHeads + i / kLines < a.gq)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(qp + i / kLines * a.q_h +
                                                          i % kLines * 64));
      }
      // a warp's copy instruction: kRows rows, lane / CH the row, lane % CH its piece
      constexpr int kRows = 32 / X::CH, kSteps = X::KT / kRows;
      const int lr = lane / X::CH, c = lane % X::CH;
      const uint32_t kd = smem_u32(ring) + lr * X::RB, vd = kd + X::KT * X::RB;
      // the rows of 16 keys follow one another in their block: one address for each 16, then
      // steps of kRows rows (what does not count is zeros; 16 keys that share a block with one
      // that counts lie in the cache)
      auto rows = [&](auto every) {
#pragma unroll
        for (int g16 = 0; g16 < X::KT / 16; ++g16) {
          int64_t b = __shfl_sync(~0u, id, 16 * g16);
          const int64_t o = __shfl_sync(~0u, off, 16 * g16) + lr;
          if (!every.value && (mask >> 16 * g16 & 0xffffu) == 0) b = 0;  // no address to take
          const char* ks = (const char*)a.kc +
                           (b * a.kc_b + o * a.kc_t + (int64_t)hk * a.kc_h) * (int)sizeof(C) + c * 16;
          const char* vs = (const char*)a.vc +
                           (b * a.vc_b + o * a.vc_t + (int64_t)hk * a.vc_h) * (int)sizeof(C) + c * 16;
#pragma unroll
          for (int i = 0; i < 16 / kRows; ++i) {
            const int row = 16 * g16 + i * kRows;  // and lr more: swz is a xor of the two
            const int at = row * X::RB + ((c ^ swz<X::RB>(lr) ^ swz<X::RB>(row)) << 4);
            if constexpr (every.value) {
              copy16(kd + at, ks);
              copy16(vd + at, vs);
            } else {
              const bool there = mask >> (row + lr) & 1;
              copy16(kd + at, ks, there);
              copy16(vd + at, vs, there);
            }
            ks += a.k_step;
            vs += a.v_step;
          }
        }
      };
      // (blocks of whole 16 keys; by one address per key, below, the batch of 64 takes 357 us
      // instead of 330)
      if (a.whole16 && mask == kAll) {
        rows(std::true_type());
      } else if (a.whole16) {
        rows(std::false_type());
      } else {
        int64_t ko = 0, vo = 0;
        if (in) {
          ko = id * a.kc_b + off * a.kc_t + hk * a.kc_h;
          vo = id * a.vc_b + off * a.vc_t + hk * a.vc_h;
        }
#pragma unroll 1
        for (int i = 0; i < kSteps; ++i) {
          const int row = i * kRows + lr;
          const int64_t k1 = __shfl_sync(~0u, ko, row), v1 = __shfl_sync(~0u, vo, row);
          const bool there = mask >> row & 1;
          const int at = i * kRows * X::RB + ((c ^ swz<X::RB>(row)) << 4);
          copy16(kd + at, (const char*)a.kc + k1 * (int)sizeof(C) + c * 16, there);
          copy16(vd + at, (const char*)a.vc + v1 * (int)sizeof(C) + c * 16, there);
        }
      }
      next(a, Hg, lane);
      if (lane == 0) {
        *st = about;
        if (at >= end) {
          st->flags |= 8u;
          *item_end = ends_at;
        }
      }
    } else if (lane == 0) {
      st->r = -1;
    }
    cp_async_commit();
  }
};

// ------------------------------------------------------------------ results
// One 16 x 8 fragment of an item's output: lane (g, t) = (lane / 4, lane % 4)
// holds heads 2t and 2t+1 of group nt at two d's: 16j + g and that + 8 (16-bit
// caches), or 16j + 2g and that + 1 (8-bit).  All lanes of a warp call it.
template <typename T, typename C>
__device__ __forceinline__ void store_fragment(T* out, int64_t o_h, int heads, int nt, int j,
                                               int lane, float4 c) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (sizeof(C) == 1) {
    const int h = nt * 8 + 2 * t;
    uint32_t* p = reinterpret_cast<uint32_t*>(out + h * o_h + 16 * j + 2 * g);
    if (h < heads) *p = pack2<T>(c.x, c.z);
    if (h + 1 < heads) *reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p) + o_h) =
        pack2<T>(c.y, c.w);
  } else {
    const uint32_t lo = transpose8x8(pack2<T>(c.x, c.y));
    const uint32_t hi = transpose8x8(pack2<T>(c.z, c.w));
    const int h = nt * 8 + g;
    if (h < heads) {
      T* p = out + h * o_h + 16 * j + 2 * t;
      *reinterpret_cast<uint32_t*>(p) = lo;
      *reinterpret_cast<uint32_t*>(p + 8) = hi;
    }
  }
}

// The exponent that a softmax's weights 2^(s - m) count from, for a largest score `top`.  For bf16
// pieces top itself.  For f16 pieces 14 below it, so that weights lie below 2^15 and those down to
// 2^-38 of the largest are seen (131072 keys of 2^-24 each may outweigh it); sums, products and
// their joins all count from the same m, so nothing takes the factor off.  Scores that large that
// 14 is lost in their rounding keep m = top.
template <typename T, typename C>
__device__ __forceinline__ float exponent_of(float top) {
  constexpr bool kF16 = sizeof(C) == 1 || std::is_same<T, __half>::value;
  return kF16 && fabsf(top) < 8388608.0f ? top - 14.0f : top;
}

__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}
// 2^(m - top), where top may be -inf (then so is m: nothing was seen).
__device__ __forceinline__ float weight(float m, float top) {
  return exp2_ftz(m - (top == -INFINITY ? 0.0f : top));
}

// Adds a part (its maxima and sums of two heads, and its products) to the parts so far.
__device__ __forceinline__ void join_part(float4& c, float& m0, float& m1, float& l0, float& l1,
                                          float2 pm, float2 pl, float4 v) {
  const float t0 = fmaxf(m0, pm.x), t1 = fmaxf(m1, pm.y);
  const float a0 = weight(m0, t0), a1 = weight(m1, t1);
  const float b0 = weight(pm.x, t0), b1 = weight(pm.y, t1);
  c.x = c.x * a0 + v.x * b0;
  c.y = c.y * a1 + v.y * b1;
  c.z = c.z * a0 + v.z * b0;
  c.w = c.w * a1 + v.w * b1;
  l0 = l0 * a0 + pl.x * b0;
  l1 = l1 * a1 + pl.y * b1;
  m0 = t0;
  m1 = t1;
}

// A partial result: fragments [nt][j][lane] as float4, then m[8 NT], l[8 NT].
template <int D, int NT>
constexpr int kPartFloats = NT * 8 * (D + 2);

// The CTA's share of the join: what crosses into the next CTA.
struct Cross {
  int32_t item, last;  // an item that goes on (-1: none), and the last CTA that has a part
};

// Workspace: [workers] first parts | [CTAs][2] parts that cross CTAs | [CTAs] Cross.
struct Room {
  float* first;
  float* cross;
  Cross* about;
};

template <typename T, typename C, int D, int NT>
__global__ void __launch_bounds__(Shape<C, D, NT>::W * 32, 1)
    k_paged_split(const __grid_constant__ Args a, const Room room) {
  using X = Shape<C, D, NT>;
  using M = typename std::conditional<sizeof(C) == 1, __half, T>::type;  // the product's type
  constexpr int W = X::W, S = X::S, KT = X::KT, PF = kPartFloats<D, NT>;
  constexpr bool F8 = sizeof(C) == 1;
  extern __shared__ __align__(128) char ring_all[];
  __shared__ int64_t before[kMaxRequests / 32 + 1];
  __shared__ Stage stages[W][S];
  __shared__ int32_t p_item[2 * W], p_flag[2 * W];
  __shared__ int64_t p_end[W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int gq = a.gq, ngr = (gq + 8 * NT - 1) / (8 * NT), Hg = a.Hkv * ngr;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the kernel before is done

  // The work in shares: each tile one, and kItemCost for each item (request and group of heads)
  // in front of its tiles.  Every worker (warp) gets the same number of shares, a range of them,
  // and with it the tiles in that range.  Shares before each group of 32 requests:
  const int groups = (a.R + 31) / 32;
  for (int i = warp; i < groups; i += W) {
    const int r = i * 32 + lane;
    const int64_t c = warp_sum(r < a.R ? shares_of(a, a.lens[r], KT) : 0) * Hg;
    if (lane == 0) before[i + 1] = c;
  }
  if (threadIdx.x < 2 * W) p_item[threadIdx.x] = -1;
  if (threadIdx.x == 0) before[0] = 0;
  __syncthreads();
  if (groups > 1 && warp == 0) {
    int64_t sum = 0;
    for (int i = 0; i < groups; i += 32) {
      int64_t c = i + lane < groups ? before[i + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(~0u, c, o);
        if (lane >= o) c += y;
      }
      if (i + lane < groups) before[i + lane + 1] = sum + c;
      sum += __shfl_sync(~0u, c, 31);
    }
  }
  if (groups > 1) __syncthreads();
  const int64_t total = before[groups];
  const int64_t workers = (int64_t)gridDim.x * W, worker = (int64_t)blockIdx.x * W + warp;
  const int64_t quota = (total + workers - 1) / workers;
  const int64_t begin = worker * quota;

  // requests without keys; lengths that are out of range
  for (int64_t r = worker; r < a.R; r += workers) {
    const int32_t len = a.lens[r];
    int t0, t1;
    tiles_of(a, len, KT, t0, t1);
    if (lane == 0 && (len < 0 || len > (int64_t)a.max_blocks * a.bs))
      atomicExch(&g_device_error, 3);
    if (t0 >= t1) {
      for (int i = lane; i < a.Hq * (D / 8); i += 32) {
        const int h = i / (D / 8), d = i % (D / 8);
        *reinterpret_cast<uint4*>((T*)a.out + r * a.o_t + h * a.o_h + d * 8) =
            make_uint4(0, 0, 0, 0);
      }
      if (a.lse)
        for (int i = lane; i < a.Hq; i += 32) a.lse[r * a.Hq + i] = -INFINITY;
    }
  }

  char* ring = ring_all + (size_t)warp * X::kRing;
  if (begin < total) {
    Walk<T, C, D, 8 * NT> w;
    w.at = w.end = min(begin + quota, total);
    {
      int lo = 0, hi = groups;  // before[lo] <= begin < before[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= begin) lo = mid;
        else hi = mid;
      }
      w.g = lo;
      w.load_group(a, lane);
      int64_t c = (int64_t)shares_of(a, w.glen, KT) * Hg;
      const int64_t mine = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(~0u, c, o);
        if (lane >= o) c += y;
      }
      const int64_t want = begin - before[lo];
      // (a request that holds the share: there is one unless the lengths change under the call)
      const int l = max(__ffs(__ballot_sync(~0u, c > want)) - 1, 0);
      const int64_t in = want - __shfl_sync(~0u, c - mine, l);
      w.r = lo * 32 + l;
      w.set_request(a);
      // in / each, below 2^16: the float quotient is off by less than one
      const int64_t each = max(w.t1 - w.t0, 1) + kItemCost;
      w.h = (int)__fdividef((float)in, (float)each);
      if (w.h * each > in) --w.h;
      else if ((w.h + 1) * each <= in) ++w.h;
      const int skip = max((int)(in - w.h * each) - kItemCost, 0);  // tiles of earlier workers
      w.t = w.t0 + skip;
      w.fresh = true;
      const int64_t at = begin - in + w.h * each + kItemCost + skip;
      if (w.r < a.R && w.t < w.t1 && in >= 0 && w.h >= 0 && w.h < Hg && at < w.end) {
        w.at = at;
        w.look_up(a, lane);
      }
    }
    uint32_t q[D / 16][2 * NT];
    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2], sc[NT][2];  // of heads 2 t4 and 2 t4 + 1 of each group of eight
    bool began = false;
    int head0 = 0, heads = 0;  // the item's query heads
    const int lrow = lane & 7, lhalf = (lane >> 3) & 1, lsec = lane >> 4;
    // where this lane points ldmatrix, from a tile's keys (values) on.  Four 8 x 8 matrices: the
    // keys' are [keys 0-7 | 8-15] x [d's | the next], in that order (an A operand: keys x d's);
    // the values' of 16 bits [d's | the next] x [keys 0-7 | 8-15] (its transpose: d's x keys), of
    // 8 bits as the keys'.
    constexpr int kStep = F8 ? 2 : 1;  // 16 d's of 8 bits are one 16-byte piece, of 16 bits two
    uint32_t kpiece[D / 16 / kStep], vpiece[D / 16 / kStep];
#pragma unroll
    for (int j = 0; j < D / 16; j += kStep) {
      const int base = F8 ? j : 2 * j;
      kpiece[j / kStep] = (lhalf * 8 + lrow) * X::RB + (((base + lsec) ^ swz<X::RB>(lrow)) << 4);
      vpiece[j / kStep] = F8 ? kpiece[j / kStep]
                             : (lsec * 8 + lrow) * X::RB +
                                   (((base + lhalf) ^ swz<X::RB>(lrow)) << 4);
    }
    // an item's queries, as they are
    auto load_queries = [&](const Stage& st) {
      const int hk = ngr == 1 ? st.h : st.h / ngr, sub = st.h - hk * ngr;
      head0 = hk * gq + sub * 8 * NT;
      heads = min(8 * NT, gq - sub * 8 * NT);
      const T* qp = (const T*)a.q + st.r * a.q_t + head0 * a.q_h;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int row = g + 8 * n;
        const T* qr = qp + row * a.q_h;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) q[j][2 * n] = q[j][2 * n + 1] = 0;
        if (row < heads) {
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            if constexpr (F8) {  // pairs in the order of the keys' 8-bit pieces
              const uint2 v = *reinterpret_cast<const uint2*>(qr + 16 * j + 4 * t4);
              q[j][2 * n] = v.x;
              q[j][2 * n + 1] = v.y;
            } else {
              const uint32_t* p = reinterpret_cast<const uint32_t*>(qr + 16 * j + 2 * t4);
              q[j][2 * n] = p[0];
              q[j][2 * n + 1] = p[4];
            }
          }
        }
      }
    };
    // nothing seen of the item yet; its queries as the product takes them
    auto start_item = [&](const Stage& st) {
      began = st.flags & 2;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float fac = 1.0f;
        if constexpr (F8 && !std::is_same<T, __half>::value) {
          // bf16 queries against keys widened to f16: the row is brought to [2^14, 2^15), the top
          // of f16, by a power of two (put back on the scores), so that elements down to 2^-31 of
          // the largest keep all of a bf16's 8 bits
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t v = q[j][2 * n + e] & 0x7fff7fffu;
              top = max(top, max(v & 0xffffu, v >> 16));
            }
          top = max(top, __shfl_xor_sync(~0u, top, 1));
          top = max(top, __shfl_xor_sync(~0u, top, 2));
          const uint32_t ex = min(max(top << 16 & 0x7f800000u, 0x07800000u), 0x7f000000u);
          fac = __uint_as_float(ex - 0x07000000u);             // 2^-14 of it
          const float inv = __uint_as_float(0x86000000u - ex);  // 1 / fac
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t v = q[j][2 * n + e];
              q[j][2 * n + e] = pack2<__half>(__uint_as_float(v << 16) * inv,
                                              __uint_as_float(v & 0xffff0000u) * inv);
            }
        }
        // the scale's sign goes to the queries, so that the maximum is found before scaling; a
        // scale of zero is queries of zero.  The factor of this lane's row, head g, is neither zero
        // nor infinite: a masked score stays -inf, and a product of zero a score of zero
        const float f = fminf(fmaxf(fabsf(a.scale2) * fac, 1.4e-45f), 3.4e38f);
        sc[n][0] = __shfl_sync(~0u, f, 8 * t4);
        sc[n][1] = __shfl_sync(~0u, f, 8 * t4 + 4);
        if (a.scale2 <= 0.0f) {
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              q[j][2 * n + e] = a.scale2 == 0.0f ? 0u : q[j][2 * n + e] ^ 0x80008000u;
        }
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][j][e] = 0.0f;
      }
    };
    int rs = 0, ws = 0;        // stage to read, stage to fill
    Stage st{0, -1, 0, 0};     // the tile at hand
    for (int ahead = S - 1;; ahead -= ahead > 0) {  // tiles to start before the first is awaited
      if (ahead == 0) {
        cp_async_wait<S - 2>();
        __syncwarp();
      }
      w.fetch(a, Hg, ngr, ring + ws * X::SB, &stages[warp][ws], &p_end[warp], lane);
      ws = ws + 1 == S ? 0 : ws + 1;
      if (ahead > 1) continue;
      if (ahead == 1) {  // the first tile is under way: its queries
        __syncwarp();
        st = stages[warp][rs];
        if (st.r < 0) break;
        load_queries(st);
        continue;
      }
      const uint32_t kb = smem_u32(ring + rs * X::SB);
      rs = rs + 1 == S ? 0 : rs + 1;
      if (st.flags & 1) start_item(st);

      // scores: rows = keys, columns = heads
      float s[KT / 16][NT][4];
#pragma unroll
      for (int k2 = 0; k2 < KT / 16; ++k2)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[k2][n][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < D / 16; j += kStep) {
        const uint32_t at = kb + kpiece[j / kStep];
#pragma unroll
        for (int k2 = 0; k2 < KT / 16; ++k2) {
          uint32_t b[4];
          ldm_x4(b, at + k2 * 16 * X::RB);
          if constexpr (F8) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t a0 = f16x2_lo(b[2 * u]), a1 = f16x2_lo(b[2 * u + 1]);
              const uint32_t a2 = f16x2_hi(b[2 * u]), a3 = f16x2_hi(b[2 * u + 1]);
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mma16816<M>(s[k2][n], a0, a1, a2, a3, q[j + u][2 * n], q[j + u][2 * n + 1]);
            }
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma16816<M>(s[k2][n], b[0], b[1], b[2], b[3], q[j][2 * n], q[j][2 * n + 1]);
          }
        }
      }

      // softmax over the keys: this lane has keys g and g + 8 of each 16, and two heads
      if (st.mask != (KT == 32 ? ~0u : 0xffffu)) {
#pragma unroll
        for (int k2 = 0; k2 < KT / 16; ++k2)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(st.mask >> (16 * k2 + g + 8 * (e >> 1)) & 1))
#pragma unroll
              for (int n = 0; n < NT; ++n) s[k2][n][e] = -INFINITY;
      }
      bool grew = false;
      float base[NT][2], c[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = fmaxf(s[0][n][h], s[0][n][h + 2]);
#pragma unroll
          for (int k2 = 1; k2 < KT / 16; ++k2)
            top = fmaxf(top, fmaxf(s[k2][n][h], s[k2][n][h + 2]));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
          // sc > 0: the largest score is that of the largest product
          const float now = fmaxf(m[n][h], exponent_of<T, C>(__fmul_rn(top, sc[n][h])));
          base[n][h] = now == -INFINITY ? 0.0f : now;
          c[n][h] = exp2_ftz(m[n][h] - base[n][h]);
          grew |= now > m[n][h];
          m[n][h] = now;
        }
      if (__any_sync(~0u, grew)) {  // a maximum rose: what was summed shrinks
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          l[n][0] *= c[n][0];
          l[n][1] *= c[n][1];
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            o[n][j][0] *= c[n][0];
            o[n][j][1] *= c[n][1];
            o[n][j][2] *= c[n][0];
            o[n][j][3] *= c[n][1];
          }
        }
      }
      // The weights enter the second product as two pieces of the 16-bit type: off by 2^-17 of a
      // weight (bf16) or 2^-22 (f16).  One f16 piece, off by 2^-12, is hidden by a bf16 output's
      // rounding only where the values do not cancel: of 3 long requests over e4m3 it let 4.9 % of
      // the outputs round the other way (two: 0.2 %, torch in 32 bits: 0.2 %).  The second costs 1 %
      // there (119 us; 5 % at the clocks of a lasting load), 5 % for e4m3 rows of 64 and 12 % for 16
      // heads per kv head.
      uint32_t ph[NT][KT / 8], pl[NT][KT / 8];
#pragma unroll
      for (int k = 0; k < KT / 8; ++k)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float* p = &s[k / 2][n][k % 2 * 2];
          // rounded as the largest was: fused, scores of 2^24 and more would be off it by their
          // rounding, and their weights by any factor
          const float x = exp2_ftz(__fsub_rn(__fmul_rn(p[0], sc[n][0]), base[n][0]));
          const float y = exp2_ftz(__fsub_rn(__fmul_rn(p[1], sc[n][1]), base[n][1]));
          l[n][0] += x;
          l[n][1] += y;
          const uint32_t w = pack2<M>(x, y);
          ph[n][k] = transpose8x8(w);  // keys x heads -> a B operand's heads x keys
          const float2 r = unpack2<M>(w);
          pl[n][k] = transpose8x8(pack2<M>(x - r.x, y - r.y));
        }

      // values: rows = d's, columns = heads
#pragma unroll
      for (int k2 = 0; k2 < KT / 16; ++k2) {
#pragma unroll
        for (int j = 0; j < D / 16; j += kStep) {
          uint32_t v[4];
          ldm_x4_t(v, kb + vpiece[j / kStep] + KT * X::RB + k2 * 16 * X::RB);
          if constexpr (F8) {
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = __byte_perm(v[u], 0, 0x3120);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t a0 = f16x2_lo(v[2 * u]), a1 = f16x2_hi(v[2 * u]);
              const uint32_t a2 = f16x2_lo(v[2 * u + 1]), a3 = f16x2_hi(v[2 * u + 1]);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma16816<M>(o[n][j + u], a0, a1, a2, a3, ph[n][2 * k2], ph[n][2 * k2 + 1]);
                mma16816<M>(o[n][j + u], a0, a1, a2, a3, pl[n][2 * k2], pl[n][2 * k2 + 1]);
              }
            }
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma16816<M>(o[n][j], v[0], v[1], v[2], v[3], ph[n][2 * k2], ph[n][2 * k2 + 1]);
              mma16816<M>(o[n][j], v[0], v[1], v[2], v[3], pl[n][2 * k2], pl[n][2 * k2 + 1]);
            }
          }
        }
      }

      const bool ends = st.flags & 4, last = st.flags & 8;
      if (ends || last) {  // the end of this warp's part of the item
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[n][h] += __shfl_xor_sync(~0u, l[n][h], x);
        if (began && ends) {
          T* out = (T*)a.out + st.r * a.o_t + head0 * a.o_h;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float i0 = l[n][0] == 0.0f ? 0.0f : a.v_scale / l[n][0];
            const float i1 = l[n][1] == 0.0f ? 0.0f : a.v_scale / l[n][1];
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
              store_fragment<T, C>(out, a.o_h, heads, n, j, lane,
                                   make_float4(o[n][j][0] * i0, o[n][j][1] * i1, o[n][j][2] * i0,
                                               o[n][j][3] * i1));
            if (a.lse && g < 2 && 8 * n + 2 * t4 + g < heads)
              a.lse[(int64_t)st.r * a.Hq + head0 + 8 * n + 2 * t4 + g] =
                  g ? lse_of(m[n][1], l[n][1]) : lse_of(m[n][0], l[n][0]);
          }
        } else {
          // a part: the first of several is put aside in the workspace, the last one in this
          // warp's ring, which is then free
          if (last) {
            cp_async_wait<0>();
            __syncwarp();
          }
          float* to = last ? reinterpret_cast<float*>(ring) : room.first + worker * PF;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
              reinterpret_cast<float4*>(to)[(n * (D / 16) + j) * 32 + lane] =
                  make_float4(o[n][j][0], o[n][j][1], o[n][j][2], o[n][j][3]);
            if (g == 0) {
              *reinterpret_cast<float2*>(to + NT * 8 * D + 8 * n + 2 * t4) =
                  make_float2(m[n][0], m[n][1]);
              *reinterpret_cast<float2*>(to + NT * 8 * (D + 1) + 8 * n + 2 * t4) =
                  make_float2(l[n][0], l[n][1]);
            }
          }
          if (lane == 0) {
            const int e = 2 * warp + (last ? 1 : 0);
            p_item[e] = st.r * Hg + st.h;
            p_flag[e] = (began ? 1 : 0) | (ends ? 2 : 0);
          }
        }
      }
      if (last) break;
      if (S == 2) __syncwarp();  // written in this turn; with more tiles, before the last wait
      st = stages[warp][rs];
      if (st.r < 0) break;
      if (st.flags & 1) load_queries(st);
    }
    if (p_item[2 * warp] >= 0) {  // the first part joins the last in the ring
      cp_async_wait<0>();
      __syncwarp();
      const float4* from = reinterpret_cast<const float4*>(room.first + worker * PF);
      float4* to = reinterpret_cast<float4*>(ring) + PF / 4;
#pragma unroll
      for (int i = 0; i < (PF / 4 + 31) / 32; ++i)
        if (i * 32 + lane < PF / 4) to[i * 32 + lane] = from[i * 32 + lane];
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // Join the CTA's own parts: entry 2w is warp w's first part, 2w + 1 its last.  Parts of one
  // item are neighbours in that order; a run that lacks the item's first or last tile crosses
  // into another CTA.  The code is met once a launch and comes from memory, so it is kept short:
  // a warp takes a fragment of a run and sums the parts as they come, each with its maximum.
  auto part = [&](int e) {
    return reinterpret_cast<const float*>(ring_all + (size_t)(e >> 1) * X::kRing) +
           (e & 1 ? 0 : PF);
  };
  static_assert(2 * W <= 32, "a lane per entry");
  constexpr int kFrags = NT * (D / 16);
  const int entry = lane < 2 * W ? p_item[lane] : -1;
  Cross cross{-1, 0};
  int turn = 0;  // fragments so far, of all runs
  for (uint32_t todo = __ballot_sync(~0u, entry >= 0); todo; turn += kFrags) {
    const int e0 = __ffs(todo) - 1, item = __shfl_sync(~0u, entry, e0);
    const uint32_t run = __ballot_sync(~0u, entry == item);
    todo &= ~run;
    const int tail = 31 - __clz(run);
    const bool has0 = p_flag[e0] & 1, has1 = p_flag[tail] & 2;
    if (has0 && !has1) {
      cross.item = item;
      // (no further than the last CTA, should the lengths change under the call)
      cross.last = (int)min(p_end[tail >> 1] / (W * quota), (int64_t)gridDim.x - 1);
    }
#pragma unroll 1
    for (int f = (warp + W * 32 - turn % W) % W; f < kFrags; f += W) {
      const int n = f / (D / 16), j = f % (D / 16), hh = n * 8 + 2 * t4;
      float4 c = make_float4(0, 0, 0, 0);
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0, l1 = 0;
#pragma unroll 1
      for (uint32_t b = run; b; b &= b - 1) {
        const float* p = part(__ffs(b) - 1);
        const float2 pm = *reinterpret_cast<const float2*>(p + NT * 8 * D + hh);
        const float2 pl = *reinterpret_cast<const float2*>(p + NT * 8 * (D + 1) + hh);
        const float4 v = reinterpret_cast<const float4*>(p)[f * 32 + lane];
        join_part(c, m0, m1, l0, l1, pm, pl, v);
      }
      const int r = item / Hg, h = item - r * Hg, sub = h % ngr;
      const int head0 = h / ngr * gq + sub * 8 * NT, heads = min(8 * NT, gq - sub * 8 * NT);
      if (has0 && has1) {
        const float i0 = l0 == 0.0f ? 0.0f : a.v_scale / l0;
        const float i1 = l1 == 0.0f ? 0.0f : a.v_scale / l1;
        store_fragment<T, C>((T*)a.out + r * a.o_t + head0 * a.o_h, a.o_h, heads, n, j, lane,
                             make_float4(c.x * i0, c.y * i1, c.z * i0, c.w * i1));
        if (a.lse && j == 0 && g == 0) {
          if (hh < heads) a.lse[(int64_t)r * a.Hq + head0 + hh] = lse_of(m0, l0);
          if (hh + 1 < heads) a.lse[(int64_t)r * a.Hq + head0 + hh + 1] = lse_of(m1, l1);
        }
      } else {
        float* to = room.cross + ((int64_t)blockIdx.x * 2 + (has0 ? 1 : 0)) * PF;
        reinterpret_cast<float4*>(to)[f * 32 + lane] = c;
        if (j == 0 && g == 0) {
          *reinterpret_cast<float2*>(to + NT * 8 * D + hh) = make_float2(m0, m1);
          *reinterpret_cast<float2*>(to + NT * 8 * (D + 1) + hh) = make_float2(l0, l1);
        }
      }
    }
  }
  if (threadIdx.x == 0) room.about[blockIdx.x] = cross;
}

// Joins the items whose parts lie in several CTAs.  Block (c, f): the item that
// starts in CTA c and goes on, its fragment f; the warps share the parts.
constexpr int kJoinWarps = 8;

template <typename T, typename C, int D, int NT>
__global__ void __launch_bounds__(kJoinWarps * 32)
    k_paged_join(const __grid_constant__ Args a, const Room room) {
  constexpr int PF = kPartFloats<D, NT>;
  __shared__ float4 sc[kJoinWarps][32];
  __shared__ float sm[kJoinWarps][32][2], sl[kJoinWarps][32][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gq = a.gq, ngr = (gq + 8 * NT - 1) / (8 * NT), Hg = a.Hkv * ngr;
  const int cta = blockIdx.x, f = blockIdx.y;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int item = __ldcg(&room.about[cta].item), last = __ldcg(&room.about[cta].last);
  if (item < 0) return;
  const int n = f / (D / 16), j = f % (D / 16), hh = n * 8 + 2 * (lane & 3);
  float4 c = make_float4(0, 0, 0, 0);
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0, l1 = 0;
#pragma unroll 4
  for (int b = cta + warp; b <= last; b += kJoinWarps) {
    const float* p = room.cross + ((int64_t)b * 2 + (b == cta ? 1 : 0)) * PF;
    const float2 pm = __ldcg(reinterpret_cast<const float2*>(p + NT * 8 * D + hh));
    const float2 pl = __ldcg(reinterpret_cast<const float2*>(p + NT * 8 * (D + 1) + hh));
    const float4 v = __ldcg(reinterpret_cast<const float4*>(p) + f * 32 + lane);
    join_part(c, m0, m1, l0, l1, pm, pl, v);
  }
  sc[warp][lane] = c;
  sm[warp][lane][0] = m0;
  sm[warp][lane][1] = m1;
  sl[warp][lane][0] = l0;
  sl[warp][lane][1] = l1;
  __syncthreads();
  if (warp) return;
  for (int w = 1; w < kJoinWarps; ++w) {
    m0 = fmaxf(m0, sm[w][lane][0]);
    m1 = fmaxf(m1, sm[w][lane][1]);
  }
  c = make_float4(0, 0, 0, 0);
  l0 = l1 = 0;
  for (int w = 0; w < kJoinWarps; ++w) {
    const float w0 = weight(sm[w][lane][0], m0), w1 = weight(sm[w][lane][1], m1);
    const float4 v = sc[w][lane];
    c.x += w0 * v.x;
    c.y += w1 * v.y;
    c.z += w0 * v.z;
    c.w += w1 * v.w;
    l0 += w0 * sl[w][lane][0];
    l1 += w1 * sl[w][lane][1];
  }
  const int r = item / Hg, h = item - r * Hg, sub = h % ngr, head0 = h / ngr * gq + sub * 8 * NT;
  const int heads = min(8 * NT, gq - sub * 8 * NT);
  const float i0 = l0 == 0.0f ? 0.0f : a.v_scale / l0, i1 = l1 == 0.0f ? 0.0f : a.v_scale / l1;
  store_fragment<T, C>((T*)a.out + r * a.o_t + head0 * a.o_h, a.o_h, heads, n, j, lane,
                       make_float4(c.x * i0, c.y * i1, c.z * i0, c.w * i1));
  if (a.lse && j == 0 && (lane >> 2) == 0) {
    if (hh < heads) a.lse[(int64_t)r * a.Hq + head0 + hh] = lse_of(m0, l0);
    if (hh + 1 < heads) a.lse[(int64_t)r * a.Hq + head0 + hh + 1] = lse_of(m1, l1);
  }
}

// Groups of eight query heads that a warp takes at once: two where a kv head has more than eight
// and registers allow (16 heads per kv head, 16 x 4k: 59 us against 91 in two items of eight, each
// reading the keys).
inline int head_tiles(int64_t Hq, int64_t Hkv, int64_t D) { return Hq / Hkv > 8 && D <= 128 ? 2 : 1; }

// One CTA per SM, but no more than the block tables' room could have tiles for.
inline int split_grid(int64_t R, int64_t Hq, int64_t Hkv, int64_t D, int elem, int64_t room) {
  const int nt = head_tiles(Hq, Hkv, D), ngr = (int)((Hq / Hkv + 8 * nt - 1) / (8 * nt));
  const int rb = (int)D * elem;
  const int64_t tiles = (room + tile_keys(rb) - 1) / tile_keys(rb) + 1;
  const int64_t most = (tiles + kItemCost) * R * Hkv * ngr / split_warps(rb, elem, nt) + 1;
  return (int)std::min<int64_t>(num_sms(), most);
}

// Floats of one partial result.
inline int64_t part_floats(int64_t Hq, int64_t Hkv, int64_t D) {
  return head_tiles(Hq, Hkv, D) * 8 * (D + 2);
}

template <typename T, typename C, int D, int NT>
int launch(Args& a, void* workspace, cudaStream_t st) {
  using X = Shape<C, D, NT>;
  a.k_step = a.kc_t * (int64_t)sizeof(C) * (32 / X::CH);
  a.v_step = a.vc_t * (int64_t)sizeof(C) * (32 / X::CH);
  constexpr int PF = kPartFloats<D, NT>;
  auto split = k_paged_split<T, C, D, NT>;
  RB_CUDA(cudaFuncSetAttribute(split, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)X::kSmem));
  const int sms = num_sms();
  const int grid = split_grid(a.R, a.Hq, a.Hkv, D, sizeof(C), (int64_t)a.max_blocks * a.bs);
  Room room;
  room.first = static_cast<float*>(workspace);
  room.cross = room.first + (int64_t)sms * X::W * PF;
  room.about = reinterpret_cast<Cross*>(room.cross + (int64_t)sms * 2 * PF);
  // both may be set up while the kernel before is ending; they wait for its end themselves
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(X::W * 32);
  cfg.dynamicSmemBytes = X::kSmem;
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  RB_CUDA(cudaLaunchKernelEx(&cfg, split, a, room));
  if (grid == 1) return REMORA_B200_OK;  // nothing crosses
  cfg.gridDim = dim3(grid, NT * (D / 16));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.dynamicSmemBytes = 0;
  RB_CUDA(cudaLaunchKernelEx(&cfg, k_paged_join<T, C, D, NT>, a, room));
  return REMORA_B200_OK;
}

template <typename T, typename C>
int launch_shape(Args& a, void* ws, cudaStream_t st) {
  const int nt = head_tiles(a.Hq, a.Hkv, a.D);
  if (a.D == 64) return nt == 2 ? launch<T, C, 64, 2>(a, ws, st) : launch<T, C, 64, 1>(a, ws, st);
  if (a.D == 128)
    return nt == 2 ? launch<T, C, 128, 2>(a, ws, st) : launch<T, C, 128, 1>(a, ws, st);
  return launch<T, C, 256, 1>(a, ws, st);
}

inline bool shape_ok(int64_t R, int64_t Hq, int64_t Hkv, int64_t D) {
  return R >= 0 && R <= kMaxRequests && Hkv >= 1 && Hq >= 1 && Hq <= 65536 && Hq % Hkv == 0 &&
         (D == 64 || D == 128 || D == 256);
}

}  // namespace paged
}  // namespace rb

extern "C" size_t remora_b200_paged_attention_workspace_bytes(int64_t R, int64_t Hq, int64_t Hkv,
                                                              int64_t D) {
  using namespace rb::paged;
  if (!shape_ok(R, Hq, Hkv, D)) return 0;
  const int64_t sms = rb::num_sms();
  return (size_t)(sms * (kMostWarps + 2) * part_floats(Hq, Hkv, D) * 4 + sms * (int64_t)sizeof(Cross));
}

extern "C" int remora_b200_paged_attention(const remora_b200_paged_attention_args* args,
                                           void* stream) {
  using namespace rb;
  using namespace rb::paged;
  clear_error();
  RB_CHECK_ARG(args, "paged_attention: args is null");
  const remora_b200_paged_attention_args& p = *args;
  const int64_t R = p.R, Hq = p.Hq, Hkv = p.Hkv, D = p.D;
  RB_CHECK_ARG(p.dtype == REMORA_B200_BF16 || p.dtype == REMORA_B200_F16,
               "paged_attention: dtype must be BF16 or F16");
  RB_CHECK_ARG(p.cache_dtype == p.dtype || p.cache_dtype == REMORA_B200_E4M3,
               "paged_attention: cache_dtype must be dtype or E4M3");
  RB_CHECK_ARG(shape_ok(R, Hq, Hkv, D),
               "paged_attention: needs R in [0, %d], Hq a multiple of Hkv and head_dim 64, 128 or "
               "256 (got R %lld, Hq %lld, Hkv %lld, head_dim %lld)",
               kMaxRequests, (long long)R, (long long)Hq, (long long)Hkv, (long long)D);
  RB_CHECK_ARG(p.block_size >= 1 && p.num_blocks >= 1 && p.block_size <= 0x7fffffff &&
                   p.num_blocks <= 0x7fffffff / p.block_size,
               "paged_attention: num_blocks * block_size must be in [1, 2^31)");
  RB_CHECK_ARG(p.max_blocks >= 1 && p.max_blocks <= 0x7fffffff / p.block_size && p.ld_table >= p.max_blocks,
               "paged_attention: max_blocks * block_size must be in [1, 2^31) and ld_table at "
               "least max_blocks");
  RB_CHECK_ARG(std::isfinite(p.scale), "paged_attention: scale is not finite");
  RB_CHECK_ARG(std::isfinite(p.scale * 1.4426950408889634f * p.k_scale),
               "paged_attention: scale, and scale times k_scale, must be below 2.3e38");
  RB_CHECK_ARG(p.window >= 0, "paged_attention: window must not be negative");
  RB_CHECK_ARG(rope::scale_ok(p.k_scale) && rope::scale_ok(p.v_scale),
               "paged_attention: the cache scales must lie in [1e-30, 1e30]");
  RB_CHECK_ARG(p.cache_dtype == REMORA_B200_E4M3 || (p.k_scale == 1.0f && p.v_scale == 1.0f),
               "paged_attention: the scales must be 1 unless the cache is E4M3");
  if (R == 0) return REMORA_B200_OK;
  RB_CHECK_ARG(p.q && p.k_cache && p.v_cache && p.block_table && p.lens && p.out,
               "paged_attention: null pointer");
  RB_CHECK_ARG(p.q != p.out, "paged_attention: out must not be q");
  RB_CHECK_ARG(aligned16(p.q) && aligned16(p.k_cache) && aligned16(p.v_cache) && aligned16(p.out),
               "paged_attention: q, the caches and out must be 16-byte aligned");
  RB_CHECK_ARG(aligned4(p.block_table, p.lens, p.lse),
               "paged_attention: a pointer is not aligned to its elements");
  const int64_t ce = p.cache_dtype == REMORA_B200_E4M3 ? 16 : 8;
  RB_CHECK_ARG(p.q_t % 8 == 0 && p.q_h % 8 == 0 && p.out_t % 8 == 0 && p.out_h % 8 == 0 &&
                   p.kc_block % ce == 0 && p.kc_token % ce == 0 && p.kc_head % ce == 0 &&
                   p.vc_block % ce == 0 && p.vc_token % ce == 0 && p.vc_head % ce == 0,
               "paged_attention: strides must be multiples of 16 bytes");
  RB_CHECK_ARG(!rows_overlap(R, p.out_t, D) && !rows_overlap(Hq, p.out_h, D),
               "paged_attention: the rows of out overlap");
  const size_t need = remora_b200_paged_attention_workspace_bytes(R, Hq, Hkv, D);
  RB_CHECK_ARG(p.workspace && p.workspace_bytes >= need && aligned16(p.workspace),
               "paged_attention: workspace of %zu bytes, 16-byte aligned, is needed", need);
  Args a = {};
  a.q = p.q;
  a.kc = p.k_cache;
  a.vc = p.v_cache;
  a.table = p.block_table;
  a.lens = p.lens;
  a.out = p.out;
  a.lse = p.lse;
  a.q_t = p.q_t;
  a.q_h = p.q_h;
  a.o_t = p.out_t;
  a.o_h = p.out_h;
  a.kc_b = p.kc_block;
  a.kc_t = p.kc_token;
  a.kc_h = p.kc_head;
  a.vc_b = p.vc_block;
  a.vc_t = p.vc_token;
  a.vc_h = p.vc_head;
  a.ld_table = p.ld_table;
  a.window = p.window;
  a.R = (int32_t)R;
  a.Hq = (int32_t)Hq;
  a.Hkv = (int32_t)Hkv;
  a.D = (int32_t)D;
  a.gq = (int32_t)(Hq / Hkv);
  a.num_blocks = (int32_t)p.num_blocks;
  a.bs = (int32_t)p.block_size;
  a.max_blocks = (int32_t)p.max_blocks;
  a.page = Divisor((uint32_t)p.block_size);
  a.whole16 = p.block_size % 16 == 0;
  a.scale2 = p.scale * 1.4426950408889634f * p.k_scale;
  a.v_scale = p.v_scale;
  cudaStream_t st = as_stream(stream);
  const bool f8 = p.cache_dtype == REMORA_B200_E4M3;
  if (p.dtype == REMORA_B200_BF16)
    return f8 ? launch_shape<__nv_bfloat16, __nv_fp8_e4m3>(a, p.workspace, st)
              : launch_shape<__nv_bfloat16, __nv_bfloat16>(a, p.workspace, st);
  return f8 ? launch_shape<__half, __nv_fp8_e4m3>(a, p.workspace, st)
            : launch_shape<__half, __half>(a, p.workspace, st);
}
