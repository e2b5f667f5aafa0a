// Attention over the paged 4-bit K / V cache for few query rows per K / V head (decoding).
//
//   s_j = scale q . k_j (softcapped), p_j = 2^(s_j log2 e - m), out = sum p_j v_j / sum p_j
//
// with the running maximum m and sum of a one-pass softmax.  The cache is read once: 17/16 d
// bytes per token and K / V head are the traffic, and what bounds the kernel next to it is the
// work of turning codes into operands.  So:
//
// * A warp owns 16 query rows (the G = H / Hk heads of a K / V head, times T tokens) and walks
//   over tiles of 32 keys on its own: copies four tiles ahead (cp.async), no block-wide waits.
//   A block's four warps take turns over the tiles of one slice of the keys and join at its end;
//   a long sequence is cut into slices over blocks, joined by a second small kernel.
// * Products run on mma.sync m16n8k16 in fp16, fp32 sums: with one to sixteen rows per head a
//   128-row tcgen05 tile would be 7/8 empty.  Codes become fp16 pairs with cvt.e2m1x2, exact.
// * K and V scales are powers of two, applied to the fp16 pairs: exact while the exponent is in
//   [-14, 13].  A tile with scales outside takes other exponents for K (28 from its own largest
//   down) and runs its V product once per window of 28 exponents, the sums moved from unit to
//   unit by powers of two.
// * q is scaled by a power of two per row to the top of fp16's range (bf16 keeps its 8 bits, what
//   falls below 2^-38 of the row's largest is lost).  p is held times 2^15: fp16's 11 bits for
//   weights down to 2^-29 of the largest.
// * Operand order: dims and keys may be summed in any order, so a thread's operands are chosen to
//   lie together: 4 bytes of a block per key for K; for V the d/16 bytes of its d/8 output dims,
//   two keys' nibbles merged into the bytes that cvt turns into a pair.
#include "fp4_kv.cuh"

#include "common.cuh"

namespace sv4 {
namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;  // keys per warp step
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct Cfg {
  static constexpr int kC = D / 32;           // scale blocks per row
  static constexpr int kCode = kTile * D / 2;  // bytes of K (or V) codes per stage
  static constexpr int kScale = kTile * kC;
  static constexpr int kStage = 2 * kCode + 2 * kScale;
  static constexpr int kStages = 4;
  static constexpr int kKTable = kTile * kC * 4;    // K scales as fp16 pairs, (row, block)
  static constexpr int kVStride = kTile + 4;        // V scales fp16, (block, row), rows in pairs
  static constexpr int kVTable = kC * kVStride * 2;
  static constexpr int kWarpBytes = (kStages * kStage + kKTable + kVTable + 15) / 16 * 16;
  static constexpr int kJoin = kWarps * 16 * D * 4 + kWarps * 16 * 8;
  static constexpr int kSmem = kWarps * kWarpBytes > kJoin ? kWarps * kWarpBytes : kJoin;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Four bytes of two codes each -> four fp16 pairs (low code in the low half).
__device__ __forceinline__ void codes_to_half2(uint32_t w, uint32_t (&o)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ float2 two_floats(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
__device__ __forceinline__ float2 two_floats(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// What the keys keep of the whole when a sink logit joins the denominator: their maximum is `top`
// (log2 units) and their sum of p (times 2^15) is l.
__device__ __forceinline__ float share_beside(float sink, float top, float l) {
  if (l == 0.f) return 0.f;  // no key
  const float s2 = sink * kLog2e;
  if (s2 <= top) return l / (l + ex2(s2 - top + 15.f));
  const float mine = l * ex2(top - s2);
  return mine / (mine + 32768.f);
}

// Swizzled byte offset of 16-byte piece `piece` of row `row` in a tile of codes, such that what a
// warp reads at once falls into different banks.
template <int D>
__device__ __forceinline__ int k_at(int row, int piece) {
  constexpr int C = D / 32;
  const int x = C == 4 ? (row >> 1) & 3 : C == 2 ? (row >> 2) & 1 : 0;
  return row * (D / 2) + ((piece ^ x) << 4);
}
template <int D>
__device__ __forceinline__ int v_at(int row, int piece) {
  const int x = D == 128 ? (row & 2) : 0;
  return row * (D / 2) + ((piece ^ x) << 4);
}

// Extremes of the scale bytes of the tile's rows (NaN blocks and zero blocks, bytes 0 and 1, left out).
__device__ __forceinline__ void scale_range(uint32_t word, int n, int& lo, int& hi, bool& nan) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= n) break;
    const int b = (word >> (8 * i)) & 255;
    if (b == 255) nan = true;
    else if (b > 1) {
      lo = min(lo, b);
      hi = max(hi, b);
    }
  }
}

// fp16 bits of 2^(byte - bias - 15) for bytes in (bias, bias + 28], else 0.
__device__ __forceinline__ uint32_t scale_bits(int byte, int bias) {
  const uint32_t f = static_cast<uint32_t>(byte - bias);
  return f <= 28u ? f << 10 : 0u;
}

// The sums' unit moved from 2^from to 2^to: exact but for what leaves fp32's range at the small
// end.  Towards smaller units only as far as the largest sum stays finite; returns the unit.
template <int N>
__device__ __forceinline__ int to_unit(float (&acc)[N][4], int from, int to) {
  float big = 0.f;
#pragma unroll
  for (int x = 0; x < N; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) big = fmaxf(big, fabsf(acc[x][y]));
  const int top = static_cast<int>(__reduce_max_sync(0xffffffffu, __float_as_uint(big)) >> 23) - 127;
  int up = max(-126, min(126, from - to));
  up = min(up, max(0, 96 - top));
  const float f = pow2f(up);
#pragma unroll
  for (int x = 0; x < N; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) acc[x][y] *= f;
  return from - up;
}

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32, D == 128 ? 3 : 4) fp4_attn_rows_kernel(const Fp4AttnArgs a) {
  using C = Cfg<D>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int G = a.H / a.Hk;
  const int tiles_per_head = (G * a.T + 15) / 16;
  const int split = blockIdx.x % a.splits, tile = blockIdx.x / a.splits, b = blockIdx.y;
  const int head = tile / tiles_per_head, row0 = (tile % tiles_per_head) * 16;
  const int rows = min(16, G * a.T - row0);

  int len = max(0, a.lengths[b]);
  const int cap = a.P * a.R;
  if (len > cap) {
    if (threadIdx.x == 0) record_error(a.err, kErrBounds);
    len = cap;
  }
  // keys that row i (token t) may see: [lo, hi)
  auto limits = [&](int i, int& lo, int& hi) {
    const int t = (row0 + min(i, rows - 1)) / G;
    hi = len - a.T + t + 1;
    lo = a.window > 0 ? max(0, hi - a.window) : 0;
  };
  int lo0, hi0, lo1, hi1, first, last, inner_lo, inner_hi;
  limits(g, lo0, hi0);
  limits(g + 8, lo1, hi1);
  limits(0, first, inner_hi);
  limits(15, inner_lo, last);
  last = max(last, 0);
  const int start = first & ~15;
  const int n_tiles = (last - start + kTile - 1) / kTile;  // 0 when no row has a key
  const int per = (n_tiles + a.splits - 1) / a.splits;
  const int t_begin = min(n_tiles, split * per), t_end = min(n_tiles, t_begin + per);
  const int mine = t_end - t_begin > warp ? (t_end - t_begin - warp + kWarps - 1) / kWarps : 0;

  // ---- q as the A operand: row g and g + 8, dims 32 b + 8 c .. + 7, scaled to fp16's top
  uint32_t qf[C::kC][8];
  float unit0, unit1;
  {
    const T* q = static_cast<const T*>(a.q) + b * a.q_b;
    float unit[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = row0 + min(g + 8 * r, rows - 1);
      const T* row = q + (head * G + i % G) * a.q_h + (i / G) * a.q_t;
      uint4 raw[C::kC];
      float amax = 0.f;
#pragma unroll
      for (int k = 0; k < C::kC; ++k) {
        raw[k] = *reinterpret_cast<const uint4*>(row + 32 * k + 8 * c);
        const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float2 f = two_floats(w[x], T{});
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int x = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
      const int up = amax > 0.f && x < 128 ? min(14 - x, 126) : 0;
      const float f = pow2f(up);
      unit[r] = pow2f(max(-up, -126));
#pragma unroll
      for (int k = 0; k < C::kC; ++k) {
        const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float2 v = two_floats(w[y], T{});
          // pair y: step y / 2, k half y % 2 -> A register 2 * (y % 2) + r
          qf[k][(y >> 1) * 4 + (y & 1) * 2 + r] = pack_half2(v.x * f, v.y * f);
        }
      }
    }
    unit0 = unit[0];
    unit1 = unit[1];
  }
  const float nat = a.softcap > 0.f ? a.scale : a.scale * kLog2e;  // softcap works on natural units

  // ---- per-warp ring of key tiles
  uint8_t* ring = smem + warp * C::kWarpBytes;
  uint32_t* ktab = reinterpret_cast<uint32_t*>(ring + C::kStages * C::kStage);
  __half* vtab = reinterpret_cast<__half*>(ring + C::kStages * C::kStage + C::kKTable);
  const uint32_t ring_u = smem_u32(ring);
  const int* table = a.table + static_cast<int64_t>(b) * a.P;

  // Where the halves (16 keys) of sixteen coming tiles lie: lane 2 i + h holds half h of tile i.
  auto look_up = [&](int batch, const uint8_t*& at, int& in_page) {
    const int i = batch * 16 + (lane >> 1);
    const int key = start + (t_begin + warp + i * kWarps) * kTile + (lane & 1) * 16;
    at = nullptr;
    in_page = -1;
    if (i < mine && key < last) {
      const int slot = key / a.R;
      const int page = table[slot];
      if (index_ok(page, 0, a.n_pages, a.err)) {
        at = a.pages + page * a.page_stride + static_cast<int64_t>(head) * a.slab;
        in_page = key - slot * a.R;
      }
    }
  };
  const uint8_t *at_now, *at_next;
  int in_now, in_next;
  look_up(0, at_now, in_now);
  look_up(1, at_next, in_next);
  uint32_t present = 0;  // two bits per stage: its halves that were copied

  auto issue = [&](int i) {
    if (i < mine) {
      if ((i & 15) == 0 && i > 0) {
        at_now = at_next;
        in_now = in_next;
        look_up((i >> 4) + 1, at_next, in_next);
      }
      const int stage = i % C::kStages;
      const uint32_t dst = ring_u + stage * C::kStage;
      present &= ~(3u << (2 * stage));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int from = ((i & 15) << 1) | h;
        const uint8_t* slab = reinterpret_cast<const uint8_t*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(at_now), from));
        const int r = __shfl_sync(0xffffffffu, in_now, from);
        if (slab == nullptr) continue;
        present |= 1u << (2 * stage + h);
        const uint8_t* k = slab + r * (D / 2);
        const uint8_t* v = k + a.R * (D / 2);
#pragma unroll
        for (int x = lane; x < 16 * C::kC; x += 32) {  // 16 rows of kC pieces
          const int row = h * 16 + x / C::kC, piece = x % C::kC;
          copy16(dst + k_at<D>(row, piece), k + x * 16);
          copy16(dst + C::kCode + v_at<D>(row, piece), v + x * 16);
        }
        // 16 rows of kC scale bytes: kC pieces for K and for V
        if (lane < 2 * C::kC) {
          const int kv = lane / C::kC, piece = lane % C::kC;
          copy16(dst + 2 * C::kCode + kv * C::kScale + h * 16 * C::kC + piece * 16,
                 slab + a.R * D + (kv * a.R + r) * C::kC + piece * 16);
        }
      }
    }
    copy_commit();
  };

  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float acc[D / 8][4];
#pragma unroll
  for (int x = 0; x < D / 8; ++x) acc[x][0] = acc[x][1] = acc[x][2] = acc[x][3] = 0.f;
  int out_unit = 0;                  // acc holds sums times 2^-out_unit
  float poison0 = 0.f, poison1 = 0.f;  // NaN once a visible V block was NaN

#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) issue(i);

  for (int i = 0; i < mine; ++i) {
    issue(i + C::kStages - 1);
    copy_wait<C::kStages - 1>();
    __syncwarp();
    const int stage = i % C::kStages;
    const uint8_t* buf = ring + stage * C::kStage;
    const int key0 = start + (t_begin + warp + i * kWarps) * kTile;
    const uint32_t halves = (present >> (2 * stage)) & 3u;

    // ---- scales: lane = row
    uint32_t kw = 0, vw = 0;
    const int my_key = key0 + lane;
    if (((halves >> (lane >> 4)) & 1u) && my_key >= first && my_key < last) {
      if constexpr (C::kC == 4) {
        kw = *reinterpret_cast<const uint32_t*>(buf + 2 * C::kCode + lane * 4);
        vw = *reinterpret_cast<const uint32_t*>(buf + 2 * C::kCode + C::kScale + lane * 4);
      } else if constexpr (C::kC == 2) {
        kw = *reinterpret_cast<const uint16_t*>(buf + 2 * C::kCode + lane * 2);
        vw = *reinterpret_cast<const uint16_t*>(buf + 2 * C::kCode + C::kScale + lane * 2);
      } else {
        kw = buf[2 * C::kCode + lane];
        vw = buf[2 * C::kCode + C::kScale + lane];
      }
    }
    int klo = 255, khi = 0, vlo = 255, vhi = 0;
    bool knan = false, vnan = false;
    scale_range(kw, C::kC, klo, khi, knan);
    scale_range(vw, C::kC, vlo, vhi, vnan);
    // exponents [-14, 13] are bytes 113 .. 140
    const bool plain = __all_sync(0xffffffffu, min(klo, vlo) > 112 && max(khi, vhi) <= 140 && !knan && !vnan);
    int kbias = 112, vbias = 112;
    if (!plain) {
      khi = __reduce_max_sync(0xffffffffu, khi);
      vhi = __reduce_max_sync(0xffffffffu, vhi);
      kbias = max(khi - 28, -14);
      vbias = max(vhi - 28, 2);
    }
    {
      uint32_t s[C::kC];
#pragma unroll
      for (int x = 0; x < C::kC; ++x) {
        const int byte = (kw >> (8 * x)) & 255;
        s[x] = scale_bits(byte, kbias) * 0x10001u;
        if (byte == 255) s[x] = 0x7e007e00u;
      }
      if constexpr (C::kC == 4) *reinterpret_cast<uint4*>(ktab + lane * 4) = make_uint4(s[0], s[1], s[2], s[3]);
      else if constexpr (C::kC == 2) *reinterpret_cast<uint2*>(ktab + lane * 2) = make_uint2(s[0], s[1]);
      else ktab[lane] = s[0];
    }
    const int pair_at = (lane & ~7) | ((lane & 3) * 2) | ((lane >> 2) & 1);  // keys c and c + 4 side by side
    auto put_v_scales = [&](int bias) {
#pragma unroll
      for (int x = 0; x < C::kC; ++x)
        vtab[x * C::kVStride + pair_at] = __ushort_as_half(static_cast<uint16_t>(scale_bits((vw >> (8 * x)) & 255, bias)));
    };
    put_v_scales(vbias);
    __syncwarp();

    // ---- scores: column n of key group j is key 8 j + n / 2 + 4 (n % 2)
    float s[4][4];
    const int k_row = (g >> 1) + 4 * (g & 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
      const int row = 8 * j + k_row;
      uint32_t sc[C::kC];
      if constexpr (C::kC == 4) {
        const uint4 t = *reinterpret_cast<const uint4*>(ktab + row * 4);
        sc[0] = t.x; sc[1] = t.y; sc[2] = t.z; sc[3] = t.w;
      } else if constexpr (C::kC == 2) {
        const uint2 t = *reinterpret_cast<const uint2*>(ktab + row * 2);
        sc[0] = t.x; sc[1] = t.y;
      } else {
        sc[0] = ktab[row];
      }
#pragma unroll
      for (int k = 0; k < C::kC; ++k) {
        uint32_t h[4];
        codes_to_half2(*reinterpret_cast<const uint32_t*>(buf + k_at<D>(row, k) + c * 4), h);
#pragma unroll
        for (int y = 0; y < 4; ++y) h[y] = mul2(h[y], sc[k]);
        mma16816(s[j], qf[k][0], qf[k][1], qf[k][2], qf[k][3], h[0], h[1]);
        mma16816(s[j], qf[k][4], qf[k][5], qf[k][6], qf[k][7], h[2], h[3]);
      }
    }

    // ---- softmax in units of log2
    float f0 = unit0 * nat, f1 = unit1 * nat;
    if (!plain) {
      const float km = pow2f(max(kbias - 112, -126));
      f0 *= km;
      f1 *= km;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j][0] *= f0;
      s[j][1] *= f0;
      s[j][2] *= f1;
      s[j][3] *= f1;
    }
    if (a.softcap > 0.f) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[j][x] = a.softcap * kLog2e * tanhf(s[j][x] / a.softcap);
    }
    if (halves != 3u || key0 < inner_lo || key0 + kTile > inner_hi) {  // some row does not see some key
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int key = key0 + 8 * j + c + 4 * x;
          const bool there = (halves >> (j >> 1)) & 1u;
          if (!there || key < lo0 || key >= hi0) s[j][x] = -INFINITY;
          if (!there || key < lo1 || key >= hi1) s[j][2 + x] = -INFINITY;
        }
      }
    }
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x0 = fmaxf(x0, fmaxf(s[j][0], s[j][1]));
      x1 = fmaxf(x1, fmaxf(s[j][2], s[j][3]));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
    }
    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
    const bool moved = n0 != m0 || n1 != m1;
    if (__any_sync(0xffffffffu, moved)) {
      const float keep0 = n0 == m0 ? 1.f : ex2(m0 - n0), keep1 = n1 == m1 ? 1.f : ex2(m1 - n1);
      l0 *= keep0;
      l1 *= keep1;
#pragma unroll
      for (int x = 0; x < D / 8; ++x) {
        acc[x][0] *= keep0;
        acc[x][1] *= keep0;
        acc[x][2] *= keep1;
        acc[x][3] *= keep1;
      }
      m0 = n0;
      m1 = n1;
    }
    // p times 2^15, a row without a key so far keeps p = 0
    const float d0 = m0 == -INFINITY ? 0.f : 15.f - m0, d1 = m1 == -INFINITY ? 0.f : 15.f - m1;
    uint32_t p[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s[j][x] = ex2(s[j][x] + d0);
        s[j][2 + x] = ex2(s[j][2 + x] + d1);
      }
      l0 += s[j][0] + s[j][1];
      l1 += s[j][2] + s[j][3];
      p[j][0] = pack_half2(s[j][0], s[j][1]);
      p[j][1] = pack_half2(s[j][2], s[j][3]);
    }

    // ---- sums of p v: column n of dim group x is dim n d/8 + x
    auto add_values = [&]() {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        constexpr int kWords = D >= 64 ? D / 64 : 1;
        uint32_t w[4][kWords];  // keys c, c + 4, c + 8, c + 12 of the half
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int row = 16 * k + c + 4 * y;
          if constexpr (D == 128) {
            const uint2 t = *reinterpret_cast<const uint2*>(buf + C::kCode + v_at<D>(row, g >> 1) + (g & 1) * 8);
            w[y][0] = t.x;
            w[y][1] = t.y;
          } else if constexpr (D == 64) {
            w[y][0] = *reinterpret_cast<const uint32_t*>(buf + C::kCode + row * 32 + g * 4);
          } else {
            w[y][0] = *reinterpret_cast<const uint16_t*>(buf + C::kCode + row * 16 + g * 2);
          }
        }
        const __half* vs = vtab + (g * D / 256) * C::kVStride + 16 * k + 2 * c;
        const uint32_t sa = *reinterpret_cast<const uint32_t*>(vs), sb = *reinterpret_cast<const uint32_t*>(vs + 8);
#pragma unroll
        for (int z = 0; z < kWords; ++z) {
          uint32_t even_a[4], odd_a[4], even_b[4], odd_b[4];
          codes_to_half2((w[0][z] & 0x0f0f0f0fu) | ((w[1][z] << 4) & 0xf0f0f0f0u), even_a);
          codes_to_half2(((w[0][z] >> 4) & 0x0f0f0f0fu) | (w[1][z] & 0xf0f0f0f0u), odd_a);
          codes_to_half2((w[2][z] & 0x0f0f0f0fu) | ((w[3][z] << 4) & 0xf0f0f0f0u), even_b);
          codes_to_half2(((w[2][z] >> 4) & 0x0f0f0f0fu) | (w[3][z] & 0xf0f0f0f0u), odd_b);
#pragma unroll
          for (int y = 0; y < (D >= 64 ? 4 : 2); ++y) {
            mma16816(acc[8 * z + 2 * y], p[2 * k][0], p[2 * k][1], p[2 * k + 1][0], p[2 * k + 1][1],
                     mul2(even_a[y], sa), mul2(even_b[y], sb));
            mma16816(acc[8 * z + 2 * y + 1], p[2 * k][0], p[2 * k][1], p[2 * k + 1][0], p[2 * k + 1][1],
                     mul2(odd_a[y], sa), mul2(odd_b[y], sb));
          }
        }
      }
    };
    if (plain && out_unit == 0) {
      add_values();
    } else {
      // windows of 28 exponents, the largest first, the sums in the unit of each
      int bias = vbias;
      while (true) {
        const int got = out_unit = to_unit(acc, out_unit, bias - 112);
        const bool limited = got != bias - 112;
        if (limited || bias != vbias) {
          __syncwarp();
          put_v_scales(got + 112);
          __syncwarp();
        }
        add_values();
        if (plain || limited) break;
        int next = 0;  // the largest byte that no window has held yet
#pragma unroll
        for (int x = 0; x < C::kC; ++x) {
          const int byte = (vw >> (8 * x)) & 255;
          if (byte <= bias && byte > 1) next = max(next, byte);
        }
        next = __reduce_max_sync(0xffffffffu, next);
        if (next == 0) break;
        bias = next - 28;
      }
      if (__any_sync(0xffffffffu, vnan)) {
        // a NaN block reaches the rows that see its key: this thread's sums lie in block c d/128
        const int mine_block = c * D / 128;
        for (int y = 0; y < kTile; ++y) {
          const uint32_t word = __shfl_sync(0xffffffffu, vw, y);
          if (((word >> (8 * mine_block)) & 255u) != 255u) continue;
          const int key = key0 + y;
          if (key >= lo0 && key < hi0) poison0 = NAN;
          if (key >= lo1 && key < hi1) poison1 = NAN;
        }
      }
    }
    __syncwarp();  // the stage and the scale tables are free again
  }

  // ---- join the block's warps
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, o);
    l1 += __shfl_xor_sync(0xffffffffu, l1, o);
  }
  copy_wait<0>();
  __syncthreads();  // all rings are free
  float* sum = reinterpret_cast<float*>(smem);                            // (warp, row, dim)
  float2* ml = reinterpret_cast<float2*>(smem + kWarps * 16 * D * 4);  // (warp, row)
  if (c == 0) {
    ml[warp * 16 + g] = make_float2(m0, l0);
    ml[warp * 16 + g + 8] = make_float2(m1, l1);
  }
  __syncthreads();
  // every part divided by the block's sum of p, so that no unit can overflow
  float big[2] = {-INFINITY, -INFINITY}, part[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) big[r] = fmaxf(big[r], ml[w * 16 + g + 8 * r].x);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 x = ml[w * 16 + g + 8 * r];
      l += x.y * (x.x == big[r] ? 1.f : ex2(x.x - big[r]));
    }
    const float m = r == 0 ? m0 : m1;
    part[r] = l == 0.f ? 0.f : (m == big[r] ? 1.f : ex2(m - big[r])) / l;
  }
  const float unit = pow2f(max(-126, min(126, out_unit)));
#pragma unroll
  for (int x = 0; x < D / 8; ++x) {
    float* row = sum + (warp * 16 + g) * D + x;
    row[2 * c * (D / 8)] = acc[x][0] * part[0] * unit + poison0;
    row[(2 * c + 1) * (D / 8)] = acc[x][1] * part[0] * unit + poison0;
    row += 8 * D;
    row[2 * c * (D / 8)] = acc[x][2] * part[1] * unit + poison1;
    row[(2 * c + 1) * (D / 8)] = acc[x][3] * part[1] * unit + poison1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += kWarps * 32) {
    const int r = i / D, d = i % D;
    float top = -INFINITY, l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * 16 + r].x);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 x = ml[w * 16 + r];
      l += x.y * (x.x == top ? 1.f : ex2(x.x - top));
      o += sum[(w * 16 + r) * D + d];
    }
    const int h = head * G + (row0 + r) % G, t = (row0 + r) / G;
    const int64_t at = (static_cast<int64_t>(b) * a.H + h) * a.T + t;
    if (a.splits > 1) {
      a.part_out[(at * a.splits + split) * D + d] = o;
      if (d == 0) a.part_ml[at * a.splits + split] = make_float2(top, l);
    } else {
      if (a.sink != nullptr) o *= share_beside(a.sink[h], top, l);
      static_cast<T*>(a.out)[at * D + d] = static_cast<T>(o);
    }
  }
}

// Joins the slices of one row, in their order: thread = dim.
template <typename T, int D>
__global__ void __launch_bounds__(D) fp4_attn_join_kernel(const Fp4AttnArgs a) {
  const int64_t row = blockIdx.x;
  const int d = threadIdx.x;
  const float2* ml = a.part_ml + row * a.splits;
  float top = -INFINITY, l = 0.f, o = 0.f;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[s].x);
  for (int s = 0; s < a.splits; ++s) {
    const float2 x = ml[s];
    if (x.y != 0.f) l += x.y * (x.x == top ? 1.f : ex2(x.x - top));
  }
  for (int s = 0; s < a.splits; ++s) {
    const float2 x = ml[s];
    if (x.y == 0.f) continue;  // an empty slice
    o += a.part_out[(row * a.splits + s) * D + d] * (x.y * (x.x == top ? 1.f : ex2(x.x - top)) / l);
  }
  if (a.sink != nullptr) o *= share_beside(a.sink[row / a.T % a.H], top, l);
  static_cast<T*>(a.out)[row * D + d] = static_cast<T>(o);
}

template <typename T, int D>
void launch(const Fp4AttnArgs& a, cudaStream_t stream) {
  const int G = a.H / a.Hk;
  const unsigned blocks = static_cast<unsigned>(a.Hk * ((G * a.T + 15) / 16) * a.splits);
  cudaFuncSetAttribute(fp4_attn_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem);
  fp4_attn_rows_kernel<T, D><<<dim3(blocks, a.B), kWarps * 32, Cfg<D>::kSmem, stream>>>(a);
  if (a.splits > 1)
    fp4_attn_join_kernel<T, D><<<static_cast<unsigned>(static_cast<int64_t>(a.B) * a.H * a.T), D, 0, stream>>>(a);
}

}  // namespace

void fp4_attn_rows(const Fp4AttnArgs& a, int d, bool half, cudaStream_t stream) {
  if (half) {
    if (d == 32) launch<__half, 32>(a, stream);
    else if (d == 64) launch<__half, 64>(a, stream);
    else launch<__half, 128>(a, stream);
  } else {
    if (d == 32) launch<__nv_bfloat16, 32>(a, stream);
    else if (d == 64) launch<__nv_bfloat16, 64>(a, stream);
    else launch<__nv_bfloat16, 128>(a, stream);
  }
}

}  // namespace sv4
