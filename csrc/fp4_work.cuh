// Shared by the attention kernels over the 4-bit K / V cache: small conversions, the list of work
// that blocks take equal parts of, and the kernel that joins what is cut between them.
#pragma once
#include "common.cuh"
#include "fp4_kv.cuh"

namespace sv4 {
namespace fp4 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMaxFloat = 3.4028235e38f;   // factors of scores stay finite and above zero: 0 times
constexpr float kMinFloat = 1.1754944e-38f;  // infinity (a mask's, too) would be NaN

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
// 2^(a - b) for a <= b, both possibly -inf
__device__ __forceinline__ float shrink(float a, float b) { return a == b ? 1.f : ex2(a - b); }

// c tanh(s / c) in log2 units, s = v f (natural units).  1 - 2 / (1 + e^2x) has an error of some 2^-21 whatever its size
// (two approximations and what the 1 leaves of them), which c repeats: 3e-5 at kRoundCap.  Above that, and
// where it costs little, x below 1/4 takes the series of tanh, whose next term is 2^-26 of it.
constexpr float kRoundCap = 64.f;
struct Cap {
  float size, twice, once;
  __device__ __forceinline__ Cap() {}
  __device__ __forceinline__ Cap(float c, float f) {
    size = fminf(c * kLog2e, kMaxFloat);
    once = fminf(f * fminf(1.f / c, kMaxFloat), kMaxFloat);
    twice = fminf(once * (2.f * kLog2e), kMaxFloat);
  }
  __device__ __forceinline__ float tanh_of(float v) const { return 1.f - __fdividef(2.f, 1.f + ex2(v * twice)); }
  __device__ __forceinline__ float round(float v) const { return __fmul_rn(size, tanh_of(v)); }
  __device__ __forceinline__ float exact(float v) const {
    const float x = v * once, y = x * x;
    const float series = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
    return __fmul_rn(size, fabsf(x) < 0.25f ? series : tanh_of(v));
  }
};

// Maxima above this are spaced by 2^-7 and more.  How far a row's maximum may lag behind the scores: fp16
// holds p (times 2^15) up to 2^15.99, and 0.9 is 0.9 only where fp32 is fine enough.
constexpr float kCoarse = 65536.f, kLag = 0.9f;

__device__ __forceinline__ float2 two_floats(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
__device__ __forceinline__ float2 two_floats(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Few {
  T v[N];
};

// What the keys keep of the whole when a sink logit joins the denominator: their maximum is `top`
// (log2 units) and their sum of p (times 2^15) is l.
__device__ __forceinline__ float share_beside(float sink, float top, float l) {
  if (l == 0.f) return 0.f;  // no key
  const float s2 = sink * kLog2e;
  if (s2 <= top) return l / (l + ex2(s2 - top + 15.f));
  const float mine = l * ex2(top - s2);
  return mine / (mine + 32768.f);
}

// A block of zeros is written with the smallest scale, byte 1, which blocks of up to 6 * 2^-126 have too.
__device__ __forceinline__ bool zero_block(uint4 codes) { return ((codes.x | codes.y | codes.z | codes.w) & 0x77777777u) == 0; }
// A row's scale bytes, 0 for its blocks of zeros.
__device__ __forceinline__ uint32_t without_zeros(uint32_t word, int n, const uint8_t* codes) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n && ((word >> (8 * i)) & 255u) == 1u && zero_block(*reinterpret_cast<const uint4*>(codes + 16 * i)))
      word &= ~(255u << (8 * i));
  return word;
}

// Extremes of the scale bytes of a row (NaN blocks, and zero blocks as byte 0, left out).
__device__ __forceinline__ void scale_range(uint32_t word, int n, int& lo, int& hi, bool& nan) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= n) break;
    const int b = (word >> (8 * i)) & 255;
    if (b == 255) nan = true;
    else if (b > 0) {
      lo = min(lo, b);
      hi = max(hi, b);
    }
  }
}

// The lowest window of exponents: its unit, 2^(bias - 112), is fp32's smallest power (2^-126), and every
// byte up to 14 lies in it.
constexpr int kLeastBias = -14;

// Windows are added to the sums in fp32, in units of 1, or of 2^kLargeUnit from the first tile on that has a
// V scale above kLargeByte: with 2^24 keys and p up to 2^16 sums stay below 2^122 either way.  Beside such
// values (2^79 and up) what is below 2^-110 is lost.
constexpr int kLargeByte = 206, kLargeUnit = 48;
// x 2^e + y for e in [-252, 127]
struct Power {
  float a, b;
  __device__ __forceinline__ explicit Power(int e) : a(pow2f(max(e, -126))), b(pow2f(max(min(e + 126, 0), -126))) {}
  __device__ __forceinline__ float add(float x, float y) const { return fmaf(x * a, b, y); }
};

// fp16 bits of 2^(byte - bias - 15) for bytes in (bias, bias + 28], else 0; byte 0 is never written and reads as 0.
__device__ __forceinline__ uint32_t scale_bits(int byte, int bias) {
  const uint32_t f = static_cast<uint32_t>(byte - bias);
  return f <= 28u && byte != 0 ? f << 10 : 0u;
}

// The work as one list: for every sequence b, `row_tiles` (K / V head, Rows query rows) segments of
// Cost + tiles(b) units each, the last tiles(b) of them tiles of Tile keys; Cost is what a segment
// costs beside its tiles (queries, first copies, join).  Block i of the grid takes the units
// [i per, (i + 1) per), so blocks have equal work whatever the lengths; a segment whose tiles lie in
// several blocks is joined by the second kernel.  tiles(b) spans what any of the T tokens may see.
struct Span {
  int len, start, tiles;  // sequence length, the tile boundary at or before the first key that anyone sees
};

template <int Tile, int Cost, int Rows, int Least>
struct Work {
  static constexpr int kTile = Tile, kRows = Rows;

  __device__ static int row_tiles_of(const Fp4AttnArgs& a) { return a.Hk * ((a.H / a.Hk * a.T + Rows - 1) / Rows); }

  __device__ static Span span_of(const Fp4AttnArgs& a, int b) {
    Span s;
    s.len = min(max(0, a.lengths[b]), a.P * a.R);
    const int first = a.window > 0 ? max(0, s.len - a.T + 1 - a.window) : 0;
    s.start = first & ~(a.R % 32 == 0 ? 31 : 15);
    s.tiles = s.len > 0 ? (s.len - s.start + Tile - 1) / Tile : 0;
    return s;
  }
  __device__ static int units_of(const Span& s) { return s.tiles > 0 ? s.tiles + Cost : 0; }

  // Sum of a segment's units for b < upto and over all b (every thread gets both).  Each warp counts for
  // itself while that takes few loads, else the block's warps share them and meet.
  __device__ static void count_units(const Fp4AttnArgs& a, int upto, int& before, int& all) {
    __shared__ int part[2][32];
    const bool alone = a.B <= 256;
    const int step = alone ? 32 : blockDim.x;
    int mine = 0, below = 0;
#pragma unroll 2
    for (int b = alone ? threadIdx.x & 31 : threadIdx.x; b < a.B; b += step) {
      const int n = units_of(span_of(a, b));
      mine += n;
      if (b < upto) below += n;
    }
    all = __reduce_add_sync(0xffffffffu, mine);
    before = __reduce_add_sync(0xffffffffu, below);
    if (alone) return;
    if ((threadIdx.x & 31) == 0) {
      part[0][threadIdx.x >> 5] = before;
      part[1][threadIdx.x >> 5] = all;
    }
    __syncthreads();
    before = all = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x + 31) / 32; ++w) {
      before += part[0][w];
      all += part[1][w];
    }
  }

  // Units per block: at least `Least` tiles.
  __device__ static int units_per_block(const Fp4AttnArgs& a, int total) {
    return max(Least, static_cast<int>((static_cast<uint32_t>(total) + a.blocks - 1) / a.blocks));
  }

  // A block's place in the list, and the steps from segment to segment.
  int left, b, y, from_unit;  // units left; the segment (sequence, row tile) and the unit in it
  Span sp;

  // False if there is nothing for this block.
  __device__ bool begin(const Fp4AttnArgs& a, int row_tiles) {
    const int lane = threadIdx.x & 31;
    int ignored, total;
    count_units(a, 0, ignored, total);
    total *= row_tiles;
    const int per = units_per_block(a, total);
    if (static_cast<int64_t>(blockIdx.x) * per >= total) return false;
    int skip = blockIdx.x * per;  // into the sequences from b on
    left = min(total - skip, per);
    b = 0;
    while (true) {  // 32 sequences at a time
      const int n = b + lane < a.B ? units_of(span_of(a, b + lane)) * row_tiles : 0;
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, skip < upto);
      if (past != 0) {
        const int here = __ffs(past) - 1;
        skip -= __shfl_sync(0xffffffffu, upto - n, here);
        b += here;
        break;
      }
      skip -= __shfl_sync(0xffffffffu, upto, 31);
      b += 32;
    }
    sp = span_of(a, b);
    y = skip / units_of(sp);
    from_unit = skip - y * units_of(sp);
    return true;
  }
  __device__ int units() const { return min(left, units_of(sp) - from_unit); }
  __device__ int from_tile() const { return max(0, from_unit - Cost); }
  // Tiles of this segment; 0 or less: only the segment's cost.
  __device__ int take() const { return from_unit + units() - Cost - from_tile(); }
  // False if that was the last segment.
  __device__ bool next(const Fp4AttnArgs& a, int row_tiles) {
    left -= units();
    if (left == 0) return false;
    from_unit = 0;
    if (++y == row_tiles) {
      y = 0;
      do sp = span_of(a, ++b);
      while (sp.tiles == 0);
    }
    return true;
  }
  // The part of this block that takes the segment's rows: 1 if its first tile is here, else 0.
  __device__ int64_t part_row() const { return (blockIdx.x * 2 + (from_tile() == 0 ? 1 : 0)) * static_cast<int64_t>(Rows); }
  __device__ bool whole() const { return from_tile() == 0 && take() == sp.tiles; }

  // Host: segments, a bound on the units, and blocks for `per_sm` of them on an SM.
  static int64_t segments(const Fp4AttnArgs& a) {
    return static_cast<int64_t>(a.B) * a.Hk * ((static_cast<int64_t>(a.H / a.Hk) * a.T + Rows - 1) / Rows);
  }
  static int64_t most_units(const Fp4AttnArgs& a) {
    const int64_t rows = static_cast<int64_t>(a.P) * a.R, seen = static_cast<int64_t>(a.window) + a.T + 31;
    const int64_t keys = a.window > 0 && seen < rows ? seen : rows;
    return segments(a) * ((keys + Tile - 1) / Tile + Cost);
  }
  static int blocks(const Fp4AttnArgs& a, int per_sm) {
    const int64_t few = (most_units(a) + Least - 1) / Least;
    return static_cast<int>(few < 1 ? 1 : few < 148 * per_sm ? few : 148 * per_sm);
  }
};

// Joins the parts of a segment's rows, always in the same order; a segment that one block had whole
// is done, one without keys is zero.  A block takes kRowsHere rows, so that each has 8 / kRowsHere
// warps for its parts: one row where a segment may be cut into 16 parts or more, else eight (64
// segments of 16 rows: 1024 blocks 12 us, 128 blocks 10 us, of which all but 2 hide behind the tiles).
constexpr int kJoinWarps = 8;

template <typename T, int D, typename W, int kRowsHere>
__global__ void __launch_bounds__(kJoinWarps * 32) fp4_attn_join_kernel(const Fp4AttnArgs a) {
  constexpr int kX = D / 32, kRows = W::kRows, kDeep = kJoinWarps / kRowsHere;
  __shared__ float sum[kJoinWarps][D];
  __shared__ float2 ml[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, deep = warp % kDeep;
  const int G = a.H / a.Hk;
  const int tiles_per_head = (G * a.T + kRows - 1) / kRows, row_tiles = a.Hk * tiles_per_head;
  constexpr int kPerSegment = kRows / kRowsHere;
  const int in_tile = blockIdx.x % kPerSegment * kRowsHere + warp / kDeep;
  const int seg = blockIdx.x / kPerSegment, b = seg / row_tiles, y = seg - b * row_tiles;
  const int i = (y % tiles_per_head) * kRows + in_tile;  // query row of the head
  const int h = y / tiles_per_head * G + i % G;

  int before, total;
  W::count_units(a, b, before, total);
  if (threadIdx.x == 0 && a.lengths[b] > a.P * a.R) record_error(a.err, kErrBounds);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Span sp = W::span_of(a, b);
  T* out = static_cast<T*>(a.out) + ((static_cast<int64_t>(b) * a.H + h) * a.T + i / G) * D + lane * kX;
  const bool here = i < G * a.T;
  if (sp.tiles == 0) {
    Few<T, kX> zero;
#pragma unroll
    for (int d = 0; d < kX; ++d) zero.v[d] = static_cast<T>(0.f);
    if (here && deep == 0) *reinterpret_cast<Few<T, kX>*>(out) = zero;
    return;
  }
  const int per = W::units_per_block(a, total * row_tiles);
  const int begin = before * row_tiles + (y + 1) * W::units_of(sp) - sp.tiles;  // its first tile
  const int block0 = begin / per, block1 = (begin + sp.tiles - 1) / per;
  if (block0 == block1) return;

  float top = -INFINITY, l = 0.f, o[kX] = {};
  if (here) {
#pragma unroll 4
    for (int x = block0 + deep; x <= block1; x += kDeep) {
      // only the first can have begun at or behind its block's first unit
      const int64_t slot = (static_cast<int64_t>(x) * 2 + (x == block0 && begin >= x * per ? 1 : 0)) * kRows + in_tile;
      const float2 p = a.part_ml[slot];
      const Few<float, kX> v = *reinterpret_cast<const Few<float, kX>*>(a.part_out + slot * D + lane * kX);
      const float next = fmaxf(top, p.x);
      const float keep = l * shrink(top, next), add = p.y * shrink(p.x, next);  // a part without keys adds 0
      top = next;
      l = keep + add;
      const float old = l == 0.f ? 0.f : keep / l, now = l == 0.f ? 0.f : add / l;  // o is the mean so far
#pragma unroll
      for (int d = 0; d < kX; ++d) o[d] = o[d] * old + v.v[d] * now;
    }
  }
  if constexpr (kDeep > 1) {
#pragma unroll
    for (int d = 0; d < kX; ++d) sum[warp][lane * kX + d] = o[d];
    if (lane == 0) ml[warp] = make_float2(top, l);
    __syncthreads();
    if (deep != 0) return;
    for (int w = warp + 1; w < warp + kDeep; ++w) {
      const float2 p = ml[w];
      const float next = fmaxf(top, p.x);
      const float keep = l * shrink(top, next), add = p.y * shrink(p.x, next);
      top = next;
      l = keep + add;
      const float old = l == 0.f ? 0.f : keep / l, now = l == 0.f ? 0.f : add / l;
#pragma unroll
      for (int d = 0; d < kX; ++d) o[d] = o[d] * old + sum[w][lane * kX + d] * now;
    }
  }
  if (!here) return;
  const float keep = a.sink != nullptr ? share_beside(a.sink[h], top, l) : 1.f;
  Few<T, kX> r;
#pragma unroll
  for (int d = 0; d < kX; ++d) r.v[d] = static_cast<T>(o[d] * keep);
  *reinterpret_cast<Few<T, kX>*>(out) = r;
}

// The join of segments of W, which may be set up while the last blocks run: it waits where it reads.
template <typename T, int D, typename W>
void launch_join(const Fp4AttnArgs& a, cudaStream_t stream) {
  const int64_t segments = W::segments(a);
  const bool deep = a.blocks >= 16 * segments;
  cudaLaunchConfig_t join{};
  join.gridDim = dim3(static_cast<unsigned>(segments * W::kRows / (deep ? 1 : 8)));
  join.blockDim = dim3(kJoinWarps * 32);
  join.stream = stream;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  join.attrs = &early;
  join.numAttrs = 1;
  if (deep) cudaLaunchKernelEx(&join, fp4_attn_join_kernel<T, D, W, 1>, a);
  else cudaLaunchKernelEx(&join, fp4_attn_join_kernel<T, D, W, 8>, a);
}

}  // namespace fp4
}  // namespace sv4
