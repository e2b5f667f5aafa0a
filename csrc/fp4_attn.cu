// Attention over the paged 4-bit K / V cache for few query rows per K / V head (decoding).
//
//   s_j = scale q . k_j (softcapped), p_j = 2^(s_j log2 e - m), out = sum p_j v_j / sum p_j
//
// with the running maximum m and sum of a one-pass softmax.  The cache is read once: 17/16 d
// bytes per token and K / V head are the traffic, and what bounds the kernel next to it is the
// work of turning codes into operands.  So:
//
// * A warp owns 8 or 16 query rows (the G = H / Hk heads of a K / V head, times T tokens) and
//   walks over tiles of 32 keys on its own: copies (cp.async) two tiles ahead, no block-wide waits.
//   A block's four warps take turns over its tiles and join at their end.  Blocks take equal parts
//   of the list of all tiles; what is cut between blocks is joined by a second small kernel.
// * Products run on mma.sync m16n8k16 in fp16 with fp32 sums, keys (then dims) as the 16 rows and
//   query rows as the 8 columns: with one to sixteen rows a 128-row tcgen05 tile would be 7/8
//   empty.  Codes become fp16 pairs with cvt.e2m1x2, exact.
// * K and V scales are powers of two, applied to the fp16 pairs: exact while the exponent is in
//   [-14, 13].  A tile with scales outside takes other exponents for K (28 from each key's own
//   largest down, so that no key's size touches another's score) and runs its V product once per window of
//   28 exponents, each added to the sums in fp32.
// * q is scaled by a power of two per row to the top of fp16's range (bf16 keeps its 8 bits, what
//   falls below 2^-38 of the row's largest is lost).  p is held times 2^15: fp16's 11 bits for
//   weights down to 2^-29 of the largest.  A row's maximum is left as it is while the new one is at
//   most 0.9 larger (log2), for which fp16 has room: the sums are rescaled less often.  (Above 2^16
//   fp32 rounds that 0.9: no lag there, and the maximum is taken from the scores before 15 is added.)
// * Operand order: dims and keys may be summed in any order, so a thread's operands are chosen to
//   lie together: d/4 dims of a key for K; for V the d/16 bytes of its d/8 output dims, two keys'
//   nibbles merged into the bytes that cvt turns into a pair.
#include "fp4_work.cuh"

namespace sv4 {
namespace {

using namespace fp4;

constexpr int kWarps = 4;
constexpr int kTile = 32;  // keys per warp step
// What a segment costs a block beside its tiles (queries, first copies, join), in tiles: with 8 blocks
// that begin many short segments come last (prefill chunk 207 us, 176 with 16, 182 with 28).
constexpr int kSegmentCost = 16;

template <int D, int NT>
struct Cfg {
  static constexpr int kRows = 8 * NT;  // query rows of a segment
  using List = Work<kTile, kSegmentCost, kRows, kWarps>;
  static constexpr int kC = D / 32;            // scale blocks per row
  static constexpr int kCode = kTile * D / 2;  // bytes of K (or V) codes per stage
  static constexpr int kScale = kTile * kC;
  static constexpr int kStage = 2 * kCode + 2 * kScale;
  static constexpr int kStages = 3;
  static constexpr int kKTable = kTile * kC * 4;  // K scales as fp16 pairs, (row, block)
  static constexpr int kVStride = kTile + 4;      // V scales fp16, (block, row), rows in pairs
  static constexpr int kVTable = kC * kVStride * 2;
  static constexpr int kWarpBytes = (kStages * kStage + kKTable + kVTable + 15) / 16 * 16;
  static constexpr int kJoin = kWarps * kRows * (D * 4 + 8);
  static constexpr int kSmem = kWarps * kWarpBytes > kJoin ? kWarps * kWarpBytes : kJoin;  // the join reuses the rings
  // Per SM.  16 rows: two blocks with all the registers they want beat three with spills (131072 keys of
  // 8 heads and as many of another length: 99 and 110 us); 8 rows: four beat three (71 and 90 us).
  static constexpr int kBlocks = D == 128 && NT == 2 ? 2 : 4;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The low four bits of every byte from a, the high ones from b.
__device__ __forceinline__ uint32_t low_nibbles_of(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xca;" : "=r"(d) : "r"(0x0f0f0f0fu), "r"(a), "r"(b));  // mask ? a : b
  return d;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 fp16 matrix, a row in four neighbouring lanes' pairs, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, Cfg<D, NT>::kBlocks) fp4_attn_rows_kernel(const Fp4AttnArgs a) {
  using C = Cfg<D, NT>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int G = a.H / a.Hk;
  const int tiles_per_head = (G * a.T + C::kRows - 1) / C::kRows, row_tiles = a.Hk * tiles_per_head;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- per-warp ring of key tiles
  uint8_t* ring = smem + warp * C::kWarpBytes;
  uint32_t* ktab = reinterpret_cast<uint32_t*>(ring + C::kStages * C::kStage);
  __half* vtab = reinterpret_cast<__half*>(ring + C::kStages * C::kStage + C::kKTable);
  const uint32_t ring_u = smem_u32(ring);

  const int scale_half = (lane / C::kC) & 1, scale_kv = lane / (2 * C::kC);
  const int64_t scale_src = static_cast<int64_t>(a.R) * D + scale_kv * a.R * C::kC + lane % C::kC * 16;

  // ---- this block's part of the list
  typename C::List list;
  if (!list.begin(a, row_tiles)) return;
  // the scale's sign (or zero) goes into q; softcap works on natural units
  const float nat = (a.scale != 0.f ? fabsf(a.scale) : 1.f) * (a.softcap > 0.f ? 1.f : kLog2e);

  while (true) {
    const int take = list.take(), from_tile = list.from_tile(), b = list.b, y = list.y;
    const Span sp = list.sp;
    if (take > 0) {
      const int head = y / tiles_per_head, row0 = (y % tiles_per_head) * C::kRows;
      const int rows = min(C::kRows, G * a.T - row0);
      // one past the last key that row i (token t) may see; rows behind the last repeat it
      auto end_of = [&](int i) { return a.T == 1 ? sp.len : sp.len - a.T + (row0 + min(i, rows - 1)) / G + 1; };
      const int last = end_of(C::kRows - 1), inner_hi = end_of(0);
      const int first = a.window > 0 ? max(0, inner_hi - a.window) : 0, inner_lo = a.window > 0 ? max(0, last - a.window) : 0;
      const int mine = take > warp ? (take - warp + kWarps - 1) / kWarps : 0;
      const int base = sp.start + (from_tile + warp) * kTile;  // the warp's first key
      const int* table = a.table + static_cast<int64_t>(b) * a.P;

      // this thread's part of the queries, on its way while the first tiles are found: rows 8 z + g, dims
      // c d/4 .. (c + 1) d/4
      uint4 raw[NT][C::kC];
#pragma unroll
      for (int z = 0; z < NT; ++z) {
        const int i = row0 + min(8 * z + g, rows - 1), t = a.T == 1 ? 0 : i / G;
        const T* row = static_cast<const T*>(a.q) + b * a.q_b + (head * G + i - t * G) * a.q_h + t * a.q_t;
#pragma unroll
        for (int k = 0; k < C::kC; ++k) raw[z][k] = *reinterpret_cast<const uint4*>(row + c * (D / 4) + 8 * k);
      }

      // Where the halves (16 keys) of sixteen coming tiles lie: lane 2 i + h holds half h of tile i.
      auto look_up = [&](int batch, const uint8_t*& slab, int& in_page) {
        const int i = batch * 16 + (lane >> 1);
        const int key = base + i * kWarps * kTile + (lane & 1) * 16;
        slab = nullptr;
        in_page = 0;
        if (i < mine && key < last) {
          const int slot = key / a.R;
          const int page = table[slot];
          if (index_ok(page, 0, a.n_pages, a.err)) {
            slab = a.pages + page * a.page_stride + static_cast<int64_t>(head) * a.slab;
            in_page = key - slot * a.R;
          }
        }
      };
      const uint8_t *slab_now, *slab_next = nullptr;
      int in_now, in_next = 0;
      uint32_t present = 0;  // two bits per stage: its halves that were copied
      int fill = 0, stage = 0;  // the next stages to copy into and to compute

      auto issue = [&](int i) {
        if (i >= mine) return;
        if ((i & 15) == 0 && i > 0) {
          slab_now = slab_next;
          in_now = in_next;
          look_up((i >> 4) + 1, slab_next, in_next);
        }
        const int from = (i & 15) << 1;
        const uint8_t* s0 = reinterpret_cast<const uint8_t*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(slab_now), from));
        const int r0 = __shfl_sync(0xffffffffu, in_now, from);
        const uint8_t* s1 = s0;
        int r1 = r0 + 16;
        if (a.R % kTile != 0) {  // else tiles start at multiples of 32 and lie in one page
          s1 = reinterpret_cast<const uint8_t*>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(slab_now), from + 1));
          r1 = __shfl_sync(0xffffffffu, in_now, from + 1);
        }
        const uint32_t dst = ring_u + fill * C::kStage;
        auto copy_codes = [&](const uint8_t* slab, int r, int to) {  // 16 rows of d/2 bytes
          const uint8_t* k = slab + r * (D / 2) + lane * 16;
          const uint8_t* v = k + a.R * (D / 2);
          if (D >= 64 || lane < 16) {
#pragma unroll
            for (int x = 0; x < (D + 63) / 64; ++x) {
              copy16(dst + to * (D / 2) + lane * 16 + x * 512, k + x * 512);
              copy16(dst + C::kCode + to * (D / 2) + lane * 16 + x * 512, v + x * 512);
            }
          }
        };
        if (s0 != nullptr) copy_codes(s0, r0, 0);
        if (s1 != nullptr) copy_codes(s1, r1, 16);
        // scales: lane (K / V, half, 16-byte piece)
        const uint8_t* sc = scale_half ? s1 : s0;
        if (lane < 4 * C::kC && sc != nullptr)
          copy16(dst + 2 * C::kCode + lane * 16, sc + scale_src + (scale_half ? r1 : r0) * C::kC);
        present = (present & ~(3u << (2 * fill))) | (((s0 != nullptr ? 1u : 0u) | (s1 != nullptr ? 2u : 0u)) << (2 * fill));
        fill = fill + 1 == C::kStages ? 0 : fill + 1;
      };
      look_up(0, slab_now, in_now);
#pragma unroll
      for (int i = 0; i < C::kStages - 1; ++i) {
        issue(i);
        copy_commit();
      }
      if (mine > 16) look_up(1, slab_next, in_next);

      // ---- q as the B operand, scaled to fp16's top
      uint32_t qf[NT][C::kC][4];
      float factor[NT][2];  // raw score -> softmax units, rows 8 z + 2 c + x
      int hi[NT][2];        // one past the last visible key, for the same rows
#pragma unroll
      for (int z = 0; z < NT; ++z) {
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < C::kC; ++k) {
          const uint32_t w[4] = {raw[z][k].x, raw[z][k].y, raw[z][k].z, raw[z][k].w};
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
        const float f = a.scale > 0.f ? pow2f(up) : a.scale < 0.f ? -pow2f(up) : 0.f;
        const float unit = fmaxf(pow2f(max(-up, -126)) * nat, kMinFloat);
#pragma unroll
        for (int k = 0; k < C::kC; ++k) {
          const uint32_t w[4] = {raw[z][k].x, raw[z][k].y, raw[z][k].z, raw[z][k].w};
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const float2 v = two_floats(w[p], T{});
            qf[z][k][p] = pack_half2(v.x * f, v.y * f);
          }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          factor[z][n] = __shfl_sync(0xffffffffu, unit, (2 * c + n) * 4);
          hi[z][n] = end_of(8 * z + 2 * c + n);
        }
      }

      float m[NT][2], sums[NT][4];  // maximum and sum of p (elements 0, 1) of rows 8 z + 2 c + x
      float acc[D / 16][NT][4];     // dims g d/8 + 2 x (elements 0, 1) and + 1 (2, 3), the same rows
      float poison[NT][2];          // NaN once a visible V block of this thread's dims was NaN
      int out_unit = 0;             // acc holds sums times 2^-out_unit: 0 or kLargeUnit
      float kept[D / 16 * NT * 4];  // the sums, while acc takes a window's product
      asm volatile("" ::"l"(kept) : "memory");  // in memory, not in registers that all tiles would miss
      bool out_of_range = false;    // maxima above kCoarse
#pragma unroll
      for (int z = 0; z < NT; ++z) {
        m[z][0] = m[z][1] = -INFINITY;
        poison[z][0] = poison[z][1] = 0.f;
#pragma unroll
        for (int p = 0; p < 4; ++p) sums[z][p] = 0.f;
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
#pragma unroll
          for (int p = 0; p < 4; ++p) acc[x][z][p] = 0.f;
      }

      for (int i = 0; i < mine; ++i) {
        issue(i + C::kStages - 1);
        copy_commit();  // an empty group too, so that the wait counts tiles
        copy_wait<C::kStages - 1>();
        __syncwarp();
        const uint8_t* buf = ring + stage * C::kStage;
        const int key0 = base + i * kWarps * kTile;
        const uint32_t halves = (present >> (2 * stage)) & 3u;
        stage = stage + 1 == C::kStages ? 0 : stage + 1;

        // ---- scales, as fp16 pairs: of K for the rows 8 j + k_row and this thread's block c d/128, of V
        // for the row pairs (16 j + c, + 4) and (+ 8, + 12) and its block g d/256.  Exponents
        // [-14, 13] are bytes 113 .. 140; bytes of both are checked by lane = row.
        const int k_row = (g >> 1) + 4 * (g & 1);
        const uint8_t *kbytes = buf + 2 * C::kCode, *vbytes = kbytes + C::kScale;
        uint32_t kw, vw;
        if constexpr (C::kC == 4) {
          kw = *reinterpret_cast<const uint32_t*>(kbytes + lane * 4);
          vw = *reinterpret_cast<const uint32_t*>(vbytes + lane * 4);
        } else if constexpr (C::kC == 2) {
          kw = *reinterpret_cast<const uint16_t*>(kbytes + lane * 2) * 0x10001u;
          vw = *reinterpret_cast<const uint16_t*>(vbytes + lane * 2) * 0x10001u;
        } else {
          kw = kbytes[lane] * 0x1010101u;
          vw = vbytes[lane] * 0x1010101u;
        }
        // All four bytes in [113, 140] at once: b + 16 and b + 19 both have 100 as their top bits, and
        // b + 15 the highest.  (A byte that carries or borrows fails itself.)
        const uint32_t k16 = kw + 0x10101010u, v16 = vw + 0x10101010u;
        const uint32_t odd = ((k16 ^ 0x80808080u) | ((k16 + 0x03030303u) ^ 0x80808080u) | (v16 ^ 0x80808080u) |
                              ((v16 + 0x03030303u) ^ 0x80808080u)) & 0xe0e0e0e0u;
        const uint32_t low = ((k16 - 0x01010101u) & (v16 - 0x01010101u) & 0x80808080u) ^ 0x80808080u;
        const bool inner = halves == 3u && key0 >= first && key0 + kTile <= last;  // every row was written
        bool plain = true, vnan = false;
        int kbias = 112, vbias = 112, vhi = 0;  // kbias: of key key0 + lane
        uint32_t ksc[4], vsc[2][2];
        const int pair_at = (lane & ~7) | ((lane & 3) * 2) | ((lane >> 2) & 1);  // keys c and c + 4 side by side
        auto put_v_scales = [&](int bias, int most) {  // of the blocks whose byte is `most` or less
#pragma unroll
          for (int x = 0; x < C::kC; ++x) {
            const int byte = (vw >> (8 * x)) & 255;
            vtab[x * C::kVStride + pair_at] = __ushort_as_half(static_cast<uint16_t>(byte <= most ? scale_bits(byte, bias) : 0));
          }
        };
        auto get_v_scales = [&]() {
          const __half* from = vtab + (g * D / 256) * C::kVStride + 2 * c;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) vsc[j][x] = *reinterpret_cast<const uint32_t*>(from + 16 * j + 8 * x);
        };
        if (__all_sync(0xffffffffu, inner && (odd | low) == 0)) {
          // (byte - 112) << 10 in one or both halves
          constexpr uint32_t kOne = 0x0400u, kBoth = 0x04000400u;
#pragma unroll
          for (int j = 0; j < 4; ++j) ksc[j] = kbytes[(8 * j + k_row) * C::kC + c * C::kC / 4] * kBoth - 112u * kBoth;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint8_t* from = vbytes + (16 * j + 8 * x + c) * C::kC + g * D / 256;
              vsc[j][x] = from[0] * kOne + (from[4 * C::kC] * (kOne << 16) - 112u * kBoth);
            }
        } else {
          const int my_key = key0 + lane;
          if (!((halves >> (lane >> 4)) & 1u) || my_key < first || my_key >= last) kw = vw = 0;  // nobody sees it: a row of zeros
          kw = without_zeros(kw, C::kC, buf + lane * (D / 2));
          vw = without_zeros(vw, C::kC, buf + C::kCode + lane * (D / 2));
          int klo = 255, khi = 0, vlo = 255;
          bool knan = false;
          scale_range(kw, C::kC, klo, khi, knan);
          scale_range(vw, C::kC, vlo, vhi, vnan);
          plain = __all_sync(0xffffffffu, min(klo, vlo) > 112 && max(khi, vhi) <= 140 && !knan && !vnan);  // but for zero blocks
          if (!plain) {
            vhi = __reduce_max_sync(0xffffffffu, vhi);
            kbias = max(khi - 28, kLeastBias);
            vbias = max(vhi - 28, kLeastBias);
          }
#pragma unroll
          for (int x = 0; x < C::kC; ++x) {
            const int byte = (kw >> (8 * x)) & 255;
            ktab[lane * C::kC + x] = byte == 255 ? 0x7e007e00u : scale_bits(byte, kbias) * 0x10001u;
          }
          put_v_scales(vbias, 254);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 4; ++j) ksc[j] = ktab[(8 * j + k_row) * C::kC + c * C::kC / 4];
          get_v_scales();
        }

        // ---- scores: row n of key group j (8 keys) is key 8 j + n / 2 + 4 (n % 2)
        uint32_t kc[4][C::kC];
        float s[2][NT][4];  // key groups 2 j (elements 0, 1) and 2 j + 1 (2, 3), rows 8 z + 2 c + x
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 8 * j + k_row;
          const uint8_t* from = buf + row * (D / 2) + c * (D / 8);
          if constexpr (C::kC == 4) {
            const uint4 t = *reinterpret_cast<const uint4*>(from);
            kc[j][0] = t.x; kc[j][1] = t.y; kc[j][2] = t.z; kc[j][3] = t.w;
          } else if constexpr (C::kC == 2) {
            const uint2 t = *reinterpret_cast<const uint2*>(from);
            kc[j][0] = t.x; kc[j][1] = t.y;
          } else {
            kc[j][0] = *reinterpret_cast<const uint32_t*>(from);
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int z = 0; z < NT; ++z) s[j][z][0] = s[j][z][1] = s[j][z][2] = s[j][z][3] = 0.f;
#pragma unroll
        for (int k = 0; k < C::kC; ++k) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t ha[4], hb[4];
            codes_to_half2(kc[2 * j][k], ha);
            codes_to_half2(kc[2 * j + 1][k], hb);
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              ha[p] = mul2(ha[p], ksc[2 * j]);
              hb[p] = mul2(hb[p], ksc[2 * j + 1]);
            }
#pragma unroll
            for (int z = 0; z < NT; ++z) {
              mma16816(s[j][z], ha[0], hb[0], ha[1], hb[1], qf[z][k][0], qf[z][k][1]);
              mma16816(s[j][z], ha[2], hb[2], ha[3], hb[3], qf[z][k][2], qf[z][k][3]);
            }
          }
        }

        // ---- softmax in units of log2: score s f
        float f[NT][2];
#pragma unroll
        for (int z = 0; z < NT; ++z)
#pragma unroll
          for (int n = 0; n < 2; ++n) f[z][n] = factor[z][n];
        auto each_score = [&](auto&& change) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int z = 0; z < NT; ++z)
#pragma unroll
              for (int p = 0; p < 4; ++p) s[j][z][p] = change(s[j][z][p], j, z, p);
        };
        auto unit_factors = [&]() {
#pragma unroll
          for (int z = 0; z < NT; ++z) f[z][0] = f[z][1] = 1.f;
        };
        if (!plain) {
          float km[4];  // units of the keys 8 j + k_row
#pragma unroll
          for (int j = 0; j < 4; ++j) km[j] = pow2f(__shfl_sync(0xffffffffu, kbias, 8 * j + k_row) - 112);
          each_score([&](float v, int j, int z, int p) { return v * fminf(f[z][p & 1] * km[2 * j + (p >> 1)], kMaxFloat); });
          unit_factors();
        }
        if (a.softcap > 0.f) {
          Cap cap[NT][2];
#pragma unroll
          for (int z = 0; z < NT; ++z)
#pragma unroll
            for (int n = 0; n < 2; ++n) cap[z][n] = Cap(a.softcap, f[z][n]);
          if (a.softcap <= kRoundCap) each_score([&](float v, int, int z, int p) { return cap[z][p & 1].round(v); });
          else each_score([&](float v, int, int z, int p) { return cap[z][p & 1].exact(v); });
          unit_factors();
        }
        if (halves != 3u || key0 < inner_lo || key0 + kTile > inner_hi) {  // some row does not see some key
          each_score([&](float v, int j, int z, int p) {
            const int key = key0 + 16 * j + 8 * (p >> 1) + k_row, end = hi[z][p & 1];
            const bool seen = ((halves >> j) & 1u) && key < end && (a.window == 0 || key >= end - a.window);
            return seen ? v : -INFINITY;
          });
        }
        float next[NT][2];
        const float lag = out_of_range ? 0.f : kLag;
        bool moved = false;
        float most = 0.f;
#pragma unroll
        for (int z = 0; z < NT; ++z) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            float x = fmaxf(fmaxf(s[0][z][n], s[0][z][2 + n]), fmaxf(s[1][z][n], s[1][z][2 + n]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            const float now = __fmul_rn(x, f[z][n]);
            next[z][n] = now > m[z][n] + lag ? now : m[z][n];
            moved = moved || next[z][n] != m[z][n];
            most = fmaxf(most, next[z][n] == -INFINITY ? 0.f : fabsf(next[z][n]));
          }
        }
        if (__any_sync(0xffffffffu, moved)) {
          if (__any_sync(0xffffffffu, most > kCoarse)) out_of_range = true;
#pragma unroll
          for (int z = 0; z < NT; ++z) {
            const float keep0 = shrink(m[z][0], next[z][0]), keep1 = shrink(m[z][1], next[z][1]);
            sums[z][0] *= keep0;
            sums[z][1] *= keep1;
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
              acc[x][z][0] *= keep0;
              acc[x][z][1] *= keep1;
              acc[x][z][2] *= keep0;
              acc[x][z][3] *= keep1;
            }
            m[z][0] = next[z][0];
            m[z][1] = next[z][1];
          }
        }
        float d[NT][2];
#pragma unroll
        for (int z = 0; z < NT; ++z)
#pragma unroll
          for (int n = 0; n < 2; ++n) d[z][n] = m[z][n] == -INFINITY ? 0.f : 15.f - m[z][n];
        if (out_of_range) {
          // The maximum is taken off first, from scores that were rounded as it was: 15 - m below would be rounded
          // to the spacing of m, 16 - m from 2^24 on, and p would pass fp16's end.
          each_score([&](float v, int, int z, int p) {
            return __fsub_rn(__fmul_rn(v, f[z][p & 1]), m[z][p & 1] == -INFINITY ? 0.f : m[z][p & 1]);
          });
          unit_factors();
#pragma unroll
          for (int z = 0; z < NT; ++z) d[z][0] = d[z][1] = 15.f;
        }
        // p times 2^15 (a row without a key so far keeps p = 0), as the B operand of the next product
        uint32_t p[2][NT][2];
#pragma unroll
        for (int z = 0; z < NT; ++z) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
              p[j][z][x] = transpose8(pack_half2(ex2(fmaf(s[j][z][2 * x], f[z][0], d[z][0])), ex2(fmaf(s[j][z][2 * x + 1], f[z][1], d[z][1]))));
          }
          // the rounded weights' sums, as a product with ones
#pragma unroll
          for (int j = 0; j < 2; ++j)
            mma16816(sums[z], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, p[j][z][0], p[j][z][1]);
        }

        // ---- sums of p v: rows n and n + 8 of dim group x are dims n d/8 + 2 x and + 1
        auto add_values = [&]() {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            constexpr int kWords = D >= 64 ? D / 64 : 1;
            uint32_t w[4][kWords];  // keys c, c + 4, c + 8, c + 12 of the half
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint8_t* from = buf + C::kCode + (16 * j + c + 4 * x) * (D / 2) + g * (D / 16);
              if constexpr (D == 128) {
                const uint2 t = *reinterpret_cast<const uint2*>(from);
                w[x][0] = t.x;
                w[x][1] = t.y;
              } else if constexpr (D == 64) {
                w[x][0] = *reinterpret_cast<const uint32_t*>(from);
              } else {
                w[x][0] = *reinterpret_cast<const uint16_t*>(from);
              }
            }
            const uint32_t sa = vsc[j][0], sb = vsc[j][1];
#pragma unroll
            for (int k = 0; k < kWords; ++k) {
              uint32_t even_a[4], odd_a[4], even_b[4], odd_b[4];
              codes_to_half2(low_nibbles_of(w[0][k], w[1][k] << 4), even_a);
              codes_to_half2(low_nibbles_of(w[0][k] >> 4, w[1][k]), odd_a);
              codes_to_half2(low_nibbles_of(w[2][k], w[3][k] << 4), even_b);
              codes_to_half2(low_nibbles_of(w[2][k] >> 4, w[3][k]), odd_b);
#pragma unroll
              for (int x = 0; x < (D >= 64 ? 4 : 2); ++x) {
                const uint32_t a0 = mul2(even_a[x], sa), a1 = mul2(odd_a[x], sa), a2 = mul2(even_b[x], sb), a3 = mul2(odd_b[x], sb);
#pragma unroll
                for (int z = 0; z < NT; ++z) mma16816(acc[4 * k + x][z], a0, a1, a2, a3, p[j][z][0], p[j][z][1]);
              }
            }
          }
        };
        // Ordinarily one product, onto the sums.  Else one for each window of 28 exponents, the largest first, by
        // itself: no size of one block, key or row limits another's.
        const bool windows = !plain || out_unit != 0;
        int bias = vbias, most_byte = 254;
        auto each_sum = [&](auto&& change) {
#pragma unroll
          for (int x = 0; x < D / 16; ++x)
#pragma unroll
            for (int z = 0; z < NT; ++z)
#pragma unroll
              for (int y = 0; y < 4; ++y) acc[x][z][y] = change(acc[x][z][y], (x * NT + z) * 4 + y);
        };
        if (!plain && vhi > kLargeByte && out_unit == 0) {
          out_unit = kLargeUnit;
          each_sum([&](float v, int) { return v * pow2f(-kLargeUnit); });
        }
        while (true) {
          if (windows)
            each_sum([&](float v, int at) {
              kept[at] = v;
              return 0.f;
            });
          add_values();
          if (!windows) break;
          const Power unit(bias - 112 - out_unit);
          each_sum([&](float v, int at) { return unit.add(v, kept[at]); });
          if (plain) break;
          int below = 0;  // the largest byte that no window has held yet
#pragma unroll
          for (int x = 0; x < C::kC; ++x) {
            const int byte = (vw >> (8 * x)) & 255;
            if (byte <= bias) below = max(below, byte);
          }
          below = __reduce_max_sync(0xffffffffu, below);
          if (below == 0) break;
          most_byte = bias;
          bias = max(below - 28, kLeastBias);
          __syncwarp();
          put_v_scales(bias, most_byte);
          __syncwarp();
          get_v_scales();
        }
        if (!plain) {
          if (__any_sync(0xffffffffu, vnan)) {
            // a NaN block reaches the rows that see its key: this thread's dims lie in block g d/256
            for (int x = 0; x < kTile; ++x) {
              const uint32_t word = __shfl_sync(0xffffffffu, vw, x);
              if (((word >> (8 * (g * D / 256))) & 255u) != 255u) continue;
              const int key = key0 + x;
#pragma unroll
              for (int z = 0; z < NT; ++z)
#pragma unroll
                for (int n = 0; n < 2; ++n)
                  if (key < hi[z][n] && (a.window == 0 || key >= hi[z][n] - a.window)) poison[z][n] = NAN;
            }
          }
        }
        __syncwarp();  // the stage and the scale tables are free again
      }

      // ---- join the block's warps: every part divided by the block's sum of p, so that no unit can overflow
      __syncthreads();  // all rings are free
      float* sum = reinterpret_cast<float*>(smem);                                     // (warp, register, lane)
      float2* ml = reinterpret_cast<float2*>(smem + kWarps * C::kRows * D * 4);  // (warp, row)
      if (g == 0) {
#pragma unroll
        for (int z = 0; z < NT; ++z)
#pragma unroll
          for (int n = 0; n < 2; ++n) ml[warp * C::kRows + 8 * z + 2 * c + n] = make_float2(m[z][n], sums[z][n]);
      }
      __syncthreads();
      const float unit = pow2f(out_unit);
      float top[NT][2], whole_l[NT][2];
#pragma unroll
      for (int z = 0; z < NT; ++z) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float2* part = ml + 8 * z + 2 * c + n;
          top[z][n] = -INFINITY;
          whole_l[z][n] = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) top[z][n] = fmaxf(top[z][n], part[w * C::kRows].x);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) whole_l[z][n] += part[w * C::kRows].y * shrink(part[w * C::kRows].x, top[z][n]);
          const float share = whole_l[z][n] == 0.f ? 0.f : shrink(m[z][n], top[z][n]) / whole_l[z][n];
#pragma unroll
          for (int x = 0; x < D / 16; ++x)
#pragma unroll
            for (int p = 0; p < 2; ++p)
              sum[(((warp * (D / 16) + x) * NT + z) * 4 + 2 * p + n) * 32 + lane] = acc[x][z][2 * p + n] * share * unit + poison[z][n];
        }
      }
      __syncthreads();
      // This warp's part of the dim groups, of all warps' sums: the result, or a part of it.
      constexpr int kX = D >= 64 ? D / 64 : 1;
      const bool whole = list.whole();
      const int64_t slot = list.part_row();
      if (warp * kX < D / 16) {
#pragma unroll
        for (int z = 0; z < NT; ++z) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int i = 8 * z + 2 * c + n;
            if (i >= rows) continue;
            const int t = a.T == 1 ? 0 : (row0 + i) / G, h = head * G + row0 + i - t * G;
            const int64_t row = (static_cast<int64_t>(b) * a.H + h) * a.T + t;
            const float keep = whole && a.sink != nullptr ? share_beside(a.sink[h], top[z][n], whole_l[z][n]) : 1.f;
            Few<float, 2 * kX> o;
#pragma unroll
            for (int x = 0; x < kX; ++x) {
#pragma unroll
              for (int p = 0; p < 2; ++p) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w)
                  v += sum[(((w * (D / 16) + warp * kX + x) * NT + z) * 4 + 2 * p + n) * 32 + lane];
                o.v[2 * x + p] = v;
              }
            }
            const int d = g * (D / 8) + 2 * warp * kX;
            if (whole) {
              Few<T, 2 * kX> r;
#pragma unroll
              for (int x = 0; x < 2 * kX; ++x) r.v[x] = static_cast<T>(o.v[x] * keep);
              *reinterpret_cast<Few<T, 2 * kX>*>(static_cast<T*>(a.out) + row * D + d) = r;
            } else {
              *reinterpret_cast<Few<float, 2 * kX>*>(a.part_out + (slot + i) * D + d) = o;
              if (warp == 0 && g == 0) a.part_ml[slot + i] = make_float2(top[z][n], whole_l[z][n]);
            }
          }
        }
      }
    }

    // ---- the next segment
    if (!list.next(a, row_tiles)) return;
    __syncthreads();  // the join's sums have been read
  }
}

template <typename T, int D, int NT>
void launch(const Fp4AttnArgs& a, cudaStream_t stream) {
  using C = Cfg<D, NT>;
  cudaFuncSetAttribute(fp4_attn_rows_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  fp4_attn_rows_kernel<T, D, NT><<<a.blocks, kWarps * 32, C::kSmem, stream>>>(a);
  launch_join<T, D, typename C::List>(a, stream);
}

// f(D, NT) for the head dim and the query rows of a K / V head: eight or fewer take 8-row segments
// (2 x 131072 keys of 8 heads, 4 rows: 71 us, with 16-row segments 97).
template <typename F>
auto by_shape(const Fp4AttnArgs& a, int d, F&& f) {
  using std::integral_constant;
  const bool few = a.H / a.Hk * a.T <= 8;
  if (d == 32) return few ? f(integral_constant<int, 32>{}, integral_constant<int, 1>{}) : f(integral_constant<int, 32>{}, integral_constant<int, 2>{});
  if (d == 64) return few ? f(integral_constant<int, 64>{}, integral_constant<int, 1>{}) : f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  return few ? f(integral_constant<int, 128>{}, integral_constant<int, 1>{}) : f(integral_constant<int, 128>{}, integral_constant<int, 2>{});
}

}  // namespace

Fp4AttnPlan fp4_attn_rows_plan(const Fp4AttnArgs& a, int d) {
  return by_shape(a, d, [&](auto dim, auto nt) {
    using C = Cfg<decltype(dim)::value, decltype(nt)::value>;
    return Fp4AttnPlan{C::List::most_units(a), C::List::blocks(a, C::kBlocks), C::kRows};
  });
}

void fp4_attn_rows(const Fp4AttnArgs& a, int d, bool half, cudaStream_t stream) {
  by_shape(a, d, [&](auto dim, auto nt) {
    if (half) launch<__half, decltype(dim)::value, decltype(nt)::value>(a, stream);
    else launch<__nv_bfloat16, decltype(dim)::value, decltype(nt)::value>(a, stream);
  });
}

}  // namespace sv4
