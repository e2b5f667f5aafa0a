// Attention over the paged 4-bit K / V cache for many query rows per K / V head (prefill chunks):
// the products on tcgen05, 128 rows by 128 keys.
//
// The mathematics, the list of work and the join are those of fp4_attn.cu.  Here 4 * 128 * 128 * d
// operations per tile stand against 128 * 17/16 d bytes, so the tensor cores bound it, and next to
// them the exponentials (128 * 128 per tile, 16 a clock) and the turning of codes into operands:
//
// * A block has 128 threads and one 128-row tile of queries (the G heads of a K / V head, times
//   tokens); thread = row = TMEM lane.  Two blocks per SM, one's products under the other's
//   softmax.  S and O accumulate in TMEM (fp32), the operands lie in shared memory as 64-column
//   128B-swizzled atoms, V contracted over its rows; P takes K's place.
// * Codes go from global memory to registers a tile ahead (eight rows of one 32-value block per
//   eight threads: coalesced reads, conflict-free swizzled writes), through cvt.e2m1x2 to fp16,
//   exact, times their scale 2^e, exact for exponents in [-14, 13].  V is written while S = Q K^T runs.
// * A tile with other exponents takes K's from its own largest 28 down, and runs P V once per window
//   of 28 exponents, each row's sums moved from unit to unit by powers of two; a row whose sums are
//   too large to follow to a small unit has no use for what is 2^-126 of them.
#include "fp4_work.cuh"

namespace sv4 {
namespace {

using namespace fp4;

constexpr int kThreads = 128;
constexpr int kKeys = 128, kRows = 128;
constexpr int kSegmentCost = 4;       // in tiles
constexpr uint32_t kAtom = 16384;     // 128 rows x 128 bytes
using List = Work<kKeys, kSegmentCost, kRows, 1>;

// Operand descriptors: contraction over columns (step s of 16), over rows.
__device__ __forceinline__ uint64_t desc_cols(uint32_t base, int s) {
  return make_smem_desc(base + (s >> 2) * kAtom + (s & 3) * 32, 16, 1024, 2);
}
__device__ __forceinline__ uint64_t desc_rows(uint32_t base, int s) {
  return make_smem_desc(base + s * 2048, kAtom, 1024, 2);
}
// Where 16-byte piece q (of the 64-column atom's eight) of row r lies.
__device__ __forceinline__ uint8_t* piece_at(uint8_t* tile, int r, int column) {
  return tile + (column >> 6) * kAtom + r * 128 + ((((column & 63) >> 3) ^ (r & 7)) << 4);
}

template <int D>
struct Cfg {
  static constexpr int kAtoms = D / 64;
  static constexpr int kQ = kAtoms * kAtom, kKP = 2 * kAtom, kV = kAtoms * kAtom;  // P: two atoms whatever D
  // alignment, barriers and flags; as much for every D, so that two blocks' TMEM is all an SM is asked for
  static constexpr int kSmem = 6 * kAtom + 1024 + 1024;
  static constexpr int kC = D / 32;
  static constexpr int kRowsAtOnce = 32 / kC;         // a warp's rows per pass: lane = (block, row)
  static constexpr int kPasses = 32 / kRowsAtOnce;    // a warp writes 32 rows
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) fp4_attn_tile_kernel(const Fp4AttnArgs a) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sq = smem, *sk = sq + C::kQ, *sv = sk + C::kKP, *sp = sk;
  uint64_t* bar = reinterpret_cast<uint64_t*>(sv + C::kV);  // 0: S is there, 1: P V is done
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bar + 2);
  int* red = reinterpret_cast<int*>(tslot + 1);                // (4)
  uint32_t* nan_keys = reinterpret_cast<uint32_t*>(red + 4);   // (128) blocks of V that are NaN
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.H / a.Hk, tiles_per_head = (G * a.T + kRows - 1) / kRows, row_tiles = a.Hk * tiles_per_head;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  List list;
  if (!list.begin(a, row_tiles)) return;
  if (tid == 0) {
    mbar_init(bar, 1);
    mbar_init(bar + 1, 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(tslot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tslot, lanes = static_cast<uint32_t>(warp * 32) << 16;
  const uint32_t ts = tbase + lanes, to = tbase + 128 + lanes;
  constexpr uint32_t kIdS = make_idesc_f16(128, 128, 0, 0, false, false);
  constexpr uint32_t kIdO = make_idesc_f16(128, D, 0, 0, false, true);
  const uint32_t uq = smem_u32(sq), uk = smem_u32(sk), uv = smem_u32(sv), up_ = smem_u32(sp);
  uint32_t n_s = 0, n_o = 0;  // products so far: parities of the two barriers
  bool alive = true;
  auto wait = [&](int which, uint32_t n) {
    if (!mbar_wait(bar + which, n & 1, nullptr, 0)) {
      record_error(a.err, kErrTimeoutAccum);
      alive = false;
    }
    __syncwarp();
    tc_fence_after();
  };
  const float nat = (a.scale != 0.f ? fabsf(a.scale) : 1.f) * (a.softcap > 0.f ? 1.f : kLog2e);
  const int in_row = lane % C::kRowsAtOnce, blk = lane / C::kRowsAtOnce;  // of a pass: row, 32-value block

  while (true) {
    const int take = list.take(), from_tile = list.from_tile(), b = list.b;
    if (take > 0) {
      const int head = list.y / tiles_per_head, row0 = (list.y % tiles_per_head) * kRows;
      const int rows = min(kRows, G * a.T - row0), len = list.sp.len;
      auto end_of = [&](int i) { return len - a.T + (row0 + min(i, rows - 1)) / G + 1; };  // one past the last key of row i
      const int hi = end_of(tid), lo = a.window > 0 ? max(0, hi - a.window) : 0;
      const int last = end_of(kRows - 1), inner_hi = end_of(0);
      const int first = a.window > 0 ? max(0, inner_hi - a.window) : 0, inner_lo = a.window > 0 ? max(0, last - a.window) : 0;
      const int* table = a.table + static_cast<int64_t>(b) * a.P;
      const int key_begin = list.sp.start + from_tile * kKeys;

      // ---- codes and scale bytes of a tile: pass x of this warp has rows 32 warp + kRowsAtOnce x + in_row
      uint4 kcode[C::kPasses], vcode[C::kPasses];
      uint32_t kbyte = 0, vbyte = 0;   // one byte per pass
      uint32_t here = 0;               // passes whose row may be seen, of the tile that K is loaded for
      uint32_t vhere = 0;
      uint32_t lost = 0;               // passes whose page id is bad
      const uint8_t* at[C::kPasses];   // the slab, or null, for the tile after
      int at_row[C::kPasses];
      auto find = [&](int key0) {
#pragma unroll
        for (int x = 0; x < C::kPasses; ++x) {
          const int key = key0 + 32 * warp + C::kRowsAtOnce * x + in_row;
          at[x] = nullptr;
          at_row[x] = 0;
          if (key < last) {
            const int slot = key / a.R, page = table[slot];
            if (index_ok(page, 0, a.n_pages, a.err)) {
              at[x] = a.pages + page * a.page_stride + static_cast<int64_t>(head) * a.slab;
              at_row[x] = key - slot * a.R;
            }
          }
        }
      };
      auto load = [&](uint4 (&code)[C::kPasses], uint32_t& bytes, int kv) {
        bytes = 0;
#pragma unroll
        for (int x = 0; x < C::kPasses; ++x) {
          code[x] = make_uint4(0, 0, 0, 0);
          if (at[x] != nullptr) {
            code[x] = *reinterpret_cast<const uint4*>(at[x] + (kv * a.R + at_row[x]) * (D / 2) + blk * 16);
            bytes |= static_cast<uint32_t>(at[x][a.R * D + (kv * a.R + at_row[x]) * C::kC + blk]) << (8 * x);
          }
        }
      };
      auto seen_mask = [&](int key0) {
        uint32_t m = 0, gone = 0;
#pragma unroll
        for (int x = 0; x < C::kPasses; ++x) {
          const int key = key0 + 32 * warp + C::kRowsAtOnce * x + in_row;
          if (key >= first && key < last) {
            if (at[x] != nullptr) m |= 1u << x;
            else gone |= 1u << x;
          }
        }
        lost = gone;
        return m;
      };
      // fp16 values of this thread's rows into a swizzled tile; scale(byte) gives the scale's fp16 bits
      auto write = [&](uint8_t* tile, const uint4 (&code)[C::kPasses], auto&& scale) {
#pragma unroll
        for (int x = 0; x < C::kPasses; ++x) {
          const int row = 32 * warp + C::kRowsAtOnce * x + in_row;
          const uint32_t s = scale(x) * 0x10001u;
          const uint32_t w[4] = {code[x].x, code[x].y, code[x].z, code[x].w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t h[4];
            codes_to_half2(w[q], h);
            *reinterpret_cast<uint4*>(piece_at(tile, row, blk * 32 + q * 8)) =
                make_uint4(mul2(h[0], s), mul2(h[1], s), mul2(h[2], s), mul2(h[3], s));
          }
        }
      };
      auto byte_of = [](uint32_t bytes, int x) { return static_cast<int>((bytes >> (8 * x)) & 255u); };
      auto block_max = [&](int v) {
        v = __reduce_max_sync(0xffffffffu, v);
        if (lane == 0) red[warp] = v;
        __syncthreads();
        v = max(max(red[0], red[1]), max(red[2], red[3]));
        __syncthreads();
        return v;
      };

      find(key_begin);
      load(kcode, kbyte, 0);
      load(vcode, vbyte, 1);

      // ---- q: thread = row, scaled by a power of two to fp16's top, into the swizzled tile
      float factor;  // raw score -> softmax units
      {
        const int i = row0 + min(tid, rows - 1);
        const T* row = static_cast<const T*>(a.q) + b * a.q_b + (head * G + i % G) * a.q_h + (i / G) * a.q_t;
        float amax = 0.f;
#pragma unroll 4
        for (int k = 0; k < D / 8; ++k) {
          const uint4 raw = *reinterpret_cast<const uint4*>(row + 8 * k);
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float2 f = two_floats(w[x], T{});
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        const int x = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
        const int up = amax > 0.f && x < 128 ? min(14 - x, 126) : 0;
        const float f = a.scale > 0.f ? pow2f(up) : a.scale < 0.f ? -pow2f(up) : 0.f;
        factor = pow2f(max(-up, -126)) * nat;
#pragma unroll 4
        for (int k = 0; k < D / 8; ++k) {
          const uint4 raw = *reinterpret_cast<const uint4*>(row + 8 * k);
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
          uint32_t h[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float2 v = two_floats(w[y], T{});
            h[y] = pack_half2(v.x * f, v.y * f);
          }
          *reinterpret_cast<uint4*>(piece_at(sq, tid, 8 * k)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
      }

      float m = -INFINITY, l = 0.f;
      int unit = 0;           // this row's sums are held times 2^-unit
      uint32_t poison = 0;    // blocks of d whose sums are NaN
      bool careful = false;   // units have moved: the block's tiles take the careful way
      bool out_of_range = false;
      uint32_t n_tile = 0;    // P V products of this segment

      for (int t = 0; t < take && alive; ++t) {
        const int key0 = key_begin + t * kKeys;
        if (key0 >= last) break;  // behind what this row tile sees (the list spans all T tokens)
        here = seen_mask(key0);
        vhere = here;
        bool ok = lost == 0;
#pragma unroll
        for (int x = 0; x < C::kPasses; ++x) {
          const int k = byte_of(kbyte, x), v = byte_of(vbyte, x);
          // exponents [-14, 13], or a block of zeros
          ok = ok && (!((here >> x) & 1u) || ((k <= 1 || (k > 112 && k <= 140)) && (v <= 1 || (v > 112 && v <= 140))));
        }
        if (n_tile > 0) wait(1, n_o - 1);  // P V of the last tile: its operands are free
        const bool plain = __syncthreads_and(ok) && !careful;
        int kbias = 112, vbias = 112;
        if (!plain) {
          int khi = 0, vhi = 0;
#pragma unroll
          for (int x = 0; x < C::kPasses; ++x) {
            if (!((here >> x) & 1u)) continue;
            const int k = byte_of(kbyte, x), v = byte_of(vbyte, x);
            if (k != 255) khi = max(khi, k);
            if (v != 255) vhi = max(vhi, v);
          }
          kbias = max(block_max(khi) - 28, -14);
          vbias = max(block_max(vhi) - 28, 2);
          nan_keys[tid] = 0;
          __syncthreads();
#pragma unroll
          for (int x = 0; x < C::kPasses; ++x) {
            const int row = 32 * warp + C::kRowsAtOnce * x + in_row;
            if (((here >> x) & 1u) && byte_of(vbyte, x) == 255) atomicOr(nan_keys + row, 1u << blk);
            if ((lost >> x) & 1u) atomicOr(nan_keys + row, 0x80000000u);  // a key that is not there
          }
        }
        write(sk, kcode, [&](int x) {
          const int k = byte_of(kbyte, x);
          if (plain) return (here >> x) & 1u ? scale_bits(k, 112) : 0u;
          return !((here >> x) & 1u) ? 0u : k == 255 ? 0x7e00u : scale_bits(k, kbias);
        });
        fence_proxy_async_smem();
        tc_fence_before();
        __syncthreads();
        if (tid == 0) {
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < D / 16; ++s) mma_bf16(tbase, desc_cols(uq, s), desc_cols(uk, s), kIdS, s > 0 ? 1u : 0u);
          mma_commit(bar);
        }
        __syncwarp();
        // under the product: V's operand, and the next tile's codes
        find(key0 + kKeys);
        load(kcode, kbyte, 0);
        if (plain) {
          write(sv, vcode, [&](int x) { return (vhere >> x) & 1u ? scale_bits(byte_of(vbyte, x), 112) : 0u; });
          load(vcode, vbyte, 1);
        }
        wait(0, n_s++);

        // ---- softmax of this thread's row, two passes over S
        float f = factor;
        if (!plain) f = fmaxf(f * pow2f(kbias - 112), 1.1754944e-38f);
        const bool masked = key0 < inner_lo || key0 + kKeys > inner_hi;
        const float cap = a.softcap * kLog2e, squeeze = a.softcap > 0.f ? 2.f * kLog2e / a.softcap : 0.f;
        auto score = [&](uint32_t raw, int key) {
          float v = __uint_as_float(raw);
          if (a.softcap > 0.f) v = cap * (1.f - __fdividef(2.f, 1.f + ex2(v * f * squeeze)));  // tanh
          if (masked) v = key >= lo && key < hi ? v : -INFINITY;
          if (!plain && (nan_keys[key - key0] >> 31)) v = -INFINITY;
          return v;
        };
        float most = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t r[32];
          tmem_ld32(ts + c * 32, r);
          tmem_ld_wait();
          if (!masked && plain && !(a.softcap > 0.f)) {
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j & 3] = fmaxf(x[j & 3], __uint_as_float(r[j]));
            most = fmaxf(most, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) most = fmaxf(most, score(r[j], key0 + c * 32 + j));
          }
        }
        if (a.softcap > 0.f) f = 1.f;
        const float next = fmaxf(m, most * f);
        out_of_range = out_of_range || (next != -INFINITY && fabsf(next) > 65536.f);
        if (n_tile > 0 && __any_sync(0xffffffffu, next != m)) {
          const float keep = shrink(m, next);
          l *= keep;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(to + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep);
            tmem_st32(to + c * 32, r);
          }
          tmem_st_wait();
        }
        m = next;
        const float d0 = m == -INFINITY ? 0.f : 15.f - m;  // p times 2^15
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t r[32];
          tmem_ld32(ts + c * 32, r);
          tmem_ld_wait();
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t h[16];
          if (!masked && plain && !(a.softcap > 0.f) && !out_of_range) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float x = ex2(fmaf(__uint_as_float(r[2 * j]), f, d0)), y = ex2(fmaf(__uint_as_float(r[2 * j + 1]), f, d0));
              sum[(2 * j) & 3] += x;
              sum[(2 * j + 1) & 3] += y;
              h[j] = pack_half2(x, y);
            }
          } else {
            // the product rounded before the maximum is taken off: a fused one would keep the bits
            // that rounding took from the maximum
            f = a.softcap > 0.f ? factor * (plain ? 1.f : pow2f(kbias - 112)) : f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float g = a.softcap > 0.f ? 1.f : f;
              const float x = ex2(__fmul_rn(score(r[2 * j], key0 + c * 32 + 2 * j), g) + d0);
              const float y = ex2(__fmul_rn(score(r[2 * j + 1], key0 + c * 32 + 2 * j + 1), g) + d0);
              sum[0] += x;
              sum[1] += y;
              h[j] = pack_half2(x, y);
            }
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(piece_at(sp, tid, c * 32 + 8 * q)) = make_uint4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]);
        }

        // ---- P V: ordinarily one product, else one for each window of V's exponents, the largest first
        int bias = vbias, most_byte = 254;
        bool dropped = false;  // this row's sums are too large for smaller units
        while (true) {
          if (!plain) {
            careful = true;
            if (n_tile > 0) wait(1, n_o - 1);
            // the row's sums to the unit of this window
            const int want = bias - 112;
            float big = 0.f;
            if (n_tile > 0) {
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                tmem_ld32(to + c * 32, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) big = fmaxf(big, fabsf(__uint_as_float(r[j])));
              }
            }
            if (big == 0.f) unit = want;  // nothing to move
            const int top = static_cast<int>(__float_as_uint(big) >> 23) - 127;
            if (unit - want > min(126, max(0, 96 - top))) dropped = true;
            const int by = dropped ? 0 : unit - want;
            const float s0 = pow2f(max(by, -126)), s1 = pow2f(max(min(by + 126, 0), -126));
            if (n_tile > 0 && __any_sync(0xffffffffu, by != 0)) {
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                tmem_ld32(to + c * 32, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * s0 * s1);
                tmem_st32(to + c * 32, r);
              }
              tmem_st_wait();
            }
            unit -= by;
            if (dropped) {
#pragma unroll
              for (int q = 0; q < 16; ++q) *reinterpret_cast<uint4*>(piece_at(sp, tid, 8 * q)) = make_uint4(0, 0, 0, 0);
            }
            write(sv, vcode, [&](int x) {
              const int v = byte_of(vbyte, x);
              return !((vhere >> x) & 1u) || v > most_byte ? 0u : scale_bits(v, bias);
            });
          }
          fence_proxy_async_smem();
          tc_fence_before();
          __syncthreads();
          if (tid == 0) {
            tc_fence_after();
#pragma unroll
            for (int s = 0; s < 8; ++s)
              mma_bf16(tbase + 128, desc_cols(up_, s), desc_rows(uv, s), kIdO, (n_tile > 0 || s > 0) ? 1u : 0u);
            mma_commit(bar + 1);
          }
          __syncwarp();
          ++n_o;
          ++n_tile;
          if (plain) break;
          int below = 0;  // the largest byte that no window has held yet
#pragma unroll
          for (int x = 0; x < C::kPasses; ++x) {
            const int v = byte_of(vbyte, x);
            if (((vhere >> x) & 1u) && v <= bias && v > 1) below = max(below, v);
          }
          below = block_max(below);
          if (below == 0) break;
          most_byte = bias;
          bias = below - 28;
        }
        if (!plain) {
          for (int j = 0; j < kKeys; ++j)
            if (key0 + j >= lo && key0 + j < hi) poison |= nan_keys[j] & 0xfu;
          load(vcode, vbyte, 1);
        }
      }

      // ---- the result, or a part of it
      if (n_tile > 0) wait(1, n_o - 1);
      const bool whole = list.whole();
      const float keep = (l == 0.f ? 0.f : 1.f / l) * (whole && a.sink != nullptr ? share_beside(a.sink[head * G + (row0 + min(tid, rows - 1)) % G], m, l) : 1.f);
      const float power = pow2f(max(-126, min(126, unit)));
      const int i = row0 + tid;
      const int64_t row = (static_cast<int64_t>(b) * a.H + head * G + i % G) * a.T + i / G;
      const int64_t slot = list.part_row() + tid;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        if (n_tile > 0) {
          tmem_ld32(to + c * 32, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = 0;
        }
        if (tid >= rows) continue;
        const float add = (poison >> c) & 1u ? NAN : 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float o[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = __uint_as_float(r[8 * q + j]) * keep * power + add;
          if (whole) {
            Few<T, 8> y;
#pragma unroll
            for (int j = 0; j < 8; ++j) y.v[j] = static_cast<T>(o[j]);
            *reinterpret_cast<Few<T, 8>*>(static_cast<T*>(a.out) + row * D + c * 32 + 8 * q) = y;
          } else {
            float4* to_part = reinterpret_cast<float4*>(a.part_out + slot * D + c * 32 + 8 * q);
            to_part[0] = make_float4(o[0], o[1], o[2], o[3]);
            to_part[1] = make_float4(o[4], o[5], o[6], o[7]);
          }
        }
      }
      if (!whole && tid < rows) a.part_ml[slot] = make_float2(m, l);
      tc_fence_before();  // the next segment's products overwrite the sums
    }
    if (!alive || !list.next(a, row_tiles)) break;
    __syncthreads();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tbase, 256);
}

template <typename T, int D>
void launch(const Fp4AttnArgs& a, cudaStream_t stream) {
  cudaFuncSetAttribute(fp4_attn_tile_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem);
  fp4_attn_tile_kernel<T, D><<<a.blocks, kThreads, Cfg<D>::kSmem, stream>>>(a);
  launch_join<T, D, List>(a, stream);
}

}  // namespace

Fp4AttnPlan fp4_attn_tile_plan(const Fp4AttnArgs& a) { return Fp4AttnPlan{List::most_units(a), List::blocks(a, 2), kRows}; }

void fp4_attn_tile(const Fp4AttnArgs& a, int d, bool half, cudaStream_t stream) {
  if (d == 64) half ? launch<__half, 64>(a, stream) : launch<__nv_bfloat16, 64>(a, stream);
  else half ? launch<__half, 128>(a, stream) : launch<__nv_bfloat16, 128>(a, stream);
}

}  // namespace sv4
