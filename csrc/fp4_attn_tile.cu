// Attention over the paged 4-bit K / V cache for many query rows per K / V head (prefill chunks):
// the products on tcgen05, 128 rows by 128 keys.
//
// The mathematics, the list of work and the join are those of fp4_attn.cu.  Here 4 * 128 * 128 * d
// operations per tile stand against 128 * 17/16 d bytes, so the tensor cores bound it, and next to
// them the exponentials (128 * 128 per tile, 16 a clock) and the turning of codes into operands.
// A block has two roles, two blocks share an SM:
//
// * Warps 0 - 3, the softmax of a 128-row tile of queries (the G heads of a K / V head, times
//   tokens): thread = row = TMEM lane.  S is read from TMEM, P (fp16, times 2^15) written over it as
//   the A operand of P V; O accumulates in TMEM too.  A row's maximum is left as it is while the new
//   one is at most 0.9 larger (log2), for which fp16 has room: most tiles then leave O alone.
//   One thread issues the products.
// * Warps 4 - 7, operands: codes from global memory to registers a tile ahead (eight rows of one
//   32-value block per eight threads: coalesced reads, conflict-free swizzled writes), through
//   cvt.e2m1x2 to fp16, exact, times their scale 2^e, exact for exponents in [-14, 13].  K and V lie
//   as 64-column 128B-swizzled atoms, V contracted over its rows.
//
// A tile with other exponents takes K's from each key's own largest 28 down, and runs P V once per window
// of 28 exponents, 64 dims at a time into the half of S that P leaves free; the softmax warps add that to
// O in fp32.
#include "fp4_work.cuh"

namespace sv4 {
namespace {

using namespace fp4;

constexpr int kThreads = 256;
constexpr int kKeys = 128, kRows = 128;
constexpr int kSegmentCost = 4;       // in tiles
constexpr uint32_t kAtom = 16384;     // 128 rows x 128 bytes
constexpr int kWindows = 10;          // 28 exponents each, from byte 254 down: -14 is the tenth's bias
using List = Work<kKeys, kSegmentCost, kRows, 1>;

// Operand descriptors, contracted over columns or over rows, and how far step s of 16 is from the
// first (the address field counts 16 bytes, and no step leaves it).
__device__ __forceinline__ uint64_t desc_cols(uint32_t base) { return make_smem_desc(base, 16, 1024, 2); }
__device__ __forceinline__ uint64_t desc_rows(uint32_t base) { return make_smem_desc(base, kAtom, 1024, 2); }
constexpr uint32_t step_cols(int s) { return ((s >> 2) * kAtom + (s & 3) * 32) >> 4; }
constexpr uint32_t step_rows(int s) { return s * 2048 >> 4; }
// Where the 16-byte piece of `column` (a multiple of 8) of row r lies.
__device__ __forceinline__ uint8_t* piece_at(uint8_t* tile, int r, int column) {
  return tile + (column >> 6) * kAtom + r * 128 + ((((column & 63) >> 3) ^ (r & 7)) << 4);
}
// D += A B with A (fp16 pairs, a row per lane) in TMEM.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// What the operand warps say about a tile.
struct Tile {
  int plain;   // all exponents in [-14, 13] and every page there, O in units of 1
  int large;   // O is held in units of 2^kLargeUnit
  int windows; // products P V
  int bias[kWindows];
  float kunit[kKeys];  // what a key's scores are multiplied by
  uint32_t nan_keys[kKeys];  // bits 0 - 3: blocks of V that are NaN; bit 31: a key whose page id is bad
};

template <int D>
struct Cfg {
  static constexpr int kAtoms = D / 64;
  static constexpr int kQ = kAtoms * kAtom;
  static constexpr int kC = D / 32;
  static constexpr int kRowsAtOnce = 32 / kC;       // a warp's rows per pass: lane = (block, row)
  static constexpr int kPasses = 32 / kRowsAtOnce;  // a warp writes 32 rows
  // q, K, V, alignment, barriers and tiles; as much for every D, so that two blocks' TMEM is all an SM is asked for
  static constexpr int kSmem = 6 * kAtom + 1024 + 3072;
};

// The largest v over the four operand warps.
__device__ __forceinline__ int most_of(int v, int* red, int part, int lane) {
  v = __reduce_max_sync(0xffffffffu, v);
  asm volatile("bar.sync 1, 128;" ::: "memory");
  if (lane == 0) red[part] = v;
  asm volatile("bar.sync 1, 128;" ::: "memory");
  return max(max(red[0], red[1]), max(red[2], red[3]));
}

// A tile with exponents outside [-14, 13], NaN blocks or missing keys: the keys' units and
// marks and V's windows, from the scale bytes (one per pass) of all operand threads.  Returns the biases of
// this thread's keys (K's scales are 2^(byte - bias - 15)), 14 more in a byte per pass, and the windows with
// 256 added for V scales above kLargeByte.
// Not inlined: its registers would be taken from every tile.
template <int D>
__device__ __noinline__ int2 describe(Tile& tile, int* red, uint32_t kbytes, uint32_t vbytes, uint32_t seen, uint32_t lost,
                                      int part, int lane) {
  using C = Cfg<D>;
  const int in_row = lane % C::kRowsAtOnce, blk = lane / C::kRowsAtOnce;
  int vhi = 0;
  uint32_t kbias = 0;
  for (int x = 0; x < C::kPasses; ++x) {
    const bool mine = (seen >> x) & 1u;
    const int k = (kbytes >> (8 * x)) & 255u, v = (vbytes >> (8 * x)) & 255u;
    int khi = mine && k != 255 ? k : 0;
    for (int o = C::kRowsAtOnce; o < 32; o <<= 1) khi = max(khi, __shfl_xor_sync(0xffffffffu, khi, o));
    const int bias = max(khi - 28, kLeastBias);
    kbias |= static_cast<uint32_t>(bias - kLeastBias) << (8 * x);
    if (blk == 0) tile.kunit[32 * part + C::kRowsAtOnce * x + in_row] = pow2f(bias - 112);
    if (mine && v != 255) vhi = max(vhi, v);
  }
  vhi = most_of(vhi, red, part, lane);
  int bias = max(vhi - 28, kLeastBias), windows = 1;
  const bool scribe = part == 0 && lane == 0;
  if (scribe) tile.bias[0] = bias;
  while (windows < kWindows) {
    int below = 0;  // the largest byte that no window holds yet
    for (int x = 0; x < C::kPasses; ++x) {
      const int v = (vbytes >> (8 * x)) & 255u;
      if (((seen >> x) & 1u) && v <= bias) below = max(below, v);
    }
    below = most_of(below, red, part, lane);
    if (below == 0) break;
    bias = max(below - 28, kLeastBias);
    if (scribe) tile.bias[windows] = bias;
    ++windows;
  }
  tile.nan_keys[32 * part + lane] = 0;
  asm volatile("bar.sync 1, 128;" ::: "memory");
  for (int x = 0; x < C::kPasses; ++x) {
    const int row = 32 * part + C::kRowsAtOnce * x + in_row;
    if (((seen >> x) & 1u) && ((vbytes >> (8 * x)) & 255u) == 255u) atomicOr(tile.nan_keys + row, 1u << blk);
    if ((lost >> x) & 1u) atomicOr(tile.nan_keys + row, 0x80000000u);
  }
  return make_int2(static_cast<int>(kbias), windows + (vhi > kLargeByte ? 256 : 0));
}

// kReady: every softmax warp has seen kKFull of the tile.  Without it warp 0 and the operand warps could
// complete kKFull once more before a warp that was held up looks, and a wait by parity would miss both.
enum Barrier { kQFull, kKFull, kReady, kSFull, kPFull, kVFull, kTFull, kOFull, kBarriers };

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) fp4_attn_tile_kernel(const Fp4AttnArgs a) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sq = smem, *sk = sq + C::kQ, *sv = sk + C::kQ;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + 6 * kAtom);
  Tile* tiles = reinterpret_cast<Tile*>(bar + kBarriers);  // (2), by turns
  uint32_t* tslot = reinterpret_cast<uint32_t*>(tiles + 2);
  int* red = reinterpret_cast<int*>(tslot + 1);  // (4)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.H / a.Hk, tiles_per_head = (G * a.T + kRows - 1) / kRows, row_tiles = a.Hk * tiles_per_head;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  List list;
  if (!list.begin(a, row_tiles)) return;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBarriers; ++i) mbar_init(bar + i, i == kSFull || i == kTFull || i == kOFull ? 1 : 4);
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(tslot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tslot;
  // The n-th completion of a barrier.  A wait that runs out records itself, and the warp (all of its lanes:
  // what follows is done together) does nothing more; the operand warps, which meet at a named barrier,
  // agree on that first.
  bool alive = true;
  auto wait = [&](int which, uint32_t n) {
    const bool done = alive && mbar_wait(bar + which, n & 1, nullptr, 0);  // errors of other kinds do not end it
    if (alive && !done) record_error(a.err, kErrTimeoutAccum);
    alive = __all_sync(0xffffffffu, done);
  };
  auto arrive = [&](int which) {  // one per warp
    __syncwarp();
    if (lane == 0) mbar_arrive(bar + which);
  };
  // Every role counts the same: segments, tiles and P V windows so far; the softmax warps also what they
  // let P be read for, and the products beside O.
  uint32_t n_seg = 0, n_tile = 0, n_pv = 0, n_p = 0, n_t = 0;

  while (true) {
    const int take = list.take(), from_tile = list.from_tile(), b = list.b;
    const int head = list.y / tiles_per_head, row0 = (list.y % tiles_per_head) * kRows;
    const int rows = min(kRows, G * a.T - row0), len = list.sp.len;
    auto end_of = [&](int i) { return len - a.T + (row0 + min(i, rows - 1)) / G + 1; };  // one past the last key of row i
    const int last = end_of(kRows - 1), inner_hi = end_of(0);
    const int first = a.window > 0 ? max(0, inner_hi - a.window) : 0;
    const int key_begin = list.sp.start + from_tile * kKeys;
    // tiles behind what this row tile sees are left out (the list spans all T tokens)
    const int count = take > 0 && key_begin < last ? min(take, (last - key_begin + kKeys - 1) / kKeys) : 0;

    if (warp >= 4) {
      // ============================================================ operands
      const int part = warp - 4, in_row = lane % C::kRowsAtOnce, blk = lane / C::kRowsAtOnce;
      const int* table = a.table + static_cast<int64_t>(b) * a.P;
      // Rows of a pass x: 32 part + kRowsAtOnce x + in_row of a tile.  A warp's 32 rows lie in one page if
      // pages have multiples of 32 rows (tiles then start at one), else 16 by 16.
      const bool one_page = a.R % 32 == 0;
      int page[2] = {-1, -1}, in_page[2] = {0, 0};       // of the tile to load next: its 16-row halves
      auto find = [&](int key0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1 && one_page) {
            page[1] = page[0];
            in_page[1] = in_page[0] + 16;
            break;
          }
          const int key = key0 + 32 * part + 16 * h;
          const int slot = key / a.R;
          page[h] = key < last ? table[slot] : -2;  // -2: nobody sees it
          in_page[h] = key - slot * a.R;
        }
      };
      // Loads without branches between them, so that all are in flight at once: a row that nobody may
      // see, or whose page id is bad, is read from the pool's first page and left out where it is used.
      uint4 code[C::kPasses];  // K's, then V's
      uint8_t kraw[C::kPasses], vraw[C::kPasses];
      uint32_t seen = 0, lost = 0;  // passes whose row may be seen; whose page id is bad
      const uint8_t* rows_at[2];    // this thread's first K codes of each half
      auto load_codes = [&](int64_t offset) {
#pragma unroll
        for (int x = 0; x < C::kPasses; ++x)
          code[x] = *reinterpret_cast<const uint4*>(rows_at[x / (C::kPasses / 2)] + offset +
                                                    x % (C::kPasses / 2) * C::kRowsAtOnce * (D / 2));
      };
      auto load = [&](int key0) {
        seen = lost = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool wanted = page[h] != -2, ok = wanted && index_ok(page[h], 0, a.n_pages, a.err);
          const uint8_t* slab = a.pages + (ok ? page[h] : 0) * a.page_stride + static_cast<int64_t>(head) * a.slab;
          const int r = (ok ? in_page[h] : 0) + in_row;
          const uint8_t* scales = slab + a.R * D + r * C::kC + blk;
          rows_at[h] = slab + r * (D / 2) + blk * 16;
#pragma unroll
          for (int y = 0; y < C::kPasses / 2; ++y) {
            const int x = h * (C::kPasses / 2) + y, key = key0 + 32 * part + C::kRowsAtOnce * x + in_row;
            kraw[x] = scales[y * C::kRowsAtOnce * C::kC];
            vraw[x] = scales[a.R * C::kC + y * C::kRowsAtOnce * C::kC];
            if (key >= first && key < last) (ok ? seen : lost) |= 1u << x;
          }
        }
        load_codes(0);
      };
      // fp16 values of this thread's rows into a swizzled tile (at `offset` from K's); scale(x) gives the
      // scale's fp16 bits.  A row's eight-row phase does not depend on the pass: four addresses do.
      uint32_t to_piece[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) to_piece[q] = smem_u32(piece_at(sk, 32 * part + in_row, blk * 32 + q * 8));
      auto write = [&](uint32_t offset, auto&& scale) {
#pragma unroll
        for (int x = 0; x < C::kPasses; ++x) {
          const uint32_t s = scale(x) * 0x10001u;
          const uint32_t w[4] = {code[x].x, code[x].y, code[x].z, code[x].w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t h[4];
            codes_to_half2(w[q], h);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                         ::"r"(to_piece[q] + offset + C::kRowsAtOnce * 128 * x), "r"(mul2(h[0], s)), "r"(mul2(h[1], s)),
                           "r"(mul2(h[2], s)), "r"(mul2(h[3], s)) : "memory");
          }
        }
      };
      bool large = false;  // a tile of this segment had such V scales: its O has another unit
      if (count > 0) {
        find(key_begin);
        load(key_begin);
        find(key_begin + kKeys);
      }
      for (int t = 0; t < count; ++t) {
        const int key0 = key_begin + t * kKeys;
        Tile& tile = tiles[n_tile & 1];
        bool ok = lost == 0;
#pragma unroll
        for (int x = 0; x < C::kPasses; ++x) {
          if ((seen >> x) & 1u) {
            const uint8_t* codes = rows_at[x / (C::kPasses / 2)] + x % (C::kPasses / 2) * C::kRowsAtOnce * (D / 2);
            if (kraw[x] == 1 && zero_block(code[x])) kraw[x] = 0;
            if (vraw[x] == 1 && zero_block(*reinterpret_cast<const uint4*>(codes + a.R * (D / 2)))) vraw[x] = 0;
            const int k = static_cast<int>(kraw[x]), v = static_cast<int>(vraw[x]);
            // exponents [-14, 13], or a block of zeros
            ok = ok && (k == 0 || (k > 112 && k <= 140)) && (v == 0 || (v > 112 && v <= 140));
          }
        }
        if (n_tile > 0) wait(kSFull, n_tile - 1);  // K is free
        const int word = most_of(!alive ? 2 : ok ? 0 : 1, red, part, lane);
        if (word == 2) {
          alive = false;
          break;
        }
        const bool plain = word == 0 && !large;
        uint32_t kbias = (112u - kLeastBias) * 0x01010101u;
        int windows = 1;
        const bool scribe = part == 0 && lane == 0;
        if (!plain) {
          uint32_t kbytes = 0, vbytes = 0;
#pragma unroll
          for (int x = 0; x < C::kPasses; ++x) {
            kbytes |= static_cast<uint32_t>(kraw[x]) << (8 * x);
            vbytes |= static_cast<uint32_t>(vraw[x]) << (8 * x);
          }
          const int2 found = describe<D>(tile, red, kbytes, vbytes, seen, lost, part, lane);
          kbias = static_cast<uint32_t>(found.x);
          windows = found.y & 255;
          large = large || found.y >= 256;
        }
        if (scribe) {
          tile.plain = plain;
          tile.large = large;
          tile.windows = windows;
        }
        write(0, [&](int x) {
          const int k = static_cast<int>(kraw[x]);
          return !((seen >> x) & 1u) ? 0u : k == 255 ? 0x7e00u : scale_bits(k, static_cast<int>((kbias >> (8 * x)) & 255u) + kLeastBias);
        });
        load_codes(a.R * (D / 2));
        fence_proxy_async_smem();
        arrive(kKFull);
        for (int w = 0; w < windows && alive; ++w) {
          if (n_pv > 0) wait(kOFull, n_pv - 1);  // V is free
          // (or the conversions, the same for all windows, would be kept in registers)
#pragma unroll
          for (int x = 0; x < C::kPasses; ++x) asm volatile("" : "+r"(code[x].x), "+r"(code[x].y), "+r"(code[x].z), "+r"(code[x].w));
          const int least = plain ? 112 : tile.bias[w], most = w == 0 ? 254 : tile.bias[w - 1];
          write(C::kQ, [&](int x) {
            const int v = static_cast<int>(vraw[x]);
            return !((seen >> x) & 1u) || v > most ? 0u : scale_bits(v, least);
          });
          fence_proxy_async_smem();
          arrive(kVFull);
          ++n_pv;
        }
        if (t + 1 < count) {
          load(key0 + kKeys);
          find(key0 + 2 * kKeys);
        }
        ++n_tile;
      }
    } else {
      // ============================================================ softmax
      constexpr uint32_t kIdS = make_idesc_f16(128, 128, 0, 0, false, false);
      constexpr uint32_t kIdO = make_idesc_f16(128, D, 0, 0, false, true), kIdT = make_idesc_f16(128, 64, 0, 0, false, true);
      const uint64_t dq = desc_cols(smem_u32(sq)), dk = desc_cols(smem_u32(sk)), dv = desc_rows(smem_u32(sv));
      const int row = threadIdx.x;  // of the tile; the warp's TMEM lanes
      const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16, ts = tbase + lanes, to = tbase + 128 + lanes;
      const int hi = end_of(row), lo = a.window > 0 ? max(0, hi - a.window) : 0;
      const int inner_lo = a.window > 0 ? max(0, last - a.window) : 0;
      const float nat = (a.scale != 0.f ? fabsf(a.scale) : 1.f) * (a.softcap > 0.f ? 1.f : kLog2e);
      float factor = 0.f;  // raw score -> softmax units
      if (count > 0) {
        const int i = row0 + min(row, rows - 1);
        const T* from = static_cast<const T*>(a.q) + b * a.q_b + (head * G + i % G) * a.q_h + (i / G) * a.q_t;
        float amax = 0.f;
#pragma unroll 4
        for (int k = 0; k < D / 8; ++k) {
          const uint4 raw = *reinterpret_cast<const uint4*>(from + 8 * k);
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float2 f = two_floats(w[x], T{});
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        const int x = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
        const int up = amax > 0.f && x < 128 ? min(14 - x, 126) : 0;  // to fp16's top
        const float f = a.scale > 0.f ? pow2f(up) : a.scale < 0.f ? -pow2f(up) : 0.f;
        factor = fmaxf(pow2f(max(-up, -126)) * nat, kMinFloat);
#pragma unroll 4
        for (int k = 0; k < D / 8; ++k) {
          const uint4 raw = *reinterpret_cast<const uint4*>(from + 8 * k);
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
          uint32_t h[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float2 v = two_floats(w[y], T{});
            h[y] = pack_half2(v.x * f, v.y * f);
          }
          *reinterpret_cast<uint4*>(piece_at(sq, row, 8 * k)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_proxy_async_smem();
        arrive(kQFull);
        if (warp == 0) wait(kQFull, n_seg);
      }

      float m = -INFINITY, l = 0.f;
      int unit = 0;                // O holds sums times 2^-unit: 0 or kLargeUnit
      uint32_t poison = 0;         // blocks of d whose sums are NaN
      bool out_of_range = false;   // maxima above kCoarse
      auto each_sum = [&](auto&& change) {  // of this row in TMEM
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(to + c * 32, r);
          tmem_ld_wait();
          change(r);
          tmem_st32(to + c * 32, r);
        }
        tmem_st_wait();
      };
      for (int t = 0; t < count && alive; ++t) {
        const int key0 = key_begin + t * kKeys;
        wait(kKFull, n_tile);  // the operand warps' word on the tile
        tc_fence_before();  // what S overwrites has been read
        arrive(kReady);
        if (warp == 0) {
          wait(kReady, n_tile);
          if (n_pv > 0) wait(kOFull, n_pv - 1);  // P lies where S goes
          if (alive && elect_one()) {
            tc_fence_after();
#pragma unroll
            for (int s = 0; s < D / 16; ++s) mma_bf16(tbase, dq + step_cols(s), dk + step_cols(s), kIdS, s > 0 ? 1u : 0u);
            mma_commit(bar + kSFull);
          }
          __syncwarp();
        }
        wait(kSFull, n_tile);
        tc_fence_after();
        const Tile& tile = tiles[n_tile & 1];
        const bool plain = tile.plain;
        const float f = plain ? factor : 1.f;  // or every key has its own
        const bool masked = key0 < inner_lo || key0 + kKeys > inner_hi, simple = !masked && plain;
        const Cap cap = a.softcap > 0.f ? Cap(a.softcap, f) : Cap();
        auto visible = [&](uint32_t raw, int j) {  // the score of key key0 + j (times f), or -inf
          float v = __uint_as_float(raw);
          if (!plain) v *= fminf(factor * tile.kunit[j], kMaxFloat);
          if (masked) v = key0 + j >= lo && key0 + j < hi ? v : -INFINITY;
          if (!plain && (tile.nan_keys[j] >> 31)) v = -INFINITY;
          return v;
        };
        float most = -INFINITY;
        if (simple) {  // 64 columns in flight
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t r[32], r2[32];
            tmem_ld32(ts + c * 64, r);
            tmem_ld32(ts + c * 64 + 32, r2);
            tmem_ld_wait();
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j & 3] = fmaxf(x[j & 3], fmaxf(__uint_as_float(r[j]), __uint_as_float(r2[j])));
            most = fmaxf(most, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t r[32];
            tmem_ld32(ts + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) most = fmaxf(most, visible(r[j], c * 32 + j));
          }
        }
        if (a.softcap > 0.f) most = most == -INFINITY ? most : cap.exact(most);  // tanh keeps the order
        else most = __fmul_rn(most, f);
        const float next = most > m + (out_of_range ? 0.f : kLag) ? most : m;
        out_of_range = out_of_range || (next != -INFINITY && fabsf(next) > kCoarse);
        if (t > 0 && __any_sync(0xffffffffu, next != m)) {
          const float keep = shrink(m, next);
          l *= keep;
          each_sum([&](uint32_t (&r)[32]) {
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * keep);
          });
        }
        m = next;
        const float m0 = m == -INFINITY ? 0.f : m, d0 = m == -INFINITY ? 0.f : 15.f - m;  // p times 2^15
        // For coarse maxima: taken off first, from scores that were rounded as they were (15 - m would be 16 - m from
        // 2^24 on).  Capped scores may pass the maximum by their own rounding: fp16's end holds them.
        auto below_maximum = [&](float v) {
          const float x = __fsub_rn(v, m0);
          return (x > 0.99f ? 0.99f : x) + 15.f;
        };
        const bool fine = simple && !__any_sync(0xffffffffu, out_of_range);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t r[32], h[16];
          tmem_ld32(ts + c * 32, r);
          tmem_ld_wait();
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          auto weigh = [&](auto&& exponent) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float x = ex2(exponent(2 * j)), y = ex2(exponent(2 * j + 1));
              sum[(2 * j) & 3] += x;
              sum[(2 * j + 1) & 3] += y;
              h[j] = pack_half2(x, y);
            }
          };
          if (a.softcap > 0.f) {
            if (fine && a.softcap <= kRoundCap) weigh([&](int j) { return cap.round(__uint_as_float(r[j])) + d0; });
            else weigh([&](int j) {
              const float v = visible(r[j], c * 32 + j);
              return v == -INFINITY ? v : below_maximum(cap.exact(v));
            });
          } else if (fine) {
            weigh([&](int j) { return fmaf(__uint_as_float(r[j]), f, d0); });
          } else {
            weigh([&](int j) { return below_maximum(__fmul_rn(visible(r[j], c * 32 + j), f)); });
          }
          // before rounding to fp16: roundings of 2^-12 either way, which the outputs' own hide (the other kernel sums
          // the rounded ones, for there a product with ones is the cheaper sum)
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tmem_st16(ts + c * 16, h);  // over columns of S that have been read
        }
        tmem_st_wait();

        // The product of window w (its V is complete), into O or, for 64 dims at `half`, beside P.
        auto multiply = [&](bool beside, int half) {
          tc_fence_before();
          arrive(kPFull);
          if (warp == 0) {
            wait(kVFull, n_pv);
            wait(kPFull, n_p);
            if (alive && elect_one()) {
              tc_fence_after();
#pragma unroll
              for (int s = 0; s < kKeys / 16; ++s)
                mma_f16_ts(tbase + (beside ? 64 : 128), tbase + 8 * s, dv + (half * kAtom >> 4) + step_rows(s),
                           beside ? kIdT : kIdO, beside ? s > 0 : t > 0 || s > 0);
              if (beside) mma_commit(bar + kTFull);
              if (!beside || half == C::kAtoms - 1) mma_commit(bar + kOFull);
            }
            __syncwarp();
          }
          ++n_p;
        };
        if (plain) {
          multiply(false, 0);
          ++n_pv;
        } else {
          for (int j = 0; j < kKeys; ++j)
            if (key0 + j >= lo && key0 + j < hi) poison |= tile.nan_keys[j] & 0xfu;
          if (tile.large && unit == 0) {
            unit = kLargeUnit;
            if (t > 0)
              each_sum([&](uint32_t (&r)[32]) {
#pragma unroll
                for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * pow2f(-kLargeUnit));
              });
          }
          const int windows = tile.windows;
          for (int w = 0; w < windows && alive; ++w) {
            const Power power(tile.bias[w] - 112 - unit);
            const bool first = t == 0 && w == 0;
            for (int half = 0; half < C::kAtoms && alive; ++half) {
              multiply(true, half);
              wait(kTFull, n_t++);
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < 2; ++c) {
                uint32_t r[32], o[32];
                tmem_ld32(ts + 64 + c * 32, r);
                tmem_ld32(to + half * 64 + c * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  o[j] = __float_as_uint(power.add(__uint_as_float(r[j]), first ? 0.f : __uint_as_float(o[j])));
                tmem_st32(to + half * 64 + c * 32, o);
              }
              tmem_st_wait();
            }
            ++n_pv;
          }
        }
        ++n_tile;
      }

      // ---- the result, or a part of it
      if (take > 0) {
        if (count > 0) {
          wait(kOFull, n_pv - 1);
          tc_fence_after();
        }
        const bool whole = list.whole();
        const int i = row0 + row, h = head * G + min(i, G * a.T - 1) % G;
        const float keep = (l == 0.f ? 0.f : 1.f / l) * (whole && a.sink != nullptr ? share_beside(a.sink[h], m, l) : 1.f);
        const float power = pow2f(unit);
        const int64_t at = (static_cast<int64_t>(b) * a.H + h) * a.T + i / G, slot = list.part_row() + row;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          __syncwarp();
          if (count > 0) {
            tmem_ld32(to + c * 32, r);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = 0;
          }
          const float add = (poison >> c) & 1u ? NAN : 0.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = __uint_as_float(r[8 * q + j]) * keep * power + add;
            if (row >= rows) {
              // nothing to write; the lane stays, for the next turn's load is the whole warp's
            } else if (whole) {
              Few<T, 8> y;
#pragma unroll
              for (int j = 0; j < 8; ++j) y.v[j] = static_cast<T>(o[j]);
              *reinterpret_cast<Few<T, 8>*>(static_cast<T*>(a.out) + at * D + c * 32 + 8 * q) = y;
            } else {
              float4* out = reinterpret_cast<float4*>(a.part_out + slot * D + c * 32 + 8 * q);
              out[0] = make_float4(o[0], o[1], o[2], o[3]);
              out[1] = make_float4(o[4], o[5], o[6], o[7]);
            }
          }
        }
        if (!whole && row < rows) a.part_ml[slot] = make_float2(m, l);
      }
      tc_fence_before();  // the next segment's products overwrite the sums
    }
    if (count > 0) ++n_seg;
    if (!__syncthreads_and(alive)) break;
    if (!list.next(a, row_tiles)) break;
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
