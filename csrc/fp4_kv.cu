// A paged K / V cache held in 4 bits (MXFP4): rows quantised into pages, rows read back, and
// attention that reads the pages as they are (fp4_attn.cu).  The page format: fp4_kv.cuh.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"
#include "fp4_kv.cuh"

namespace sv4 {
namespace {


template <typename T>
__device__ __forceinline__ float as_float(T v);
template <>
__device__ __forceinline__ float as_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float as_float<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half(v); }

// Eight values in one or two 16-byte accesses.
template <typename T>
struct alignas(16) Eight {
  T v[8];
};

// 2^(byte - 127); 255 is NaN.  Byte 0 (2^-127 in E8M0) is never written and reads as 0.
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}

// Eight values (to be multiplied by `inv`, a power of two) as E2M1 codes, the first in the lowest four
// bits.  cvt rounds ties to the even code, the format to the smaller one: they differ at 0.75, 1.75
// and 3.5.  A value of eleven bits or fewer (16-bit types) times 1 - 2^-20 is below the tie if it was
// a tie, and on its side of it otherwise; fp32 values are first cut to twelve bits, what is cut off
// leaving a one in the last, which keeps them on their side of every tie.  A negative zero becomes zero.
template <typename T>
__device__ __forceinline__ uint32_t e2m1_codes(const float (&f)[8], float inv) {
  float a[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float x = f[j];
    if constexpr (sizeof(T) == 4) {
      const uint32_t bits = __float_as_uint(x);
      x = __uint_as_float((bits & 0xfffff000u) | (((bits & 0xfffu) + 0xfffu) & 0x1000u));
    }
    a[j] = x * (inv * (1.f - 0x1p-20f));
  }
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w) : "f"(a[0]), "f"(a[1]), "f"(a[2]), "f"(a[3]), "f"(a[4]), "f"(a[5]), "f"(a[6]), "f"(a[7]));
  const uint32_t some = ((w & 0x77777777u) + 0x77777777u) & 0x88888888u;  // the sign bit where the magnitude is not 0
  return w & (some | 0x77777777u);
}

// Eight codes -> values.
__device__ __forceinline__ void e2m1_values(uint32_t w, float (&f)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
    f[2 * j] = v.x;
    f[2 * j + 1] = v.y;
  }
}

struct RowsArgs {
  const void* src[2];     // write: K, V rows
  void* dst[2];           // read: K, V rows
  int64_t row_stride[2];  // elements
  int64_t head_stride[2];
  uint8_t* pages;
  int64_t page_stride;
  const int64_t* slots;
  int64_t rows, n_slots;  // n_slots: pages * R
  int heads, R, slab;
  int* err;
};

// Where a slot's row lies: the slabs of its page, and the row in it; null: skipped.
__device__ __forceinline__ uint8_t* page_of(const RowsArgs& a, int64_t slot, int& r) {
  r = 0;
  if (slot == -1 || !index_ok(slot, 0, a.n_slots, a.err)) return nullptr;
  int64_t page;
  if (a.n_slots <= UINT32_MAX) page = static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.R);
  else page = slot / a.R;
  r = static_cast<int>(slot - page * a.R);
  return a.pages + page * a.page_stride;
}

// Both kernels move bytes (16.5 to 32.5 bits a value) and are bound by them and by what a thread
// does besides: one thread handles eight values of kRowsEach rows (accesses of 16 and 4 bytes, neighbours
// next to one another) in kUnits of the rows' parts (K or V of a head), so that finding a row's page is
// paid once for all its parts and four to eight loads are in flight before the first is used.  65537
// rows of 8 heads in fp32: written in 99 us (537 MB in, 143 out), read in 124 us, 6.9 and 5.5 TB/s;
// with one part of four rows to a thread 169 us each.
constexpr int kRowThreads = 256;

// Four neighbouring threads share a scale: the largest magnitude over them.
template <typename T, int D, int kRowsEach, int kUnits>
__global__ void __launch_bounds__(kRowThreads) fp4_kv_write_kernel(const RowsArgs a) {
  constexpr int kPer = D / 8, kRows = kRowThreads / kPer;
  const int part = threadIdx.x % kPer, unit0 = blockIdx.y * kUnits, units = 2 * a.heads;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kRows * kRowsEach) + threadIdx.x / kPer;
  uint8_t* page[kRowsEach];
  int in_page[kRowsEach];
  Eight<T> x[kRowsEach][kUnits];
#pragma unroll
  for (int y = 0; y < kRowsEach; ++y) {
    const int64_t row = row0 + y * kRows;
    const int64_t slot = row < a.rows ? a.slots[row] : -1;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int kv = (unit0 + u) & 1, head = (unit0 + u) >> 1;
      if (row < a.rows && unit0 + u < units)
        x[y][u] = *reinterpret_cast<const Eight<T>*>(static_cast<const T*>(a.src[kv]) + row * a.row_stride[kv] +
                                                     head * a.head_stride[kv] + part * 8);
    }
    page[y] = page_of(a, slot, in_page[y]);
  }
#pragma unroll
  for (int y = 0; y < kRowsEach; ++y) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int kv = (unit0 + u) & 1, head = (unit0 + u) >> 1;
      const bool live = page[y] != nullptr && unit0 + u < units;
      float f[8];
      uint32_t most = 0;  // bits of the largest magnitude; infinity's or above: not finite
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = live ? as_float<T>(x[y][u].v[j]) : 0.f;
        most = max(most, __float_as_uint(f[j]) & 0x7fffffffu);
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      if (!live) continue;
      const bool bad = most >= 0x7f800000u;
      // the magnitude is 1.m * 2^x: the exponent is x - 2 while 1.m <= 1.5
      const int e = max(-126, static_cast<int>(most >> 23) - 129 + ((most & 0x7fffffu) > 0x400000u ? 1 : 0));
      const uint32_t word = bad ? 0u : e2m1_codes<T>(f, __uint_as_float(static_cast<uint32_t>(127 - e) << 23));
      uint8_t* slab = page[y] + static_cast<int64_t>(head) * a.slab;
      const int r = kv * a.R + in_page[y];
      *reinterpret_cast<uint32_t*>(slab + r * (D / 2) + part * 4) = word;
      if ((part & 3) == 0) slab[a.R * D + r * (D / 32) + part / 4] = static_cast<uint8_t>(bad ? 255 : e + 127);
    }
  }
}

template <typename T, int D, int kRowsEach, int kUnits>
__global__ void __launch_bounds__(kRowThreads) fp4_kv_read_kernel(const RowsArgs a) {
  constexpr int kPer = D / 8, kRows = kRowThreads / kPer;
  const int part = threadIdx.x % kPer, unit0 = blockIdx.y * kUnits, units = 2 * a.heads;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kRows * kRowsEach) + threadIdx.x / kPer;
  uint32_t word[kRowsEach][kUnits];
  uint8_t byte[kRowsEach][kUnits];
#pragma unroll
  for (int y = 0; y < kRowsEach; ++y) {
    const int64_t row = row0 + y * kRows;
    int r;
    const uint8_t* page = page_of(a, row < a.rows ? a.slots[row] : -1, r);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      word[y][u] = 0;
      byte[y][u] = 127;
      if (page != nullptr && unit0 + u < units) {
        const uint8_t* slab = page + static_cast<int64_t>((unit0 + u) >> 1) * a.slab;
        const int at = ((unit0 + u) & 1) * a.R + r;
        word[y][u] = *reinterpret_cast<const uint32_t*>(slab + at * (D / 2) + part * 4);
        byte[y][u] = slab[a.R * D + at * (D / 32) + part / 4];
      }
    }
  }
#pragma unroll
  for (int y = 0; y < kRowsEach; ++y) {
    const int64_t row = row0 + y * kRows;
    if (row >= a.rows) continue;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (unit0 + u >= units) continue;
      float f[8];
      e2m1_values(word[y][u], f);
      const float s = scale_of(byte[y][u]);
      Eight<T> z;
#pragma unroll
      for (int j = 0; j < 8; ++j) z.v[j] = from_float<T>(f[j] * s);
      *reinterpret_cast<Eight<T>*>(static_cast<T*>(a.dst[(unit0 + u) & 1]) + (row * a.heads + ((unit0 + u) >> 1)) * D + part * 8) = z;
    }
  }
}

// Numbers in messages go through std::to_string: the stream operators of the toolchain's
// libstdc++ and torch's do not agree on the locale's number facets.
std::string num(int64_t v) { return std::to_string(v); }

// Checks of a pages tensor; returns the rows per page.
int page_rows_of(const torch::Tensor& pages, int64_t d, const char* who) {
  TORCH_CHECK(pages.is_cuda() && pages.scalar_type() == at::kByte && pages.dim() == 3, who,
              ": pages must be a CUDA uint8 tensor (n_pages, kv_heads, slab)");
  TORCH_CHECK(d == 32 || d == 64 || d == 128, who, ": head_dim must be 32, 64 or 128, got ", num(d));
  const int64_t slab = pages.size(2), rows = slab * 16 / (17 * d);
  TORCH_CHECK(rows > 0 && rows % 16 == 0 && rows * d * 17 / 16 == slab, who, ": a slab of ", num(slab),
              " bytes is not a multiple of 16 rows of head_dim ", num(d));
  TORCH_CHECK(rows <= 65536, who, ": at most 65536 rows per page");
  TORCH_CHECK(pages.stride(2) == 1 && (pages.size(1) == 1 || pages.stride(1) == slab) &&
                  (pages.size(0) <= 1 || (pages.stride(0) % 16 == 0 && pages.stride(0) >= pages.size(1) * slab)) &&
                  reinterpret_cast<uintptr_t>(pages.data_ptr()) % 16 == 0,
              who, ": pages must be contiguous within a page, with pages on 16-byte boundaries");
  return static_cast<int>(rows);
}

template <typename F>
void by_dim(int64_t d, F&& f) {
  if (d == 32) f(std::integral_constant<int, 32>{});
  else if (d == 64) f(std::integral_constant<int, 64>{});
  else f(std::integral_constant<int, 128>{});
}

// f(T, D) for the rows' type and head dim.
template <typename F>
void by_type(at::ScalarType t, F&& f) {
  if (t == at::kFloat) f(float{});
  else if (t == at::kHalf) f(__half{});
  else f(__nv_bfloat16{});
}

// A tensor whose rows of eight values can be read in 16-byte pieces.
torch::Tensor rows_aligned(const torch::Tensor& t) {
  const int64_t w = 16 / t.element_size();
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) == 1 || t.stride(i) % w == 0);
  return ok ? t : t.contiguous();
}

// Which of the two attention kernels.  One time grows with 16-row tiles times 32-key steps (about 2 ns
// each at d = 128, behind 10 us), the other with 128-row tiles times 128 keys (20 ns behind 20 us):
// 64 sequences of 4096 keys and 16 heads take 47 and 54 us with 3 tokens each (28k steps), 58 and 55
// with 4 (37k), 78 and 58 with 6 (55k); 8 sequences of 8192 keys 43 and 48 us with 16 tokens (33k).
constexpr int64_t kManySteps = 36000;

bool many_rows(int64_t groups, int64_t rows, int64_t keys) {
  return rows > 32 && groups * ((rows + 15) / 16) * ((keys + 31) / 32) >= kManySteps;
}

RowsArgs rows_args(const torch::Tensor& pages, const torch::Tensor& slots, int64_t d, const char* who) {
  RowsArgs a{};
  a.R = page_rows_of(pages, d, who);
  TORCH_CHECK(slots.is_cuda() && slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.is_contiguous() &&
                  slots.device() == pages.device(), who, ": slots must be a contiguous int64 vector on the pages' device");
  a.pages = pages.data_ptr<uint8_t>();
  a.page_stride = pages.size(0) > 1 ? pages.stride(0) : pages.size(1) * pages.size(2);
  a.slots = slots.data_ptr<int64_t>();
  a.rows = slots.size(0);
  a.n_slots = pages.size(0) * a.R;
  TORCH_CHECK(pages.size(1) <= 32767, who, ": at most 32767 K/V heads");
  a.heads = static_cast<int>(pages.size(1));
  a.slab = static_cast<int>(pages.size(2));
  return a;
}

// A tensor on like's device, without the dispatcher's cost (the calls are short).
torch::Tensor uninitialised(at::IntArrayRef sizes, at::ScalarType dtype, const torch::Tensor& like) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt);
}

// f(T, rows each, units): one head takes two rows of a thread's, more heads two of them of one row.
template <typename F>
void by_rows(const RowsArgs& a, int64_t d, at::ScalarType type, F&& f) {
  const int rows_each = a.heads == 1 ? 2 : 1, units = a.heads == 1 ? 2 : 4;
  const int64_t per = kRowThreads / (d / 8) * rows_each;
  const dim3 grid(static_cast<unsigned>((a.rows + per - 1) / per), static_cast<unsigned>((2 * a.heads + units - 1) / units));
  by_dim(d, [&](auto dim) {
    by_type(type, [&](auto t) {
      if (a.heads == 1) f(t, dim, std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{}, grid);
      else f(t, dim, std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{}, grid);
    });
  });
}

}  // namespace

// Quantise rows k, v (N, kv_heads, d) into `pages` at slots (N) = page * R + row; -1 skips a row.
void fp4_kv_write(torch::Tensor k, torch::Tensor v, torch::Tensor pages, torch::Tensor slots, torch::Tensor err) {
  TORCH_CHECK(k.dim() == 3 && v.sizes() == k.sizes() && k.scalar_type() == v.scalar_type() && k.is_cuda() &&
                  v.device() == k.device() && k.device() == pages.device(),
              "fp4_kv_write: k and v must be (rows, kv_heads, head_dim) of one type on the pages' device");
  TORCH_CHECK(k.scalar_type() == at::kFloat || k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16,
              "fp4_kv_write: rows must be bf16, fp16 or fp32");
  const int64_t d = k.size(2);
  RowsArgs a = rows_args(pages, slots, d, "fp4_kv_write");
  TORCH_CHECK(k.size(1) == a.heads && k.size(0) == a.rows, "fp4_kv_write: ", num(k.size(0)), " rows of ",
              num(k.size(1)), " heads for ", num(a.rows), " slots and pages of ", num(a.heads), " heads");
  if (k.numel() == 0) return;
  c10::cuda::CUDAGuard guard(k.device());
  k = rows_aligned(k);
  v = rows_aligned(v);
  a.src[0] = k.data_ptr();
  a.src[1] = v.data_ptr();
  a.row_stride[0] = k.stride(0);
  a.row_stride[1] = v.stride(0);
  a.head_stride[0] = k.stride(1);
  a.head_stride[1] = v.stride(1);
  a.err = err.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
  by_rows(a, d, k.scalar_type(), [&](auto t, auto dim, auto each, auto units, dim3 grid) {
    fp4_kv_write_kernel<decltype(t), decltype(dim)::value, decltype(each)::value, decltype(units)::value>
        <<<grid, kRowThreads, 0, stream>>>(a);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// The rows at `slots` as k, v (N, kv_heads, d) of type `dtype`; a slot of -1 gives zeros.
std::tuple<torch::Tensor, torch::Tensor> fp4_kv_read(torch::Tensor pages, torch::Tensor slots, int64_t d,
                                                     at::ScalarType dtype, torch::Tensor err) {
  TORCH_CHECK(dtype == at::kFloat || dtype == at::kHalf || dtype == at::kBFloat16,
              "fp4_kv_read: rows are read in bf16, fp16 or fp32");
  RowsArgs a = rows_args(pages, slots, d, "fp4_kv_read");
  c10::cuda::CUDAGuard guard(pages.device());
  auto k = uninitialised({a.rows, a.heads, d}, dtype, pages), v = uninitialised({a.rows, a.heads, d}, dtype, pages);
  if (k.numel() == 0) return {k, v};
  a.dst[0] = k.data_ptr();
  a.dst[1] = v.data_ptr();
  a.err = err.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
  by_rows(a, d, k.scalar_type(), [&](auto t, auto dim, auto each, auto units, dim3 grid) {
    fp4_kv_read_kernel<decltype(t), decltype(dim)::value, decltype(each)::value, decltype(units)::value>
        <<<grid, kRowThreads, 0, stream>>>(a);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {k, v};
}

// q (B, H, T, d) bf16 / fp16; table (B, P) int32; lengths (B) int32, the T tokens included.
torch::Tensor fp4_kv_attention(torch::Tensor q, torch::Tensor pages, torch::Tensor table, torch::Tensor lengths,
                               int64_t window, c10::optional<torch::Tensor> sink, double softcap, double scale,
                               torch::Tensor err) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 4 && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf),
              "fp4_kv_attention: q must be a CUDA (B, H, T, head_dim) tensor in bf16 or fp16");
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), d = q.size(3);
  Fp4AttnArgs a{};
  a.R = page_rows_of(pages, d, "fp4_kv_attention");
  const int64_t Hk = pages.size(1);
  TORCH_CHECK(Hk > 0 && H % Hk == 0, "fp4_kv_attention: ", num(H), " query heads over ", num(Hk),
              " K/V heads");
  TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == B && table.is_contiguous() &&
                  table.device() == q.device() && pages.device() == q.device(),
              "fp4_kv_attention: table must be a contiguous (B, pages) int32 tensor on q's device");
  TORCH_CHECK(lengths.scalar_type() == at::kInt && lengths.dim() == 1 && lengths.size(0) == B &&
                  lengths.is_contiguous() && lengths.device() == q.device(),
              "fp4_kv_attention: lengths must be a contiguous int32 vector of ", num(B), " on q's device");
  TORCH_CHECK(table.size(1) * a.R + T <= INT32_MAX - 1024 && window >= 0 && softcap >= 0,
              "fp4_kv_attention: window and softcap must not be negative, table rows and tokens below 2^31 - 1024");
  // A window of the whole table sees what no window sees.  Positions, -T at the least, less a smaller
  // window stay within 32 bits.
  if (window >= table.size(1) * a.R) window = 0;
  if (sink.has_value())
    TORCH_CHECK(sink->scalar_type() == at::kFloat && sink->numel() == H && sink->is_contiguous() &&
                    sink->device() == q.device(), "fp4_kv_attention: sink must be ", num(H), " contiguous fp32 values");
  c10::cuda::CUDAGuard guard(q.device());
  torch::Tensor out = uninitialised({B, H, T, d}, q.scalar_type(), q);
  if (out.numel() == 0) return out;
  q = rows_aligned(q);
  a.q = q.data_ptr();
  a.q_b = q.stride(0);
  a.q_h = q.stride(1);
  a.q_t = q.stride(2);
  a.pages = pages.data_ptr<uint8_t>();
  a.page_stride = pages.size(0) > 1 ? pages.stride(0) : Hk * pages.size(2);
  a.n_pages = pages.size(0);
  a.table = table.data_ptr<int>();
  a.lengths = lengths.data_ptr<int>();
  a.sink = sink.has_value() ? sink->data_ptr<float>() : nullptr;
  a.out = out.data_ptr();
  a.B = static_cast<int>(B);
  a.H = static_cast<int>(H);
  a.Hk = static_cast<int>(Hk);
  a.T = static_cast<int>(T);
  a.P = static_cast<int>(table.size(1));
  a.slab = static_cast<int>(pages.size(2));
  a.window = static_cast<int>(window);
  a.scale = static_cast<float>(scale);
  a.softcap = static_cast<float>(softcap);
  a.err = err.data_ptr<int>();
  TORCH_CHECK(B <= 65535 && H * T <= (1 << 26), "fp4_kv_attention: at most 65535 sequences and 2^26 query rows in each");
  const int64_t keys = window > 0 ? std::min<int64_t>(table.size(1) * a.R, window + T) : table.size(1) * a.R;
  const bool many = d >= 64 && pages.size(0) > 0 && many_rows(B * Hk, H / Hk * T, keys);
  const Fp4AttnPlan plan = many ? fp4_attn_tile_plan(a) : fp4_attn_rows_plan(a, static_cast<int>(d));
  TORCH_CHECK(plan.units < INT32_MAX, "fp4_kv_attention: the table has room for more than 2^31 tiles of work (its width counts, not the lengths); "
              "split the batch");
  a.blocks = plan.blocks;
  const int64_t part_rows = static_cast<int64_t>(plan.blocks) * 2 * plan.rows;
  torch::Tensor parts = uninitialised({part_rows * (d + 2)}, at::kFloat, q);
  a.part_ml = reinterpret_cast<float2*>(parts.data_ptr<float>());
  a.part_out = parts.data_ptr<float>() + 2 * part_rows;
  (many ? fp4_attn_tile : fp4_attn_rows)(a, static_cast<int>(d), q.scalar_type() == at::kHalf, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

}  // namespace sv4
