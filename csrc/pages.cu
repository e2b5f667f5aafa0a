// Page bookkeeping of a paged cache, on the device: sequences forked (full pages shared by
// reference counts, a partial last page copied), freed, and the pool compacted.  The pool is
// any tensor whose first dimension is the page: its bytes are only moved.
//
// State: table (S, P) int32 page ids, -1 behind a row's last page; lengths (S) rows;
// refcount (n_pages) rows of the table that hold a page, 0 = free.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"

namespace sv4 {
namespace {

constexpr int kPlan = 1024;  // threads of the planning block

// Exclusive prefix sum of `v` over a block of kPlan threads; *total gets the block's sum.
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int sums[kPlan / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the last call's sums have been read
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    sums[lane] = s;
  }
  __syncthreads();
  *total = sums[kPlan / 32 - 1];
  return x - v + (warp > 0 ? sums[warp - 1] : 0);
}

// The second kernel of a pair may be set up while the first runs, and waits for its results.
__device__ __forceinline__ void release_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

constexpr int kCopyThreads = 256, kPiece = 16384;  // bytes: four 16-byte loads in flight per thread

// Up to kPiece bytes (a multiple of 16) by the whole block.
__device__ __forceinline__ void copy_piece(uint8_t* to, const uint8_t* from, int64_t bytes) {
  const uint4* src = reinterpret_cast<const uint4*>(from);
  uint4* dst = reinterpret_cast<uint4*>(to);
  constexpr int kEach = kPiece / 16 / kCopyThreads;
  const int n = static_cast<int>(bytes / 16);
  uint4 v[kEach];
#pragma unroll
  for (int x = 0; x < kEach; ++x)
    if (static_cast<int>(threadIdx.x) + x * kCopyThreads < n) v[x] = src[threadIdx.x + x * kCopyThreads];
#pragma unroll
  for (int x = 0; x < kEach; ++x)
    if (static_cast<int>(threadIdx.x) + x * kCopyThreads < n) dst[threadIdx.x + x * kCopyThreads] = v[x];
}

// The first `need` free pages in ascending order, by the planning block; returns how many were found.
__device__ __forceinline__ int find_free(const int* refcount, int n_pages, int need, int* found) {
  int have = 0;
  for (int p0 = 0; p0 < n_pages && have < need; p0 += kPlan) {
    const int p = p0 + threadIdx.x;
    int total;
    const int is_free = p < n_pages && refcount[p] == 0;
    const int rank = have + block_scan(is_free, &total);
    if (is_free && rank < need) found[rank] = p;
    have += total;
  }
  __syncthreads();
  return min(have, need);
}

struct ReserveArgs {
  int* table;
  int* lengths;
  int* refcount;
  const int* rows;
  int64_t* slots;  // (n, count)
  int* found;      // (n * pages that `count` rows can open)
  int S, P, n, n_pages, R, count;
  int* err;
};

// One block: the pages that `count` more rows of each sequence open, in the order of the sequences;
// all or nothing.  The pages' ids go into the table, the rows' slots out.
__global__ void __launch_bounds__(kPlan) reserve_rows_kernel(const ReserveArgs a) {
  // pages that sequence i needs, with its row and length; -1: out of range.  Rows and a page more take 32 bits.
  const uint32_t more = static_cast<uint32_t>(a.R) - 1u;
  auto needs = [&](int i, int& row, int& len, int* err) {
    row = a.rows[i];
    len = 0;
    if (!index_ok(row, 0, a.S, err)) return -1;
    len = a.lengths[row];
    if (!index_ok(len, 0, static_cast<int64_t>(a.P) * a.R - a.count + 1, err)) return -1;
    return static_cast<int>((static_cast<uint32_t>(len) + a.count + more) / a.R - (static_cast<uint32_t>(len) + more) / a.R);
  };
  int need = 0, bad = 0;
  for (int i0 = 0; i0 < a.n; i0 += kPlan) {
    const int i = i0 + threadIdx.x;
    int row, len, total;
    const int pages = i < a.n ? needs(i, row, len, a.err) : 0;
    bad += __syncthreads_count(pages < 0);
    block_scan(max(pages, 0), &total);
    need += total;
  }
  const bool fits = bad == 0 && find_free(a.refcount, a.n_pages, need, a.found) == need;
  if (bad == 0 && !fits) record_error(a.err, kErrPages);
  int before = 0;
  for (int i0 = 0; i0 < a.n && fits; i0 += kPlan) {
    const int i = i0 + threadIdx.x;
    int row = 0, len = 0, total;
    const int pages = i < a.n ? needs(i, row, len, nullptr) : 0;
    const int first = before + block_scan(pages, &total);
    for (int x = 0; x < pages; ++x) {
      const int page = a.found[first + x];
      a.table[static_cast<int64_t>(row) * a.P + (static_cast<uint32_t>(len) + more) / a.R + x] = page;
      a.refcount[page] = 1;
    }
    before += total;
  }
  __syncthreads();
  for (int64_t x = threadIdx.x; x < static_cast<int64_t>(a.n) * a.count; x += kPlan) {
    int64_t slot = -1;
    if (fits) {
      const int row = a.rows[x / a.count];
      const int pos = a.lengths[row] + static_cast<int>(x % a.count);
      slot = static_cast<int64_t>(a.table[static_cast<int64_t>(row) * a.P + pos / a.R]) * a.R + pos % a.R;
    }
    a.slots[x] = slot;
  }
  __syncthreads();
  if (fits)
    for (int i = threadIdx.x; i < a.n; i += kPlan) a.lengths[a.rows[i]] += a.count;
}

struct ForkArgs {
  uint8_t* pool;
  int64_t page_bytes;
  const int* table;
  const int* lengths;
  const int* refcount;
  const int* parents;
  const int* children;
  int* new_table;
  int* new_lengths;
  int* new_refcount;
  int* fresh;  // (F + 1): the page that takes the copied tail of fork i, or -1; [F]: 1 if all fitted
  int S, P, F, n_pages, R;
  int* err;
};

// What fork i does: false if its rows are out of range (recorded by `err`, when given).
__device__ __forceinline__ bool fork_rows(const ForkArgs& a, int i, int* err, int* parent, int* child, int* len) {
  *parent = a.parents[i];
  *child = a.children[i];
  *len = 0;
  if (!index_ok(*child, 0, a.S, err) || !index_ok(*parent, -1, a.S, err)) return false;
  if (*parent >= 0) {
    *len = a.lengths[*parent];
    if (!index_ok(*len, 0, static_cast<int64_t>(a.P) * a.R + 1, err)) return false;
  }
  return true;
}

// Block 0 gives every fork that copies a tail the next free page in ascending order; the other
// blocks copy the state that the forks then change.
__global__ void __launch_bounds__(kPlan) fork_plan_kernel(const ForkArgs a) {
  release_next();
  if (blockIdx.x > 0) {
    const int64_t step = static_cast<int64_t>(gridDim.x - 1) * kPlan;
    const int64_t first = static_cast<int64_t>(blockIdx.x - 1) * kPlan + threadIdx.x;
    for (int64_t i = first; i < static_cast<int64_t>(a.S) * a.P; i += step) a.new_table[i] = a.table[i];
    for (int64_t i = first; i < a.S; i += step) a.new_lengths[i] = a.lengths[i];
    for (int64_t i = first; i < a.n_pages; i += step) a.new_refcount[i] = a.refcount[i];
    return;
  }
  int need = 0;
  for (int i0 = 0; i0 < a.F; i0 += kPlan) {
    const int i = i0 + threadIdx.x;
    int parent = -1, child = -1, len = 0, copies = 0, total;
    if (i < a.F && fork_rows(a, i, a.err, &parent, &child, &len)) copies = parent != child && len % a.R != 0;
    const int rank = need + block_scan(copies, &total);
    if (i < a.F) a.fresh[i] = copies ? rank : -1;  // the rank now, the page below
    need += total;
  }
  int* found = a.fresh + a.F + 1;  // the tail of `fresh`
  const bool fits = find_free(a.refcount, a.n_pages, need, found) == need;
  if (!fits) record_error(a.err, kErrPages);
  for (int i = threadIdx.x; i < a.F; i += kPlan) {
    const int rank = a.fresh[i];
    a.fresh[i] = rank >= 0 && fits ? found[rank] : -1;
  }
  if (threadIdx.x == 0) a.fresh[a.F] = fits;
}

// Block (i, y): fork i.  Every block copies pieces of the tail page; block y = 0 also rewrites
// the child's row and counts the pages that it leaves and takes (sums of whole numbers: their
// order does not matter).
__global__ void __launch_bounds__(kCopyThreads) fork_apply_kernel(const ForkArgs a) {
  wait_previous();
  if (a.fresh[a.F] == 0) return;  // too few free pages: nothing changes
  const int i = blockIdx.x;
  int parent, child, len;
  if (!fork_rows(a, i, nullptr, &parent, &child, &len) || parent == child) return;
  const int fresh = a.fresh[i];
  const int tail = len / a.R;
  const int* from = a.table + static_cast<int64_t>(max(parent, 0)) * a.P;
  if (blockIdx.y == 0) {
    const int* old = a.table + static_cast<int64_t>(child) * a.P;
    int* row = a.new_table + static_cast<int64_t>(child) * a.P;
    for (int c = threadIdx.x; c < a.P; c += blockDim.x) {
      const int gone = old[c];
      if (gone >= 0 && index_ok(gone, 0, a.n_pages, a.err)) atomicSub(a.new_refcount + gone, 1);
      int page = parent >= 0 ? from[c] : -1;
      if (fresh >= 0 && c == tail) page = fresh;
      row[c] = page;
      if (page >= 0 && index_ok(page, 0, a.n_pages, a.err)) atomicAdd(a.new_refcount + page, 1);
    }
    if (threadIdx.x == 0) a.new_lengths[child] = len;
  }
  if (fresh < 0) return;
  const int source = from[tail];
  if (!index_ok(source, 0, a.n_pages, a.err)) return;
  for (int64_t at = static_cast<int64_t>(blockIdx.y) * kPiece; at < a.page_bytes; at += static_cast<int64_t>(gridDim.y) * kPiece)
    copy_piece(a.pool + fresh * a.page_bytes + at, a.pool + source * a.page_bytes + at,
               min(static_cast<int64_t>(kPiece), a.page_bytes - at));
}

struct CompactArgs {
  uint8_t* pool;
  int64_t page_bytes;
  const int* table;
  const int* refcount;
  int* new_table;
  int* new_refcount;
  int* live;   // scalar: pages in use
  int* where;  // (n_pages): where a page's contents go; -1: free
  int* moves;  // count, then (target, source) pairs
  int64_t entries;
  int n_pages;
  int* err;
};

// One block: a thread classifies four neighbouring pages, two counts share a scan.  The k-th hole
// below the live count takes the k-th live page from it on.
__global__ void __launch_bounds__(kPlan) compact_plan_kernel(const CompactArgs a) {
  __shared__ int live_s;
  release_next();
  if (threadIdx.x == 0) live_s = 0;
  __syncthreads();
  int mine = 0;
  for (int p = threadIdx.x; p < a.n_pages; p += kPlan) mine += a.refcount[p] > 0;
  mine = __reduce_add_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) atomicAdd(&live_s, mine);
  __syncthreads();
  const int live = live_s;
  if (threadIdx.x == 0) *a.live = live;
  int* target = a.moves + 1;
  int* source = a.moves + 1 + a.n_pages;
  int holes = 0, lates = 0;
  for (int p0 = 0; p0 < a.n_pages; p0 += 4 * kPlan) {
    const int p = p0 + 4 * threadIdx.x;
    uint32_t counts = 0;  // holes in the low half, late pages in the high half: at most 4096 each
    bool hole[4], late[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const bool in = p + x < a.n_pages, used = in && a.refcount[p + x] > 0;
      hole[x] = in && !used && p + x < live;
      late[x] = used && p + x >= live;
      if (in) a.where[p + x] = used && !late[x] ? p + x : -1;
      counts += (hole[x] ? 1u : 0u) + (late[x] ? 0x10000u : 0u);
    }
    int total;
    const uint32_t before = block_scan(static_cast<int>(counts), &total);
    int h = holes + (before & 0xffffu), t = lates + (before >> 16);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (hole[x]) target[h++] = p + x;
      if (late[x]) source[t++] = p + x;
    }
    holes += total & 0xffff;
    lates += static_cast<uint32_t>(total) >> 16;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < lates; k += kPlan) a.where[source[k]] = target[k];
  if (threadIdx.x == 0) a.moves[0] = lates;
}

// Sources are at or behind the live count and targets before it, so the copies are independent.
// Bound by the pool's bytes: blocks take 16 KB pieces of the moved pages in turn.
__global__ void __launch_bounds__(kCopyThreads) compact_apply_kernel(const CompactArgs a) {
  wait_previous();
  const int live = *a.live;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = first; i < a.entries; i += step) {
    const int p = a.table[i];
    a.new_table[i] = p < 0 ? -1 : index_ok(p, 0, a.n_pages, a.err) ? a.where[p] : -1;
  }
  for (int64_t p = first; p < a.n_pages; p += step) {
    const int to = a.where[p];
    if (p >= live) a.new_refcount[p] = 0;
    if (to >= 0) a.new_refcount[to] = a.refcount[p];
  }
  const int64_t pieces = (a.page_bytes + kPiece - 1) / kPiece, n = a.moves[0] * pieces;
  for (int64_t x = blockIdx.x; x < n; x += gridDim.x) {
    const int64_t k = x / pieces, at = (x - k * pieces) * kPiece;
    copy_piece(a.pool + a.moves[1 + k] * a.page_bytes + at, a.pool + a.moves[1 + a.n_pages + k] * a.page_bytes + at,
               min(static_cast<int64_t>(kPiece), a.page_bytes - at));
  }
}

// An int32 tensor like `like`, without the dispatcher's cost (the calls are short).
torch::Tensor ints(at::IntArrayRef sizes, const torch::Tensor& like) {
  return at::detail::empty_cuda(sizes, at::kInt, like.device(), std::nullopt);
}

template <typename A>
void launch_after(void (*kernel)(A), dim3 grid, const A& args, cudaStream_t stream) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(kCopyThreads);
  config.stream = stream;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, args));
}

// The kernels count pages and sequences in 32 bits, and step past the last by a block's share.
void check_counts(int64_t n_pages, int64_t sequences, int64_t forks, const char* who) {
  TORCH_CHECK(std::max({n_pages, sequences, forks}) <= INT32_MAX - 4 * kPlan, who,
              ": more pages or sequences than 32 bits count");
}

// The pool as pages of bytes; returns the bytes of a page.
int64_t check_pool(const torch::Tensor& pool, const torch::Tensor& table, const torch::Tensor& refcount, const char* who) {
  TORCH_CHECK(pool.is_cuda() && pool.dim() >= 2 && pool.is_contiguous(), who,
              ": pool must be a contiguous CUDA tensor (n_pages, ...)");
  const int64_t bytes = pool.size(0) > 0 ? pool.numel() / pool.size(0) * pool.element_size() : 0;
  TORCH_CHECK(bytes % 16 == 0 && reinterpret_cast<uintptr_t>(pool.data_ptr()) % 16 == 0, who,
              ": pages must be multiples of 16 bytes on 16-byte boundaries, got ", std::to_string(bytes));
  TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2 && table.is_contiguous() &&
                  table.device() == pool.device(), who, ": table must be a contiguous (rows, pages) int32 tensor on the pool's device");
  TORCH_CHECK(refcount.scalar_type() == at::kInt && refcount.dim() == 1 && refcount.is_contiguous() &&
                  refcount.device() == pool.device() && refcount.size(0) == pool.size(0), who,
              ": refcount must be a contiguous int32 vector of one count per page");
  check_counts(pool.size(0), table.size(0), 0, who);
  return bytes;
}

}  // namespace

// In place: `count` more rows for each of `rows`; returns their slots (n, count).
torch::Tensor reserve_rows(torch::Tensor table, torch::Tensor lengths, torch::Tensor refcount, torch::Tensor rows,
                           int64_t count, int64_t page_rows, torch::Tensor err) {
  TORCH_CHECK(table.is_cuda() && table.scalar_type() == at::kInt && table.dim() == 2 && table.is_contiguous(),
              "reserve_rows: table must be a contiguous CUDA (rows, pages) int32 tensor");
  auto vec = [&](const torch::Tensor& t) {
    return t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.device() == table.device();
  };
  TORCH_CHECK(vec(lengths) && lengths.size(0) == table.size(0) && vec(refcount) && vec(rows),
              "reserve_rows: lengths, refcount and rows must be contiguous int32 vectors on the table's device");
  TORCH_CHECK(count > 0 && page_rows > 0 && table.size(1) * page_rows <= INT32_MAX && count <= INT32_MAX / 2,
              "reserve_rows: count and page_rows must be positive");
  check_counts(refcount.size(0), table.size(0), rows.size(0) * ((count + page_rows - 1) / page_rows), "reserve_rows");
  c10::cuda::CUDAGuard guard(table.device());
  auto slots = at::detail::empty_cuda({rows.size(0), count}, at::kLong, table.device(), std::nullopt);
  if (rows.size(0) == 0) return slots;
  auto found = ints({rows.size(0) * ((count + page_rows - 1) / page_rows)}, table);
  ReserveArgs a{};
  a.table = table.data_ptr<int>();
  a.lengths = lengths.data_ptr<int>();
  a.refcount = refcount.data_ptr<int>();
  a.rows = rows.data_ptr<int>();
  a.slots = slots.data_ptr<int64_t>();
  a.found = found.data_ptr<int>();
  a.S = static_cast<int>(table.size(0));
  a.P = static_cast<int>(table.size(1));
  a.n = static_cast<int>(rows.size(0));
  a.n_pages = static_cast<int>(refcount.size(0));
  a.R = static_cast<int>(page_rows);
  a.count = static_cast<int>(count);
  a.err = err.data_ptr<int>();
  reserve_rows_kernel<<<1, kPlan, 0, at::cuda::getCurrentCUDAStream()>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return slots;
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> fork_pages(torch::Tensor pool, torch::Tensor table,
                                                                   torch::Tensor lengths, torch::Tensor refcount,
                                                                   torch::Tensor parents, torch::Tensor children,
                                                                   int64_t page_rows, torch::Tensor err) {
  ForkArgs a{};
  a.page_bytes = check_pool(pool, table, refcount, "fork_pages");
  const int64_t F = parents.numel();
  auto vec = [&](const torch::Tensor& t, int64_t n) {
    return t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.size(0) == n && t.device() == pool.device();
  };
  TORCH_CHECK(vec(lengths, table.size(0)), "fork_pages: lengths must be a contiguous int32 vector, one per table row");
  TORCH_CHECK(vec(parents, F) && vec(children, F),
              "fork_pages: parents and children must be contiguous int32 vectors of one length on the pool's device");
  TORCH_CHECK(page_rows > 0 && table.size(1) * page_rows <= INT32_MAX, "fork_pages: page_rows must be positive");
  check_counts(0, 0, F, "fork_pages");
  c10::cuda::CUDAGuard guard(pool.device());
  if (F == 0) return {table.clone(), lengths.clone(), refcount.clone()};
  auto new_table = ints(table.sizes(), table), new_lengths = ints(lengths.sizes(), table), new_refs = ints(refcount.sizes(), table);
  auto fresh = ints({2 * F + 1}, table);
  a.pool = static_cast<uint8_t*>(pool.data_ptr());
  a.table = table.data_ptr<int>();
  a.lengths = lengths.data_ptr<int>();
  a.refcount = refcount.data_ptr<int>();
  a.parents = parents.data_ptr<int>();
  a.children = children.data_ptr<int>();
  a.new_table = new_table.data_ptr<int>();
  a.new_lengths = new_lengths.data_ptr<int>();
  a.new_refcount = new_refs.data_ptr<int>();
  a.fresh = fresh.data_ptr<int>();
  a.S = static_cast<int>(table.size(0));
  a.P = static_cast<int>(table.size(1));
  a.F = static_cast<int>(F);
  a.n_pages = static_cast<int>(pool.size(0));
  a.R = static_cast<int>(page_rows);
  a.err = err.data_ptr<int>();
  const int64_t copied = std::max<int64_t>({table.numel(), lengths.numel(), refcount.numel()});
  auto stream = at::cuda::getCurrentCUDAStream();
  fork_plan_kernel<<<1 + static_cast<unsigned>(std::min<int64_t>(147, (copied + kPlan - 1) / kPlan)), kPlan, 0, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  const int64_t pieces = std::max<int64_t>(1, std::min<int64_t>(64, (a.page_bytes + kPiece - 1) / kPiece));
  launch_after(fork_apply_kernel, dim3(static_cast<unsigned>(F), static_cast<unsigned>(pieces)), a, stream);
  return {new_table, new_lengths, new_refs};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> compact_pages(torch::Tensor pool, torch::Tensor table,
                                                                      torch::Tensor refcount, torch::Tensor err) {
  CompactArgs a{};
  a.page_bytes = check_pool(pool, table, refcount, "compact_pages");
  c10::cuda::CUDAGuard guard(pool.device());
  auto new_table = ints(table.sizes(), table), new_refs = ints(refcount.sizes(), table), live = ints({}, table);
  if (pool.size(0) == 0) return {table.clone(), new_refs, live.zero_()};
  auto work = ints({3 * pool.size(0) + 1}, table);
  a.pool = static_cast<uint8_t*>(pool.data_ptr());
  a.table = table.data_ptr<int>();
  a.refcount = refcount.data_ptr<int>();
  a.new_table = new_table.data_ptr<int>();
  a.new_refcount = new_refs.data_ptr<int>();
  a.live = live.data_ptr<int>();
  a.where = work.data_ptr<int>();
  a.moves = a.where + pool.size(0);
  a.entries = table.numel();
  a.n_pages = static_cast<int>(pool.size(0));
  a.err = err.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
  compact_plan_kernel<<<1, kPlan, 0, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  launch_after(compact_apply_kernel, dim3(148 * 8), a, stream);
  return {new_table, new_refs, live};
}

}  // namespace sv4
