// A step's addressing tensors from request lengths, in one launch: cumulative query lengths, the
// position and pool slot of every new token, the padded block tables and the last row of each request.
//
// Every block scans all request lengths into shared memory (B is at most a few thousand and the
// lengths sit in L2), then fills its share of the tokens (binary search for the request) and of the
// table rows.  A few tens of kilobytes: launch latency bounds it, which is why it is one kernel.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <tuple>

#include "int4_pages.cuh"

namespace lsb {

int* status_ptr(const at::Tensor& status);

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 8192;        // 64 KiB of prefix sums in shared memory

// Sum of two counts (not negative) that stays at INT32_MAX once it gets there: sums of any lengths are in order, and one
// past int32 is past every limit.
__device__ __forceinline__ int2 add_sat(int2 a, int2 b) {
  return make_int2((int)min((uint32_t)a.x + (uint32_t)b.x, (uint32_t)INT32_MAX),
                   (int)min((uint32_t)a.y + (uint32_t)b.y, (uint32_t)INT32_MAX));
}

// Block-wide scan of pairs: the sum of the threads before this one and, through `total`, of all.
__device__ __forceinline__ int2 block_scan(int2 v, int2* scratch, int2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, s.x, o), b = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) s = add_sat(s, make_int2(a, b));
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = s;
  __syncthreads();
  int2 before = make_int2(__shfl_up_sync(0xffffffffu, s.x, 1), __shfl_up_sync(0xffffffffu, s.y, 1));
  if (lane == 0) before = make_int2(0, 0);
  total = make_int2(0, 0);
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before = add_sat(before, scratch[w]);
    total = add_sat(total, scratch[w]);
  }
  return before;
}

__global__ void __launch_bounds__(kThreads) step_maps_kernel(
    const int* __restrict__ q_lens, const int* __restrict__ k_lens, const int* __restrict__ ids, int num_ids, int B,
    int bs, int T, int width, int* __restrict__ cu, int64_t* __restrict__ positions, int* __restrict__ slots,
    int* __restrict__ tables, int64_t* __restrict__ last, int* status) {
  extern __shared__ int2 first[];          // [B + 1]: (first token, first block id) of each request
  __shared__ int2 scratch[kThreads / 32];
  __shared__ int first_bad;                // requests from the first contradicting one on count as empty
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x == 0) first_bad = B;
  __syncthreads();
  const int per = (B + kThreads - 1) / kThreads, lo = min(B, (int)threadIdx.x * per), hi = min(B, lo + per);
  for (int i = lo; i < hi; ++i) {
    const int q = q_lens[i], k = k_lens[i];
    if (q < 0 || k < q || q > T) {
      atomicMin(&first_bad, i);
      break;
    }
  }
  __syncthreads();
  const int good = first_bad;
  auto lengths = [&](int i) {              // (new tokens, blocks) of request i
    return i < good ? make_int2(q_lens[i], (int)(((int64_t)k_lens[i] + bs - 1) / bs)) : make_int2(0, 0);
  };
  int2 mine = make_int2(0, 0), total;
  for (int i = lo; i < hi; ++i) mine = add_sat(mine, lengths(i));
  int2 at = block_scan(mine, scratch, total);
  for (int i = lo; i < hi; ++i) {
    first[i] = at;
    at = add_sat(at, lengths(i));
  }
  if (threadIdx.x == 0) first[B] = total;
  if (blockIdx.x == 0 && (good < B || total.x > T || total.y > num_ids)) record_error(status, kBadIndex);
  __syncthreads();
  const int stride = gridDim.x * kThreads, start = blockIdx.x * kThreads + threadIdx.x;
  for (int t = start; t < T; t += stride) {
    int64_t pos = 0;
    int slot = -1;
    if (t < total.x) {
      int a = 0, b = B;                    // the last request whose first token is <= t (an empty one never is last)
      while (b - a > 1) {
        const int m = (a + b) >> 1;
        if (first[m].x <= t) a = m;
        else b = m;
      }
      const int p = k_lens[a] - q_lens[a] + (t - first[a].x);
      pos = p;
      if (p / bs < num_ids - first[a].y) {         // more blocks than ids: the list ends before the sums do
        const int64_t s = (int64_t)ids[first[a].y + p / bs] * bs + p % bs;
        slot = s >= 0 && s <= INT32_MAX ? (int)s : -1;
      }
    }
    positions[t] = pos;
    slots[t] = slot;
  }
  for (int i = start; i < B * width; i += stride) {
    const int row = i / width, c = i - row * width, at_row = first[row].y;
    tables[i] = c < min(first[row + 1].y, num_ids) - at_row ? ids[at_row + c] : 0;
  }
  for (int i = start; i <= B; i += stride) {
    cu[i] = min(first[i].x, T);
    if (i < B) last[i] = max(0, min(first[i + 1].x, T) - 1);
  }
}

}  // namespace

// q_lens / k_lens int32 [B] (new tokens, keys after the step); ids int32 [N]: each request's block ids
// in order, ceil(k_len / block_size) of them, back to back.  Returns cu_seqlens_q, positions, slot_mapping,
// block_tables, last_token_indices (allocated here: five tensors from Python cost more than the kernel).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> step_maps(at::Tensor q_lens, at::Tensor k_lens,
                                                                                 at::Tensor ids, int64_t bs, int64_t T,
                                                                                 int64_t width, at::Tensor status) {
  const at::Device dev = q_lens.device();
  LSB_INT4_CHECK(q_lens.is_cuda(), "q_lens must be a CUDA tensor");
  int4::check_int32(q_lens, "q_lens", 1, dev);
  int4::check_int32(k_lens, "k_lens", 1, dev);
  int4::check_int32(ids, "block_ids", 1, dev);
  const int64_t B = q_lens.size(0);
  LSB_INT4_CHECK(k_lens.size(0) == B, "q_lens and k_lens differ in length");
  LSB_INT4_CHECK(bs >= 1 && bs <= INT32_MAX, "block_size must be positive");
  LSB_INT4_CHECK(T >= 0 && width >= 0, "num_tokens and table_width must not be negative");
  LSB_INT4_CHECK(B <= kMaxRequests, "more than 8192 requests in one step");
  LSB_INT4_CHECK(T <= INT32_MAX - (1 << 20) && B * width <= INT32_MAX - (1 << 20) && ids.size(0) < INT32_MAX,
                 "step maps exceed int32");
  const at::cuda::CUDAGuard g(dev);
  const auto i32 = q_lens.options(), i64 = i32.dtype(at::kLong);
  at::Tensor cu = at::empty({B + 1}, i32), positions = at::empty({T}, i64), slots = at::empty({T}, i32),
             tables = at::empty({B, width}, i32), last = at::empty({B}, i64);
  const int64_t items = std::max(std::max(T, B * width), B + 1);
  // four items to a thread: a block's scan of the lengths is worth a thousand of them
  const unsigned grid = (unsigned)std::min<int64_t>(148, (items + 4 * kThreads - 1) / (4 * kThreads));
  const int smem = (int)(B + 1) * (int)sizeof(int2);
  ensure_dynamic_smem((const void*)step_maps_kernel, smem);
  launch_pdl(step_maps_kernel, dim3(grid), dim3(kThreads), smem, at::cuda::getCurrentCUDAStream(),
             q_lens.data_ptr<int>(), k_lens.data_ptr<int>(), ids.data_ptr<int>(), (int)ids.size(0), (int)B, (int)bs,
             (int)T, (int)width, cu.data_ptr<int>(), positions.data_ptr<int64_t>(), slots.data_ptr<int>(),
             tables.data_ptr<int>(), last.data_ptr<int64_t>(), status_ptr(status));
  const cudaError_t e = cudaGetLastError();
  LSB_INT4_CHECK(e == cudaSuccess, std::string("step_maps launch failed: ") + cudaGetErrorString(e));
  return {cu, positions, slots, tables, last};
}

}  // namespace lsb
