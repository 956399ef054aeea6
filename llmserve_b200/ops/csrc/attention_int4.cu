// Causal attention of packed query rows against 4-bit KV pages (format: int4_pages.cuh).
//
// One block per (query row, head): four warps take every fourth key, a lane holds head_dim / 32
// neighbouring dims of the query and the output, and each warp keeps its running maximum and sum
// (fp32); the warps merge through shared memory at the end.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "int4_pages.cuh"

namespace lsb {

int* status_ptr(const at::Tensor& status);

namespace {

using namespace int4;
constexpr int kWarps = 4;

// cu_q == nullptr: exactly nq query rows per sequence.
template <int HD>
__global__ void __launch_bounds__(kWarps * 32) attention_int4_kernel(
    bf16* __restrict__ out, const bf16* __restrict__ q, Pages kp, Pages vp, const int* __restrict__ cu_q, int nq,
    const int* __restrict__ k_lens, const int* __restrict__ tables, int width, int B, float scale_log2, int nh, int nkv,
    int bs, int nblk, int* status) {
  pdl_trigger();
  pdl_wait();
  constexpr int kD = HD / 32;
  __shared__ float sm_o[kWarps][HD], sm_m[kWarps], sm_l[kWarps];
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, kvh = h / (nh / nkv), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int seq, row, q_len;
  if (cu_q == nullptr) {
    seq = (int)(t / nq), row = (int)(t % nq), q_len = nq;
  } else {
    if (t >= cu_q[B]) return;                      // rows behind the last sequence stay as they are
    int a = 0, b = B;
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (cu_q[m] <= t) a = m;
      else b = m;
    }
    seq = a, row = (int)t - cu_q[a], q_len = cu_q[a + 1] - cu_q[a];
  }
  const int k_len = k_lens[seq];
  const int end = min(min(k_len, k_len - q_len + row + 1), (int)min((int64_t)width * bs, (int64_t)INT32_MAX));
  float x[kD], o[kD], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kD; ++i) {
    x[i] = to_f(q[(t * nh + h) * HD + lane * kD + i]) * scale_log2;
    o[i] = 0.f;
  }
  for (int j = warp; j < end; j += kWarps) {
    const int blk = tables[(int64_t)seq * width + j / bs];
    if (blk < 0 || blk >= nblk) {
      if (lane == 0) record_error(status, kBadIndex);
      continue;
    }
    const size_t r = ((size_t)blk * nkv + kvh) * bs + j % bs;
    auto value = [&](const Pages& p, int i) {
      const int d = lane * kD + i;
      const uint32_t w = (uint16_t)p.words[r * (HD / kGroup) + d / kGroup];
      const uint32_t c = (p.codes[r * (HD / 2) + d / 2] >> (4 * (d & 1))) & 15u;
      return word_scale(w) * (float)((int)c - (int)word_zero(w));
    };
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kD; ++i) s += x[i] * value(kp, i);
    s = warp_sum(s);
    const float mn = fmaxf(m, s), a = m == -INFINITY ? 0.f : exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * a + p;
#pragma unroll
    for (int i = 0; i < kD; ++i) o[i] = o[i] * a + p * value(vp, i);
  }
#pragma unroll
  for (int i = 0; i < kD; ++i) sm_o[warp][lane * kD + i] = o[i];
  if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
  __syncthreads();
  for (int d = threadIdx.x; d < HD; d += kWarps * 32) {
    float mx = -INFINITY, sum = 0.f, acc = 0.f;
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm_m[w]);
    for (int w = 0; w < kWarps; ++w) {
      const float a = sm_l[w] == 0.f ? 0.f : exp2f(sm_m[w] - mx);
      sum += a * sm_l[w];
      acc += a * sm_o[w][d];
    }
    out[(t * nh + h) * HD + d] = to_b(sum == 0.f ? 0.f : acc / sum);
  }
}

}  // namespace

void attention_int4(at::Tensor out, at::Tensor q, at::Tensor kc, at::Tensor kw, at::Tensor vc, at::Tensor vw,
                    at::Tensor cu_q, int64_t nq, at::Tensor k_lens, at::Tensor tables, double scale,
                    at::Tensor status) {
  const at::Device dev = q.device();
  check_page_pair(kc, kw, vc, vw, dev);
  LSB_INT4_CHECK(q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.is_contiguous(),
                 "q must be contiguous bfloat16 [rows, heads, head_dim]");
  LSB_INT4_CHECK(q.size(2) == kc.size(3) * 2 && q.size(1) >= 1 && q.size(1) % kc.size(1) == 0,
                 "query heads do not match the pages");
  LSB_INT4_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.is_contiguous() &&
                     out.device() == dev, "bad output");
  check_int32(k_lens, "sequence lengths", 1, dev);
  check_int32(tables, "block_tables", 2, dev);
  const int64_t B = k_lens.size(0), T = q.size(0);
  LSB_INT4_CHECK(tables.size(0) >= B, "block_tables must hold one row per sequence");
  if (nq > 0) {
    LSB_INT4_CHECK(T == B * nq, "q must hold nq rows per sequence");
  } else {
    check_int32(cu_q, "cu_seqlens_q", 1, dev);
    LSB_INT4_CHECK(cu_q.size(0) == B + 1, "cu_seqlens_q must hold one entry more than there are sequences");
  }
  if (T == 0 || B == 0) return;
  const at::cuda::CUDAGuard g(dev);
  auto go = [&](auto kern) {
    launch_pdl(kern, dim3((unsigned)T, (unsigned)q.size(1)), dim3(kWarps * 32), 0, at::cuda::getCurrentCUDAStream(),
               (bf16*)out.data_ptr(), (const bf16*)q.data_ptr(),
               Pages{kc.data_ptr<uint8_t>(), kw.data_ptr<int16_t>()}, Pages{vc.data_ptr<uint8_t>(), vw.data_ptr<int16_t>()},
               nq > 0 ? (const int*)nullptr : (const int*)cu_q.data_ptr<int>(), (int)nq, k_lens.data_ptr<int>(),
               tables.data_ptr<int>(), (int)tables.size(1), (int)B, (float)(scale * 1.4426950408889634),
               (int)q.size(1), (int)kc.size(1), (int)kc.size(2), (int)kc.size(0), status_ptr(status));
  };
  if (q.size(2) == 128) go(attention_int4_kernel<128>);
  else go(attention_int4_kernel<64>);
  const cudaError_t e = cudaGetLastError();
  LSB_INT4_CHECK(e == cudaSuccess, std::string("attention_int4 launch failed: ") + cudaGetErrorString(e));
}

}  // namespace lsb
