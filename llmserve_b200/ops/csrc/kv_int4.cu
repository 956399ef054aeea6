// Filling and reading back 4-bit KV pages (format: int4_pages.cuh).
//
// A lane holds eight consecutive dims of a row (one 16-byte access of bf16, one 4-byte word of codes), so a
// group of 64 dims is eight lanes and its range two three-step butterflies.  Each byte moves once.  For a step's
// rows launch latency bounds the kernels; for prompts the quantiser's arithmetic (the store issues in 77% of the
// cycles, integer pipe 62%) and, in the fused store, waiting for loads with half the warps.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <tuple>

#include "int4_pages.cuh"

namespace lsb {

int* status_ptr(const at::Tensor& status);

namespace {

using namespace int4;
constexpr int kThreads = 128;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Codes (eight nibbles, dim order) and scale word of a group of 64 held eight values to a lane by
// eight neighbouring lanes; every lane of the group gets the word.
//   range widened to hold zero; s = range / 15 rounded UP to four significant bits, so no code
//   saturates by more than the half step that rounding both ends can cost; z = rint(-min / s);
//   c = min(15, rint(x / s) + z).
// A group whose range is below 15 times the smallest normal number is stored as zeros, one that holds
// an infinity or a NaN as NaN (scale NaN), so that a broken row stays visible.
//
// x / s is x * (1 / s): for bf16 inputs (kSnap) a quotient that lies exactly half way between two
// codes must stay there.  x has eight significant bits and s four, so a quotient above 1/4 that is
// not half way is at least 2^-6 / 30 = 5.2e-4 away from it; rounding to a multiple of 2^-13 (the sum with
// 1536) moves it by 6.1e-5 at most and removes the 4e-6 that an approximate reciprocal adds, which gives
// the division's result.  The sum with 1.5 * 2^23 then rounds to the integer, half to even, and leaves it
// in the low mantissa bits: no conversion instruction (a quarter of the rate) and no division (16384 rows
// of 8 heads of 128, store and read-back: 73 us with them and 64-bit indexing, 43 us without).
template <bool kSnap>
__device__ __forceinline__ int round_code(float x, float inv) {
  const float y = kSnap ? __fadd_rn(fmaf(x, inv, 1536.f), 12582912.f - 1536.f) : fmaf(x, inv, 12582912.f);
  return __float_as_int(y) - 0x4b400000;
}
template <bool kSnap>
__device__ __forceinline__ uint32_t quantise8(const float* x, uint32_t& word) {
  float mx = 0.f, mn = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    mx = max_nan(mx, x[i]);
    mn = min_nan(mn, x[i]);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  // r = (range / 2) / 7.5: product with the reciprocal and one correction, exact where the quotient is
  const float half = 0.5f * mx - 0.5f * mn, q = half * 0.13333334f, r = fmaf(fmaf(-q, 7.5f, half), 0.13333334f, q);
  if (!(r <= 3.402823466e38f)) {          // NaN or infinity in the group
    word = 0x7fc0u;
    return 0u;
  }
  word = 0u;
  if (r < 1.17549435e-38f) return 0u;
  const uint32_t sbits = (__float_as_uint(r) + 0xfffffu) & 0x7ff00000u;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(__uint_as_float(sbits)));
  const int z = round_code<kSnap>(-mn, inv);
  word = (sbits >> 16) | (uint32_t)z;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) codes = codes * 16u + (uint32_t)min(round_code<kSnap>(x[i], inv) + z, 15);
  return codes;
}

__device__ __forceinline__ void unpack_bf16x8(const uint4& u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Row (slot, kv head) of a pool; false for a skipped slot (< 0) or one outside the pool (recorded).
__device__ __forceinline__ bool page_row(int slot, int64_t num_slots, int nkv, int h, uint32_t bs, int* status,
                                         size_t& row) {
  if (slot < 0) return false;
  if (slot >= num_slots) {
    record_error(status, kBadIndex);
    return false;
  }
  const uint32_t blk = (uint32_t)slot / bs, off = (uint32_t)slot - blk * bs;
  row = ((size_t)blk * nkv + h) * bs + off;
  return true;
}

// Unit u of 8 dims: (token, head, part) in row-major order; a lane takes it of K and of V, two independent
// chains on one slot look-up.
template <int HD>
__global__ void __launch_bounds__(kThreads) store_int4_kernel(
    const bf16* __restrict__ k, const bf16* __restrict__ v, int64_t kst, int64_t ksh, int64_t vst, int64_t vsh,
    uint8_t* __restrict__ kc, int16_t* __restrict__ kw, uint8_t* __restrict__ vc, int16_t* __restrict__ vw,
    const int* __restrict__ slots, uint32_t rows, uint32_t nkv, uint32_t bs, int64_t num_slots, int* status) {
  pdl_trigger();
  pdl_wait();
  constexpr int kLanes = HD / 8;
  const uint32_t th0 = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const bool live = th0 < rows;
  const uint32_t th = live ? th0 : rows - 1;       // tail lanes take part in the butterflies
  const uint32_t t = th / nkv, h = th - t * nkv;
  const int slot = slots[t];
  float x[8], y[8];
  unpack_bf16x8(*reinterpret_cast<const uint4*>(k + t * kst + h * ksh + lane * 8), x);
  unpack_bf16x8(*reinterpret_cast<const uint4*>(v + t * vst + h * vsh + lane * 8), y);
  uint32_t word_k, word_v;
  const uint32_t codes_k = quantise8<true>(x, word_k), codes_v = quantise8<true>(y, word_v);
  size_t row;
  if (!live || !page_row(slot, num_slots, nkv, h, bs, status, row)) return;
  reinterpret_cast<uint32_t*>(kc + row * (HD / 2))[lane] = codes_k;
  reinterpret_cast<uint32_t*>(vc + row * (HD / 2))[lane] = codes_v;
  if (lane % 8 == 0) {
    kw[row * (HD / kGroup) + lane / 8] = (int16_t)word_k;
    vw[row * (HD / kGroup) + lane / 8] = (int16_t)word_v;
  }
}

// eight codes of one group as bf16.  128 + c is a bf16 with c in its low mantissa bits; pairs (n, n + 4) of
// nibbles, put in order at the end
__device__ __forceinline__ uint4 dequantise8(uint32_t c, uint32_t w) {
  const uint32_t dup = __byte_perm(w, 0, 0x1010), s2 = dup & 0x7ff07ff0u, z2 = (dup & 0x000f000fu) | 0x43004300u;
  uint32_t y[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) y[n] = mul2(sub2(((c >> (4 * n)) & 0x000f000fu) | 0x43004300u, z2), s2);
  return make_uint4(__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410), __byte_perm(y[0], y[1], 0x7632),
                    __byte_perm(y[2], y[3], 0x7632));
}

template <int HD>
__global__ void __launch_bounds__(kThreads) load_int4_kernel(
    bf16* __restrict__ k, bf16* __restrict__ v, const uint8_t* __restrict__ kc, const int16_t* __restrict__ kw,
    const uint8_t* __restrict__ vc, const int16_t* __restrict__ vw, const int* __restrict__ slots, uint32_t rows,
    uint32_t nkv, uint32_t bs, int64_t num_slots, int* status) {
  pdl_trigger();
  pdl_wait();
  constexpr int kLanes = HD / 8;
  const uint32_t th = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  if (th >= rows) return;
  const uint32_t t = th / nkv, h = th - t * nkv;
  uint32_t ck = 0, cv = 0, wk = 0, wv = 0;         // scale 0: zeros
  size_t row;
  if (page_row(slots[t], num_slots, nkv, h, bs, status, row)) {
    ck = reinterpret_cast<const uint32_t*>(kc + row * (HD / 2))[lane];
    cv = reinterpret_cast<const uint32_t*>(vc + row * (HD / 2))[lane];
    wk = (uint16_t)kw[row * (HD / kGroup) + lane / 8];
    wv = (uint16_t)vw[row * (HD / kGroup) + lane / 8];
  }
  reinterpret_cast<uint4*>(k)[(size_t)th * kLanes + lane] = dequantise8(ck, wk);
  reinterpret_cast<uint4*>(v)[(size_t)th * kLanes + lane] = dequantise8(cv, wv);
}

// Whole pages in the layout of a bf16 pool, [n, nkv, bs, HD], and the table that addresses them: i for page i, -1
// where its id lies outside the pool (its rows are zeros), so that the reader skips and records it.
template <int HD>
__global__ void __launch_bounds__(kThreads) load_pages_int4_kernel(
    bf16* __restrict__ k, bf16* __restrict__ v, int* __restrict__ table, const uint8_t* __restrict__ kc,
    const int16_t* __restrict__ kw, const uint8_t* __restrict__ vc, const int16_t* __restrict__ vw,
    const int* __restrict__ ids, uint32_t rows, uint32_t page_rows, uint32_t nblk) {
  pdl_trigger();
  pdl_wait();
  constexpr int kLanes = HD / 8;
  const uint32_t th = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  if (th >= rows) return;
  const uint32_t page = th / page_rows, in_page = th - page * page_rows;
  const uint32_t blk = (uint32_t)ids[page];
  const bool there = blk < nblk;
  if (in_page == 0 && lane == 0) table[page] = there ? (int)page : -1;
  uint32_t ck = 0, cv = 0, wk = 0, wv = 0;         // scale 0: zeros
  if (there) {
    const size_t row = (size_t)blk * page_rows + in_page;
    ck = reinterpret_cast<const uint32_t*>(kc + row * (HD / 2))[lane];
    cv = reinterpret_cast<const uint32_t*>(vc + row * (HD / 2))[lane];
    wk = (uint16_t)kw[row * (HD / kGroup) + lane / 8];
    wv = (uint16_t)vw[row * (HD / kGroup) + lane / 8];
  }
  reinterpret_cast<uint4*>(k)[(size_t)th * kLanes + lane] = dequantise8(ck, wk);
  reinterpret_cast<uint4*>(v)[(size_t)th * kLanes + lane] = dequantise8(cv, wv);
}

// One step's projection rows [T, (nh + 2 nkv) * HD] (bf16, or S fp32 split-K planes that are summed
// here): per-head RMS norm of q and k (optional), rotation, q out as bf16, k and v into the pages.
// Everything between the load and the one rounding at the end is fp32.  HD / 8 lanes hold a head;
// the rotation's partner dim (d, d + HD/2) is HD / 16 lanes away.  A block takes `steps` heads per lane
// group of one token, so that the angles are loaded once for them: several for a prompt's rows, one for
// a step's, where more blocks are worth more (8191 rows of 48 heads with their read-back: 85 us with one, 69 with
// six).
template <int HD, bool kPlanes>
__global__ void __launch_bounds__(kThreads) rope_store_int4_kernel(
    bf16* __restrict__ q_out, const void* __restrict__ qkv, int S, const int64_t* __restrict__ positions,
    const float* __restrict__ cos_sin, int64_t max_pos, const bf16* __restrict__ q_w, const bf16* __restrict__ k_w,
    float eps, uint8_t* __restrict__ kc, int16_t* __restrict__ kw, uint8_t* __restrict__ vc, int16_t* __restrict__ vw,
    const int* __restrict__ slots, int T, int nh, int nkv, int steps, uint32_t bs, int64_t num_slots, int* status) {
  pdl_trigger();
  pdl_wait();
  constexpr int kLanes = HD / 8, kHalf = HD / 2, kGroups = kThreads / kLanes;
  const int heads = nh + 2 * nkv, t = blockIdx.x;
  const int head0 = blockIdx.y * kGroups * steps + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes, d0 = lane * 8;
  auto load = [&](int head, float* x) {
    const int64_t at = ((int64_t)t * heads + min(head, heads - 1)) * HD + d0;
    if constexpr (kPlanes) {
      const float* p = (const float*)qkv + at;
      const int64_t plane = (int64_t)T * heads * HD;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
#pragma unroll 4
      for (int s = 0; s < S; ++s) {
        const float4 a = *reinterpret_cast<const float4*>(p + s * plane);
        const float4 b = *reinterpret_cast<const float4*>(p + s * plane + 4);
        x[0] += a.x, x[1] += a.y, x[2] += a.z, x[3] += a.w;
        x[4] += b.x, x[5] += b.y, x[6] += b.z, x[7] += b.w;
      }
    } else {
      unpack_bf16x8(*reinterpret_cast<const uint4*>((const bf16*)qkv + at), x);
    }
  };
  float x[8], c[8], s[8];
  load(head0, x);
  const int slot = slots[t];
  int64_t pos = positions[t];
  const bool pos_ok = pos >= 0 && pos < max_pos;
  if (!pos_ok) {                                   // never read outside the table; the row is not stored
    if (head0 == 0) record_error(status, kBadIndex);
    pos = 0;
  }
  const float* cs = cos_sin + pos * HD + (d0 & (kHalf - 1));
  const float sign = d0 < kHalf ? -1.f : 1.f;      // x1 c - x2 s | x2 c + x1 s
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(cs + i);
    const float4 v = *reinterpret_cast<const float4*>(cs + kHalf + i);
    s[i] = sign * v.x, s[i + 1] = sign * v.y, s[i + 2] = sign * v.z, s[i + 3] = sign * v.w;
  }
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    const int head = head0 + i * kGroups;
    if (head - threadIdx.x / kLanes >= heads) break;       // the same for the whole block
    float next[8];
    if (i + 1 < steps) load(head + kGroups, next);
    const bool live = head < heads, is_v = head >= nh + nkv;
    if (q_w != nullptr) {                          // uniform over the grid: both weights or neither
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (!is_v) {
        const float inv = rsqrtf(ss / HD + eps);
        float g[8];
        unpack_bf16x8(*reinterpret_cast<const uint4*>((head < nh ? q_w : k_w) + d0), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * g[e];
      }
    }
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __shfl_xor_sync(0xffffffffu, x[e], kLanes / 2);
    if (!is_v)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * c[e] + y[e] * s[e];
    uint32_t word = 0, codes = 0;
    if (__any_sync(0xffffffffu, head >= nh)) {     // a warp of query heads has nothing to quantise
      // values that are bf16 already (V of a bf16 projection) take the exact-tie form
      const bool all_v = !kPlanes && __all_sync(0xffffffffu, is_v), some_v = !kPlanes && __any_sync(0xffffffffu, is_v);
      if (!all_v) codes = quantise8<false>(x, word);
      if (some_v) {
        uint32_t word_v;
        const uint32_t codes_v = quantise8<true>(x, word_v);
        if (is_v) codes = codes_v, word = word_v;
      }
    }
    if (live && head < nh) {
      *reinterpret_cast<uint4*>(q_out + ((int64_t)t * nh + head) * HD + d0) =
          pos_ok ? make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]))
                 : make_uint4(0, 0, 0, 0);
    } else if (live) {
      const int h = is_v ? head - nh - nkv : head - nh;
      size_t row;
      if (pos_ok && page_row(slot, num_slots, nkv, h, bs, status, row)) {
        reinterpret_cast<uint32_t*>((is_v ? vc : kc) + row * (HD / 2))[lane] = codes;
        if (lane % 8 == 0) (is_v ? vw : kw)[row * (HD / kGroup) + lane / 8] = (int16_t)word;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = next[e];
  }
}

// Accepted tree nodes' rows of every layer into the pools, codes and words as they are (quantising what was
// quantised before need not give the same codes).  grid (layers, committed nodes, kv heads); lanes 0..15 take K,
// 16..31 V.  A few kilobytes: launch latency bounds it.
__global__ void commit_tree_int4_kernel(
    const uint8_t* __restrict__ tkc, const int16_t* __restrict__ tkw, const uint8_t* __restrict__ tvc,
    const int16_t* __restrict__ tvw, uint8_t* __restrict__ kc, int16_t* __restrict__ kw, uint8_t* __restrict__ vc,
    int16_t* __restrict__ vw, const int* __restrict__ nodes, const int* __restrict__ slots, int n_nodes, int nkv, int hd,
    uint32_t bs, int64_t num_slots, int* status) {
  pdl_trigger();
  pdl_wait();
  const int layer = blockIdx.x, h = blockIdx.z, lane = threadIdx.x & 15;
  const bool is_v = threadIdx.x >= 16;
  const int node = nodes[blockIdx.y];
  if (node < 0 || node >= n_nodes) {
    if (threadIdx.x == 0) record_error(status, kBadIndex);
    return;
  }
  size_t to;
  if (!page_row(slots[blockIdx.y], num_slots, nkv, h, bs, status, to)) return;
  to += (size_t)layer * num_slots * nkv;
  const size_t from = ((size_t)layer * n_nodes + node) * nkv + h;
  if (lane < hd / 8)
    reinterpret_cast<uint32_t*>((is_v ? vc : kc) + to * (hd / 2))[lane] =
        reinterpret_cast<const uint32_t*>((is_v ? tvc : tkc) + from * (hd / 2))[lane];
  if (lane < hd / kGroup) (is_v ? vw : kw)[to * (hd / kGroup) + lane] = (is_v ? tvw : tkw)[from * (hd / kGroup) + lane];
}

inline bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// [T, nkv, hd] rows whose last dim is dense and whose rows start on 16 bytes, else a dense copy
at::Tensor rows_for_store(const at::Tensor& x) {
  if (x.stride(2) == 1 && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0 && x.stride(0) >= 0 && x.stride(1) >= 0 &&
      aligned16(x))
    return x;
  return x.clone(at::MemoryFormat::Contiguous);
}

void launch_check(const char* what) {
  const cudaError_t e = cudaGetLastError();
  LSB_INT4_CHECK(e == cudaSuccess, std::string(what) + " launch failed: " + cudaGetErrorString(e));
}

}  // namespace

void store_kvcache_int4(at::Tensor k, at::Tensor v, at::Tensor kc, at::Tensor kw, at::Tensor vc, at::Tensor vw,
                        at::Tensor slots, at::Tensor status) {
  check_page_pair(kc, kw, vc, vw, k.device());
  LSB_INT4_CHECK(k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16 && k.dim() == 3 &&
                     v.sizes() == k.sizes() && v.device() == k.device(),
                 "k and v must be bfloat16 [tokens, kv_heads, head_dim]");
  LSB_INT4_CHECK(k.size(1) == kc.size(1) && k.size(2) == kc.size(3) * 2, "k / v heads do not match the pages");
  check_int32(slots, "slot_mapping", 1, k.device());
  LSB_INT4_CHECK(slots.size(0) == k.size(0), "slot_mapping must hold one slot per token");
  const int64_t rows = k.size(0) * k.size(1), per = kThreads / (k.size(2) / 8);
  if (rows == 0) return;
  LSB_INT4_CHECK(rows < INT32_MAX, "too many rows for one launch");
  const at::cuda::CUDAGuard g(k.device());
  k = rows_for_store(k);
  v = rows_for_store(v);
  const dim3 grid((unsigned)((rows + per - 1) / per));
  auto go = [&](auto kern) {
    launch_pdl(kern, grid, dim3(kThreads), 0, at::cuda::getCurrentCUDAStream(), (const bf16*)k.data_ptr(),
               (const bf16*)v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), kc.data_ptr<uint8_t>(),
               kw.data_ptr<int16_t>(), vc.data_ptr<uint8_t>(), vw.data_ptr<int16_t>(), slots.data_ptr<int>(),
               (uint32_t)rows, (uint32_t)kc.size(1), (uint32_t)kc.size(2), kc.size(0) * kc.size(2), status_ptr(status));
  };
  if (k.size(2) == 128) go(store_int4_kernel<128>);
  else go(store_int4_kernel<64>);
  launch_check("store_kvcache_int4");
}

std::tuple<at::Tensor, at::Tensor> load_kvcache_int4(at::Tensor kc, at::Tensor kw, at::Tensor vc, at::Tensor vw,
                                                     at::Tensor slots, at::Tensor status) {
  const at::Device dev = kc.device();
  check_page_pair(kc, kw, vc, vw, dev);
  check_int32(slots, "slot_mapping", 1, dev);
  const at::cuda::CUDAGuard g(dev);
  at::Tensor k = at::empty({slots.size(0), kc.size(1), kc.size(3) * 2}, kc.options().dtype(at::kBFloat16)),
             v = at::empty_like(k);
  const int64_t rows = k.size(0) * k.size(1), per = kThreads / (k.size(2) / 8);
  if (rows == 0) return {k, v};
  LSB_INT4_CHECK(rows < INT32_MAX, "too many rows for one launch");
  const dim3 grid((unsigned)((rows + per - 1) / per));
  auto go = [&](auto kern) {
    launch_pdl(kern, grid, dim3(kThreads), 0, at::cuda::getCurrentCUDAStream(), (bf16*)k.data_ptr(),
               (bf16*)v.data_ptr(), kc.data_ptr<uint8_t>(), kw.data_ptr<int16_t>(), vc.data_ptr<uint8_t>(),
               vw.data_ptr<int16_t>(), slots.data_ptr<int>(), (uint32_t)rows, (uint32_t)kc.size(1), (uint32_t)kc.size(2),
               kc.size(0) * kc.size(2), status_ptr(status));
  };
  if (k.size(2) == 128) go(load_int4_kernel<128>);
  else go(load_int4_kernel<64>);
  launch_check("load_kvcache_int4");
  return {k, v};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> load_pages_int4(at::Tensor kc, at::Tensor kw, at::Tensor vc, at::Tensor vw,
                                                               at::Tensor ids) {
  const at::Device dev = kc.device();
  check_page_pair(kc, kw, vc, vw, dev);
  check_int32(ids, "block_table", 1, dev);
  const int64_t hd = kc.size(3) * 2, page_rows = kc.size(1) * kc.size(2), rows = ids.size(0) * page_rows;
  LSB_INT4_CHECK(rows < INT32_MAX, "too many rows for one launch");
  const at::cuda::CUDAGuard g(dev);
  at::Tensor k = at::empty({ids.size(0), kc.size(1), kc.size(2), hd}, kc.options().dtype(at::kBFloat16)),
             v = at::empty_like(k), table = at::empty_like(ids);
  if (rows == 0) return {k, v, table};
  const int64_t per = kThreads / (hd / 8);
  const dim3 grid((unsigned)((rows + per - 1) / per));
  auto go = [&](auto kern) {
    launch_pdl(kern, grid, dim3(kThreads), 0, at::cuda::getCurrentCUDAStream(), (bf16*)k.data_ptr(),
               (bf16*)v.data_ptr(), table.data_ptr<int>(), kc.data_ptr<uint8_t>(), kw.data_ptr<int16_t>(),
               vc.data_ptr<uint8_t>(), vw.data_ptr<int16_t>(), ids.data_ptr<int>(), (uint32_t)rows, (uint32_t)page_rows,
               (uint32_t)kc.size(0));
  };
  if (hd == 128) go(load_pages_int4_kernel<128>);
  else go(load_pages_int4_kernel<64>);
  launch_check("load_pages_int4");
  return {k, v, table};
}

void qkv_rope_int4(at::Tensor q_out, at::Tensor qkv, at::Tensor positions, at::Tensor cos_sin, at::Tensor q_w,
                   at::Tensor k_w, double eps, at::Tensor kc, at::Tensor kw, at::Tensor vc, at::Tensor vw,
                   at::Tensor slots, int64_t nh, at::Tensor status) {
  const at::Device dev = qkv.device();
  check_page_pair(kc, kw, vc, vw, dev);
  const bool planes = qkv.scalar_type() == at::kFloat;
  const int64_t nkv = kc.size(1), hd = kc.size(3) * 2;
  LSB_INT4_CHECK((planes ? qkv.dim() == 3 : qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16) &&
                     qkv.is_contiguous() && aligned16(qkv),
                 "qkv must be contiguous bfloat16 [T, width] or float32 planes [S, T, width]");
  LSB_INT4_CHECK(nh >= 1 && qkv.size(-1) == (nh + 2 * nkv) * hd, "qkv width does not match the heads");
  const int64_t T = qkv.size(-2), S = planes ? qkv.size(0) : 0;
  LSB_INT4_CHECK(!planes || S >= 1, "no split-K planes");
  LSB_INT4_CHECK(q_out.scalar_type() == at::kBFloat16 && q_out.is_contiguous() && q_out.numel() == T * nh * hd &&
                     q_out.device() == dev,
                 "q_out must be contiguous bfloat16 [T, heads, head_dim]");
  LSB_INT4_CHECK(positions.scalar_type() == at::kLong && positions.is_contiguous() && positions.numel() == T &&
                     positions.device() == dev,
                 "positions must be contiguous int64 [T]");
  LSB_INT4_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.is_contiguous() && cos_sin.dim() == 2 &&
                     cos_sin.size(1) == hd && cos_sin.size(0) >= 1 && aligned16(cos_sin) && cos_sin.device() == dev,
                 "cos_sin must be contiguous float32 [positions, head_dim]");
  check_int32(slots, "slot_mapping", 1, dev);
  LSB_INT4_CHECK(slots.size(0) == T, "slot_mapping must hold one slot per token");
  LSB_INT4_CHECK((q_w.numel() == 0) == (k_w.numel() == 0), "q and k norm weights go together");
  for (const at::Tensor* w : {&q_w, &k_w})
    LSB_INT4_CHECK(w->numel() == 0 || (w->scalar_type() == at::kBFloat16 && w->is_contiguous() && w->numel() == hd &&
                                       aligned16(*w) && w->device() == dev),
                   "norm weights must be contiguous bfloat16 [head_dim]");
  if (T == 0) return;
  const int64_t rows = T * (nh + 2 * nkv), groups = kThreads / (hd / 8), chunks = (nh + 2 * nkv + groups - 1) / groups;
  // heads per lane group: as many as leave sixteen blocks a SM
  const int64_t steps = std::max<int64_t>(1, std::min<int64_t>(chunks, T * chunks / (148 * 16)));
  LSB_INT4_CHECK(rows < INT32_MAX, "too many rows for one launch");
  const at::cuda::CUDAGuard g(dev);
  auto go = [&](auto kern) {
    launch_pdl(kern, dim3((unsigned)T, (unsigned)((chunks + steps - 1) / steps)), dim3(kThreads), 0, at::cuda::getCurrentCUDAStream(),
               (bf16*)q_out.data_ptr(), (const void*)qkv.data_ptr(), (int)S, positions.data_ptr<int64_t>(),
               cos_sin.data_ptr<float>(), cos_sin.size(0), q_w.numel() ? (const bf16*)q_w.data_ptr() : nullptr,
               k_w.numel() ? (const bf16*)k_w.data_ptr() : nullptr, (float)eps, kc.data_ptr<uint8_t>(),
               kw.data_ptr<int16_t>(), vc.data_ptr<uint8_t>(), vw.data_ptr<int16_t>(), slots.data_ptr<int>(), (int)T,
               (int)nh, (int)nkv, (int)steps, (uint32_t)kc.size(2), kc.size(0) * kc.size(2), status_ptr(status));
  };
  if (hd == 128) planes ? go(rope_store_int4_kernel<128, true>) : go(rope_store_int4_kernel<128, false>);
  else planes ? go(rope_store_int4_kernel<64, true>) : go(rope_store_int4_kernel<64, false>);
  launch_check("qkv_rope_int4");
}

// tree rows [layers, nodes, kv_heads, ..] into pools [layers, blocks, kv_heads, block_size, ..]
void commit_tree_kv_int4(at::Tensor tkc, at::Tensor tkw, at::Tensor tvc, at::Tensor tvw, at::Tensor kc, at::Tensor kw,
                         at::Tensor vc, at::Tensor vw, at::Tensor nodes, at::Tensor slots, at::Tensor status) {
  const at::Device dev = kc.device();
  LSB_INT4_CHECK(kc.dim() == 5 && kw.dim() == 5 && vc.dim() == 5 && vw.dim() == 5 && kc.is_contiguous() && kw.is_contiguous() &&
                     vc.is_contiguous() && vw.is_contiguous(),
                 "pools must be contiguous [layers, blocks, kv_heads, block_size, ..]");
  const int64_t L = kc.size(0), nkv = kc.size(2), hd = kc.size(4) * 2, m = nodes.numel();
  if (L == 0) return;
  check_page_pair(kc[0], kw[0], vc[0], vw[0], dev);
  LSB_INT4_CHECK(kw.size(0) == L && vc.size(0) == L && vw.size(0) == L, "pools differ in layers");
  LSB_INT4_CHECK(tkc.dim() == 4 && tkc.size(0) == L && tkc.size(2) == nkv && tkc.size(3) * 2 == hd && tvc.sizes() == tkc.sizes() &&
                     tkw.sizes() == at::IntArrayRef({L, tkc.size(1), nkv, hd / kGroup}) && tvw.sizes() == tkw.sizes(),
                 "tree rows must be [layers, nodes, kv_heads, ..] of the pools' heads");
  for (const at::Tensor* t : {&tkc, &tvc})
    LSB_INT4_CHECK(t->scalar_type() == at::kByte && t->is_contiguous() && t->device() == dev && aligned16(*t),
                   "tree codes must be contiguous, 16-byte aligned uint8 on the pools' device");
  for (const at::Tensor* t : {&tkw, &tvw})
    LSB_INT4_CHECK(t->scalar_type() == at::kShort && t->is_contiguous() && t->device() == dev,
                   "tree scale words must be contiguous int16 on the pools' device");
  check_int32(nodes, "node_indices", 1, dev);
  check_int32(slots, "slot_mapping", 1, dev);
  LSB_INT4_CHECK(slots.numel() == m, "slot_mapping must hold one slot per node");
  LSB_INT4_CHECK(m <= 65535 && nkv <= 65535 && L <= INT32_MAX && tkc.size(1) <= INT32_MAX, "too many nodes or heads for one launch");
  if (m == 0 || nkv == 0) return;
  const at::cuda::CUDAGuard g(dev);
  launch_pdl(commit_tree_int4_kernel, dim3((unsigned)L, (unsigned)m, (unsigned)nkv), dim3(32), 0,
             at::cuda::getCurrentCUDAStream(), tkc.data_ptr<uint8_t>(), tkw.data_ptr<int16_t>(), tvc.data_ptr<uint8_t>(),
             tvw.data_ptr<int16_t>(), kc.data_ptr<uint8_t>(), kw.data_ptr<int16_t>(), vc.data_ptr<uint8_t>(),
             vw.data_ptr<int16_t>(), nodes.data_ptr<int>(), slots.data_ptr<int>(), (int)tkc.size(1), (int)nkv, (int)hd,
             (uint32_t)kc.size(3), kc.size(1) * kc.size(3), status_ptr(status));
  launch_check("commit_tree_kv_int4");
}

}  // namespace lsb
