// The 4-bit KV page format and its host-side checks, shared by the kernels that fill and read it.
//
// A pool is two tensors: codes uint8 [blocks, kv_heads, block_size, head_dim / 2] (dim 2i in the low
// nibble of byte i) and scale words int16 [blocks, kv_heads, block_size, head_dim / 64], one per
// token, KV head and group of 64 dims.  A word is the bf16 pattern of the group's scale s with the
// four low mantissa bits replaced by the zero code z; a code c stands for s * (c - z).  s keeps four
// significant bits, so s * (c - z) (four bits times at most four bits and a sign) is exact in bf16:
// a kernel may feed the dequantised value to the tensor cores as bf16, or feed the integer and scale
// the product, and both are the same number.
#pragma once
#include <ATen/ATen.h>

#include <cmath>

#include "common.cuh"

namespace lsb {
namespace int4 {

constexpr int kGroup = 64;

// a pair of bf16 at a time
__device__ __forceinline__ uint32_t sub2(uint32_t x, uint32_t z) {
  uint32_t y;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(z));
  return y;
}
__device__ __forceinline__ uint32_t mul2(uint32_t x, uint32_t z) {
  uint32_t y;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(z));
  return y;
}
// global to shared memory, counted by an mbarrier; both addresses and the size are multiples of 16 bytes
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

struct Pages {
  const uint8_t* codes;
  const int16_t* words;
};

#define LSB_INT4_CHECK(cond, msg) TORCH_CHECK(cond, "llmserve_b200: ", msg)

inline void check_pages(const at::Tensor& codes, const at::Tensor& words, const char* name, const at::Device& dev) {
  LSB_INT4_CHECK(codes.is_cuda() && codes.device() == dev && words.device() == dev,
                 std::string(name) + " pages must be on the device of the other arguments");
  LSB_INT4_CHECK(codes.scalar_type() == at::kByte && words.scalar_type() == at::kShort,
                 std::string(name) + " pages must be uint8 codes and int16 scale words");
  LSB_INT4_CHECK(codes.dim() == 4 && words.dim() == 4 && codes.is_contiguous() && words.is_contiguous(),
                 std::string(name) + " pages must be contiguous [blocks, kv_heads, block_size, ..]");
  const int64_t hd = codes.size(3) * 2;
  LSB_INT4_CHECK(hd == 64 || hd == 128, "4-bit pages need head_dim 64 or 128");
  LSB_INT4_CHECK(words.size(0) == codes.size(0) && words.size(1) == codes.size(1) && words.size(2) == codes.size(2) &&
                     words.size(3) == hd / kGroup,
                 std::string(name) + " pages: scale words must be [blocks, kv_heads, block_size, head_dim / 64]");
  LSB_INT4_CHECK(codes.size(2) >= 16 && codes.size(2) % 16 == 0, "block_size must be a multiple of 16");
  LSB_INT4_CHECK(codes.size(0) * codes.size(2) <= INT32_MAX, "more slots than an int32 slot can name");
  LSB_INT4_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(words.data_ptr()) % 16 == 0,
                 std::string(name) + " pages must be 16-byte aligned");
}

inline void check_page_pair(const at::Tensor& kc, const at::Tensor& kw, const at::Tensor& vc, const at::Tensor& vw,
                            const at::Device& dev) {
  check_pages(kc, kw, "K", dev);
  check_pages(vc, vw, "V", dev);
  LSB_INT4_CHECK(kc.sizes() == vc.sizes(), "K and V pages differ in shape");
}

inline void check_int32(const at::Tensor& t, const char* name, int64_t dim, const at::Device& dev) {
  LSB_INT4_CHECK(t.scalar_type() == at::kInt && t.dim() == dim && t.is_contiguous() && t.device() == dev,
                 std::string(name) + " must be contiguous int32 with " + std::to_string(dim) +
                     " dimension(s) on the device of the other arguments");
}

// What scores are multiplied by, for exponentials of base two: `times` times the scale in float32, which must not
// round to zero (a hidden score, minus infinity, would become NaN) or to infinity.
inline float scale_log2(double scale, double times) {
  const float s = (float)(scale * times * 1.4426950408889634);
  LSB_INT4_CHECK(s >= 1.17549435e-38f && std::isfinite(s), "scale must be positive and within the range of float32");
  return s;
}

}  // namespace int4
}  // namespace lsb
