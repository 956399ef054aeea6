// Decode and verify attention against 4-bit KV pages (format: int4_pages.cuh).
//
// The query rows of one KV head (nq new tokens x heads per KV head) are the narrow side of the tensor
// core products and the keys and head dims the wide one, with mma.sync and fp32 sums:
//   S^T [16 keys x 8 rows] = C_K [16 x HD] Q^T        O^T [16 dims x 8 rows] += (C_V - z)^T [16 x 16 keys] W^T
// so a tile of 16 keys costs 8 rows of padding at most (16 from nine rows on).  A tcgen05 tile would
// need 128 of them.
//
// What bounds it next to memory is the integer pipe (64 lanes a clock) that turns nibbles into operands.
//   K: a byte 0..15 read as e4m3 is c 2^-9 exactly (subnormals and the first binade are one even grid),
//      so masking alone makes the operand: 3 instructions for 8 codes where a 16-bit form takes 7.  The
//      query, eight significant bits, becomes two e4m3 terms after scaling the row by a power of two;
//      values below 2^-10 of the row's largest lose what lies under 2^-17 of it.
//      s = sum_g sk_g (sum_d q_d c_d - zk_g sum_d q_d)     g: groups of 64 dims
//   V: 128 + c is a bf16 with c in its low mantissa bits (a mask-or for two nibbles); less 128 + zv of its
//      key and group it is the exact c - zv.  The other operand is w_jg = p_j sv_jg in bf16, the one
//      rounding besides the output's.  e4m3 has too few bits for w.
//
// A warp's operand layout asks K for 8 dims of a key (a code word as it lies) and V for pairs of keys (one
// PRMT joins the half words of two rows): neither needs a shuffle, and the order of dims or keys inside a
// product is free as long as both operands share it.
//
// One producer warp copies 128-key chunks (codes and words of K and V, a contiguous run per page) into
// a ring with bulk copies; four consumer warps take 32 keys of every chunk and never meet until a
// segment ends.  Work is the list of (sequence, KV head, chunk), cut into equal contiguous shares over a
// grid that fills the GPU once, whatever the lengths: lengths are read on the device, so one captured
// launch serves any batch.  A (sequence, head) that is cut leaves fp32 partials; the block that
// finishes last merges them in their order (results do not depend on who is last) and resets the
// counter.  Bound by memory for long contexts, by instruction issue (about 280 for 16 keys a warp) just
// behind it.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cuda_fp16.h>

#include <cmath>
#include <type_traits>

#include "int4_pages.cuh"
#include "umma.cuh"

namespace lsb {

int* status_ptr(const at::Tensor& status);

namespace {

using namespace int4;
using umma::wait_phase;

constexpr int kChunk = 128;               // keys of a ring stage, the unit of work
constexpr int kWarps = 4;                 // consumer warps
constexpr int kWarpKeys = kChunk / kWarps;
constexpr int kThreads = (kWarps + 1) * 32;
constexpr float kRescaleLog2 = 8.f;

template <int HD, int NT>
struct DecLayout {
  static constexpr int kGroups = HD / kGroup;
  static constexpr int kStages = 3;
  static constexpr int kBlocks = NT == 2 ? 2 : 3;          // resident blocks per SM that registers are held to
  static constexpr int kCodes = kChunk * HD / 2;           // bytes of one tensor's codes in a stage
  static constexpr int kWords = kChunk * kGroups * 2;
  static constexpr int kStage = 2 * kCodes + 2 * kWords;
  static constexpr int kRow = HD + 4;                      // floats of a merge row (padded)
  static constexpr int kMergeOff = kStages * kStage;
  static constexpr int kMlOff = kMergeOff + kWarps * 8 * NT * kRow * 4;
  static constexpr int kBarOff = kMlOff + kWarps * 8 * NT * 8;
  static constexpr int kBytes = kBarOff + 128;
};

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// (x & mask) | bits, one instruction
__device__ __forceinline__ uint32_t mask_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t x, uint32_t z) {
  uint32_t y;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(z));
  return y;
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t x, uint32_t z) {
  uint32_t y;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(z));
  return y;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t x, uint32_t m, uint32_t z) {
  uint32_t y;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(x), "r"(m), "r"(z));
  return y;
}
// nibbles s and s + 4 of a word as the bf16 pair (128 + low, 128 + high)
__device__ __forceinline__ uint32_t nibbles(uint32_t w, int s) { return mask_or(w >> (4 * s), 0x000f000fu, 0x43004300u); }
// the eight nibbles of a word less z as fp16 pairs (s, s + 4): nz = -(1024 + z) twice, nz64 = -(64 + z) twice
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t nz, uint32_t nz64, uint32_t* y) {
  const uint32_t h = w >> 8;
  y[0] = add_f16x2(mask_or(w, 0x000f000fu, 0x64006400u), nz);
  y[1] = fma_f16x2(mask_or(w, 0x00f000f0u, 0x64006400u), 0x2c002c00u, nz64);      // (1024 + 16 c) / 16
  y[2] = add_f16x2(mask_or(h, 0x000f000fu, 0x64006400u), nz);
  y[3] = fma_f16x2(mask_or(h, 0x00f000f0u, 0x64006400u), 0x2c002c00u, nz64);
}
__device__ __forceinline__ uint32_t pack2_f16(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

struct Args {
  bf16* out;
  const bf16* q;
  Pages kp, vp;
  const int* lens;
  const int* tables;
  float* part_o;
  float* part_ml;
  int* counters;
  int* status;
  float scale_log2;
  int width, B, nq, nh, nkv, bs, nblk, max_splits, row_tiles;
};

__device__ __forceinline__ int key_count(const Args& a, int b) {
  return max(0, min(a.lens[b], (int)min((int64_t)a.width * a.bs, (int64_t)INT32_MAX - kChunk)));
}
__device__ __forceinline__ int chunk_count(const Args& a, int b) { return (key_count(a, b) + kChunk - 1) / kChunk; }

// This block's share [c0, c1) of all chunks and where it starts; the same in every lane of a warp.
struct Share {
  int c0, c1, total;
  int b;             // sequence of chunk c0
  int before;        // chunks of all heads before sequence b
};
__device__ __forceinline__ int share_begin(int total, int grid, int i) { return (int)((int64_t)total * i / grid); }

__device__ __forceinline__ Share find_share(const Args& a, int lane, int& grid) {
  int sum = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) sum += b0 + lane < a.B ? chunk_count(a, b0 + lane) : 0;
  Share s;
  s.total = __reduce_add_sync(0xffffffffu, sum) * a.nkv;
  grid = min((int)gridDim.x, s.total);
  s.c0 = s.c1 = s.b = s.before = 0;
  if ((int)blockIdx.x >= grid) return s;
  s.c0 = share_begin(s.total, grid, blockIdx.x);
  s.c1 = share_begin(s.total, grid, blockIdx.x + 1);
  const int want = s.c0 / a.nkv;          // the sequence whose per-head chunks hold this one
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int n = b0 + lane < a.B ? chunk_count(a, b0 + lane) : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, base + incl > want);
    if (hit) {
      const int l = __ffs(hit) - 1;
      s.b = b0 + l;
      s.before = (base + __shfl_sync(0xffffffffu, incl - n, l)) * a.nkv;
      return s;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  return s;
}

// One stretch of chunks of a (sequence, head) inside the share.
struct Segment {
  int b, h, keys, chunks;      // the sequence's keys and chunks
  int first, n;                // chunks [first, first + n) of them
  int pair0;                   // index of the pair's first chunk in the whole list
};
__device__ __forceinline__ bool next_segment(const Args& a, Share& s, Segment& g) {
  if (s.c0 >= s.c1) return false;
  g.b = s.b;
  g.keys = key_count(a, g.b);
  g.chunks = (g.keys + kChunk - 1) / kChunk;
  g.h = (s.c0 - s.before) / g.chunks;
  g.pair0 = s.before + g.h * g.chunks;
  g.first = s.c0 - g.pair0;
  g.n = min(g.chunks - g.first, s.c1 - s.c0);
  s.c0 += g.n;
  if (g.h == a.nkv - 1 && g.first + g.n == g.chunks) {      // on to the next sequence that has keys
    s.before = s.c0;
    ++s.b;
    while (s.c0 < s.c1 && chunk_count(a, s.b) == 0) ++s.b;
  }
  return true;
}

template <int HD, int NT>
__global__ void __launch_bounds__(kThreads, DecLayout<HD, NT>::kBlocks) decode_int4_kernel(const Args a) {
  using L = DecLayout<HD, NT>;
  constexpr int kG = L::kGroups, kQ = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* empty = full + L::kStages;
  volatile uint32_t* bad_tiles = reinterpret_cast<uint32_t*>(empty + L::kStages);    // a bit per 16 keys of the stage
  __shared__ int abort_flag;
  __shared__ int merge_me;
  volatile int* abort_v = &abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    fence_barrier_init();
  }
  pdl_trigger();
  pdl_wait();
  __syncthreads();
  int grid;
  Share share = find_share(a, lane, grid);
  Segment g;

  if (warp == kWarps) {
    // ---------------- producer ----------------
    int it = 0;
    int issued[L::kStages] = {};
    bool ok = true;
    while (ok && next_segment(a, share, g)) {
      const int* table = a.tables + (int64_t)g.b * a.width;
      for (int c = g.first; ok && c < g.first + g.n; ++c, ++it) {
        const int s = it % L::kStages, u = it / L::kStages;
        if (u >= 1) ok = __all_sync(0xffffffffu, wait_phase(&empty[s], (u - 1) & 1, abort_v, a.status, kTimeoutSmemEmpty));
        if (!ok) break;
        // lane i takes the i-th page that the chunk touches; runs are whole 16-key tiles of a page
        const int k0 = c * kChunk, kend = min(k0 + kChunk, (g.keys + 15) & ~15);
        const int page = k0 / a.bs + lane;
        const int from = max(k0, page * a.bs), to = min(kend, (page + 1) * a.bs);
        const bool mine = lane < kChunk / 16 + 1 && from < to;
        int blk = 0;
        bool bad = false;
        if (mine) {
          blk = table[page];
          bad = blk < 0 || blk >= a.nblk;
          if (bad) record_error(a.status, kBadIndex);
        }
        uint32_t flags = 0;
        if (bad) flags = ((1u << ((to - k0) / 16)) - 1u) & ~((1u << ((from - k0) / 16)) - 1u);
        flags = __reduce_or_sync(0xffffffffu, flags);
        const int keys = mine && !bad ? to - from : 0;
        const int total = __reduce_add_sync(0xffffffffu, keys);
        if (lane == 0) {
          bad_tiles[s] = flags;                    // published by the arrival below
          mbar_expect_tx(&full[s], (uint32_t)total * (HD + 4 * kG));
        }
        __syncwarp();
        if (keys > 0) {
          const size_t row = ((size_t)blk * a.nkv + g.h) * a.bs + (from - page * a.bs);
          const uint32_t st = smem_u32(smem) + s * L::kStage;
          const int at = from - k0;
          bulk_copy(st + at * (HD / 2), a.kp.codes + row * (HD / 2), keys * (HD / 2), &full[s]);
          bulk_copy(st + 2 * L::kCodes + at * 2 * kG, a.kp.words + row * kG, keys * 2 * kG, &full[s]);
          bulk_copy(st + L::kCodes + at * (HD / 2), a.vp.codes + row * (HD / 2), keys * (HD / 2), &full[s]);
          bulk_copy(st + 2 * L::kCodes + L::kWords + at * 2 * kG, a.vp.words + row * kG, keys * 2 * kG, &full[s]);
        }
        issued[s] = u + 1;
      }
    }
    // every copy has landed before the block may end
    for (int s = 0; s < L::kStages; ++s)
      if (issued[s] > 0) mbar_wait(&full[s], (issued[s] - 1) & 1);
    return;
  }

  // ---------------- consumers ----------------
  const int gid = lane >> 2, t4 = lane & 3;
  const int group_heads = a.nh / a.nkv;
  const int row0 = blockIdx.y * kQ, rows = min(kQ, a.nq * group_heads - row0);
  float* merge = reinterpret_cast<float*>(smem + L::kMergeOff);
  float2* ml = reinterpret_cast<float2*>(smem + L::kMlOff);

  // sequences without keys: zeros
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (key_count(a, b) == 0)
      for (int i = threadIdx.x; i < a.nkv * rows * (HD / 8); i += kWarps * 32) {
        const int r = i / (HD / 8) % rows + row0, h = i / (HD / 8) / rows;
        const size_t at = ((size_t)b * a.nq + r / group_heads) * a.nh + h * group_heads + r % group_heads;
        *reinterpret_cast<uint4*>(a.out + at * HD + (i % (HD / 8)) * 8) = make_uint4(0, 0, 0, 0);
      }

  int it = 0;
  bool ok = true;
  while (next_segment(a, share, g)) {
    // address of query row r (< rows) of this pair, in rows of HD
    auto row_of = [&](int r) {
      r += row0;
      return ((size_t)g.b * a.nq + r / group_heads) * a.nh + g.h * group_heads + r % group_heads;
    };
    // Q^T operand: row gid of each 8-row tile as fp16 after scaling it by a power of two to a largest value
    // in [2^14, 2^15); for group g and word i the dims 64 g + 16 t4 + 8 i + (s, s + 4)
    uint32_t qf[NT][kG][2][4];
    float back[NT][2];                             // rows 2 t4, 2 t4 + 1: what a score is multiplied by
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool live = n * 8 + gid < rows;
      const uint4* src = reinterpret_cast<const uint4*>(a.q + row_of(live ? n * 8 + gid : 0) * HD);
      uint4 v[kG][2];
      uint32_t most = 0;                           // bit pattern of the largest magnitude
#pragma unroll
      for (int gr = 0; gr < kG; ++gr)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          v[gr][i] = live ? src[(gr * 64 + t4 * 16 + i * 8) / 8] : make_uint4(0, 0, 0, 0);
          const uint32_t w[4] = {v[gr][i].x, v[gr][i].y, v[gr][i].z, v[gr][i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) most = max(most, max(w[e] & 0x7fffu, w[e] >> 16 & 0x7fffu));
        }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // 2^k in two factors, k = 14 - exponent (subnormals count as 2^-126)
      const int k = 14 + 127 - max(1, (int)(most >> 7)), k0 = k >> 1, k1 = k - k0;
      const float up0 = __uint_as_float((uint32_t)(127 + k0) << 23), up1 = __uint_as_float((uint32_t)(127 + k1) << 23);
#pragma unroll
      for (int gr = 0; gr < kG; ++gr)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t w[4] = {v[gr][i].x, v[gr][i].y, v[gr][i].z, v[gr][i].w};
          float x[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[2 * e] = __uint_as_float(w[e] << 16) * up0 * up1;
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u) * up0 * up1;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[n][gr][i][e] = pack2_f16(x[e], x[e + 4]);
        }
      // an infinity or NaN in the row: NaN scores
      const float down = most >= 0x7f80u ? __uint_as_float(0x7fc00000u)
                                         : __uint_as_float((uint32_t)(127 - k0) << 23) * a.scale_log2 *
                                               __uint_as_float((uint32_t)(127 - k1) << 23);
      back[n][0] = __shfl_sync(0xffffffffu, down, t4 * 8);
      back[n][1] = __shfl_sync(0xffffffffu, down, t4 * 8 + 4);
    }
    // keys that row r of the block sees
    auto limit = [&](int r) { return r < rows ? min(g.keys, a.lens[g.b] - a.nq + (row0 + r) / group_heads + 1) : 0; };
    // keys below this are seen by every row of the tile
    const int all_see = min(g.keys, a.lens[g.b] - a.nq + row0 / group_heads + 1);

    float o[NT][kG][4][4];
    // m: the reference that exponents are taken from, top: the score that moves it (-inf: none seen yet)
    float m[NT][2], top[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int gr = 0; gr < kG; ++gr)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][gr][j][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = 0.f;
        top[n][e] = -INFINITY;
        l[n][e] = 0.f;
      }
    }

    for (int c = g.first; c < g.first + g.n; ++c, ++it) {
      const int s = it % L::kStages;
      ok = ok && __all_sync(0xffffffffu, wait_phase(&full[s], (it / L::kStages) & 1, abort_v, a.status, kTimeoutTmaFull));
      if (!ok) break;
      const uint8_t* st = smem + s * L::kStage;
      const uint32_t bad = bad_tiles[s];
      // 16 keys; edge: some row of this block does not see some of them
      auto tile = [&](auto edge, int at) {
        const int k0 = c * kChunk + at;
        // Row m of the tile is key (m & 8) + ((m & 7) >> 1) + 4 (m & 1): the four rows that the four lanes
        // of a group read together for V then lie in two bank halves instead of one.
        const int key_a = (gid >> 1) + 4 * (gid & 1), key_b = key_a + 8;
        const uint8_t* ka = st + (at + key_a) * (HD / 2) + t4 * 8;
        const uint8_t* kw = st + 2 * L::kCodes;
        const uint8_t* vw = kw + L::kWords;
        // scale words of a key: group 0 in the low half word, group 1 in the high one
        auto words = [&](const uint8_t* w, int key) -> uint32_t {
          if constexpr (kG == 2) return reinterpret_cast<const uint32_t*>(w)[key];
          else return reinterpret_cast<const uint16_t*>(w)[key];
        };
        auto scale = [](uint32_t w, int gr) { return __uint_as_float((gr == 0 ? w << 16 : w) & 0x7ff00000u); };
        const uint32_t kwa = words(kw, at + key_a), kwb = words(kw, at + key_b);
        const uint32_t vwa = words(vw, at + key_a), vwb = words(vw, at + key_b);
        float p[NT][4];                            // [key a row 0, key a row 1, key b row 0, key b row 1]
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          const uint2 wa = *reinterpret_cast<const uint2*>(ka + gr * 32);
          const uint2 wb = *reinterpret_cast<const uint2*>(ka + gr * 32 + 8 * (HD / 2));
          // -(1024 + z) of each key, twice, and -(64 + z)
          const uint32_t za = mask_or(__byte_perm(kwa, 0, gr ? 0x3232 : 0x1010), 0x000f000fu, 0xe400e400u);
          const uint32_t zb = mask_or(__byte_perm(kwb, 0, gr ? 0x3232 : 0x1010), 0x000f000fu, 0xe400e400u);
          const uint32_t za64 = add_f16x2(za, 0x63806380u), zb64 = add_f16x2(zb, 0x63806380u);
          float sacc[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sacc[n][e] = 0.f;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t ya[4], yb[4];
            codes_f16(i ? wa.y : wa.x, za, za64, ya);
            codes_f16(i ? wb.y : wb.x, zb, zb64, yb);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; e += 2)
                mma_f16(sacc[n], ya[e], yb[e], ya[e + 1], yb[e + 1], qf[n][gr][i][e], qf[n][gr][i][e + 1]);
          }
          const float ska = scale(kwa, gr), skb = scale(kwb, gr);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) p[n][e] = fmaf(e < 2 ? ska : skb, sacc[n][e], gr == 0 ? 0.f : p[n][e]);
        }
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = p[n][e] * back[n][e & 1];
            if (edge.value && k0 + (e < 2 ? key_a : key_b) >= limit(n * 8 + t4 * 2 + (e & 1))) x = -INFINITY;
            p[n][e] = x;
            grow |= x > top[n][e & 1];
          }
        // the reference maximum moves only when a score passes it by 2^8 (first tile: from -inf)
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = fmaxf(p[n][e], p[n][e + 2]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
              // f = 2^(old - new); a row that has seen no key keeps reference 0 and the next score moves it
              const bool none = top[n][e] == -INFINITY;
              const float mn = none ? mx : fmaxf(m[n][e], mx), f = none ? 0.f : umma::ex2(m[n][e] - mn);
              m[n][e] = mn == -INFINITY ? 0.f : mn;
              top[n][e] = mn + kRescaleLog2;
              l[n][e] *= f;
#pragma unroll
              for (int gr = 0; gr < kG; ++gr) {
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][gr][j][e] *= f, o[n][gr][j][e + 2] *= f;
              }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[n][e] = umma::ex2(p[n][e] - m[n][e & 1]);
            l[n][e & 1] += p[n][e];
          }
        // O^T: words of keys (rows 2 t4, 2 t4 + 1, + 8) for dims 64 g + 8 gid ..; row 2 t4 is key t4, row
        // 2 t4 + 1 key t4 + 4
        const uint8_t* v0 = st + L::kCodes + (at + t4) * (HD / 2) + gid * 4;
        const uint32_t z0 = words(vw, at + t4), z1 = words(vw, at + t4 + 4), z8 = words(vw, at + t4 + 8),
                       z9 = words(vw, at + t4 + 12);
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          uint32_t w0[NT], w1[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = p[n][e] * scale(e < 2 ? vwa : vwb, gr);
              // a key that this row does not see may hold anything, NaN scales among it
              if (edge.value && k0 + (e < 2 ? key_a : key_b) >= limit(n * 8 + t4 * 2 + (e & 1))) w[e] = 0.f;
            }
            const uint32_t lo = umma::pack2_bf16(w[0], w[1]), hi = umma::pack2_bf16(w[2], w[3]);
            w0[n] = transpose8x8(lo);
            w1[n] = transpose8x8(hi);
          }
          const uint32_t x0 = *reinterpret_cast<const uint32_t*>(v0 + gr * 32),
                         x1 = *reinterpret_cast<const uint32_t*>(v0 + gr * 32 + 4 * (HD / 2)),
                         x8 = *reinterpret_cast<const uint32_t*>(v0 + gr * 32 + 8 * (HD / 2)),
                         x9 = *reinterpret_cast<const uint32_t*>(v0 + gr * 32 + 12 * (HD / 2));
          // 128 + z of the two keys of each pair
          const uint32_t z01 = mask_or(__byte_perm(z0, z1, gr ? 0x7632 : 0x5410), 0x000f000fu, 0x43004300u);
          const uint32_t z89 = mask_or(__byte_perm(z8, z9, gr ? 0x7632 : 0x5410), 0x000f000fu, 0x43004300u);
          const uint32_t lo01 = __byte_perm(x0, x1, 0x5410), hi01 = __byte_perm(x0, x1, 0x7632);
          const uint32_t lo89 = __byte_perm(x8, x9, 0x5410), hi89 = __byte_perm(x8, x9, 0x7632);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a0 = sub_bf16x2(nibbles(lo01, j), z01), a1 = sub_bf16x2(nibbles(hi01, j), z01),
                           a2 = sub_bf16x2(nibbles(lo89, j), z89), a3 = sub_bf16x2(nibbles(hi89, j), z89);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_bf16(o[n][gr][j], a0, a1, a2, a3, w0[n], w1[n]);
          }
        }
      };
      const int at0 = warp * kWarpKeys, k0 = c * kChunk + at0;
      if (k0 + kWarpKeys <= all_see && bad == 0u) {
#pragma unroll
        for (int i = 0; i < kWarpKeys; i += 16) tile(std::false_type(), at0 + i);
      } else {
#pragma unroll 1
        for (int i = 0; i < kWarpKeys; i += 16)
          if (k0 + i < g.keys && !((bad >> ((at0 + i) / 16)) & 1u)) tile(std::true_type(), at0 + i);
      }
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(&empty[s]);
    }

    // ---- the warps' results of this segment meet in shared memory ----
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = n * 8 + t4 * 2 + e;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
        if (gid == 0) ml[warp * kQ + r] = make_float2(top[n][e] - kRescaleLog2, l[n][e]);
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          float* dst = merge + (warp * kQ + r) * L::kRow + gr * 64 + gid * 8;
          *reinterpret_cast<float4*>(dst) = make_float4(o[n][gr][0][e], o[n][gr][1][e], o[n][gr][2][e], o[n][gr][3][e]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(o[n][gr][0][e + 2], o[n][gr][1][e + 2], o[n][gr][2][e + 2], o[n][gr][3][e + 2]);
        }
      }
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
    const bool whole = g.n == g.chunks;
    for (int i = threadIdx.x; i < rows * (HD / 8); i += kWarps * 32) {
      const int r = i / (HD / 8), d = (i % (HD / 8)) * 8;
      float mx = -INFINITY, sum = 0.f, acc[8] = {};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml[w * kQ + r].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 x = ml[w * kQ + r];
        const float f = x.x == -INFINITY ? 0.f : umma::ex2(x.x - mx);
        sum += f * x.y;
        const float* src = merge + (w * kQ + r) * L::kRow + d;
        if (f != 0.f)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += f * src[e];
      }
      const size_t row = row_of(r);
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint4*>(a.out + row * HD + d) =
            make_uint4(umma::pack2_bf16(acc[0] * inv, acc[1] * inv), umma::pack2_bf16(acc[2] * inv, acc[3] * inv),
                       umma::pack2_bf16(acc[4] * inv, acc[5] * inv), umma::pack2_bf16(acc[6] * inv, acc[7] * inv));
      } else {
        const size_t slot = row * a.max_splits + g.first;
        float4* dst = reinterpret_cast<float4*>(a.part_o + slot * HD + d);
        __stcg(dst, make_float4(acc[0], acc[1], acc[2], acc[3]));
        __stcg(dst + 1, make_float4(acc[4], acc[5], acc[6], acc[7]));
        if (d == 0) __stcg(reinterpret_cast<float2*>(a.part_ml) + slot, make_float2(mx, sum));
      }
    }
    if (!whole) {
      // pieces of this pair: cut where the shares of the blocks begin
      const int i0 = (int)(((int64_t)(g.pair0 + 1) * grid - 1) / share.total);
      const int i1 = (int)(((int64_t)(g.pair0 + g.chunks) * grid - 1) / share.total);
      const int pieces = i1 - i0 + 1;
      __threadfence();
      asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
      if (threadIdx.x == 0)
        merge_me = atomicInc(reinterpret_cast<unsigned*>(a.counters) + ((size_t)g.b * a.nkv + g.h) * a.row_tiles + blockIdx.y,
                             (unsigned)pieces - 1u) == (unsigned)pieces - 1u;
      asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
      if (merge_me) {
        __threadfence();
        for (int i = threadIdx.x; i < rows * (HD / 8); i += kWarps * 32) {
          const int r = i / (HD / 8), d = (i % (HD / 8)) * 8;
          const size_t row = row_of(r);
          float mx = -INFINITY, sum = 0.f, acc[8] = {};
          for (int x = 0; x < pieces; ++x) {
            const int first = max(0, share_begin(share.total, grid, i0 + x) - g.pair0);
            const size_t slot = row * a.max_splits + first;
            const float2 v = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + slot);
            if (v.y == 0.f) continue;              // saw no key
            const float mn = fmaxf(mx, v.x), f = mx == -INFINITY ? 0.f : umma::ex2(mx - mn), fx = umma::ex2(v.x - mn);
            mx = mn;
            sum = sum * f + fx * v.y;
            const float4* src = reinterpret_cast<const float4*>(a.part_o + slot * HD + d);
            const float4 y0 = __ldcg(src), y1 = __ldcg(src + 1);
            const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = acc[e] * f + fx * y[e];
          }
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          *reinterpret_cast<uint4*>(a.out + row * HD + d) =
              make_uint4(umma::pack2_bf16(acc[0] * inv, acc[1] * inv), umma::pack2_bf16(acc[2] * inv, acc[3] * inv),
                         umma::pack2_bf16(acc[4] * inv, acc[5] * inv), umma::pack2_bf16(acc[6] * inv, acc[7] * inv));
        }
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");    // the merge rows are free again
  }
}

}  // namespace

void decode_attention_int4(at::Tensor out, at::Tensor q, at::Tensor kc, at::Tensor kw, at::Tensor vc, at::Tensor vw,
                           int64_t nq, at::Tensor lens, at::Tensor tables, double scale, at::Tensor part_o,
                           at::Tensor part_ml, at::Tensor counters, int64_t max_splits, at::Tensor status) {
  const at::Device dev = q.device();
  check_page_pair(kc, kw, vc, vw, dev);
  LSB_INT4_CHECK(q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.is_contiguous() &&
                     reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
                 "q must be contiguous, 16-byte aligned bfloat16 [rows, heads, head_dim]");
  LSB_INT4_CHECK(q.size(2) == kc.size(3) * 2 && q.size(1) >= 1 && q.size(1) % kc.size(1) == 0,
                 "query heads do not match the pages");
  LSB_INT4_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.is_contiguous() &&
                     out.device() == dev, "bad output");
  check_int32(lens, "sequence lengths", 1, dev);
  check_int32(tables, "block_tables", 2, dev);
  const int64_t B = lens.size(0), T = q.size(0), nh = q.size(1), nkv = kc.size(1), hd = q.size(2), bs = kc.size(2);
  LSB_INT4_CHECK(tables.size(0) >= B, "block_tables must hold one row per sequence");
  LSB_INT4_CHECK(nq >= 1 && T == B * nq, "q must hold nq rows per sequence");
  LSB_INT4_CHECK(scale > 0 && std::isfinite(scale), "scale must be positive");
  if (T == 0) return;
  const int64_t cap = tables.size(1) * bs;
  LSB_INT4_CHECK(part_o.scalar_type() == at::kFloat && part_ml.scalar_type() == at::kFloat &&
                     counters.scalar_type() == at::kInt && part_o.is_contiguous() && part_ml.is_contiguous() &&
                     counters.is_contiguous() && part_o.device() == dev && part_ml.device() == dev &&
                     counters.device() == dev && max_splits * kChunk >= cap && part_o.numel() >= T * nh * max_splits * hd &&
                     part_ml.numel() >= T * nh * max_splits * 2 && counters.numel() >= T * nh,
                 "decode workspace too small for this batch");
  LSB_INT4_CHECK(B * nkv * ((cap + kChunk - 1) / kChunk) < INT32_MAX, "more 128-key chunks than an int32 can count");
  LSB_INT4_CHECK(T * nh < INT32_MAX && nq * (nh / nkv) <= 16 * 65535, "batch exceeds int32 rows");
  const at::cuda::CUDAGuard guard(dev);
  const int rows = (int)(nq * (nh / nkv)), nt = rows > 8 ? 2 : 1, tiles = (rows + 8 * nt - 1) / (8 * nt);
  Args a = {(bf16*)out.data_ptr(), (const bf16*)q.data_ptr(), {kc.data_ptr<uint8_t>(), kw.data_ptr<int16_t>()},
            {vc.data_ptr<uint8_t>(), vw.data_ptr<int16_t>()}, lens.data_ptr<int>(), tables.data_ptr<int>(),
            part_o.data_ptr<float>(), part_ml.data_ptr<float>(), counters.data_ptr<int>(), status_ptr(status),
            (float)(scale * 1.4426950408889634), (int)tables.size(1), (int)B, (int)nq, (int)nh, (int)nkv, (int)bs,
            (int)kc.size(0), (int)max_splits, tiles};
  auto go = [&](auto kern, int smem, int per_sm) {
    ensure_dynamic_smem((const void*)kern, smem);
    // as many blocks as fit the GPU at once, shared by the row tiles, and no more than there can be chunks
    const int64_t most = B * nkv * std::max<int64_t>(1, (cap + kChunk - 1) / kChunk);
    const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(most, 148 * per_sm / tiles));
    launch_pdl(kern, dim3((unsigned)grid, tiles), dim3(kThreads), smem, at::cuda::getCurrentCUDAStream(), a);
  };
#define LSB_DEC(HD, NT) go(decode_int4_kernel<HD, NT>, DecLayout<HD, NT>::kBytes, DecLayout<HD, NT>::kBlocks)
  if (hd == 128) {
    if (nt == 1) LSB_DEC(128, 1);
    else LSB_DEC(128, 2);
  } else {
    if (nt == 1) LSB_DEC(64, 1);
    else LSB_DEC(64, 2);
  }
#undef LSB_DEC
  const cudaError_t e = cudaGetLastError();
  LSB_INT4_CHECK(e == cudaSuccess, std::string("decode_attention_int4 launch failed: ") + cudaGetErrorString(e));
}

}  // namespace lsb
