// Decode and verify attention against 4-bit KV pages (format: int4_pages.cuh).
//
// The query rows of one KV head (nq new tokens x heads per KV head) are the narrow side of the tensor
// core products and the keys and head dims the wide one, with mma.sync and fp32 sums:
//   S^T [16 keys x 8 rows] = (C_K - z) [16 x HD] Q^T    O^T [16 dims x 8 rows] += (C_V - z)^T [16 x 16 keys] W^T
// so a tile of 16 keys costs 8 rows of padding at most, where a tcgen05 tile would need 128 of them.  More
// than eight rows are so many tiles of eight, next to one another in the grid: the second reads the keys
// from L2.
//
// What bounds it next to memory is the integer pipe (64 lanes a clock) that turns nibbles into operands.
// A nibble masked where it stands in a 16-bit lane is a bf16 (the patterns up to 255 are an even grid through
// zero), and a multiply-add by 2^127 turns it into the exact (c - z) / 64 or, four bits up, (c - z) / 4: five
// integer instructions for eight codes.  The powers of two go into the query and into O's rows.
//   s = sum_g sk_g sum_d q_d (c_d - z_g), g: groups of 64 dims      w_jg = p_j sv_jg in bf16: the one rounding
// besides the output's.
// A warp's operand layout asks K for 8 dims of a key (a code word as it lies) and V for pairs of keys (one
// PRMT joins the half words of two rows): neither needs a shuffle, and the order of dims or keys inside a
// product is free as long as both operands share it.
//
// A warp takes 32 keys of every 128-key chunk and copies them itself, bulk copies into a ring of its own (a
// producer warp would cost registers that four more computing warps need); the four warps of a block
// meet when a segment ends.  Work is the list of (sequence, KV head, chunk), cut into equal contiguous
// shares over a grid that fills the GPU once, whatever the lengths: lengths are read on the device, so one
// captured launch serves any batch.  A (sequence, head) that is cut leaves fp32 partials; the block that
// finishes last merges them in their order (results do not depend on who is last) and resets the counter.
// Where every (sequence, head) can have a block and none is far above the equal share, nothing is cut: leaving
// and merging a piece costs about kCutCost chunks, and kNextCost more where a block goes on to another one
// (on the device, cut / not: one context of 513 keys 10.4 / 11.4 us, eight of 700 15.7 / 17.1, 64 of 600 to 1200
// 33.8 / 29.8, 64 of 256 to 512 cut by an earlier form 25.6 / 17.6).
//
// Measured on a B200 with 32 query and 8 KV heads of 128: 32 contexts of 1..32768 keys 171 us (594 MB: 3.5 TB/s),
// 64 of 256..512 keys 18 us, 64 x 4 queries on 200..2048 keys 79 us.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <type_traits>

#include "int4_pages.cuh"
#include "umma.cuh"

namespace lsb {

int* status_ptr(const at::Tensor& status);

namespace {

using namespace int4;
using umma::wait_phase;

constexpr int kChunk = 128;               // keys of a unit of work
constexpr int kWarps = 4;
constexpr int kWarpKeys = kChunk / kWarps;
constexpr int kThreads = kWarps * 32;
constexpr int kBlocksPerSm = 4;           // 128 registers a thread
constexpr int kRows = 8;                  // query rows of a block
constexpr int kCutCost = 3, kNextCost = 2;
constexpr float kRescaleLog2 = 8.f;

template <int HD>
struct DecLayout {
  static constexpr int kGroups = HD / kGroup;
  static constexpr int kStages = HD == 128 ? 2 : 4;        // of a warp's ring
  static constexpr int kCodes = kWarpKeys * HD / 2;        // bytes of one tensor's codes in a stage
  static constexpr int kWords = kWarpKeys * kGroups * 2;
  static constexpr int kStage = 2 * kCodes + 2 * kWords;   // K codes, V codes, K words, V words
  static constexpr int kRow = HD + 4;                      // floats of a merge row (padded)
  static constexpr int kMergeOff = kWarps * kStages * kStage;
  static constexpr int kMlOff = kMergeOff + kWarps * kRows * kRow * 4;
  static constexpr int kBarOff = kMlOff + kWarps * kRows * 8;
  static constexpr int kBytes = kBarOff + kWarps * kStages * 8;
};

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
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t x, uint32_t m, uint32_t z) {
  uint32_t y;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(x), "r"(m), "r"(z));
  return y;
}
// The patterns 0 .. 255 of bf16 (subnormals and the first binade) are one even grid: n 2^-133.  So a nibble
// masked where it stands is c 2^-133 or, four bits up, c 2^-129, and one multiply-add by 2^127 makes the
// exact (c - z) / 64 or (c - z) / 4.
constexpr uint32_t kUp = 0x7f007f00u;      // 2^127 twice
// zero codes of a pair of 16-bit lanes (in their low four bits) as -z / 64 and -z / 4
struct Zeros {
  uint32_t low, high;
};
__device__ __forceinline__ Zeros zeros(uint32_t w) {
  const uint32_t low = mul2(w & 0x000f000fu, kUp | 0x80008000u);
  return {low, mul2(low, 0x41804180u)};
}
// nibbles (s, s + 4) of a word less the lanes' zero codes: /64 for even s, /4 for odd s
__device__ __forceinline__ void codes_bf16(uint32_t w, const Zeros& z, uint32_t* y) {
  const uint32_t h = w >> 8;
  y[0] = fma_bf16x2(w & 0x000f000fu, kUp, z.low);
  y[1] = fma_bf16x2(w & 0x00f000f0u, kUp, z.high);
  y[2] = fma_bf16x2(h & 0x000f000fu, kUp, z.low);
  y[3] = fma_bf16x2(h & 0x00f000f0u, kUp, z.high);
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
  float scale_log2;            // 16 times the scale, for scores in the log2 domain
  int width, B, nq, nh, nkv, bs, nblk, max_splits, row_tiles;
  uint32_t page_magic;         // ceil(2^32 / (bs / 16)); 0 for blocks of 16
};

__device__ __forceinline__ int key_count(const Args& a, int b) {
  return max(0, min(a.lens[b], (int)min((int64_t)a.width * a.bs, (int64_t)INT32_MAX - kChunk)));
}
__device__ __forceinline__ int chunk_count(const Args& a, int b) { return (key_count(a, b) + kChunk - 1) / kChunk; }

// This block's share [c0, c1) of all chunks and where it starts; the same in every lane of a warp.
struct Share {
  int c0, c1;
  int b;             // sequence of chunk c0
  int before;        // chunks of all heads before sequence b
};
// All chunks, and the blocks they are dealt to (0: a block per (sequence, head), nothing cut).
struct Deal {
  int total, grid;
};
__device__ __forceinline__ int share_begin(const Deal& d, int i) { return (int)((int64_t)d.total * i / d.grid); }

__device__ __forceinline__ Share find_share(const Args& a, int lane, Deal& deal) {
  int sum = 0, most = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int n = b0 + lane < a.B ? chunk_count(a, b0 + lane) : 0;
    sum += n;
    most = max(most, n);
  }
  deal.total = __reduce_add_sync(0xffffffffu, sum) * a.nkv;
  most = __reduce_max_sync(0xffffffffu, most);
  Share s = {0, 0, 0, 0};
  const int blocks = (int)gridDim.x, me = (int)blockIdx.x;
  const bool uncut = (int64_t)a.B * a.nkv <= blocks && most <= deal.total / blocks + kCutCost + (deal.total > blocks ? kNextCost : 0);
  deal.grid = uncut ? 0 : min(blocks, deal.total);
  if (uncut ? me >= a.B * a.nkv : me >= deal.grid) return s;
  if (!uncut) {
    s.c0 = share_begin(deal, me);
    s.c1 = share_begin(deal, me + 1);
  }
  // the sequence whose chunks hold c0 (uncut: sequence me / nkv)
  const int want = uncut ? me / a.nkv : s.c0 / a.nkv;
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int n = b0 + lane < a.B ? chunk_count(a, b0 + lane) : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, uncut ? b0 + lane == want : base + incl > want);
    if (hit) {
      const int l = __ffs(hit) - 1, mine = __shfl_sync(0xffffffffu, n, l);
      s.b = b0 + l;
      s.before = (base + __shfl_sync(0xffffffffu, incl - n, l)) * a.nkv;
      if (uncut) {
        s.c0 = s.before + (me % a.nkv) * mine;
        s.c1 = s.c0 + mine;
      }
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

template <int HD>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) decode_int4_kernel(const Args a) {
  using L = DecLayout<HD>;
  constexpr int kG = L::kGroups;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int abort_flag, merge_me;
  volatile int* abort_v = &abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOff) + warp * L::kStages;    // this warp's ring
  uint8_t* ring = smem + warp * L::kStages * L::kStage;
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane < L::kStages) mbar_init(&full[lane], 1);
  fence_barrier_init();
  pdl_trigger();
  pdl_wait();
  __syncthreads();
  Deal deal;
  Share share = find_share(a, lane, deal);

  // ---- copies: this warp's 32 keys of the chunks of the share, kStages of them ahead ----
  Share ahead = share;
  Segment pg;
  // chunks left of the segment; first key and keys there for the next one; a lane's block and row in it
  int left = 0, k_next = 0, there = 0, k_end = 0, blk = 0, first_row = 0, issued = 0;
  uint32_t gone = 0;                                       // two bits a stage: 16-key tiles that are not there
  bool more = true;
  // Lanes 0..7: two pages (32 keys never touch more, pages hold whole 16-key tiles) x four tensors: codes of
  // K and V, words of K and V.
  const int tensor = lane >> 1 & 3, per_key = tensor < 2 ? HD / 2 : 2 * kG;
  const uint8_t* source = tensor == 0 ? a.kp.codes : tensor == 1 ? a.vp.codes
                          : reinterpret_cast<const uint8_t*>(tensor == 2 ? a.kp.words : a.vp.words);
  const uint32_t dest = smem_u32(ring) + (tensor < 2 ? tensor * L::kCodes : 2 * L::kCodes + (tensor & 1) * L::kWords);
  const int cap = lane < 8 ? kWarpKeys : 0;
  int from = 0, to = 0;                                    // keys of this lane's page in the next chunk
  auto find_next = [&]() {
    k_next += kChunk;
    if (--left < 0) {
      more = next_segment(a, ahead, pg);
      if (!more) return;
      left = pg.n - 1;
      k_next = pg.first * kChunk + warp * kWarpKeys;
      k_end = (pg.keys + 15) & ~15;
    }
    there = max(0, min(kWarpKeys, k_end - k_next));
    const uint32_t tile = (uint32_t)k_next / 16u;
    const int page = (int)(a.page_magic ? __umulhi(tile, a.page_magic) : tile) + (lane & 1), start = page * a.bs - k_next;
    from = max(0, start);
    to = min(min(cap, there), start + a.bs);
    first_row = from - start;
    if (from < to) blk = __ldg(a.tables + (int64_t)pg.b * a.width + page);
  };
  auto issue = [&]() {
    if (!more) return;
    const int s = issued % L::kStages;
    bool mine = from < to;
    const bool bad = mine && (uint32_t)blk >= (uint32_t)a.nblk;
    int total = there;
    if (gone) gone &= ~(3u << (2 * s));
    if (__any_sync(0xffffffffu, bad)) {
      if (bad) record_error(a.status, kBadIndex);
      const uint32_t flags = bad ? ((1u << (to / 16)) - 1u) & ~((1u << (from / 16)) - 1u) : 0u;
      gone |= __reduce_or_sync(0xffffffffu, flags) << (2 * s);
      total -= 16 * __popc(gone >> (2 * s) & 3u);
      mine = mine && !bad;
    }
    if (lane == 0) mbar_expect_tx(&full[s], (uint32_t)total * (HD + 4 * kG));
    __syncwarp();
    if (mine) {
      const int64_t row = ((int64_t)blk * a.nkv + pg.h) * a.bs + first_row;
      bulk_copy(dest + s * L::kStage + from * per_key, source + row * per_key, (to - from) * per_key, &full[s]);
    }
    ++issued;
    find_next();
  };
  find_next();
#pragma unroll 1
  for (int i = 0; i < L::kStages; ++i) issue();

  const int gid = lane >> 2, t4 = lane & 3;
  const int group_heads = a.nh / a.nkv;
  const int row0 = blockIdx.y * kRows, rows = min(kRows, a.nq * group_heads - row0);
  float* merge = reinterpret_cast<float*>(smem + L::kMergeOff);
  float2* ml = reinterpret_cast<float2*>(smem + L::kMlOff);

  // sequences without keys: zeros
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (key_count(a, b) == 0)
      for (int i = threadIdx.x; i < a.nkv * rows * (HD / 8); i += kThreads) {
        const int r = i / (HD / 8) % rows + row0, h = i / (HD / 8) / rows;
        const size_t at = ((size_t)b * a.nq + r / group_heads) * a.nh + h * group_heads + r % group_heads;
        *reinterpret_cast<uint4*>(a.out + at * HD + (i % (HD / 8)) * 8) = make_uint4(0, 0, 0, 0);
      }

  Segment g;
  int it = 0;
  bool ok = true;
  while (next_segment(a, share, g)) {
    // address of query row r (< rows) of this pair, in rows of HD
    auto row_of = [&](int r) {
      r += row0;
      return ((size_t)g.b * a.nq + r / group_heads) * a.nh + g.h * group_heads + r % group_heads;
    };
    // Q^T operand: row gid; for group g and word i the dims 64 g + 16 t4 + 8 i + (s, s + 4), times 4 for even s and
    // 1/4 for odd s: with the codes' /64 and /4 every product is a sixteenth
    uint32_t qf[kG][2][4];
    {
      const bool live = gid < rows;
      const uint4* src = reinterpret_cast<const uint4*>(a.q + row_of(live ? gid : 0) * HD);
#pragma unroll
      for (int gr = 0; gr < kG; ++gr)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 v = live ? src[(gr * 64 + t4 * 16 + i * 8) / 8] : make_uint4(0, 0, 0, 0);
          qf[gr][i][0] = mul2(__byte_perm(v.x, v.z, 0x5410), 0x40804080u);
          qf[gr][i][1] = mul2(__byte_perm(v.x, v.z, 0x7632), 0x3e803e80u);
          qf[gr][i][2] = mul2(__byte_perm(v.y, v.w, 0x5410), 0x40804080u);
          qf[gr][i][3] = mul2(__byte_perm(v.y, v.w, 0x7632), 0x3e803e80u);
        }
    }
    // keys that row r of the block sees, and keys that all its rows see
    auto limit = [&](int r) { return r < rows ? min(g.keys, a.lens[g.b] - a.nq + (row0 + r) / group_heads + 1) : 0; };
    const int all_see = min(g.keys, a.lens[g.b] - a.nq + row0 / group_heads + 1);

    // m: the reference that exponents are taken from, top: the score that moves it (-inf: none seen yet)
    float o[kG][4][4], m[2] = {0.f, 0.f}, top[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int gr = 0; gr < kG; ++gr)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[gr][j][e] = 0.f;

    for (int c = g.first; c < g.first + g.n; ++c, ++it) {
      const int s = it % L::kStages;
      ok = ok && __all_sync(0xffffffffu, wait_phase(&full[s], (it / L::kStages) & 1, abort_v, a.status, kTimeoutTmaFull));
      if (!ok) break;
      const uint8_t* st = ring + s * L::kStage;
      // 16 keys; edge: some row of this block does not see some of them
      auto tile = [&](auto edge, int at) {
        const int k0 = c * kChunk + warp * kWarpKeys + at;
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
        float p[4];                                // [key a row 0, key a row 1, key b row 0, key b row 1]
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          const uint2 wa = *reinterpret_cast<const uint2*>(ka + gr * 32);
          const uint2 wb = *reinterpret_cast<const uint2*>(ka + gr * 32 + 8 * (HD / 2));
          const Zeros za = zeros(__byte_perm(kwa, 0, gr ? 0x3232 : 0x1010)), zb = zeros(__byte_perm(kwb, 0, gr ? 0x3232 : 0x1010));
          float sacc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t ya[4], yb[4];
            codes_bf16(i ? wa.y : wa.x, za, ya);
            codes_bf16(i ? wb.y : wb.x, zb, yb);
#pragma unroll
            for (int e = 0; e < 4; e += 2)
              mma_bf16(sacc, ya[e], yb[e], ya[e + 1], yb[e + 1], qf[gr][i][e], qf[gr][i][e + 1]);
          }
          const float ska = scale(kwa, gr), skb = scale(kwb, gr);
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = gr == 0 ? (e < 2 ? ska : skb) * sacc[e] : fmaf(e < 2 ? ska : skb, sacc[e], p[e]);
        }
        bool grow = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] *= a.scale_log2;
          if (edge.value && k0 + (e < 2 ? key_a : key_b) >= limit(t4 * 2 + (e & 1))) p[e] = -INFINITY;
          grow |= p[e] > top[e & 1];
        }
        // the reference maximum moves only when a score passes it by 2^8 (first tile: from -inf)
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(p[e], p[e + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            // f = 2^(old - new); a row that has seen no key keeps reference 0 and the next score moves it
            const bool none = top[e] == -INFINITY;
            const float mn = none ? mx : fmaxf(m[e], mx), f = none ? 0.f : umma::ex2(m[e] - mn);
            m[e] = mn == -INFINITY ? 0.f : mn;
            top[e] = mn + kRescaleLog2;
            l[e] *= f;
#pragma unroll
            for (int gr = 0; gr < kG; ++gr)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[gr][j][e] *= f, o[gr][j][e + 2] *= f;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = umma::ex2(p[e] - m[e & 1]);
          l[e & 1] += p[e];
        }
        // O^T: words of keys (rows 2 t4, 2 t4 + 1, + 8) for dims 64 g + 8 gid ..; row 2 t4 is key t4, row
        // 2 t4 + 1 key t4 + 4
        const uint8_t* v0 = st + L::kCodes + (at + t4) * (HD / 2) + gid * 4;
        const uint32_t z0 = words(vw, at + t4), z1 = words(vw, at + t4 + 4), z8 = words(vw, at + t4 + 8),
                       z9 = words(vw, at + t4 + 12);
#pragma unroll
        for (int gr = 0; gr < kG; ++gr) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = p[e] * scale(e < 2 ? vwa : vwb, gr);
            // a key that this row does not see may hold anything, NaN scales among it
            if (edge.value && k0 + (e < 2 ? key_a : key_b) >= limit(t4 * 2 + (e & 1))) w[e] = 0.f;
          }
          const uint32_t w0 = transpose8x8(umma::pack2_bf16(w[0], w[1])), w1 = transpose8x8(umma::pack2_bf16(w[2], w[3]));
          const uint32_t x0 = *reinterpret_cast<const uint32_t*>(v0 + gr * 32),
                         x1 = *reinterpret_cast<const uint32_t*>(v0 + gr * 32 + 4 * (HD / 2)),
                         x8 = *reinterpret_cast<const uint32_t*>(v0 + gr * 32 + 8 * (HD / 2)),
                         x9 = *reinterpret_cast<const uint32_t*>(v0 + gr * 32 + 12 * (HD / 2));
          const Zeros z01 = zeros(__byte_perm(z0, z1, gr ? 0x7632 : 0x5410)), z89 = zeros(__byte_perm(z8, z9, gr ? 0x7632 : 0x5410));
          uint32_t a0[4], a1[4], a2[4], a3[4];
          codes_bf16(__byte_perm(x0, x1, 0x5410), z01, a0);
          codes_bf16(__byte_perm(x0, x1, 0x7632), z01, a1);
          codes_bf16(__byte_perm(x8, x9, 0x5410), z89, a2);
          codes_bf16(__byte_perm(x8, x9, 0x7632), z89, a3);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_bf16(o[gr][j], a0[j], a1[j], a2[j], a3[j], w0, w1);
        }
      };
      const int k0 = c * kChunk + warp * kWarpKeys;
      const uint32_t away = gone >> (2 * s) & 3u;
      if (k0 + kWarpKeys <= all_see && away == 0u) {
#pragma unroll
        for (int i = 0; i < kWarpKeys; i += 16) tile(std::false_type(), i);
      } else {
#pragma unroll 1
        for (int i = 0; i < kWarpKeys; i += 16)
          if (k0 + i < g.keys && !(away >> (i / 16) & 1u)) tile(std::true_type(), i);
      }
      __syncwarp();                                // every lane has read the stage
      issue();
    }

    // ---- the warps' results of this segment meet in shared memory ----
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = t4 * 2 + e;
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
      if (gid == 0) ml[warp * kRows + r] = make_float2(top[e] - kRescaleLog2, l[e]);
#pragma unroll
      for (int gr = 0; gr < kG; ++gr) {
        float* dst = merge + (warp * kRows + r) * L::kRow + gr * 64 + gid * 8;
        *reinterpret_cast<float4*>(dst) = make_float4(o[gr][0][e] * 64.f, o[gr][1][e] * 4.f, o[gr][2][e] * 64.f, o[gr][3][e] * 4.f);
        *reinterpret_cast<float4*>(dst + 4) = 
            make_float4(o[gr][0][e + 2] * 64.f, o[gr][1][e + 2] * 4.f, o[gr][2][e + 2] * 64.f, o[gr][3][e + 2] * 4.f);
      }
    }
    __syncthreads();
    const bool whole = g.n == g.chunks;
    for (int i = threadIdx.x; i < rows * (HD / 8); i += kThreads) {
      const int r = i / (HD / 8), d = (i % (HD / 8)) * 8;
      float mx = -INFINITY, sum = 0.f, acc[8] = {};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml[w * kRows + r].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 x = ml[w * kRows + r];
        const float f = x.x == -INFINITY ? 0.f : umma::ex2(x.x - mx);
        sum += f * x.y;
        const float* src = merge + (w * kRows + r) * L::kRow + d;
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
      const int i0 = (int)(((int64_t)(g.pair0 + 1) * deal.grid - 1) / deal.total);
      const int i1 = (int)(((int64_t)(g.pair0 + g.chunks) * deal.grid - 1) / deal.total);
      const int pieces = i1 - i0 + 1;
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0)
        merge_me = atomicInc(reinterpret_cast<unsigned*>(a.counters) + ((size_t)g.b * a.nkv + g.h) * a.row_tiles + blockIdx.y,
                             (unsigned)pieces - 1u) == (unsigned)pieces - 1u;
      __syncthreads();
      if (merge_me) {
        __threadfence();
        for (int i = threadIdx.x; i < rows * (HD / 8); i += kThreads) {
          const int r = i / (HD / 8), d = (i % (HD / 8)) * 8;
          const size_t row = row_of(r);
          float mx = -INFINITY, sum = 0.f, acc[8] = {};
#pragma unroll 4
          for (int x = 0; x < pieces; ++x) {
            const int first = max(0, share_begin(deal, i0 + x) - g.pair0);
            const size_t slot = row * a.max_splits + first;
            const float2 v = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + slot);
            const float4* src = reinterpret_cast<const float4*>(a.part_o + slot * HD + d);
            const float4 y0 = __ldcg(src), y1 = __ldcg(src + 1);
            const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
            if (v.y == 0.f) continue;              // saw no key
            const float mn = fmaxf(mx, v.x), f = mx == -INFINITY ? 0.f : umma::ex2(mx - mn), fx = umma::ex2(v.x - mn);
            mx = mn;
            sum = sum * f + fx * v.y;
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
    __syncthreads();                               // the merge rows are free again
  }
  // after a wait ran out: the copies in flight have landed before the block may end
  for (; it < issued; ++it) mbar_wait(&full[it % L::kStages], (it / L::kStages) & 1);
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
  const float factor = scale_log2(scale, 16);
  if (T == 0) return;
  const int64_t cap = tables.size(1) * bs;
  LSB_INT4_CHECK(part_o.scalar_type() == at::kFloat && part_ml.scalar_type() == at::kFloat &&
                     counters.scalar_type() == at::kInt && part_o.is_contiguous() && part_ml.is_contiguous() &&
                     counters.is_contiguous() && part_o.device() == dev && part_ml.device() == dev &&
                     counters.device() == dev && max_splits * kChunk >= cap && part_o.numel() >= T * nh * max_splits * hd &&
                     part_ml.numel() >= T * nh * max_splits * 2 && counters.numel() >= T * nh,
                 "decode workspace too small for this batch");
  // a page is tile * magic >> 32: exact while tile * (bs / 16) stays below 2^32
  LSB_INT4_CHECK((cap / 16 + 8) * (bs / 16) < (1ll << 32) || ((bs / 16) & (bs / 16 - 1)) == 0, "context too long for this block size");
  LSB_INT4_CHECK(B * nkv * ((cap + kChunk - 1) / kChunk) < INT32_MAX, "more 128-key chunks than an int32 can count");
  LSB_INT4_CHECK(T * nh < INT32_MAX && nq * (nh / nkv) <= kRows * 65535, "batch exceeds int32 rows");
  const at::cuda::CUDAGuard guard(dev);
  const int tiles = (int)((nq * (nh / nkv) + kRows - 1) / kRows);
  Args a = {(bf16*)out.data_ptr(), (const bf16*)q.data_ptr(), {kc.data_ptr<uint8_t>(), kw.data_ptr<int16_t>()},
            {vc.data_ptr<uint8_t>(), vw.data_ptr<int16_t>()}, lens.data_ptr<int>(), tables.data_ptr<int>(),
            part_o.data_ptr<float>(), part_ml.data_ptr<float>(), counters.data_ptr<int>(), status_ptr(status),
            factor, (int)tables.size(1), (int)B, (int)nq, (int)nh, (int)nkv, (int)bs,
            (int)kc.size(0), (int)max_splits, tiles, bs == 16 ? 0u : (uint32_t)(((1ll << 32) + bs / 16 - 1) / (bs / 16))};
  auto go = [&](auto kern, int smem) {
    ensure_dynamic_smem((const void*)kern, smem);
    // as many blocks as fit the GPU at once, shared by the row tiles, and no more than there can be chunks
    const int64_t most = B * nkv * std::max<int64_t>(1, (cap + kChunk - 1) / kChunk);
    const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(most, 148 * kBlocksPerSm / tiles));
    launch_pdl(kern, dim3((unsigned)grid, tiles), dim3(kThreads), smem, at::cuda::getCurrentCUDAStream(), a);
  };
  if (hd == 128) go(decode_int4_kernel<128>, DecLayout<128>::kBytes);
  else go(decode_int4_kernel<64>, DecLayout<64>::kBytes);
  const cudaError_t e = cudaGetLastError();
  LSB_INT4_CHECK(e == cudaSuccess, std::string("decode_attention_int4 launch failed: ") + cudaGetErrorString(e));
}

}  // namespace lsb
