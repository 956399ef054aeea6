// Varlen causal attention of query chunks against 4-bit KV pages (format: int4_pages.cuh) on the
// 5th-generation tensor cores: S = Q K^T and O += P V as tcgen05.mma with fp32 accumulators in TMEM.
//
// The query rows of one KV head are (query, head of its group) pairs, query-major; a block computes two
// 128-row tiles ("A", "B") of them against the same 128-key tiles, so a key is dequantised once for
// 256 rows whatever the group size, and short chunks still fill the tile.
//   warps 0..3 / 4..7 : softmax of tile A / B, a thread per row.  Two passes over the row's 128 scores in
//                    TMEM (maximum; exponentials), 32 columns at a time, so nothing waits on 128
//                    registers.  P replaces S in TMEM as bf16 (columns 16 c .. of chunk c: behind what
//                    has been read) and is the PV product's A operand from there: it never passes
//                    through shared memory.  The reference maximum moves only when a score passes it by
//                    2^8; O is then rescaled in TMEM (its last PV is done: S of this tile was issued after).
//   warp 13        : copies the codes and words of K and V tiles (a run per page, bulk copies) into a ring of
//                    three entries, K and V by turns.
//   warps 8..11    : dequantise an entry into the two-stage rings of the 128B-swizzled tiles the products
//                    read (K K-major, V MN-major).  A code pair is (nibble s, nibble s + 4) of a word, so
//                    every 8 dims stand in the order 0 4 1 5 2 6 3 7: Q's rows are written in that order
//                    too, and O's columns are put back at the end.  128 + c is a bf16 with c in its
//                    mantissa; less 128 + z, times the scale, both exact.  Lanes of the upper group take
//                    the halves of their 16 bytes the other way round: no bank is hit twice in a store.
//   warp 12, lane 0: MMA issuer: PV_A(j), S_A(j+1), PV_B(j), S_B(j+1): while one tile's softmax works the
//                    other tile's products run.
// A 4096-token prompt of 32 / 8 heads of 128 takes 200 us (684 TFLOP/s): products 2350 of 5400 cycles a key tile.
//
// Keys past the block's last visible one, or in a block outside the pool (recorded), are zeros in both
// tiles and masked in S.  A V group that holds NaN is zeroed too and flagged: only the rows that see the
// key return NaN for that group.  Every wait is bounded; a timeout records an error and every role ends.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "int4_pages.cuh"
#include "umma.cuh"

namespace lsb {

int* status_ptr(const at::Tensor& status);

namespace {

using namespace int4;
using namespace umma;

constexpr int kBQ = 128;                  // rows of a tile (UMMA M)
constexpr int kBK = 128;                  // keys of a tile
constexpr int kDeq = 4;                   // dequantising warps, 32 keys of a tile each
constexpr int kMmaWarp = 8 + kDeq, kCopyWarp = kMmaWarp + 1;
constexpr int kThreads = (kCopyWarp + 1) * 32;
constexpr int kEntries = 3;               // ring of packed tiles
constexpr float kRescaleLog2 = 8.f;

template <int HD>
struct PfLayout {
  static constexpr int kHalves = HD / 64;
  static constexpr int kHalf = 128 * 128;                 // 128 rows of 128 bytes
  static constexpr int kTile = kHalves * kHalf;
  static constexpr int kKOff = 2 * kTile;                 // after the two Q tiles
  static constexpr int kVOff = kKOff + 2 * kTile;
  static constexpr int kRawOff = kVOff + 2 * kTile;        // packed tiles: codes, then words
  static constexpr int kRawCodes = kBK * HD / 2;
  static constexpr int kRaw = kRawCodes + kBK * kHalves * 2;
  static constexpr int kBarOff = kRawOff + kEntries * kRaw;
  static constexpr int kBytes = kBarOff + 512 + 1024;     // barriers and flags, alignment slack
};

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(acc));
}
// 32 lanes x 32 columns of fp32 (no wait)
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// two fp32 at a time (one instruction)
__device__ __forceinline__ uint64_t join2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split2(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t mask_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}

// What softmax has to know of a 128-key tile beyond its position, a bit per key: keys that are not there
// (known when K is), and those whose V group 0 / 1 is NaN (known when V is).
struct TileFlags {
  uint32_t gone[4], nan0[4], nan1[4];      // per dequantising warp
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) prefill_int4_kernel(
    bf16* __restrict__ out, const bf16* __restrict__ q, Pages kp, Pages vp, const int* __restrict__ cu_q,
    const int* __restrict__ k_lens, const int* __restrict__ tables, int width, int B, int T, int max_q, float scale_log2,
    int nh, int nkv, int bs, int nblk, int* __restrict__ status) {
  using L = PfLayout<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 7,
           *s_full = bars + 9, *p_full = bars + 11, *p_half = bars + 13, *drain = bars + 15, *raw_full = bars + 16,
           *raw_empty = raw_full + kEntries;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_empty + kEntries);
  volatile uint32_t* raw_gone = tmem_slot + 1;             // 16-key tiles of an entry that are not there
  TileFlags* flags = reinterpret_cast<TileFlags*>(smem + L::kBarOff + 256);    // four tiles' worth
  __shared__ int abort_flag;
  volatile int* abort_v = &abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_trigger();
  pdl_wait();
  // This block's sequence and pair of tiles: the grid holds (pair of tiles, KV head), heads fastest, for as many
  // pairs as the rows can make; a sequence's last pair, which sees most keys, comes first.
  const int G = nh / nkv, per_tile = kBQ / G;              // queries of a tile
  const int kvh = blockIdx.x % nkv, want = blockIdx.x / nkv;
  int seq = -1, pair = 0, base = 0;
  auto row_at = [&](int b) { return max(0, min(T, cu_q[b])); };      // first row of sequence b, whatever the table holds
  for (int b0 = 0; b0 < B && seq < 0; b0 += 32) {
    int n = 0;
    if (b0 + lane < B) n = (max(0, min(max_q, row_at(b0 + lane + 1) - row_at(b0 + lane))) + 2 * per_tile - 1) / (2 * per_tile);
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, base + incl > want);
    if (hit) {
      const int l = __ffs(hit) - 1;
      seq = b0 + l;
      pair = base + __shfl_sync(0xffffffffu, incl, l) - 1 - want;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (seq < 0) return;
  const int q0 = row_at(seq), q_len = row_at(seq + 1) - q0;
  const int first = pair * 2 * per_tile;
  const int k_cap = max(0, min(k_lens[seq], (int)min((int64_t)width * bs, (int64_t)INT32_MAX - kBK)));
  const int shift = k_lens[seq] - q_len;                   // absolute position of query 0
  int kend_t[2], nt[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int a = first + t * per_tile, last = min(q_len, a + per_tile) - 1;
    kend_t[t] = a < q_len ? max(0, min(k_cap, shift + last + 1)) : 0;
    nt[t] = (kend_t[t] + kBK - 1) / kBK;
  }
  const int kend = max(kend_t[0], kend_t[1]), ntiles = max(nt[0], nt[1]);

  // the softmax warps' query rows, on their way while the barriers are set up
  uint4 qv[HD / 8];
  if (warp < 8) {
    constexpr int kPieces = HD / 8;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int rr = (warp & 3) * 32 + i * (32 / kPieces) + lane / kPieces;
      const int qi = first + (warp >> 2) * per_tile + rr / G;
      qv[i] = make_uint4(0, 0, 0, 0);
      if (rr < per_tile * G && qi < q_len)
        qv[i] = __ldg(reinterpret_cast<const uint4*>(q + ((size_t)(q0 + qi) * nh + kvh * G + rr % G) * HD) + lane % kPieces);
    }
  }
  if (threadIdx.x == 0) {
    abort_flag = 0;
    mbar_init(q_full, 8);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], kDeq);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], kDeq);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&p_half[s], 4);
    }
    for (int e = 0; e < kEntries; ++e) {
      mbar_init(&raw_full[e], 1);
      mbar_init(&raw_empty[e], kDeq);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;                        // S (then P) of tile t at 128 t, O at 256 + 128 t

  if (warp >= 8 && warp < kMmaWarp) {
    // ---------------- dequantisation ----------------
    constexpr int kCpk = HD / 32;                          // 16-byte chunks of a key
    constexpr int kKps = 32 / kCpk;                        // keys of a step
    const int w = warp - 8;
    const int chunk = lane % kCpk, half = chunk >> 1, key0 = w * 32 + lane / kCpk;
    // words 2 h and 2 h + 1 of the chunk first (h = half), then the other two; their places in the tile
    const uint32_t src0 = key0 * (HD / 2) + chunk * 16 + half * 8;
    uint32_t place[4];
#pragma unroll
    for (int p = 0; p < 4; ++p)
      place[p] = half * L::kHalf + key0 * 128 + ((((chunk & 1) * 4 + (p ^ (half * 2))) ^ (key0 & 7)) << 4);
    bool ok = true;
#pragma unroll 1
    for (int e = 0; e < 2 * ntiles; ++e) {                 // K of tile 0, V of tile 0, K of tile 1, ..
      const int j = e >> 1, kv = e & 1, s = j & 1, u = j >> 1, re = e % kEntries;
      ok = __all_sync(0xffffffffu, wait_phase(&raw_full[re], (e / kEntries) & 1, abort_v, status, kTimeoutTmaFull));
      if (ok && u >= 1)
        ok = __all_sync(0xffffffffu, wait_phase((kv ? v_empty : k_empty) + s, (u - 1) & 1, abort_v, status, kTimeoutSmemEmpty));
      if (!ok) break;
      const uint8_t* raw = smem + L::kRawOff + re * L::kRaw;
      const uint16_t* words = reinterpret_cast<const uint16_t*>(raw + L::kRawCodes);
      uint8_t* tile = smem + (kv ? L::kVOff : L::kKOff) + s * L::kTile;
      // keys of this warp that read as zeros: past the last one, or in a block that is not there
      const uint32_t gone16 = raw_gone[re] >> (w * 2) & 3u;
      const uint32_t gone = (gone16 & 1u ? 0xffffu : 0u) | (gone16 & 2u ? 0xffff0000u : 0u);
      const int left = kend - j * kBK - w * 32;
      const uint32_t zero = gone | (left >= 32 ? 0u : left <= 0 ? ~0u : ~0u << left);
      uint32_t nan[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 32 / kKps; ++i) {
        const int in_warp = lane / kCpk + i * kKps;
        const uint2 c0 = *reinterpret_cast<const uint2*>(raw + src0 + i * kKps * (HD / 2));
        const uint2 c1 = *reinterpret_cast<const uint2*>(raw + (src0 ^ 8u) + i * kKps * (HD / 2));
        uint32_t sw = words[(key0 + i * kKps) * L::kHalves + half];
        if (zero >> in_warp & 1u) sw = 0;                  // scale 0
        const bool bad = kv && (sw & 0x7f80u) == 0x7f80u;
        if (__any_sync(0xffffffffu, bad)) {                // zeros, and a flag for the rows that see the key
          const uint32_t bit = bad ? 1u << in_warp : 0u;
          nan[0] |= __reduce_or_sync(0xffffffffu, half == 0 ? bit : 0u);
          nan[1] |= __reduce_or_sync(0xffffffffu, half == 1 ? bit : 0u);
          if (bad) sw = 0;
        }
        const uint32_t dup = __byte_perm(sw, 0, 0x1010);
        const uint32_t s2 = dup & 0x7ff07ff0u, z2 = mask_or(dup, 0x000f000fu, 0x43004300u);
        const uint32_t c[4] = {c0.x, c0.y, c1.x, c1.y};
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          uint32_t y[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) y[n] = mul2(sub2(mask_or(c[p] >> (4 * n), 0x000f000fu, 0x43004300u), z2), s2);
          *reinterpret_cast<uint4*>(tile + place[p] + i * kKps * 128) = make_uint4(y[0], y[1], y[2], y[3]);
        }
      }
      // flags of tile j (those of j - 4 are out of use: V of j - 1 was written after PV of j - 3 ended)
      if (lane == 0) {
        TileFlags& f = flags[j & 3];
        if (kv == 0) f.gone[w] = gone;
        else f.nan0[w] = nan[0], f.nan1[w] = nan[1];
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive((kv ? v_full : k_full) + s);
        mbar_arrive(&raw_empty[re]);
      }
    }
  } else if (warp == kCopyWarp) {
    // ---------------- copies ----------------
    const int* table = tables + (int64_t)seq * width;
    int issued[kEntries] = {};
    bool ok = true;
    for (int e = 0; e < 2 * ntiles; ++e) {
      const int j = e >> 1, re = e % kEntries, u = e / kEntries;
      // lane i takes the i-th page that the tile touches; runs are whole 16-key tiles of a page
      const int k0 = j * kBK, last = min(k0 + kBK, (kend + 15) & ~15), page = k0 / bs + lane;
      const int from = max(k0, page * bs), to = min(last, (page + 1) * bs);
      const bool mine = lane < kBK / 16 + 1 && from < to;
      const int blk = mine ? table[page] : 0;
      const bool bad = mine && (blk < 0 || blk >= nblk);
      uint32_t gone = 0;
      if (bad) {
        record_error(status, kBadIndex);
        gone = ((1u << ((to - k0) / 16)) - 1u) & ~((1u << ((from - k0) / 16)) - 1u);
      }
      gone = __reduce_or_sync(0xffffffffu, gone);
      const int keys = mine && !bad ? to - from : 0;
      const int total = __reduce_add_sync(0xffffffffu, keys);
      if (u >= 1) ok = __all_sync(0xffffffffu, wait_phase(&raw_empty[re], (u - 1) & 1, abort_v, status, kTimeoutSmemEmpty));
      if (!ok) break;
      if (lane == 0) {
        raw_gone[re] = gone;                               // published by the arrival below
        mbar_expect_tx(&raw_full[re], (uint32_t)total * (HD / 2 + 2 * L::kHalves));
      }
      __syncwarp();
      if (keys > 0) {
        const Pages& p = e & 1 ? vp : kp;
        const size_t row = ((size_t)blk * nkv + kvh) * bs + (from - page * bs);
        const uint32_t dst = smem_u32(smem) + L::kRawOff + re * L::kRaw;
        bulk_copy(dst + (from - k0) * (HD / 2), p.codes + row * (HD / 2), keys * (HD / 2), &raw_full[re]);
        bulk_copy(dst + L::kRawCodes + (from - k0) * 2 * L::kHalves, p.words + row * L::kHalves, keys * 2 * L::kHalves, &raw_full[re]);
      }
      issued[re] = u + 1;
    }
    // every copy has landed before the block may end
    for (int re = 0; re < kEntries; ++re)
      if (issued[re] > 0) mbar_wait(&raw_full[re], (issued[re] - 1) & 1);
  } else if (warp == kMmaWarp) {
    // ---------------- MMA issuer ----------------
    if (lane == 0 && ntiles > 0) {
      constexpr uint32_t id_s = idesc_f16(kBQ, kBK, false), id_pv = idesc_f16(kBQ, HD, true);
      // descriptors differ in the address field (16-byte units) only
      const uint64_t dq = desc_kmajor(smem_u32(smem)), dk = desc_kmajor(smem_u32(smem + L::kKOff)),
                     dv = desc_mnmajor(smem_u32(smem + L::kVOff), L::kHalf);
      bool ok = wait_phase(q_full, 0, abort_v, status, kTimeoutTmaFull);
      auto issue_s = [&](int t, int j) {
        const int s = j & 1;
        if (!wait_phase(&k_full[s], (j >> 1) & 1, abort_v, status, kTimeoutTmaFull)) return false;
        fence_after();
        const uint64_t qt = dq + t * (L::kTile / 16), kt = dk + s * (L::kTile / 16);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          mma(tmem + t * 128, qt + ((k / 4) * L::kHalf + (k % 4) * 32) / 16, kt + ((k / 4) * L::kHalf + (k % 4) * 32) / 16,
              id_s, k != 0);
        commit(&s_full[t]);
        if (t == 1 || j >= nt[1]) commit(&k_empty[s]);     // the last S that reads this K tile
        return true;
      };
      auto issue_pv = [&](int t, int j) {
        const int s = j & 1;
        if (!wait_phase(&p_half[t], j & 1, abort_v, status, kTimeoutAccum)) return false;
        if (!wait_phase(&v_full[s], (j >> 1) & 1, abort_v, status, kTimeoutTmaFull)) return false;
        const uint64_t vt = dv + s * (L::kTile / 16);
#pragma unroll
        for (int k = 0; k < kBK / 16; ++k) {
          if (k == kBK / 32 && !wait_phase(&p_full[t], j & 1, abort_v, status, kTimeoutAccum)) return false;
          if (k % (kBK / 32) == 0) fence_after();
          mma_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, vt + k * 16 * 128 / 16, id_pv, (j | k) != 0);
        }
        if (t == 1 || j >= nt[1]) commit(&v_empty[s]);
        return true;
      };
      for (int t = 0; ok && t < 2; ++t)
        if (nt[t] > 0) ok = issue_s(t, 0);
      for (int j = 0; ok && j < ntiles; ++j)
        for (int t = 0; ok && t < 2; ++t) {
          if (j < nt[t]) ok = issue_pv(t, j);
          if (ok && j + 1 < nt[t]) ok = issue_s(t, j + 1);
          else if (ok && j + 1 == nt[t]) commit(&s_full[t]);        // one more phase: O is complete
        }
      commit(drain);
      mbar_wait(drain, 0);
    }
    __syncwarp();
  } else {
    // ---------------- softmax ----------------
    const int t = warp >> 2, r = (warp & 3) * 32 + lane;
    const int qi = first + t * per_tile + r / G, head = kvh * G + r % G;
    const bool live = r < per_tile * G && qi < q_len;
    const size_t row = (size_t)(q0 + (live ? qi : 0)) * nh + head;
    // Q rows of this warp into the tile, 8 dims at a time in the order 0 4 1 5 2 6 3 7; rows without a query
    // are zeros
    {
      constexpr int kPieces = HD / 8;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int rr = (warp & 3) * 32 + i * (32 / kPieces) + lane / kPieces, c = lane % kPieces;
        *reinterpret_cast<uint4*>(smem + t * L::kTile + (c / 8) * L::kHalf + rr * 128 + (((c % 8) ^ (rr & 7)) << 4)) =
            make_uint4(__byte_perm(qv[i].x, qv[i].z, 0x5410), __byte_perm(qv[i].x, qv[i].z, 0x7632),
                       __byte_perm(qv[i].y, qv[i].w, 0x5410), __byte_perm(qv[i].y, qv[i].w, 0x7632));
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    // keys this row sees; rows without a query take whatever comes (their result is dropped)
    const int limit = live ? max(0, min(k_cap, shift + qi + 1)) : INT32_MAX;
    const int warp_limit = __reduce_min_sync(0xffffffffu, limit);
    const uint32_t base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tmem_s = tmem + t * 128 + base, tmem_o = tmem + 256 + t * 128 + base;
    float m_used = -INFINITY, l = 0.f;
    bool nan0 = false, nan1 = false, ok = true;
    // NaN groups of V(jj) that this row sees
    auto note_nan = [&](int jj) {
      const TileFlags& f = flags[jj & 3];
      const uint4 a = *reinterpret_cast<const uint4*>(f.nan0), b = *reinterpret_cast<const uint4*>(f.nan1);
      if ((a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w) == 0u) return;
      for (int c = 0; c < 4; ++c) {
        const int n = limit - jj * kBK - c * 32;
        const uint32_t seen = n >= 32 ? ~0u : n <= 0 ? 0u : ~(~0u << n);
        nan0 |= (f.nan0[c] & seen) != 0u;
        nan1 |= (f.nan1[c] & seen) != 0u;
      }
    };
    for (int j = 0; j < nt[t]; ++j) {
      ok = __all_sync(0xffffffffu, wait_phase(&s_full[t], j & 1, abort_v, status, kTimeoutAccum));
      if (!ok) break;
      fence_after();
      const int k0 = j * kBK;
      if (j > 0) note_nan(j - 1);                          // complete: S of this tile was issued after PV of that one
      const uint4 gone = *reinterpret_cast<const uint4*>(flags[j & 3].gone);
      const bool inside = (gone.x | gone.y | gone.z | gone.w) == 0u && k0 + kBK <= warp_limit;
      // keys of chunk c that this row does not see, as a bit mask
      auto hidden = [&](int c) {
        const int n = limit - k0 - c * 32;
        return (n >= 32 ? 0u : n <= 0 ? 0xffffffffu : ~0u << n) | flags[j & 3].gone[c];
      };
      // the next 32 scores are on their way while these are worked on
      uint32_t xa[32], xb[32];
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      auto largest = [&](uint32_t* x, int c) {
        if (!inside) {
          const uint32_t h = hidden(c);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (h >> e & 1u) x[e] = 0xff800000u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          mx4[e / 2 & 3] = max3(mx4[e / 2 & 3], __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
      };
      tmem_ld32(tmem_s, xa);
#pragma unroll 1
      for (int c = 0; c < 4; c += 2) {
        tmem_wait_ld();
        tmem_ld32(tmem_s + c * 32 + 32, xb);
        largest(xa, c);
        tmem_wait_ld();
        tmem_ld32(tmem_s + (c * 32 + 64) % 128, xa);       // at the end: chunk 0 again, for the exponentials
        largest(xb, c + 1);
      }
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2;
      float alpha = 1.f;
      if (mx > m_used + kRescaleLog2) {
        alpha = m_used == -INFINITY ? 0.f : ex2(m_used - mx);
        m_used = mx;
        l *= alpha;
      }
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
        for (int c = 0; c < HD; c += 16) {
          uint32_t o[16];
          tmem_ld16(tmem_o + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st16(tmem_o + c, o);
        }
      }
      const float neg_m = m_used == -INFINITY ? 0.f : -m_used;      // a row that sees nothing: all P = 0
      const uint64_t scale2 = join2(scale_log2, scale_log2), neg2 = join2(neg_m, neg_m);
      uint64_t sum2[2] = {0, 0};
      auto weights = [&](uint32_t* x, int c) {
        if (!inside) {
          const uint32_t h = hidden(c);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (h >> e & 1u) x[e] = 0xff800000u;
        }
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 y = split2(fma_pair(join2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), scale2, neg2));
          const float a = ex2(y.x), b = ex2(y.y);
          sum2[e / 2 & 1] = add_pair(sum2[e / 2 & 1], join2(a, b));
          p[e / 2] = pack2_bf16(a, b);
        }
        tmem_st16(tmem_s + c * 16, p);
      };
#pragma unroll 1
      for (int c = 0; c < 4; c += 2) {
        tmem_wait_ld();
        tmem_ld32(tmem_s + c * 32 + 32, xb);
        weights(xa, c);                                    // P's 16 columns lie in chunks already read
        tmem_wait_ld();
        if (c == 0) tmem_ld32(tmem_s + 64, xa);
        weights(xb, c + 1);
        tmem_wait_st();                                    // half of P is there: its products may start
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive((c == 0 ? p_half : p_full) + t);
      }
      const float2 sum = split2(add_pair(sum2[0], sum2[1]));
      l += sum.x + sum.y;
    }
    // O / l, columns back in order
    const bool done = ok && nt[t] > 0 &&
                      __all_sync(0xffffffffu, wait_phase(&s_full[t], nt[t] & 1, abort_v, status, kTimeoutAccum));
    fence_after();
    uint4* dst = reinterpret_cast<uint4*>(out + row * HD);
    if (done) {
      note_nan(nt[t] - 1);
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int c = 0; c < HD; c += 16) {
        const float i = (c < 64 ? nan0 : nan1) ? __uint_as_float(0x7fc00000u) : inv;
        uint32_t o[16];
        tmem_ld16(tmem_o + c, o);
        tmem_wait_ld();
        if (live)
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            auto v = [&](int d) { return __uint_as_float(o[e + d]) * i; };      // column d holds dim (0 4 1 5 2 6 3 7)[d]
            dst[(c + e) / 8] = make_uint4(pack2_bf16(v(0), v(2)), pack2_bf16(v(4), v(6)), pack2_bf16(v(1), v(3)),
                                          pack2_bf16(v(5), v(7)));
          }
      }
    } else if (live && nt[t] == 0) {
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) dst[c] = make_uint4(0, 0, 0, 0);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

}  // namespace

void prefill_attention_int4(at::Tensor out, at::Tensor q, at::Tensor kc, at::Tensor kw, at::Tensor vc, at::Tensor vw,
                            at::Tensor cu_q, at::Tensor k_lens, at::Tensor tables, double scale, int64_t max_q,
                            at::Tensor status) {
  const at::Device dev = q.device();
  check_page_pair(kc, kw, vc, vw, dev);
  LSB_INT4_CHECK(q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.is_contiguous() &&
                     reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
                 "q must be contiguous, 16-byte aligned bfloat16 [rows, heads, head_dim]");
  const int64_t T = q.size(0), nh = q.size(1), hd = q.size(2), nkv = kc.size(1), bs = kc.size(2);
  LSB_INT4_CHECK(hd == kc.size(3) * 2 && nh >= 1 && nh % nkv == 0, "query heads do not match the pages");
  LSB_INT4_CHECK(nh / nkv <= kBQ, "more than 128 query heads per KV head");
  LSB_INT4_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.is_contiguous() &&
                     out.device() == dev, "bad output");
  check_int32(k_lens, "sequence lengths", 1, dev);
  check_int32(tables, "block_tables", 2, dev);
  check_int32(cu_q, "cu_seqlens_q", 1, dev);
  const int64_t B = k_lens.size(0);
  LSB_INT4_CHECK(tables.size(0) >= B, "block_tables must hold one row per sequence");
  LSB_INT4_CHECK(cu_q.size(0) == B + 1, "cu_seqlens_q must hold one entry more than there are sequences");
  const float factor = scale_log2(scale, 1);
  LSB_INT4_CHECK(kc.numel() / (hd / 2) / 16 < INT32_MAX && T < INT32_MAX, "pages exceed int32 rows of 16 keys");
  if (T == 0 || B == 0 || max_q <= 0) return;
  const at::cuda::CUDAGuard guard(dev);
  // pairs of tiles: every sequence ends one early, and none is longer than max_q
  const int64_t per = 2 * (kBQ / (nh / nkv));
  const int64_t pairs = std::min(T / per + B, (std::min(max_q, T) + per - 1) / per * B);
  LSB_INT4_CHECK(pairs * nkv < INT32_MAX, "too many query tiles for one launch");
  auto go = [&](auto kern, int smem) {
    ensure_dynamic_smem((const void*)kern, smem);
    launch_pdl(kern, dim3((unsigned)(pairs * nkv)), dim3(kThreads), smem, at::cuda::getCurrentCUDAStream(),
               (bf16*)out.data_ptr(), (const bf16*)q.data_ptr(), Pages{kc.data_ptr<uint8_t>(), kw.data_ptr<int16_t>()},
               Pages{vc.data_ptr<uint8_t>(), vw.data_ptr<int16_t>()}, (const int*)cu_q.data_ptr<int>(),
               (const int*)k_lens.data_ptr<int>(), (const int*)tables.data_ptr<int>(), (int)tables.size(1), (int)B, (int)T,
               (int)std::min(max_q, T), factor, (int)nh, (int)nkv, (int)bs,
               (int)kc.size(0), status_ptr(status));
  };
  if (hd == 128) go(prefill_int4_kernel<128>, PfLayout<128>::kBytes);
  else go(prefill_int4_kernel<64>, PfLayout<64>::kBytes);
  const cudaError_t e = cudaGetLastError();
  LSB_INT4_CHECK(e == cudaSuccess, std::string("prefill_attention_int4 launch failed: ") + cudaGetErrorString(e));
}

}  // namespace lsb
