// Attention of new tokens over a paged K/V cache: out = softmax(scale * q k^T) v and lse, keys and values read where they lie.
//
// The query heads that share a K/V head and the new tokens of a sequence are the rows of one product, so that a key is read
// once for all of them: rows r = token * G + head of the group.
//
// paged_attn_few: bound by memory (each byte of the cache feeds as many multiply-adds as there are rows).
//   work       : a unit is 128 (or 64) keys of one (sequence, K/V head, tile of rows).  The units of all sequences, counted by every
//                workgroup from the lengths in device memory, are dealt out evenly and in order to one workgroup per CU: a
//                long sequence beside short ones, or alone, keeps all CUs reading, without the host knowing a length.  A
//                workgroup whose share ends inside an item leaves a partial result, and paged_attn_join adds those up.
//   wavefront  : every fourth (second) tile of 32 keys is its own, in a ring of LDS filled by copies that do not pass through
//                registers (buffer_load ... lds) nor stay in the caches (a key is read once): no barrier in the loop, and 64
//                to 128 KB in flight on a CU, where 25 bytes a nanosecond times the latency of a microsecond asks for 25 KB.
//   S^T = K Q^T: v_mfma_f32_16x16x32_bf16 with A = K rows from LDS and B = Q rows in registers: lane (ln, lg) then holds
//                keys 4 lg .. +3 of both halves of a tile for row ln, softmax is lane-local but for two exchanges.
//   O^T = V^T P^T: the same lane's P is the B operand, and the transposing LDS reads fetch V^T in its key order.
//   e4m3       : codes are exact in bf16 (v_cvt_scalef32_pk_bf16_fp8); a key's scale multiplies its score, a value's scale
//                its weight, in fp32.  The weights go to the product as bf16 (off by 2^-8 of each at most), up to 16 rows as
//                two bf16 numbers (2^-14); there is no other rounding below 32 bits before the last.
#include "paged_attn.hpp"

namespace mhip {
namespace {

typedef __attribute__((__vector_size__(2 * sizeof(int)))) int i32x2;

constexpr int kKeys = 32;                  // keys of a tile, one wavefront's
// Bytes of K and V tiles of a wavefront, of which a CU has 128 KB: four wavefronts of them, or eight of half as much.  Eight where there are
// registers for two on a SIMD and half as much still holds two tiles: up to 16 rows, of up to 128 bytes.  us, four / eight wavefronts:
// e4m3 64 x 100 .. 2048 H32/8 43.4 / 35.9, 32 x 300 .. 16384 111.1 / 102.3, 16 x 5 tokens at 211 .. 4099 H16/8 D80 29.1 / 24.4, 4 x 131072
// 180.6 / 181.2; bf16 D64 64 x 100 .. 2048 35.5 / 31.5, 32 x 300 .. 16384 96.5 / 94.4, 16 x 5 23.4 / 21.7, 8 x 8192 H16/2 15.3 / 15.6.
template <bool E4M3, int COLS, int NR>
constexpr int kRingOf = NR == 1 && COLS * (E4M3 ? 1 : 2) <= 128 ? 16384 : 32768;
constexpr int kNoColumn = 0x7fff0000;      // vector offset out of every descriptor's range (spans stay below 2^30)
constexpr int kWavefronts = 1024;          // of a launch with rings of 32 KB: four on a CU, in workgroups of four or two
constexpr int kFewRows = 64;               // rows of a sequence and K/V head that paged_attn_few takes, else paged_attn_chunk

// Row tiles of a sequence and K/V head, units of each, and what an item counts for: its units behind `pause` more, the time in which a
// workgroup that enters it does not read.  Without it a workgroup with many short items ends last; where there are fewer items than
// workgroups it would only spoil even shares.  us, 0 / 1 / 2 / 3 units (e4m3 with four wavefronts on a CU): 64 x 20 .. 1024 H32/8 48.6 / 35.5
// / 31.6 / 32.0, 64 x 100 .. 2048 63.1 / 55.8 / 55.2 / 54.0 (e4m3 56.2 / 49.8 / 43.7 / 42.0), 256 x 20 .. 512 72.1 / 62.4 / 54.8 / 53.4,
// 32 x 300 .. 16384 203.0 / 202.6 / 203.9 / 207.1; 8 tokens at 32768 34.4 / 35.8 / 35.7 / 35.8.  With eight wavefronts, 1 / 2 / 3 units: e4m3
// 256 x 20 .. 512 44.5 / 40.9 / 42.1, 64 x 100 .. 2048 37.2 / 36.2 / 36.3.
struct Item { int rts, steps, weight; };
template <int UNIT>
constexpr int kPauseOf = UNIT == 2 * kKeys ? 2 : 0;
template <int ROWS, int UNIT>
__device__ __forceinline__ Item item_of(const PagedAttn& p, const PagedSeq& s) {
  Item it;
  it.rts = s.n * p.G <= p.few_rows ? (s.n * p.G + ROWS - 1) / ROWS : 0;
  it.steps = s.len > UNIT ? (s.len + UNIT - 1) / UNIT : 1;
  it.weight = it.steps + kPauseOf<UNIT>;
  return it;
}
template <int ROWS, int UNIT>
__device__ __forceinline__ int64_t units_of(const PagedAttn& p, const PagedSeq& s) {
  const Item it = item_of<ROWS, UNIT>(p, s);
  return (int64_t)it.weight * it.rts * p.Hkv;
}

// The units before each lane's run of sequences, and of all of them.
struct Plan {
  int per;                   // sequences of a lane
  PagedSeq last;             // and the last of them
  int64_t before, mine, total;
};
template <int ROWS, int UNIT>
__device__ __forceinline__ Plan plan_of(const PagedAttn& p, int lane) {
  Plan plan;
  plan.per = (p.g.B + 63) / 64;
  plan.last = PagedSeq{};
  plan.mine = 0;
  for (int j = 0; j < plan.per; ++j)
    if (lane * plan.per + j < p.g.B) {
      plan.last = paged_seq<false>(p.g, lane * plan.per + j);
      plan.mine += units_of<ROWS, UNIT>(p, plan.last);
    }
  int64_t sum = plan.mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t below = __shfl_up((long long)sum, off);
    if (lane >= off) sum += below;
  }
  plan.before = sum - plan.mine;
  plan.total = __shfl((long long)sum, 63);
  return plan;
}
template <int ROWB>
__device__ __forceinline__ int swizzle(int row) {      // of the 16-byte chunks of LDS rows of ROWB bytes
  return ROWB == 256 ? lds_row_swizzle_16(row) : ROWB == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
}

template <bool E4M3, int COLS, int NR, int WAVES>
__global__ __launch_bounds__(WAVES * 64, (32768 / kRingOf<E4M3, COLS, NR>)) void paged_attn_few(const PagedAttn p) {
  constexpr int ROWS = 16 * NR, UNIT = WAVES * kKeys, kPause = kPauseOf<UNIT>;
  constexpr int kSize = E4M3 ? 1 : 2;
  constexpr int ROWB = COLS * kSize;                   // bytes of a row in LDS
  constexpr int kChunks = ROWB / 16;
  constexpr int kCopyRows = 1024 / ROWB;               // rows of one copy instruction
  constexpr int kCopies = 16 / kCopyRows;              // and instructions of half a tile
  constexpr int kTileBytes = kKeys * ROWB;
  constexpr int kStages = kRingOf<E4M3, COLS, NR> / (2 * kTileBytes);
  constexpr int kStage = 2 * kTileBytes + (E4M3 ? 256 : 0);      // K, V, 32 scales of each
  constexpr int nK = 2 * kCopies + (E4M3 ? 1 : 0), nV = 2 * kCopies;
  constexpr int KB = COLS / 32, DB = COLS / 16;
  constexpr int kPair = NR < 2 ? NR : 2;               // blocks of rows that are worked on together
  // Weights to 14 bits and more of their mantissa, in two products, where that costs next to nothing: up to 16 rows (32 sequences of 300 .. 16384
  // bf16 177.8 us and 177.8, e4m3 102.3 and 103.3).  With more rows the matrix instructions show, and weights are rounded to bf16 once.
  constexpr bool kTwice = NR == 1;
  constexpr int kRegion = kStages * kStage;
  static_assert(ROWS * COLS * 4 <= kRegion, "a wavefront's O takes the place of its ring");
  static_assert(kStages * (nK + nV) < 64, "copies in flight are counted in 6 bits");
  __shared__ __attribute__((aligned(16))) unsigned char smem[WAVES * kRegion];
  __shared__ f32x2 stats[WAVES][ROWS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, lg = lane >> 4;

  // ---- this workgroup's share ------------------------------------------------------------------------------
  // (workgroups of one XCD take neighbouring shares)
  const int w = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const Plan plan = plan_of<ROWS, UNIT>(p, lane);
  const int64_t total = uniform64(plan.total);
  const int64_t shares = total < (int64_t)gridDim.x ? total : gridDim.x;
  if (w >= shares) {
    if (threadIdx.x == 0 && !p.by_item) p.shared[w].rows = 0;
    return;
  }
  bool leaves = false;                                 // an item that begins here and ends elsewhere
  int64_t lo = total * w / shares;
  const int64_t hi = total * (w + 1) / shares;
  const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lo >= plan.before && lo < plan.before + plan.mine));
  int b = owner * plan.per;
  int64_t pos = lo - uniform64(__shfl((long long)plan.before, owner));     // inside sequence b
  // (up to 64 sequences are a lane's each, which need not be read once more)
  PagedSeq s{__builtin_amdgcn_readlane(plan.last.start, owner), __builtin_amdgcn_readlane(plan.last.n, owner),
             __builtin_amdgcn_readlane(plan.last.len, owner)};
  if (plan.per > 1) {
    for (int64_t u; b + 1 < p.g.B && pos >= (u = units_of<ROWS, UNIT>(p, paged_seq<true>(p.g, b))); ++b) pos -= u;
    s = paged_seq<true>(p.g, b);
  }

  // ---- what does not change from segment to segment -----------------------------------------------------------
  const uint32_t lds_smem = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const uint32_t ring = lds_smem + wave * kRegion;
  int voff[kCopies];
#pragma unroll
  for (int u = 0; u < kCopies; ++u) {
    const int row = u * kCopyRows + lane / kChunks, chunk = (lane % kChunks) ^ swizzle<ROWB>(row);
    voff[u] = chunk * 16 < p.D * kSize ? row * (int)p.c_ss16 * 16 + chunk * 16 : kNoColumn;
  }
  // K operand: 16 bytes of row ln; in e4m3 they serve two k-steps of 32 columns
  constexpr int KR = E4M3 ? KB / 2 : KB;               // 16-byte reads of a K row
  int k_a[KR];
#pragma unroll
  for (int i = 0; i < KR; ++i) k_a[i] = (int)ring + ln * ROWB + (((4 * i + lg) ^ swizzle<ROWB>(ln)) << 4);
  // V^T operand: keys 4 lg .. +3 of both halves of the tile, one column of a strip of 16 per lane.  bf16: within 16 lanes lane s
  // supplies the address of columns 4 (s % 4) .. +3 of row s / 4 and receives column s; e4m3: of columns 8 (s % 2) .. +7 of row s / 2.
  int v_a[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    if (E4M3) {
      const int r8 = ln >> 1, row = (r8 & 3) + 4 * lg + 16 * (r8 >> 2);
      v_a[db] = (int)ring + kTileBytes + row * ROWB + ((db ^ swizzle<ROWB>(row & 15)) << 4) + (ln & 1) * 8;
    } else {
      const int row = 4 * lg + (ln >> 2);
      v_a[db] = (int)ring + kTileBytes + row * ROWB + (((2 * db + ((ln & 3) >> 1)) ^ swizzle<ROWB>(row)) << 4) + (ln & 1) * 8;
    }
  }
  typedef __attribute__((address_space(3))) bf16x4* lds_bf16x4;
  typedef __attribute__((address_space(3))) i32x2* lds_i32x2;
  typedef __attribute__((address_space(3))) const u32x4* lds_u32x4;
  typedef __attribute__((address_space(3))) const f32x4* lds_f32x4;
  auto codes_to_bf16 = [](uint32_t a, uint32_t c) -> bf16x8 {
    const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false), x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true);
    const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, false), x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, true);
    return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
  };
  auto read_v = [&](int db, int stage_at) -> bf16x8 {
    if constexpr (E4M3) {
      const i32x2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2)(uintptr_t)(uint32_t)(v_a[db] + stage_at));
      return codes_to_bf16((uint32_t)c[0], (uint32_t)c[1]);
    } else {
      const bf16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4)(uintptr_t)(uint32_t)(v_a[db] + stage_at));
      const bf16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4)(uintptr_t)(uint32_t)(v_a[db] + stage_at + 16 * ROWB));
      return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  };
  auto mfma = [](const bf16x8& x, const bf16x8& y, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0); };

  for (;;) {
    const Item it = item_of<ROWS, UNIT>(p, s);
    const int64_t item = pos / it.weight;
    const int from = (int)(pos - item * it.weight);
    const int take = (int)(it.weight - from < hi - lo ? it.weight - from : hi - lo);
    const int first = from > kPause ? from - kPause : 0, count = from + take > kPause ? from + take - kPause - first : 0;
    const int64_t start = lo - from;                   // of the item
    lo += take;
    pos += take;
    if (count > 0) {
    const int hk = (int)(item / it.rts), rt = (int)(item - (int64_t)hk * it.rts);
    const int row0 = rt * ROWS;
    const int rows = s.n * p.G - row0 < ROWS ? s.n * p.G - row0 : ROWS;

    // ---- Q rows: B operand of S^T, lane (ln, lg) holds 8 columns of row ln, in the order of the K operand's ----------
    bf16x8 qf[NR][KB];
    int lim[NR];                                       // keys that the row sees
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int row = r * 16 + ln;
      int of_group;
      const int token = p.by_group.quotient(row0 + (row < rows ? row : 0), of_group);
      const uint16_t* src = p.q + b * p.q_sb + (int64_t)(s.start + token) * p.q_ss + (hk * p.G + of_group) * p.q_sh;
      lim[r] = p.causal ? clamped(s.len - s.n + token + 1, 0, s.len) : s.len;
#pragma unroll
      for (int ks = 0; ks < KB; ++ks) {
        const int col = E4M3 ? (ks >> 1) * 64 + lg * 16 + (ks & 1) * 8 : ks * 32 + lg * 8;
        qf[r][ks] = bf16x8{};
        if (row < rows && col < p.D) qf[r][ks] = *reinterpret_cast<const bf16x8*>(src + col);
      }
    }
    // keys that all rows see, and that some row sees
    auto sees = [&](int row) {
      return __builtin_amdgcn_readfirstlane(p.causal ? clamped(s.len - s.n + p.by_group.quotient(row) + 1, 0, s.len) : s.len);
    };
    const int seen_first = sees(row0), seen_last = sees(row0 + rows - 1);

    // ---- copies of tile t of this wavefront, 16 keys (of one page) at a time -----------------------------------------
    const int* table = p.g.table + b * p.g.t_sb;
    auto key_of = [&](int t) { return ((first + t) * WAVES + wave) * kKeys; };
    int page[2], slot[2], held[2];                     // of the tile whose copies go out next
    auto look_up = [&](int t) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = key_of(t) + 16 * h;
        held[h] = t < count ? clamped(seen_last - key, 0, 16) : 0;
        page[h] = -1;
        slot[h] = 0;
        if (held[h] > 0) page[h] = uniform_load(table, p.g.by_page.quotient(key, slot[h]));
      }
    };
    uint32_t gone = 0;                                 // two bits of each stage: that half of its tile is not here
    auto settle = [&](int stage) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool here = page[h] >= 0 && page[h] < p.g.pages;
        if (!here) held[h] = 0;
        gone = (gone & ~(1u << (2 * stage + h))) | (here ? 0u : 1u << (2 * stage + h));
      }
    };
    auto copy = [&](const uint8_t* base, int at) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* from = base + (held[h] > 0 ? row_offset(p, page[h], slot[h]) + hk * p.c_sh : 0);
        const u32x4 rs = rsrc_words(from, held[h] > 0 ? (uint32_t)((held[h] - 1) * (int)p.c_ss16 * 16 + p.D * kSize) : 0u);
#pragma unroll
        for (int u = 0; u < kCopies; ++u) copy16_once_to_lds(rs, ring + at + h * 16 * ROWB + u * 1024, voff[u], 0);
      }
    };
    auto copy_k = [&](int stage) {
      if constexpr (E4M3) {
        const int h = (lane >> 4) & 1, row = ln < held[h] ? ln : held[h] - 1;
        const float* at = (lane >> 5 ? p.v_scales : p.k_scales) + (page[h] * p.s_sp + (slot[h] + row) * p.s_ss + hk * p.s_sh);
        copy4_to_lds(held[h] > 0 ? static_cast<const void*>(at) : p.q, ring + stage * kStage + 2 * kTileBytes);
      }
      copy(p.k, stage * kStage);
    };
    auto copy_v = [&](int stage) { copy(p.v, stage * kStage + kTileBytes); };

    f32x4 o[DB][NR];
    float m[NR], l[NR];                                // maximum (times scale * log2 e), this lane's share of the sum
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db][r] = f32x4{};
    }
    look_up(0);                                        // (on its way with Q)
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int ks = 0; ks < KB; ++ks) asm volatile("" : "+v"(qf[r][ks]));      // loaded before the first copy goes out
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int t = 0; t < kStages; ++t) {
      if (t > 0) look_up(t);
      settle(t);
      copy_k(t);
      copy_v(t);
    }
    look_up(kStages);

    auto weigh = [&](int db, int r, const bf16x8& vf, const u32x4& high, const u32x4& low) __attribute__((always_inline)) {
      o[db][r] = mfma(vf, __builtin_bit_cast(bf16x8, high), o[db][r]);
      if (kTwice) o[db][r] = mfma(vf, __builtin_bit_cast(bf16x8, low), o[db][r]);
    };
    for (int t = 0; t < count; ++t) {
      const int stage = t % kStages, at = stage * kStage, key0 = key_of(t);
      const uint32_t hidden = gone >> (2 * stage) & 3u;
      asm volatile("s_waitcnt vmcnt(%0)" :: "n"(nV + (kStages - 1) * (nK + nV)) : "memory");     // K of tile t is there
      const bool cut = key0 + kKeys > seen_first;                // some row does not see some key
      f32x4 k_scale[2], v_scale[2];
      // Two blocks of rows at a time: with all four of 64 rows the registers run out.  The second time K and V are read from LDS again.
#pragma unroll
      for (int r0 = 0; r0 < NR; r0 += kPair) {
        f32x4 sc[2][kPair];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < KR; ++i) {
            const u32x4 w = *(lds_u32x4)(uintptr_t)(uint32_t)(k_a[i] + at + kb * 16 * ROWB);
#pragma unroll
            for (int e = 0; e < KB / KR; ++e) {
              const bf16x8 kf = E4M3 ? codes_to_bf16(w[2 * e], w[2 * e + 1]) : __builtin_bit_cast(bf16x8, w);
              const int ks = E4M3 ? 2 * i + e : i;
#pragma unroll
              for (int r = 0; r < kPair; ++r) sc[kb][r] = mfma(kf, qf[r0 + r][ks], ks == 0 ? f32x4{} : sc[kb][r]);
            }
          }
        if (E4M3 && r0 == 0)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            k_scale[kb] = *(lds_f32x4)(uintptr_t)(uint32_t)(ring + at + 2 * kTileBytes + kb * 64 + lg * 16);
            v_scale[kb] = *(lds_f32x4)(uintptr_t)(uint32_t)(ring + at + 2 * kTileBytes + 128 + kb * 64 + lg * 16);
            asm volatile("" : "+v"(k_scale[kb]), "+v"(v_scale[kb]));
          }
        if (r0 + kPair >= NR) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // the tile has been read: its place can be filled
          settle(stage);
          copy_k(stage);
        }

        // ---- softmax --------------------------------------------------------------------------------------------
        u32x4 pw[kPair], pl[kPair];                              // weights in bf16, and what that leaves of them
        bool moved = false;
        float alpha[kPair];
#pragma unroll
        for (int r = 0; r < kPair; ++r) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[kb][r][j] *= E4M3 ? p.scale_log2 * k_scale[kb][j] : p.scale_log2;
          if (cut || hidden) {
            asm volatile("");
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              const int left = hidden >> kb & 1 ? 0 : lim[r0 + r] - (key0 + 16 * kb) - 4 * lg;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (j >= left) sc[kb][r][j] = -INFINITY;
            }
          }
          float top = sc[0][r][0];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, sc[kb][r][j]);
          top = fmaxf(quad_max(top), m[r0 + r]);
          const float ref = top == -INFINITY ? 0.f : top;
          alpha[r] = fast_exp2(m[r0 + r] - ref);
          moved = moved || !(m[r0 + r] == top);
          m[r0 + r] = top;
          float x[8], sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = fast_exp2(sc[i >> 2][r][i & 3] - ref);
            sum += x[i];
            // (a masked key's scale may be anything; a NaN of one that the row sees counts however small its weight is)
            if constexpr (E4M3) x[i] = sc[i >> 2][r][i & 3] == -INFINITY ? 0.f : x[i] * v_scale[i >> 2][i & 3];
          }
          l[r0 + r] = l[r0 + r] * alpha[r] + sum;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (kTwice) {
              // (cut off, not rounded, and the rest a little large: both have the weight's sign and are zero only with it, so that
              // infinite values stay what they are)
              pw[r][i] = __builtin_amdgcn_perm(__float_as_uint(x[2 * i + 1]), __float_as_uint(x[2 * i]), 0x07060302u);
              pl[r][i] = pack_bf16(__builtin_fmaf(x[2 * i], 0x1.00004p0f, -bf16_lo(pw[r][i])),
                                   __builtin_fmaf(x[2 * i + 1], 0x1.00004p0f, -bf16_hi(pw[r][i])));
            } else {
              pw[r][i] = pack_bf16(x[2 * i], x[2 * i + 1]);
            }
          }
        }
        if (__builtin_amdgcn_ballot_w64(moved) != 0) {
#pragma unroll
          for (int r = 0; r < kPair; ++r)
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db][r0 + r] *= alpha[r];
        }

        // ---- O^T += V^T P^T ---------------------------------------------------------------------------------------
        if (r0 == 0)                                             // V of tile t is there
          asm volatile("s_waitcnt vmcnt(%0)" :: "n"((NR <= kPair ? nK : 0) + (kStages - 1) * (nK + nV)) : "memory");
        if (!(cut && seen_first < seen_last)) {
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const bf16x8 vf = read_v(db, at);
#pragma unroll
            for (int r = 0; r < kPair; ++r) weigh(db, r0 + r, vf, pw[r], pl[r]);
          }
        } else {
          // (some rows do not see some of the keys: see finite_part)
          uint32_t odd = 0;
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const bf16x8 vf = __builtin_bit_cast(bf16x8, finite_part(__builtin_bit_cast(u32x4, read_v(db, at)), odd));
#pragma unroll
            for (int r = 0; r < kPair; ++r) weigh(db, r0 + r, vf, pw[r], pl[r]);
            __builtin_amdgcn_sched_barrier(0);
          }
          if (__builtin_amdgcn_ballot_w64(odd != 0) != 0) {
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              const bf16x8 marks = __builtin_bit_cast(bf16x8, odd_marks(__builtin_bit_cast(u32x4, read_v(db, at))));
#pragma unroll
              for (int r = 0; r < kPair; ++r) {
                int left[2];
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) left[kb] = hidden >> kb & 1 ? 0 : lim[r0 + r] - (key0 + 16 * kb) - 4 * lg;
                const f32x4 counts = mfma(marks, __builtin_bit_cast(bf16x8, seen_marks(left[0], left[1])), f32x4{});
#pragma unroll
                for (int j = 0; j < 4; ++j) o[db][r0 + r][j] = with_odd(o[db][r0 + r][j], counts[j]);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
        if (NR > kPair) __builtin_amdgcn_sched_barrier(0);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      copy_v(stage);
      look_up(t + kStages + 1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // copies past the last tile

    // ---- the wavefronts' shares meet -------------------------------------------------------------------------------
    unsigned char* region = smem + wave * kRegion;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float sum = quad_sum(l[r]);
      if (lg == 0) stats[wave][r * 16 + ln] = f32x2{m[r], sum};
#pragma unroll
      for (int db = 0; db < DB; ++db)
        *reinterpret_cast<f32x4*>(region + (r * 16 + ln) * (COLS * 4) + (((db * 4 + lg) ^ ln) << 4)) = o[db][r];
    }
    __syncthreads();
    const bool whole = count == it.steps;
    const int64_t slot_of = 2 * (int64_t)w + (first == 0 ? 1 : 0);
    if (first == 0) {
      leaves = leaves || !whole;
      if (threadIdx.x == 0 && (p.by_item || !whole)) {
        const int last = (int)(((start + it.weight) * shares - 1) / total);        // the workgroup with its last unit
        const int64_t at = p.by_item ? (int64_t)b * it.rts * p.Hkv + item : w;
        p.shared[at] = Shared{b, hk, row0, whole ? 0 : rows, last - w + 1, 2 * w + 1, 2 * (w + 1), 2};
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS * COLS / 4 / (WAVES * 64); ++i) {
      const int unit = i * (WAVES * 64) + threadIdx.x;
      const int row = unit / (COLS / 4), c4 = unit % (COLS / 4);
      if (row >= rows) continue;
      f32x2 st[WAVES];
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) {
        st[v] = stats[v][row];
        top = fmaxf(top, st[v][0]);
      }
      const float ref = top == -INFINITY ? 0.f : top;
      f32x4 acc{};
#pragma unroll
      for (int v = 0; v < WAVES; ++v) {
        const float weight = fast_exp2(st[v][0] - ref);
        sum += st[v][1] * weight;
        acc += *reinterpret_cast<const f32x4*>(smem + v * kRegion + row * (COLS * 4) + ((c4 ^ (row & 15)) << 4)) * weight;
      }
      if (whole) {
        int of_group;
        const int token = s.start + p.by_group.quotient(row0 + row, of_group), head = hk * p.G + of_group;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if (c4 * 4 < p.D)
          *reinterpret_cast<u32x2*>(p.out + b * p.o_sb + (int64_t)token * p.o_ss + head * p.o_sh + c4 * 4) =
              u32x2{pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv)};
        if (c4 == 0) p.lse[b * p.l_sb + head * p.l_sh + token] = sum == 0.f ? -INFINITY : (top + fast_log2(sum)) * kLn2;
      } else {
        *reinterpret_cast<f32x4*>(p.part_o + (slot_of * ROWS + row) * COLS + c4 * 4) = acc;
        if (c4 == 0) p.part_ml[slot_of * ROWS + row] = f32x2{top, sum};
      }
    }

    if (lo < hi) __syncthreads();
    }
    if (lo >= hi) break;
    if (pos >= (int64_t)it.weight * it.rts * p.Hkv) {
      pos = 0;
      for (++b; b + 1 < p.g.B && units_of<ROWS, UNIT>(p, paged_seq<true>(p.g, b)) == 0;) ++b;
      s = paged_seq<true>(p.g, b);
    }
  }
  if (!leaves && threadIdx.x == 0 && !p.by_item) p.shared[w].rows = 0;
}

// Tiles of 16, 32 or 64 rows: the least that holds the rows of a sequence with `most` new tokens.
int row_blocks(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
// Workgroups of four wavefronts, one to a CU, or of two, two to a CU: the pair covers the one's pauses between items (Q, the first tiles,
// the wavefronts' results) with the other's reading, and costs twice as many partial results.  Items to a workgroup decide; us, four / two:
//   items   8: 1 x 131072 H32/8 88.0 / 89.4, e4m3 57.5 / 61.2, 8 tokens at 32768 33.1 / 37.8    16: 8 x 8192 H16/2 D64 e4m3 16.9 / 20.8
//          32: 4 x 131072 H32/8 e4m3 180.7 / 182.7    128: 16 x 5 tokens at 211 .. 4099 H16/8 D80 36.4 / 27.1, e4m3 26.4 / 24.4
//         256: 32 x 300 .. 16384 H32/8 177.9 / 177.5    512: 64 x 100 .. 2048 H32/8 64.8 / 54.1, e4m3 49.7 / 35.3
//        2048: 256 x 20 .. 512 H32/8 84.1 / 55.5, e4m3 63.9 / 40.7
// (twice as many of either where kRingOf halves the rings)
constexpr int64_t kManyItems = 128;

// One partial result at each end of a workgroup's share.
int64_t few_bytes(int64_t rows, int D) { return 2 * kWavefronts * (16 * (int64_t)row_blocks(rows) * ((D <= 64 ? 64 : 128) + 2) * 4 + 16); }

template <bool E4M3, int COLS, int NR, int WAVES>
void launch_few(PagedAttn p, int64_t rows, hipStream_t st) {
  constexpr int workgroups = kWavefronts * (32768 / kRingOf<E4M3, COLS, NR>) / WAVES;
  p.part_ml = reinterpret_cast<f32x2*>(p.part_o + 2 * (int64_t)workgroups * 16 * NR * COLS);
  p.shared = reinterpret_cast<Shared*>(p.part_ml + 2 * (int64_t)workgroups * 16 * NR);
  // Where the items are known and not more than the workgroups, the last step has one row of workgroups for each of them, not for
  // each workgroup that one might begin in (8 items of 32 rows: 34.1 us instead of 39.7, of which launching 2048 workgroups was 5).
  const int64_t items = (int64_t)p.g.B * p.Hkv * ((rows + 16 * NR - 1) / (16 * NR));
  p.by_item = !p.g.starts && items <= workgroups;
  const int blocks = !p.g.starts && rows < 16 * NR ? (int)((rows + 3) / 4) : 4 * NR;       // (packed, `rows` is a hint)
  hipLaunchKernelGGL((paged_attn_few<E4M3, COLS, NR, WAVES>), dim3(workgroups), dim3(WAVES * 64), 0, st, p);
  hipLaunchKernelGGL((paged_attn_join<COLS, 16 * NR, 1, 4>), dim3(blocks, p.by_item ? (int)items : workgroups), dim3(256), 0, st, p);
}
template <bool E4M3, int COLS, int NR>
void launch_few(const PagedAttn& p, int64_t rows, hipStream_t st) {
  if ((int64_t)p.g.B * p.Hkv >= kManyItems) launch_few<E4M3, COLS, NR, 2>(p, rows, st);
  else launch_few<E4M3, COLS, NR, 4>(p, rows, st);
}
template <bool E4M3, int COLS>
void launch_rows(const PagedAttn& p, int64_t rows, hipStream_t st) {
  const int blocks = row_blocks(rows);
  if (blocks == 1) launch_few<E4M3, COLS, 1>(p, rows, st);
  else if (blocks == 2) launch_few<E4M3, COLS, 2>(p, rows, st);
  else launch_few<E4M3, COLS, 4>(p, rows, st);
}
void launch(const PagedAttn& p, bool e4m3, int64_t rows, hipStream_t st) {
  if (e4m3) {
    if (p.D <= 64) launch_rows<true, 64>(p, rows, st);
    else launch_rows<true, 128>(p, rows, st);
  } else {
    if (p.D <= 64) launch_rows<false, 64>(p, rows, st);
    else launch_rows<false, 128>(p, rows, st);
  }
}

}  // namespace
}  // namespace mhip

using namespace mhip;

extern "C" int64_t mhip_paged_attn_workspace_bytes(int B, int n, int T, int most_new, int packed, int Hq, int Hkv, int D) {
  if (B < 0 || n < 0 || T < 0 || most_new < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return MHIP_EINVAL;
  if (D <= 0 || D > 128) return MHIP_EHEADDIM;
  const int64_t rows = (int64_t)(packed ? most_new : n) * (Hq / Hkv), few = few_bytes(rows, D);
  const int64_t chunk = rows > kFewRows ? paged_attn_chunk_bytes(B, n, T, Hq / Hkv, Hkv, D, packed != 0) : 0;
  return few > chunk ? few : chunk;
}

extern "C" int mhip_paged_attn_fwd(const void* q, const void* k_cache, const void* v_cache, const float* k_scales, const float* v_scales,
                                   const int* page_table, const int* lengths, const int* starts, void* out, float* lse,
                                   int B, int n, int T, int most_new, int Hq, int Hkv, int D, int pages, int page_size, int table_pages,
                                   int64_t t_sb, int64_t q_sb, int64_t q_ss, int64_t q_sh,
                                   int64_t c_sp, int64_t c_ss, int64_t c_sh, int64_t s_sp, int64_t s_ss, int64_t s_sh,
                                   int64_t o_sb, int64_t o_ss, int64_t o_sh,
                                   float softmax_scale, int mask, int dtype, void* workspace, void* stream) {
  PagedAttn p{};
  if (B < 0 || n < 0 || T < 0 || most_new < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return MHIP_EINVAL;
  if (!(softmax_scale > 0.f) || !(softmax_scale < INFINITY)) return MHIP_EINVAL;
  if (mask != MHIP_MASK_NONE && mask != MHIP_MASK_CAUSAL) return MHIP_EINVAL;
  if (!starts && (int64_t)B * n > 0x7fffffff) return MHIP_EUNSUPPORTED;
  if (!starts) { T = B * n; most_new = n; }
  if (int code = paged_geometry(p.g, page_table, lengths, starts, t_sb, B, n, T, pages, page_size, table_pages)) return code;
  if (int code = paged_cache_fits(k_cache, v_cache, k_scales, v_scales, pages, Hkv, D, c_sp, c_ss, c_sh, dtype)) return code;
  if (T == 0 || B == 0) return MHIP_OK;
  if (!q || !out || !lse || !workspace) return MHIP_EINVAL;
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || (reinterpret_cast<uintptr_t>(lse) & 3u)) return MHIP_EALIGN;
  for (int64_t s : {q_sb, q_ss, q_sh, o_sb, o_ss, o_sh})
    if (s % 8 != 0) return MHIP_EALIGN;
  if ((int64_t)T * Hq >= (int64_t(1) << 31) - 256) return MHIP_EUNSUPPORTED;       // (rows, up to a whole tile of them, are ints)
  const int size = dtype == MHIP_E4M3 ? 1 : 2;
  // places are counted in 16 bytes: 32 bits for a page, and for the rows of one
  if (c_sp < 0 || c_sp * size / 16 > 0xffffffffll || c_ss * size / 16 * page_size > 0xffffffffll) return MHIP_EUNSUPPORTED;
  p.k = static_cast<const uint8_t*>(k_cache); p.v = static_cast<const uint8_t*>(v_cache);
  p.k_scales = k_scales; p.v_scales = v_scales;
  p.c_sp16 = (uint32_t)(c_sp * size / 16); p.c_ss16 = (uint32_t)(c_ss * size / 16); p.c_sh = c_sh * size;
  p.s_sp = s_sp; p.s_ss = s_ss; p.s_sh = s_sh;
  p.q = static_cast<const uint16_t*>(q); p.out = static_cast<uint16_t*>(out); p.lse = lse;
  p.q_sb = starts ? 0 : q_sb; p.q_ss = q_ss; p.q_sh = q_sh;
  p.o_sb = starts ? 0 : o_sb; p.o_ss = o_ss; p.o_sh = o_sh;
  p.l_sb = starts ? 0 : (int64_t)Hq * n; p.l_sh = starts ? T : n;
  p.Hkv = Hkv; p.G = Hq / Hkv; p.D = D;
  p.causal = mask == MHIP_MASK_CAUSAL;
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * kLog2e;
  p.by_group = Divisor(p.G);
  p.part_o = static_cast<float*>(workspace);
  const int64_t rows = (int64_t)most_new * p.G;
  if (rows > kFewRows && !paged_attn_chunk_fits(B, n, T, p.G, Hkv, starts != nullptr)) return MHIP_EUNSUPPORTED;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows <= kFewRows) {                  // (a sequence with more rows all the same is several tiles of them)
    p.few_rows = 0x7fffffff;
    launch(p, dtype == MHIP_E4M3, rows, st);
  } else {
    // Packed sequences may be of either kind, such as generate a token at a time and such as take a chunk: two pairs of launches, one
    // after the other on the stream, share the workspace.
    p.few_rows = starts && p.G <= kFewRows ? 16 * row_blocks(p.G) : -1;
    if (p.few_rows > 0) launch(p, dtype == MHIP_E4M3, p.few_rows, st);
    paged_attn_chunk_launch(p, dtype == MHIP_E4M3, st);
  }
  return launch_status();
}
