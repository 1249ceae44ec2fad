// Attention of many new tokens over a paged K/V cache: more rows than paged_attn_few takes (rows r = token * G + head of the group).
//
// Bound by the matrix pipes (and the board's power), as the block forward: a key tile feeds 256 rows, 256 multiply-adds for each
// byte read.  The structure is that of attn_fwd.hip on 16 x 16 MFMA tiles:
//   workgroup  = 256 rows of one (sequence, K/V head): 8 wavefronts x 32 rows, one workgroup per CU, two wavefronts per SIMD
//   main loop  = 64-key tiles, K and V rings of four stages in LDS, rows of 256 bytes with XOR-swizzled 16-byte chunks
//   S^T = K Q^T, O^T = V^T P^T with the lane's own P as B operand; the reference score of a row is its first tile's maximum and
//                moves only when a later sum would overflow
//   ping-pong  : the matrix phase of wavefronts 0-3 runs beside the vector phase of wavefronts 4-7 and the other way round
// and what the pages change:
//   copies     : a wavefront copies 8 rows of each tile, which lie in one page; the table's entries are read through the scalar cache
//                at the start of a vector phase and used at its end, when nothing else waits on that counter
//   e4m3, e2m1 : a wavefront's 8 rows of codes come through registers, requested one tile ahead, and go into LDS as bf16 rows
//                times their scale, exact for a power of two: converted once by one wavefront, not by all eight
//   pieces     : where the items are few, or one is long, several workgroups share an item's keys: paged_attn_chunk_plan cuts
//                them and deals them out, paged_attn_join adds the partial results up
#include "paged_attn.hpp"

namespace mhip {
namespace {

constexpr int kBM = 256;                   // rows of a workgroup: 8 wavefronts of 32
constexpr int kBN = 64;                    // keys of a tile
constexpr int kTileLds = kBN * 256;        // a K or V tile in LDS, rows of 256 bytes
constexpr int kRingStages = 4;
constexpr int kVRing = kRingStages * kTileLds;
constexpr int kParts = 512;                // partial results there is room for
constexpr float kPieceCost = 8.f;          // what a piece costs besides its steps, and joining costs, in steps
constexpr float kJoinCost = 6.f;

// How the items (sequence, K/V head, tile of rows) are cut into pieces of their keys, one workgroup each: of so many steps of 64 keys at
// most, an item's all alike.
struct Pieces { int rts, parts, steps; };              // tiles of rows, pieces of each item, its steps
__device__ __forceinline__ int parts_of(int steps, int longest) {
  const int parts = (steps + longest - 1) / longest, most = steps / 4;         // (none shorter than four)
  return parts < most ? parts : most > 1 ? most : 1;
}
__device__ __forceinline__ Pieces chunk_items(const PagedAttn& p, const PagedSeq& s) {
  Pieces c;
  c.rts = s.n * p.G > p.few_rows ? (s.n * p.G + kBM - 1) / kBM : 0;
  c.steps = s.len > kBN ? (s.len + kBN - 1) / kBN : 1;
  c.parts = 1;
  return c;
}
// piece i of a sequence: K/V heads fastest (eight of them: one to an XCD's L2), then the row tiles, the last (longest) first
struct Piece { int part, rt, hk; };
__device__ __forceinline__ Piece piece_of(const Record& c, int Hkv, int64_t i) {
  Piece x;
  const int64_t of_part = (int64_t)c.rts * Hkv;
  x.part = (int)(i / of_part);
  const int rest = (int)(i - x.part * of_part);
  x.rt = c.rts - 1 - rest / Hkv;
  x.hk = rest % Hkv;
  return x;
}

// ---- the plan ------------------------------------------------------------------------------------------------------------
// One workgroup counts the items, cuts them into pieces and deals the pieces out, the longest first, since workgroups take them in order
// as CUs come free.  It leaves for every piece its sequence (-1: none), for every sequence its numbers, and the items in several pieces.
constexpr int kPlanWaves = 16, kStaged = 2048, kBuckets = 64;
__global__ __launch_bounds__(kPlanWaves * 64) void paged_attn_chunk_plan(const PagedAttn p, int places) {
  __shared__ int steps_of[kStaged], rts_of[kStaged];
  __shared__ float sums[kPlanWaves][3][64];
  __shared__ int extremes[2], longest, bucket[kBuckets], slots, items;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), threads = kPlanWaves * 64;
  if (tid == 0) { extremes[0] = 0; extremes[1] = 0x7fffffff; slots = items = 0; }
  if (tid < kBuckets) bucket[tid] = 0;
  for (int i = tid; i < places; i += threads) p.pieces[i] = -1;
  for (int i = tid; i < kParts / 2; i += threads) p.shared[i].rows = 0;
  __syncthreads();
  for (int b = tid; b < p.g.B; b += threads) {
    const Pieces c = chunk_items(p, paged_seq<false>(p.g, b));
    if (b < kStaged) { steps_of[b] = c.steps; rts_of[b] = c.rts; }
    if (c.rts > 0) {
      atomicMax(&extremes[0], c.steps);
      atomicMin(&extremes[1], c.steps);
    }
  }
  __syncthreads();
  const int most = extremes[0], least = extremes[1];
  if (most == 0) return;
  // Each lane tries a length (the longest item in 1 .. 32, then up to 256 pieces) and estimates the launch's time: one round where
  // there is a CU for each piece, whole rounds where all are alike, else the mean of the CUs and a third of the last piece.
  {
    const int tries = lane < 32 ? lane + 1 : 32 + (lane - 31) * 7, bound = (most + tries - 1) / tries;
    float pieces = 0.f, cut = 0.f, steps = 0.f;
    int length = 0;
    for (int b = wave; b < p.g.B; b += kPlanWaves) {
      int rts, of;
      if (b < kStaged) { rts = rts_of[b]; of = steps_of[b]; }
      else { const Pieces c = chunk_items(p, paged_seq<true>(p.g, b)); rts = c.rts; of = c.steps; }
      if (rts == 0) continue;
      const int parts = parts_of(of, bound), here = (of + parts - 1) / parts;
      const float n = (float)rts * parts;
      pieces += n;
      cut += parts > 1 ? n : 0.f;
      steps += (float)rts * of;
      length = here > length ? here : length;
    }
    // (the two counts are whole numbers far below 2^24 wherever they decide)
    sums[wave][0][lane] = pieces;
    sums[wave][1][lane] = cut;
    sums[wave][2][lane] = steps;
    __shared__ int lengths[kPlanWaves][64];
    lengths[wave][lane] = length;
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < kPlanWaves; ++w) {
        pieces += sums[w][0][lane];
        cut += sums[w][1][lane];
        steps += sums[w][2][lane];
        length = lengths[w][lane] > length ? lengths[w][lane] : length;
      }
      pieces *= p.Hkv;
      cut *= p.Hkv;
      steps *= p.Hkv;
      const float one = length + kPieceCost;
      float time = pieces <= 256.f ? one : least == most ? __builtin_ceilf(pieces / 256.f) * one : (steps + pieces * kPieceCost) / 256.f + one / 3.f;
      if (time < one) time = one;
      if (cut > 0.f) time += kJoinCost;
      if (cut > kParts) time = INFINITY;
      float best = time;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) best = fminf(best, __shfl_xor(best, off));
      const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(time == best));
      if (lane == at) longest = bound;
    }
    __syncthreads();
  }
  // pieces by length, in 64 buckets, the longest first
  auto seq = [&](int b) {
    Pieces c;
    if (b < kStaged) { c.rts = rts_of[b]; c.steps = steps_of[b]; c.parts = 1; }
    else c = chunk_items(p, paged_seq<false>(p.g, b));
    if (c.rts > 0) c.parts = parts_of(c.steps, longest);
    return c;
  };
  auto bucket_of = [&](const Pieces& c) { return kBuckets - 1 - (int)((int64_t)((c.steps + c.parts - 1) / c.parts) * (kBuckets - 1) / most); };
  for (int b = tid; b < p.g.B; b += threads) {
    const Pieces c = seq(b);
    if (c.rts > 0) atomicAdd(&bucket[bucket_of(c)], p.Hkv * c.rts * c.parts);
  }
  __syncthreads();
  if (wave == 0) {
    int sum = bucket[lane];
    const int own = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int below = __shfl_up(sum, off);
      if (lane >= off) sum += below;
    }
    bucket[lane] = sum - own;
  }
  __syncthreads();
  for (int b = tid; b < p.g.B; b += threads) {
    const Pieces c = seq(b);
    if (c.rts == 0) continue;
    const int n = p.Hkv * c.rts * c.parts;
    p.records[b] = Record{atomicAdd(&bucket[bucket_of(c)], n), c.parts > 1 ? atomicAdd(&slots, n) : 0, c.parts, c.rts};
  }
  __syncthreads();
  for (int b = wave; b < p.g.B; b += kPlanWaves) {
    const Pieces c = seq(b);
    if (c.rts == 0) continue;
    const Record r = p.records[b];
    const int n = p.Hkv * c.rts * c.parts, in_part = p.Hkv * c.rts;
    for (int i = lane; i < n; i += 64)
      if ((uint32_t)(r.first + i) < (uint32_t)places) p.pieces[r.first + i] = b;       // (starts that fall may count more than there are)
    if (c.parts == 1) continue;
    int at = 0;
    if (lane == 0) at = atomicAdd(&items, in_part);
    at = __builtin_amdgcn_readfirstlane(at);
    const int rows = paged_seq<true>(p.g, b).n * p.G;
    for (int i = lane; i < in_part; i += 64) {           // (as many as partial results / parts, so that there is room)
      const Piece x = piece_of(r, p.Hkv, i);
      const int left = rows - x.rt * kBM;
      if (at + i < kParts / 2)
        p.shared[at + i] = Shared{b, x.hk, x.rt * kBM, left < kBM ? left : kBM, c.parts, r.slot + i, r.slot + in_part + i, in_part};
    }
  }
}
__device__ __forceinline__ Record record_of(const PagedAttn& p, int b) {
  const int* r = reinterpret_cast<const int*>(p.records + b);
  return Record{uniform_load(r, 0), uniform_load(r, 1), uniform_load(r, 2), uniform_load(r, 3)};
}
constexpr int kNoColumn = 0x7fff0000;      // vector offset out of every descriptor's range (spans stay below 2^30)
constexpr int kFragDepth = 4;              // LDS operand reads in flight ahead of the MFMAs
constexpr int kOStride = 136;              // epilogue staging of O, bf16 elements per row

template <int TYPE, int COLS>
__global__ __launch_bounds__(512, 2) void paged_attn_chunk(const PagedAttn p) {
  constexpr bool E2M1 = TYPE == MHIP_E2M1, CODES = TYPE != MHIP_BF16;
  constexpr int KB = COLS / 32, DB = COLS / 16;        // k-steps of S^T, blocks of O^T
  constexpr int MB = kBN / 16, kSteps = kBN / 32;      // key blocks of S^T, k-steps of O^T
  constexpr int kSlotsS = MB * KB, kSlotsO = kSteps * DB;
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * kVRing];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, lg = lane >> 4;
  const bool group_b = wave >= 4;

  // ---- this workgroup's piece --------------------------------------------------------------------------------
  const int b = uniform_load(p.pieces, blockIdx.x);
  if (b < 0) return;                                   // past the last piece
  const PagedSeq s = paged_seq<true>(p.g, b);
  const Record c = record_of(p, b);
  const int pos = (int)blockIdx.x - c.first;
  const Piece piece = piece_of(c, p.Hkv, pos);
  const int hk = piece.hk, row0 = piece.rt * kBM;
  const int rows = s.n * p.G - row0 < kBM ? s.n * p.G - row0 : kBM;
  auto sees = [&](int row) {                           // keys that a row sees
    return __builtin_amdgcn_readfirstlane(p.causal ? clamped(s.len - s.n + p.by_group.quotient(row) + 1, 0, s.len) : s.len);
  };
  const int seen_last = sees(row0 + rows - 1);
  const int64_t steps = (seen_last + kBN - 1) / kBN;
  const int t0 = (int)(steps * piece.part / c.parts), ntiles = (int)(steps * (piece.part + 1) / c.parts) - t0;
  // of the wavefront's rows (those past the last repeat it): the least
  const int my_row0 = row0 + wave * 32;
  const int seen_first = sees(my_row0 < row0 + rows ? my_row0 : row0 + rows - 1);

  // ---- Q rows: B operand of S^T, lane (ln, lg) holds 8 columns of rows ln and 16 + ln --------------------------------
  bf16x8 qf[2][KB];
  int lim[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = my_row0 + r * 16 + ln, real = row < row0 + rows ? row : row0 + rows - 1;
    int of_group;
    const int token = p.by_group.quotient(real, of_group);
    lim[r] = p.causal ? clamped(s.len - s.n + token + 1, 0, s.len) : s.len;
    const uint16_t* src = p.q + b * p.q_sb + (int64_t)(s.start + token) * p.q_ss + (hk * p.G + of_group) * p.q_sh;
#pragma unroll
    for (int ks = 0; ks < KB; ++ks) {
      const int col = ks * 32 + lg * 8;
      qf[r][ks] = bf16x8{};
      if (col < p.D) qf[r][ks] = *reinterpret_cast<const bf16x8*>(src + col);
    }
  }

  // ---- tiles into LDS -----------------------------------------------------------------------------------------------
  const uint32_t lds_smem = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const uint32_t lds_rows = lds_smem + wave * 2048;    // the wavefront's 8 rows of a stage
  const int* table = p.g.table + b * p.g.t_sb;
  // A wavefront's 8 rows of a tile lie in one page.  A look-up reads its table entry (past the last key the last key's), settle() uses
  // it.  Pages that are not here are rare: whether there are any among the piece's is found out once, and only then every tile's four
  // quarters of 16 keys are looked up; gone holds four bits of each of the last eight tiles, that its quarters are not here.
  struct Entry { int page, slot; };
  struct Rows { int64_t at; int page, slot, held, bytes; };      // at: from the first row of the head; bytes: of the rows there are
  auto look_up = [&](int t) {
    const int key = (t0 + t) * kBN + 8 * wave;
    Entry e;
    e.page = uniform_load(table, p.g.by_page.quotient(key < seen_last ? key : seen_last - 1, e.slot));
    return e;
  };
  // (on their way together with Q: the entries of the first tiles, and all of the piece's)
  constexpr int kAhead = 5;
  Entry ahead[kAhead];
  if (ntiles > 0) {
#pragma unroll
    for (int t = 0; t < kAhead; ++t) ahead[t] = look_up(t);
  }
  uint32_t gone = 0;
  bool any_gone = false;
  if (ntiles > 0) {
    int rest;
    const int first = p.g.by_page.quotient(t0 * kBN, rest);
    const int end = (t0 + ntiles) * kBN < seen_last ? (t0 + ntiles) * kBN : seen_last, last = p.g.by_page.quotient(end - 1, rest);
    bool missing = false;
    for (int e = first + lane; e <= last; e += 64) missing = missing || (uint32_t)table[e] >= (uint32_t)p.g.pages;
    any_gone = __builtin_amdgcn_ballot_w64(missing) != 0;
  }
  const int row_step = (int)p.c_ss16 * 16, row_tail = p.D * 2 - row_step;        // (bf16)
  auto settle = [&](int t, Entry e) {
    asm volatile("" : "+s"(e.page));                   // waited for here
    const int left = seen_last - ((t0 + t) * kBN + 8 * wave), held = left < 8 ? left : 8;
    Rows x{0, 0, e.slot, 0, 0};
    if ((uint32_t)e.page < (uint32_t)p.g.pages && t < ntiles && left > 0) {
      x.page = e.page;
      x.held = held;
      x.bytes = held * row_step + row_tail;
    }
    x.at = row_offset(p, x.page, x.slot);
    if (any_gone) {
      uint32_t bits = 0;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int key = (t0 + t) * kBN + 16 * h;
        int slot;
        const int page = uniform_load(table, p.g.by_page.quotient(key < seen_last ? key : seen_last - 1, slot));
        bits |= (uint32_t)page < (uint32_t)p.g.pages ? 0u : 1u << h;
      }
      gone = (gone & ~(15u << (4 * (t & 7)))) | bits << (4 * (t & 7));
    }
    return x;
  };
  int voff[2];                                         // bf16: of copy instruction u, 4 rows each
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = 4 * u + (lane >> 4), chunk = (lane & 15) ^ lds_row_swizzle(8 * wave + row);
    voff[u] = chunk * 8 < p.D ? row * (int)p.c_ss16 * 16 + chunk * 16 : kNoColumn;
  }
  const uint8_t* k_head = p.k + hk * p.c_sh;
  const uint8_t* v_head = p.v + hk * p.c_sh;
  auto copy_rows = [&](const uint8_t* head, const Rows& x, uint32_t to) {
    const u32x4 rs = rsrc_words(head + x.at, (uint32_t)x.bytes);
#pragma unroll
    for (int u = 0; u < 2; ++u) copy16_to_lds(rs, to + u * 1024, voff[u], 0);
  };
  // e4m3 and e2m1: lane l takes codes 16 (l % 8) .. +15 of row l / 8, which have one scale
  const int row8 = lane >> 3, col16 = (lane & 7) * 16;
  struct Codes { u32x4 w; float scale; };
  auto request = [&](const uint8_t* head, const float* scales, const Rows& x) {
    Codes k{u32x4{}, E2M1 ? 0.f : 1.f};
    if (row8 < x.held && col16 < p.D) {
      const uint8_t* at = head + x.at + row8 * (int)p.c_ss16 * 16 + (E2M1 ? col16 / 2 : col16);
      const float* scale = scales + (x.page * p.s_sp + (int64_t)(x.slot + row8) * p.s_ss + hk * p.s_sh);
      if constexpr (E2M1) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(at);
        k.w[0] = w[0];
        k.w[1] = w[1];
        k.scale = __builtin_bit_cast(float, (uint32_t)reinterpret_cast<const uint8_t*>(scale)[col16 >> 5]);      // (the byte: nothing waits for it here)
      } else {
        k.w = *reinterpret_cast<const u32x4*>(at);
        k.scale = *scale;
      }
    }
    return k;
  };
  typedef __attribute__((address_space(3))) u32x4* lds_u32x4;
  auto put = [&](const Codes& k, uint32_t to) {
    u32x4 lo, hi;
    auto keep = [&](int i, uint32_t w0, uint32_t w1) {
      if (i < 2) { lo[2 * i] = w0; lo[2 * i + 1] = w1; } else { hi[2 * i - 4] = w0; hi[2 * i - 3] = w1; }
    };
    // scales 2^-126 .. 2^127 go into the conversion; others, and NaN, through fp32 and one rounding
    const uint32_t bits = __builtin_bit_cast(uint32_t, k.scale);
    if constexpr (E2M1) {
      lo = e2m1_to_bf16(k.w[0], e8m0(bits));
      hi = e2m1_to_bf16(k.w[1], e8m0(bits));
    } else if (__builtin_expect(__builtin_amdgcn_ballot_w64((bits & 0x807fffffu) != 0 || bits - 0x00800000u >= 0x7f000000u) == 0, 1)) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        keep(i, __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k.w[i], k.scale, false)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k.w[i], k.scale, true)));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2 x = __builtin_amdgcn_cvt_pk_f32_fp8(k.w[i], false), z = __builtin_amdgcn_cvt_pk_f32_fp8(k.w[i], true);
        keep(i, pack_bf16(x[0] * k.scale, x[1] * k.scale), pack_bf16(z[0] * k.scale, z[1] * k.scale));
      }
    }
    const int swz = lds_row_swizzle(8 * wave + row8), chunk = (lane & 7) * 2;
    *(lds_u32x4)(uintptr_t)(to + row8 * 256 + ((chunk ^ swz) << 4)) = lo;
    *(lds_u32x4)(uintptr_t)(to + row8 * 256 + (((chunk + 1) ^ swz) << 4)) = hi;
  };

  // ---- operands from LDS (addresses inside the stage that is read next move on in place) --------------------------------
  int k_a[KB];                                         // + mb * 16 rows
#pragma unroll
  for (int ks = 0; ks < KB; ++ks) k_a[ks] = (int)lds_smem + ln * 256 + (((4 * ks + lg) ^ lds_row_swizzle(ln)) << 4);
  int v_a[DB];                                         // + t * 32 rows
  {
    const int row = 4 * lg + (ln >> 2);
#pragma unroll
    for (int db = 0; db < DB; ++db)
      v_a[db] = (int)lds_smem + kVRing + row * 256 + (((2 * db + ((ln & 3) >> 1)) ^ lds_row_swizzle(row)) << 4) + (ln & 1) * 8;
  }
  typedef __attribute__((address_space(3))) bf16x4* lds_bf16x4;
  typedef __attribute__((address_space(3))) const bf16x8* lds_bf16x8;
  auto read_k = [&](int mb, int ks) -> bf16x8 { return *(lds_bf16x8)(uintptr_t)(uint32_t)(k_a[ks] + mb * 4096); };
  auto read_v = [&](int db, int t) -> bf16x8 {
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4)(uintptr_t)(uint32_t)(v_a[db] + t * 8192));
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4)(uintptr_t)(uint32_t)(v_a[db] + t * 8192 + 4096));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto stage_step = [](int t) { return (t + 1) % kRingStages == 0 ? -(kRingStages - 1) * kTileLds : kTileLds; };

  // ---- softmax state and products -------------------------------------------------------------------------------------
  f32x4 o_acc[DB][2], sc[MB][2];
  u32x4 pw[kSteps][2];                                 // P^T of the current tile
  float m_ref[2] = {}, nmsc[2] = {}, l_run[2] = {}, rs[2] = {};
#pragma unroll
  for (int i = 0; i < DB; ++i) o_acc[i][0] = o_acc[i][1] = f32x4{};
  constexpr float kTrigger = 1048576.f, kSlack = 14.f, kMost = 0x1.fffffep127f;
  float scale_log2 = p.scale_log2;
  asm volatile("" : "+s"(scale_log2));
  auto mfma = [](const bf16x8& x, const bf16x8& z, const f32x4& a) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, z, a, 0, 0, 0); };
  auto s_mfma = [&](int mb, int ks, const bf16x8& kf) {
#pragma unroll
    for (int r = 0; r < 2; ++r) sc[mb][r] = mfma(kf, qf[r][ks], ks == 0 ? f32x4{} : sc[mb][r]);
  };
  auto o_mfma = [&](int db, int t, const bf16x8& vf) {
#pragma unroll
    for (int r = 0; r < 2; ++r) o_acc[db][r] = mfma(vf, __builtin_bit_cast(bf16x8, pw[t][r]), o_acc[db][r]);
  };
  auto cuts = [&](int t) { return (t0 + t + 1) * kBN > seen_first; };      // some row of the wavefront does not see some key
  auto sm_mask = [&](int t) {
    const uint32_t bits = gone >> (4 * (t & 7)) & 15u;
    if (__builtin_expect(cuts(t) || bits, 0)) {
      asm volatile("");                                // (a branch: not 32 selections on every tile)
      const int kv0 = (t0 + t) * kBN;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const int left = bits >> mb & 1 ? 0 : lim[r] - (kv0 + mb * 16) - lg * 4;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j >= left) sc[mb][r][j] = -INFINITY;
          // (one comparison at a time: their masks would take the scalar registers that the loop's addresses are in)
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  };
  auto sm_pair = [&](int idx) {
    const int t = idx >> 3, r = (idx >> 2) & 1, d = idx & 3, mb = 2 * t + (d >> 1), e = 2 * (d & 1);
    const float x0 = fast_exp2(__builtin_fmaf(sc[mb][r][e], scale_log2, nmsc[r]));
    const float x1 = fast_exp2(__builtin_fmaf(sc[mb][r][e + 1], scale_log2, nmsc[r]));
    if (t == 0 && d == 0) rs[r] = x0 + x1; else rs[r] += x0 + x1;
    uint32_t w = pack_bf16(x0, x1);
    asm volatile("" : "+v"(w), "+v"(rs[r]));           // keeps the pair where it is written
    pw[t][r][d] = w;
  };
  constexpr int kPairs = kBN / 4;
  auto sm_exps = [&]() {
#pragma unroll
    for (int idx = 0; idx < kPairs; ++idx) sm_pair(idx);
  };
  auto sm_fix = [&](bool first) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = sc[0][r][0];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, sc[mb][r][j]);
      mx = quad_max(mx);
      const float grown = (mx - m_ref[r]) * scale_log2;
      const bool move = first || grown > kSlack;
      if (!first) {
        const float alpha = move ? fast_exp2(-grown) : 1.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) o_acc[db][r] *= alpha;
        l_run[r] *= alpha;
      }
      if (move) m_ref[r] = first ? fmaxf(mx, -kMost) : mx;
      nmsc[r] = fminf(-m_ref[r] * scale_log2, kMost);
    }
  };
  // Up to 96 columns the matrix phase is the shorter one: it takes the tile copies of the vector phase then, and on 64 columns more of
  // the exponentials.
  constexpr bool kShortMatrix = COLS < 128;
  constexpr int kEarlyPairs = COLS == 64 ? 6 : 2;
  auto sm_tile = [&]() {
#pragma unroll
    for (int idx = kEarlyPairs; idx < kPairs; ++idx) sm_pair(idx);
    if (__builtin_amdgcn_ballot_w64(!(rs[0] + rs[1] < kTrigger)) != 0) {
      sm_fix(false);
      sm_exps();
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) l_run[r] += rs[r];
  };
  // O^T of a tile that cuts (see finite_part).
  auto pv_cut = [&](int tile) __attribute__((always_inline)) {
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < kSlotsO; ++i) {
      o_mfma(i % DB, i / DB, __builtin_bit_cast(bf16x8, finite_part(__builtin_bit_cast(u32x4, read_v(i % DB, i / DB)), odd)));
      __builtin_amdgcn_sched_barrier(0);
    }
    if (__builtin_amdgcn_ballot_w64(odd != 0) == 0) return;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      f32x4 counts[2] = {};
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        const bf16x8 marks = __builtin_bit_cast(bf16x8, odd_marks(__builtin_bit_cast(u32x4, read_v(db, t))));
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          int left[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            left[h] = gone >> (4 * (tile & 7) + 2 * t + h) & 1u ? 0 : lim[r] - ((t0 + tile) * kBN + (2 * t + h) * 16) - lg * 4;
          counts[r] = mfma(marks, __builtin_bit_cast(bf16x8, seen_marks(left[0], left[1])), counts[r]);
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) o_acc[db][r][j] = with_odd(o_acc[db][r][j], counts[r][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Matrix phase of tile t: S^T(t+1) and O^T += V^T(t) P^T(t), operands kFragDepth reads ahead.
  auto read_frag = [&](int i) -> bf16x8 {
    if (i < kSlotsS) return read_k(i % MB, i / MB);
    return read_v((i - kSlotsS) % DB, (i - kSlotsS) / DB);
  };
  bf16x8 frag[kFragDepth];
  auto first_frags = [&]() {
#pragma unroll
    for (int i = 0; i < kFragDepth; ++i) frag[i] = read_frag(i);
  };
  auto early_slot = [](int idx) { return kSlotsS + DB + idx * (kSlotsO - DB) / kEarlyPairs; };
  Rows next_v{}, next_k{};                             // of the tiles whose copies go out (of codes: which are put into LDS) next
  auto copies = [&](int t) {                           // K(t + 4), V(t + 3)
    copy_rows(k_head, next_k, lds_rows + (t & 3) * kTileLds);
    copy_rows(v_head, next_v, lds_rows + kVRing + ((t + 3) & 3) * kTileLds);
    next_v = next_k;
  };
  auto matrix_phase = [&](int t) __attribute__((always_inline)) {
    const int k_step = stage_step(t + 1), v_step = stage_step(t);
#pragma unroll
    for (int i = 0; i < kSlotsS + kSlotsO; ++i) {
      if (i < kSlotsS) s_mfma(i % MB, i / MB, frag[i % kFragDepth]);
      else o_mfma((i - kSlotsS) % DB, (i - kSlotsS) / DB, frag[i % kFragDepth]);
      if (i + kFragDepth < kSlotsS + kSlotsO) frag[i % kFragDepth] = read_frag(i + kFragDepth);
      if (i >= kSlotsS && i < kSlotsS + KB) k_a[i - kSlotsS] += k_step;            // the last K read went out before slot kSlotsS
      if (i >= kSlotsS + kSlotsO - kFragDepth) {                                   // and the last V read by here
#pragma unroll
        for (int e = 0; e < DB; ++e)
          if (e % kFragDepth == i - (kSlotsS + kSlotsO - kFragDepth)) v_a[e] += v_step;
      }
      if (!CODES && kShortMatrix && i == 1) copies(t);
      if (i == kSlotsS) sm_mask(t + 1);
#pragma unroll
      for (int idx = 0; idx < kEarlyPairs; ++idx)
        if (early_slot(idx) == i) sm_pair(idx);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // the same where tile t cuts
  auto matrix_phase_cut = [&](int t) __attribute__((always_inline)) {
    if (!CODES && kShortMatrix) copies(t);
    pv_cut(t);
#pragma unroll
    for (int i = 0; i < kSlotsS; ++i) {
      s_mfma(i % MB, i / MB, read_k(i % MB, i / MB));
      __builtin_amdgcn_sched_barrier(0);
    }
    const int k_step = stage_step(t + 1), v_step = stage_step(t);
#pragma unroll
    for (int ks = 0; ks < KB; ++ks) k_a[ks] += k_step;
#pragma unroll
    for (int e = 0; e < DB; ++e) v_a[e] += v_step;
    sm_mask(t + 1);
#pragma unroll
    for (int idx = 0; idx < kEarlyPairs; ++idx) sm_pair(idx);
  };

  if (ntiles > 0) {
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int ks = 0; ks < KB; ++ks) asm volatile("" : "+v"(qf[r][ks]));      // loaded before the first copy goes out
    // Tiles 0 .. 3 of K and 0 .. 2 of V; in the loop K(t + 4) and V(t + 3) follow, whose places tile t's matrix phase and the one
    // before it were the last to read.  Codes that pass through registers are requested one tile before they are put there.
    Codes ck, cv;
    auto first_tile = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < KB; ++ks) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) s_mfma(mb, ks, read_k(mb, ks));
        k_a[ks] += kTileLds;
      }
      sm_mask(0);
      sm_fix(true);
      sm_exps();
#pragma unroll
      for (int r = 0; r < 2; ++r) l_run[r] = rs[r];
    };
    if constexpr (!CODES) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const Rows x = settle(t, ahead[t]);
        copy_rows(k_head, x, lds_rows + t * kTileLds);
        if (t < 3) copy_rows(v_head, x, lds_rows + kVRing + t * kTileLds);
        next_v = x;
      }
      next_k = settle(4, ahead[4]);
      asm volatile("s_waitcnt vmcnt(12)" ::: "memory");         // K(0)
      __builtin_amdgcn_s_barrier();
      first_tile();
      // V(0), K(1), V(1) and K(2) are read before their copiers' next wait: the first group reads K(2) in its vector phase of tile 0 and
      // V(1) in the phase after, beside the other group's vector phase of tile 0.  V(2) and K(3) may be on their way, every wavefront waits
      // for them in that phase; from there on the vector phase of tile t waits for K(t + 3) and V(t + 2), read from the next one on.
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
      __builtin_amdgcn_s_barrier();
    } else {
      Codes k[4], v[3];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const Rows x = settle(t, ahead[t]);
        k[t] = request(k_head, p.k_scales, x);
        if (t < 3) v[t] = request(v_head, p.v_scales, x);
        next_v = x;
      }
      next_k = settle(4, ahead[4]);
      put(k[0], lds_rows);
      __syncthreads();
      first_tile();
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (t > 0) put(k[t], lds_rows + t * kTileLds);
        if (t < 3) put(v[t], lds_rows + kVRing + t * kTileLds);
      }
      cv = request(v_head, p.v_scales, next_v);
      ck = request(k_head, p.k_scales, next_k);
      __syncthreads();
    }
    if (ntiles > 1) first_frags();
    if (group_b) __builtin_amdgcn_s_barrier();
    // vector phase of tile t: softmax of tile t + 1 and the copies ahead
    auto vector_phase = [&](int t) __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) asm volatile("" : "+v"(sc[0][r]), "+v"(sc[MB - 1][r]));   // keeps the exponentials behind the barrier
      if constexpr (!CODES) {
        const Entry e = look_up(t + 5);
        sm_tile();
        if (!kShortMatrix) copies(t);
        next_k = settle(t + 5, e);
        if (t + 2 < ntiles) first_frags();
        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");          // the four copies of one tile ago are done
      } else {
        const Entry e = look_up(t + 5);
        sm_tile();
        const Rows x = settle(t + 5, e);
        put(ck, lds_rows + (t & 3) * kTileLds);
        put(cv, lds_rows + kVRing + ((t + 3) & 3) * kTileLds);
        cv = request(v_head, p.v_scales, next_k);
        ck = request(k_head, p.k_scales, x);
        next_k = x;
        if (t + 2 < ntiles) first_frags();
      }
    };
    // Tiles that all rows see whole, then those that cut (of the workgroup, whose wavefronts keep step).
    const int whole = clamped(sees(row0) / kBN - t0, 0, ntiles - 1);
    int t = 0;
    for (; t < whole; ++t) {
      __builtin_amdgcn_s_setprio(2);
      matrix_phase(t);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_s_barrier();
      vector_phase(t);
      __builtin_amdgcn_s_barrier();
    }
    for (; t + 1 < ntiles; ++t) {
      matrix_phase_cut(t);
      __builtin_amdgcn_s_barrier();
      vector_phase(t);
      __builtin_amdgcn_s_barrier();
    }
    if (cuts(ntiles - 1)) pv_cut(ntiles - 1);
    else {
#pragma unroll
      for (int i = 0; i < kSlotsO; ++i) o_mfma(i % DB, i / DB, read_v(i % DB, i / DB));
    }
    if (!group_b) __builtin_amdgcn_s_barrier();
  }

  // ---- epilogue -----------------------------------------------------------------------------------------------------
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // copies past the last tile
  const PagedAttn a = arguments_again();
  __syncthreads();                                     // every wavefront is done with K and V
  if (c.parts > 1) {
    const int64_t at = ((int64_t)c.slot + pos) * kBM + wave * 32;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float l_tot = quad_sum(l_run[r]);
      if (wave * 32 + r * 16 + ln >= rows) continue;
      const int64_t row = at + r * 16 + ln;
      if (lg == 0) a.part_ml[row] = f32x2{l_tot == 0.f ? -INFINITY : m_ref[r] * scale_log2, l_tot};
#pragma unroll
      for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(a.part_o + row * COLS + db * 16 + lg * 4) = o_acc[db][r];
    }
    return;
  }
  unsigned char* os = smem + wave * (32 * kOStride * 2);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float l_tot = quad_sum(l_run[r]), inv = l_tot == 0.f ? 0.f : 1.f / l_tot;
    const int row = my_row0 + r * 16 + ln;
    if (lg == 0 && row < row0 + rows) {
      int of_group;
      const int token = s.start + a.by_group.quotient(row, of_group);
      a.lse[b * a.l_sb + (hk * a.G + of_group) * a.l_sh + token] = l_tot == 0.f ? -INFINITY : __builtin_fmaf(fast_log2(l_tot), kLn2, m_ref[r] * a.scale);
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      u32x2 w;
      w[0] = pack_bf16(o_acc[db][r][0] * inv, o_acc[db][r][1] * inv);
      w[1] = pack_bf16(o_acc[db][r][2] * inv, o_acc[db][r][3] * inv);
      *reinterpret_cast<u32x2*>(os + (r * 16 + ln) * (kOStride * 2) + (db * 16 + lg * 4) * 2) = w;
    }
  }
  __syncthreads();
  const int chunk = lane & 15;
#pragma unroll
  for (int it = 0; it < 8; ++it) {
    const int r = (lane >> 4) + 4 * it, row = my_row0 + r;
    if (row < row0 + rows && chunk * 8 < a.D) {
      int of_group;
      const int token = s.start + a.by_group.quotient(row, of_group);
      *reinterpret_cast<u32x4*>(a.out + b * a.o_sb + (int64_t)token * a.o_ss + (hk * a.G + of_group) * a.o_sh + chunk * 8) =
          *reinterpret_cast<const u32x4*>(os + r * (kOStride * 2) + chunk * 16);
    }
  }
}

int64_t places_of(int64_t B, int64_t T, int64_t n, int G, int Hkv, bool packed) {
  return Hkv * (packed ? T * G / kBM + B : B * ((n * G + kBM - 1) / kBM)) + kParts;
}
int columns_of(int D) { return D <= 64 ? 64 : D <= 96 ? 96 : 128; }
int64_t up16(int64_t x) { return (x + 15) & ~int64_t(15); }

template <int TYPE, int COLS>
void launch(const PagedAttn& p, int places, hipStream_t st) {
  hipLaunchKernelGGL(paged_attn_chunk_plan, dim3(1), dim3(kPlanWaves * 64), 0, st, p, places);
  hipLaunchKernelGGL((paged_attn_chunk<TYPE, COLS>), dim3((unsigned)places), dim3(512), 0, st, p);
  // rows of a workgroup: 4 / 8 / 16 / 32 took 57.0 / 58.6 / 65.2 / 76.4 us with 64 tokens at 32768 (8 now 56.1)
  constexpr int rows = 8;
  hipLaunchKernelGGL((paged_attn_join<COLS, kBM, 2, rows>), dim3(kBM / rows, kParts / 2), dim3(256), 0, st, p);
}
template <int TYPE>
void launch(const PagedAttn& p, int places, hipStream_t st) {
  if (p.D <= 64) launch<TYPE, 64>(p, places, st);
  else if (p.D <= 96) launch<TYPE, 96>(p, places, st);
  else launch<TYPE, 128>(p, places, st);
}

}  // namespace

// The workspace: partial results, their maxima and sums, the items that are shared, the sequences' records, the pieces.
int64_t paged_attn_chunk_bytes(int64_t B, int64_t n, int64_t T, int G, int Hkv, int D, bool packed) {
  return (int64_t)kParts * kBM * (columns_of(D) + 2) * 4 + kParts / 2 * 32 + 16 * B + up16(4 * places_of(B, T, n, G, Hkv, packed));
}
bool paged_attn_chunk_fits(int64_t B, int64_t n, int64_t T, int G, int Hkv, bool packed) {
  return grid_fits(places_of(B, T, n, G, Hkv, packed), 512);
}
void paged_attn_chunk_launch(const PagedAttn& p, int type, hipStream_t stream) {
  const int places = (int)places_of(p.g.B, p.g.T, p.g.n, p.G, p.Hkv, p.g.starts != nullptr);
  PagedAttn q = p;
  char* at = reinterpret_cast<char*>(q.part_o) + (int64_t)kParts * kBM * columns_of(p.D) * 4;
  q.part_ml = reinterpret_cast<f32x2*>(at);
  at += (int64_t)kParts * kBM * 8;
  q.shared = reinterpret_cast<Shared*>(at);
  at += kParts / 2 * 32;
  q.records = reinterpret_cast<Record*>(at);
  q.pieces = reinterpret_cast<int*>(at + 16 * (int64_t)p.g.B);
  if (type == MHIP_E2M1) launch<MHIP_E2M1>(q, places, stream);
  else if (type == MHIP_E4M3) launch<MHIP_E4M3>(q, places, stream);
  else launch<MHIP_BF16>(q, places, stream);
}

}  // namespace mhip
