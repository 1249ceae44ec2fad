// A paged K/V cache that stays within a budget.  A sequence of more than `limit` tokens is cut to `keep`: each K/V head keeps the keys
// of its `recent` last tokens and, of the others, the keep - recent with the largest weights (of equal ones the first), in their order.
//
// paged_evict_choose: one workgroup for each (sequence, K/V head).  The weights are looked at as whole numbers that order like them, read
//   once and held in registers: the number that the last kept one has is found eleven bits at a time behind those that all have in
//   common, by counting (the largest first), and a pass in order then leaves the positions that stay, each at its place in the result.
// paged_evict_move: rows that stay, with scales and weights, to their new places.  In its own pages a row moves down or not at all, so a
//   workgroup that reads a tile of rows whole, and then writes it, has read whatever it writes over, and rows of later tiles
//   lie behind everything that it writes: one workgroup walks each (sequence, K/V head, half) from the first row on.  Into other
//   pages rows are independent, and many workgroups share them.
// Measured, us: one sequence of 1040 tokens, four heads, to 1024: 7 and 4 (both chains of dependent loads); 32 x 3000 .. 8192 e4m3 H8 D128 to
// 2048: 13 and 74, the rows at 4.5 TB/s of reading and writing.
#include "paged.hpp"

namespace mhip {
namespace {

struct Evict {
  PagedGeom g;
  const int* out_table; int64_t ot_sb;                     // NULL: the sequences' own pages
  uint8_t* k; uint8_t* v; float* k_scales; float* v_scales;
  int64_t c_sp, c_ss, c_sh;        // of the cache, bytes
  int64_t s_sp, s_ss, s_sh;        // of the scales, four bytes
  float* weights;
  int64_t w_sp, w_ss, w_sh;
  int* kept; int* left;
  int Hkv, keep, recent, limit, row;       // row: bytes of a row of the cache
  Divisor by_heads;
};

constexpr int kChoosers = 1024, kChooserWaves = kChoosers / 64;

// Whole numbers that order as the weights do; NaN is above all.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t bits = __builtin_bit_cast(uint32_t, w + 0.f);           // (-0 counts as 0)
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// Lane l's with those of lanes 0 .. l - 1, by f; `none` takes no part in it.  (In registers: a shuffle is a trip through LDS.)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved_lanes(uint32_t x, uint32_t none) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, CTRL, ROWS, 0xf, false);
}
template <class F>
__device__ __forceinline__ uint32_t up_to_lane(uint32_t x, uint32_t none, F&& f) {
  x = f(x, moved_lanes<0x111, 0xf>(x, none));    // 1, 2, 4 and 8 lanes further up within rows of 16
  x = f(x, moved_lanes<0x112, 0xf>(x, none));
  x = f(x, moved_lanes<0x114, 0xf>(x, none));
  x = f(x, moved_lanes<0x118, 0xf>(x, none));
  x = f(x, moved_lanes<0x142, 0xa>(x, none));    // the last of rows 0 and 2 to rows 1 and 3
  return f(x, moved_lanes<0x143, 0xc>(x, none)); // lane 31 to rows 2 and 3
}
// Of what the wavefronts have left, the sum over those before this one.
__device__ __forceinline__ uint32_t before_wave(const uint32_t (&waves)[kChooserWaves], int wave) {
  uint32_t sum = 0;
#pragma unroll
  for (int v = 0; v < kChooserWaves; ++v) sum += v < wave ? waves[v] : 0u;
  return sum;
}

constexpr int kDigits = 2048, kListed = 24576;
struct ChooserLds {
  uint32_t count[kDigits];
  uint32_t waves[2][kChooserWaves];
  uint32_t found[3];                             // the digit, how many of it are kept, and of how many
  uint32_t listed;
  uint32_t list[kListed];
};

// The keep - recent with the largest weights of the first `others` positions into kept, in order.  A wavefront has 64 HELD positions in a
// row in registers.  HELD = 0: as many as there are, read anew each time, three times if all goes well: to count the first digits; to put
// those with the digit of the last one kept into a list, their other bits and which wavefront's they are; and to leave the positions.
// (4 x 131072 tokens to 100000, 2 heads: 237 us when every digit was counted over all, 149 so,
// 115 with the runs below.)
template <int HELD>
__device__ __forceinline__ void choose(const Evict& p, ChooserLds& lds, const int* table, int hk, int others, int* kept) {
  constexpr int kAtOnce = HELD > 0 && HELD < 16 ? HELD : 16, kRegisters = HELD > 0 ? HELD : kAtOnce;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int each = HELD > 0 ? HELD : (others + kChoosers * kAtOnce - 1) / (kChoosers * kAtOnce) * kAtOnce;
  const int first = wave * each * 64 + lane;
  // The wavefront's positions from 64 u0 on.  Runs of 16 lie in one page: a lane finds where run `lane` begins, and all take from there
  // what they need, so that the table is read and the strides are multiplied once for 16 positions.
  uint32_t x[kRegisters];
  const float* weights_of_lane = p.weights + ((int64_t)hk * p.w_sh + (lane & 15) * p.w_ss);
  auto read = [&](int u0, uint32_t* to) __attribute__((always_inline)) {
    const int run = wave * each * 64 + u0 * 64 + lane * 16;
    int slot;
    const int page = table[p.g.by_page.quotient(run < others ? run : (others - 1) & ~15, slot)];
    const int64_t at = (int64_t)page * p.w_sp + (int64_t)slot * p.w_ss;
    float w[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int from = (u * 4 + (lane >> 4)) * 4;
      const uint32_t lo = __builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)at), hi = __builtin_amdgcn_ds_bpermute(from, (int)(at >> 32));
      w[u] = weights_of_lane[(int64_t)((uint64_t)hi << 32 | lo)];
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) to[u] = order_of(w[u]);
  };
  auto all = [&](auto&& f) __attribute__((always_inline)) {              // f(position, its number, whether it is one)
    if constexpr (HELD > 0) {
#pragma unroll
      for (int u = 0; u < HELD; ++u) f(first + u * 64, x[u], first + u * 64 < others);
    } else {
      for (int u0 = 0; u0 < each; u0 += kAtOnce) {
        read(u0, x);
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) f(first + (u0 + u) * 64, x[u], first + (u0 + u) * 64 < others);
      }
    }
  };
  if constexpr (HELD > 0) {
#pragma unroll
    for (int u0 = 0; u0 < HELD; u0 += kAtOnce) read(u0, x + u0);
  }

  // ---- the bits that all have in common (of many they are not looked for) -----------------------------------------------------
  uint32_t last = 0, need = p.keep - p.recent;
  int bits = 32;                                 // that differ
  if (HELD > 0) {
    uint32_t high = 0, low = 0xffffffffu;
    all([&](int, uint32_t v, bool real) {
      high = real && v > high ? v : high;
      low = real && v < low ? v : low;
    });
    high = up_to_lane(high, 0u, [](uint32_t a, uint32_t c) { return a > c ? a : c; });
    low = up_to_lane(low, 0xffffffffu, [](uint32_t a, uint32_t c) { return a < c ? a : c; });
    if (lane == 63) {
      lds.waves[0][wave] = high;
      lds.waves[1][wave] = low;
    }
    __syncthreads();
    high = 0;
    low = 0xffffffffu;
#pragma unroll
    for (int v = 0; v < kChooserWaves; ++v) {
      high = lds.waves[0][v] > high ? lds.waves[0][v] : high;
      low = lds.waves[1][v] < low ? lds.waves[1][v] : low;
    }
    bits = high == low ? 0 : 32 - __builtin_clz(high ^ low);
    last = bits == 32 ? 0u : high >> bits << bits;
  }

  // ---- the number of the last one kept, and how many of that number are (or the number below the least kept, and none) ------------
  bool listed = false;
  uint32_t above = 0, equal = 0;                 // of this wavefront; listed: above the list's numbers
  while (bits > 0) {
    const int shift = bits > 11 ? bits - 11 : 0;
    const uint32_t digits = (1u << (bits - shift)) - 1;
    lds.count[tid] = lds.count[tid + kChoosers] = 0;
    __syncthreads();
    if (listed) {
      for (uint32_t i = tid; i < lds.listed; i += kChoosers) {
        const uint32_t v = lds.list[i];
        if (((v ^ last) & 0x1fffffu) >> bits == 0) atomicAdd(&lds.count[v >> shift & digits], 1u);
      }
    } else {
      all([&](int, uint32_t v, bool real) {
        if (real && (bits == 32 || (v ^ last) >> bits == 0)) atomicAdd(&lds.count[v >> shift & digits], 1u);
      });
    }
    __syncthreads();
    // thread t has the digits 2047 - 2 t and 2046 - 2 t: how many are above them, and in which of them the last one kept is
    const uint32_t c0 = lds.count[kDigits - 1 - 2 * tid], c1 = lds.count[kDigits - 2 - 2 * tid];
    uint32_t higher = up_to_lane(c0 + c1, 0u, [](uint32_t a, uint32_t c) { return a + c; });
    if (lane == 63) lds.waves[0][wave] = higher;
    __syncthreads();
    higher += before_wave(lds.waves[0], wave) - c0 - c1;
    if (higher < need && need <= higher + c0 + c1) {
      const bool upper = need <= higher + c0;
      lds.found[0] = kDigits - 1 - 2 * tid - (upper ? 0 : 1);
      lds.found[1] = need - higher - (upper ? 0 : c0);
      lds.found[2] = upper ? c0 : c1;
    }
    if (tid == 0 && !listed) lds.listed = 0;
    __syncthreads();
    last |= lds.found[0] << shift;
    need = lds.found[1];
    bits = shift;
    const uint32_t of = lds.found[2];
    if (HELD > 0 && need == of && last > 0) {    // all with these digits are kept
      --last;
      need = 0;
      break;
    }
    if (HELD == 0 && bits == 21 && of <= kListed) {
      listed = true;
      all([&](int, uint32_t v, bool real) {
        const uint64_t in = __builtin_amdgcn_ballot_w64(real && v >> 21 == last >> 21);
        above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(real && v >> 21 > last >> 21));
        if (in == 0) return;
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&lds.listed, (uint32_t)__builtin_popcountll(in));
        at = __builtin_amdgcn_readfirstlane(at) + __builtin_popcountll(in & ((1ull << lane) - 1));
        if (in >> lane & 1) lds.list[at] = (v & 0x1fffffu) | (uint32_t)wave << 28;
      });
    }
    __syncthreads();
  }

  // ---- the positions in order: those above, and of those equal the first `need` ------------------------------------------------
  if (listed) {
    if (tid < kChooserWaves) lds.waves[1][tid] = 0;
    if (lane == 0) lds.waves[0][wave] = above;
    __syncthreads();
    for (uint32_t i = tid; i < lds.listed; i += kChoosers) {
      const uint32_t v = lds.list[i] & 0x1fffffu, whose = lds.list[i] >> 28;
      if (v > (last & 0x1fffffu)) atomicAdd(&lds.waves[0][whose], 1u);
      if (v == (last & 0x1fffffu)) atomicAdd(&lds.waves[1][whose], 1u);
    }
  } else {
    all([&](int, uint32_t v, bool real) {
      above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(real && v > last));
      equal += __builtin_popcountll(__builtin_amdgcn_ballot_w64(real && v == last));
    });
    __syncthreads();
    if (lane == 0) {
      lds.waves[0][wave] = above;
      lds.waves[1][wave] = equal;
    }
  }
  __syncthreads();
  above = before_wave(lds.waves[0], wave);
  equal = before_wave(lds.waves[1], wave);
  const uint64_t below = (1ull << lane) - 1;
  all([&](int at, uint32_t v, bool real) {
    const uint64_t mask_above = __builtin_amdgcn_ballot_w64(real && v > last), mask_equal = __builtin_amdgcn_ballot_w64(real && v == last);
    const uint32_t here = above + __builtin_popcountll(mask_above & below), ties = equal + __builtin_popcountll(mask_equal & below);
    if (real && (v > last || (v == last && ties < need))) kept[here + (ties < need ? ties : need)] = at;
    above += __builtin_popcountll(mask_above);
    equal += __builtin_popcountll(mask_equal);
  });
}

__global__ __launch_bounds__(kChoosers) void paged_evict_choose(const Evict p) {
  __shared__ ChooserLds lds;
  const int tid = threadIdx.x;
  int hk;
  const int b = p.by_heads.quotient(blockIdx.x, hk);
  const int len = clamped(uniform_load(p.g.lengths, b), 0, p.g.width * p.g.page);
  const int* table = p.g.table + b * p.g.t_sb;
  int* kept = p.kept + (int64_t)blockIdx.x * p.limit;

  int rest;
  const int entries = len > 0 ? p.g.by_page.quotient(len - 1, rest) + 1 : 0;
  bool missing = false;
  for (int e = tid; e < entries; e += kChoosers) missing = missing || (uint32_t)table[e] >= (uint32_t)p.g.pages;
  const bool whole = __syncthreads_or(missing) == 0;
  const bool cut = whole && len > p.limit;
  if (tid == 0 && hk == 0) p.left[b] = cut ? p.keep : len;
  if (!cut) {                                    // all rows stay, or nobody knows
    for (int i = tid; i < p.limit; i += kChoosers) kept[i] = whole && i < len ? i : -1;
    return;
  }
  const int others = len - p.recent, chosen = p.keep - p.recent;         // (recent <= keep <= limit < len)
  for (int i = tid; i < p.limit - chosen; i += kChoosers) kept[chosen + i] = i < p.recent ? others + i : -1;
  if (chosen == 0) return;
  if (others <= 2 * kChoosers) choose<2>(p, lds, table, hk, others, kept);
  else if (others <= 8 * kChoosers) choose<8>(p, lds, table, hk, others, kept);
  else if (others <= 32 * kChoosers) choose<32>(p, lds, table, hk, others, kept);
  else choose<0>(p, lds, table, hk, others, kept);
}

// LANES lanes take a row, of up to 16 bytes each; a workgroup moves THREADS / LANES rows at once and DEEP times as many with their loads in flight
// together (each kind of load stands before the first that waits for one: positions, pages, rows).
template <int LANES, int DEEP, bool APART, int THREADS>
__global__ __launch_bounds__(THREADS, DEEP == 4 ? 8 : 4) void paged_evict_move(const Evict p, const int tiles) {
  constexpr int kRows = THREADS / LANES, kTile = kRows * DEEP;
  const int sub = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int half = blockIdx.x & 1;
  int item = blockIdx.x >> 1, tile = 0;
  if (APART) {
    tile = item % tiles;
    item /= tiles;
  }
  int hk;
  const int b = p.by_heads.quotient(item, hk);
  const int* kept = p.kept + (int64_t)item * p.limit;
  const int len = clamped(uniform_load(p.g.lengths, b), 0, p.g.width * p.g.page), left = uniform_load(p.left, b);
  if (!APART && left == len) return;             // (or not all of it is here, and kept is empty)
  const int count = left < p.limit ? left : p.limit;
  const int* table = p.g.table + b * p.g.t_sb;
  const int* to_table = APART ? p.out_table + b * p.ot_sb : table;
  uint8_t* rows = (half ? p.v : p.k) + (int64_t)hk * p.c_sh + sub * 16;
  float* scales = half ? p.v_scales : p.k_scales;
  const bool real = sub * 16 < p.row;
  // of a row's lanes the first moves its scales, and among the keys the second (there are four) what attention it has had
  const bool scaled = sub == 0 && scales, weighted = sub == 1 && half == 0;
  float* word = scaled ? scales + (int64_t)hk * p.s_sh : p.weights + (int64_t)hk * p.w_sh;
  const int64_t word_sp = scaled ? p.s_sp : p.w_sp, word_ss = scaled ? p.s_ss : p.w_ss;

  for (int i0 = tile * kTile; i0 < count; i0 = APART ? count : i0 + kTile) {
    const int last = i0 + kTile < count ? i0 + kTile - 1 : count - 1;
    if (!APART && kept[last] == last) continue;  // (positions rise: every row of the tile is in its place)
    int at[DEEP], slot[DEEP], page[DEEP], to_slot[DEEP], to_page[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      const int i = i0 + u * kRows + group;
      at[u] = kept[i < count ? i : count - 1];
      to_page[u] = to_table[p.g.by_page.quotient(i < count ? i : count - 1, to_slot[u])];
      if (i >= count) to_page[u] = -1;
    }
    if (at[0] < 0) break;                        // (all of them: some page of the sequence is not here)
#pragma unroll
    for (int u = 0; u < DEEP; ++u) page[u] = table[p.g.by_page.quotient(at[u], slot[u])];
    u32x4 x[DEEP];
    uint32_t y[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      x[u] = u32x4{};
      y[u] = 0;
      if (real) x[u] = *reinterpret_cast<const u32x4*>(rows + (int64_t)page[u] * p.c_sp + (int64_t)slot[u] * p.c_ss);
    }
    if (scaled || weighted) {
#pragma unroll
      for (int u = 0; u < DEEP; ++u) y[u] = *reinterpret_cast<const uint32_t*>(word + (int64_t)page[u] * word_sp + (int64_t)slot[u] * word_ss);
    }
    if (!APART) {                                // what the tile writes over has been read by all
#pragma unroll
      for (int u = 0; u < DEEP; ++u) asm volatile("" : "+v"(x[u]), "+v"(y[u]));
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      if ((uint32_t)to_page[u] >= (uint32_t)p.g.pages) continue;
      if (real) *reinterpret_cast<u32x4*>(rows + (int64_t)to_page[u] * p.c_sp + (int64_t)to_slot[u] * p.c_ss) = x[u];
      if (scaled || weighted) *reinterpret_cast<uint32_t*>(word + (int64_t)to_page[u] * word_sp + (int64_t)to_slot[u] * word_ss) = y[u];
    }
  }
}

// Rows of a lane at once, us, 8 / 4: into other pages 32 x 3000 .. 8192 tokens e4m3 H8 D128 to 2048 95.6 / 74.5, bf16 137 / 134, one row of 64
// more than its 1024 5.3 / 4.0; in its own pages, where a tile is a round of its loads and a barrier, the first 52.2 / 64.4, 4 x 8192 to
// 8000 55.9 / 68.1.  With few (sequence, K/V head) pairs workgroups of 1024 threads: 1 x 8192 H8 bf16 to 4096 101 us with 256, 46.4 with 1024.
constexpr int kDeepApart = 4, kDeep = 8, kMovers = 256, kManyMovers = 1024;
int lanes_of(int row) { return row <= 64 ? 4 : row <= 128 ? 8 : 16; }
int64_t tiles_of(const Evict& p) {
  const int tile = kMovers / lanes_of(p.row) * kDeepApart;
  return p.out_table ? ((int64_t)p.limit + tile - 1) / tile : 1;
}
template <int LANES>
void move(const Evict& p, int64_t items, hipStream_t st) {
  const int tiles = (int)tiles_of(p);
  const dim3 grid((unsigned)(items * 2 * tiles));
  if (p.out_table) hipLaunchKernelGGL((paged_evict_move<LANES, kDeepApart, true, kMovers>), grid, dim3(kMovers), 0, st, p, tiles);
  else if (items <= 128) hipLaunchKernelGGL((paged_evict_move<LANES, kDeep, false, kManyMovers>), grid, dim3(kManyMovers), 0, st, p, tiles);
  else hipLaunchKernelGGL((paged_evict_move<LANES, kDeep, false, kMovers>), grid, dim3(kMovers), 0, st, p, tiles);
}

}  // namespace
}  // namespace mhip

using namespace mhip;

extern "C" int mhip_paged_cache_evict(void* k_cache, void* v_cache, void* k_scales, void* v_scales, const int* page_table, const int* out_table,
                                      const int* lengths, float* weights, int* kept, int* left,
                                      int B, int Hkv, int D, int pages, int page_size, int table_pages, int out_pages,
                                      int64_t t_sb, int64_t ot_sb, int keep, int recent, int limit,
                                      int64_t c_sp, int64_t c_ss, int64_t c_sh, int64_t s_sp, int64_t s_ss, int64_t s_sh,
                                      int64_t w_sp, int64_t w_ss, int64_t w_sh, int dtype, void* stream) {
  Evict p{};
  if (recent < 0 || keep < recent || limit < keep) return MHIP_EINVAL;
  if (int code = paged_geometry(p.g, page_table, lengths, nullptr, t_sb, B, 0, 0, pages, page_size, table_pages)) return code;
  if (int code = paged_cache_fits(k_cache, v_cache, k_scales, v_scales, pages, Hkv, D, c_sp, c_ss, c_sh, dtype)) return code;
  if (out_table && (out_pages < 0 || (int64_t)out_pages * page_size < limit)) return MHIP_EINVAL;
  if (reinterpret_cast<uintptr_t>(out_table) & 3u) return MHIP_EALIGN;
  if (B == 0) return MHIP_OK;
  if (!left || (limit > 0 && !kept) || (pages > 0 && !weights)) return MHIP_EINVAL;
  if ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(kept) | reinterpret_cast<uintptr_t>(left)) & 3u) return MHIP_EALIGN;
  if (limit > 0x7fff0000) return MHIP_EUNSUPPORTED;
  const int64_t items = (int64_t)B * Hkv;
  const int size = dtype == MHIP_BF16 ? 2 : 1;
  p.out_table = out_table; p.ot_sb = ot_sb;
  p.k = static_cast<uint8_t*>(k_cache); p.v = static_cast<uint8_t*>(v_cache);
  p.k_scales = dtype == MHIP_BF16 ? nullptr : static_cast<float*>(k_scales); p.v_scales = dtype == MHIP_BF16 ? nullptr : static_cast<float*>(v_scales);
  p.c_sp = c_sp * size; p.c_ss = c_ss * size; p.c_sh = c_sh * size;
  p.s_sp = s_sp; p.s_ss = s_ss; p.s_sh = s_sh;
  p.weights = weights;
  p.w_sp = w_sp; p.w_ss = w_ss; p.w_sh = w_sh;
  p.kept = kept; p.left = left;
  p.Hkv = Hkv; p.keep = keep; p.recent = recent; p.limit = limit;
  p.row = row_bytes(dtype, D);
  p.by_heads = Divisor(Hkv);
  if (!grid_fits(items, kChoosers) || !grid_fits(items * 2 * tiles_of(p), kMovers)) return MHIP_EUNSUPPORTED;
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(paged_evict_choose, dim3((unsigned)items), dim3(kChoosers), 0, st, p);
  if (limit > 0 && pages > 0) {
    if (lanes_of(p.row) == 4) move<4>(p, items, st);
    else if (lanes_of(p.row) == 8) move<8>(p, items, st);
    else move<16>(p, items, st);
  }
  return launch_status();
}
