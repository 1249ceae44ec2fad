// A paged K/V cache that stays within a budget.  A sequence of more than `limit` tokens is cut to `keep`: each K/V head keeps the keys
// of its `recent` last tokens and, of the others, the keep - recent with the largest weights (of equal ones the first), in their order.
//
// paged_evict_choose: one workgroup for each (sequence, K/V head).  The weights are looked at as whole numbers that order like them: the
//   number that the last kept one has is found eight bits at a time, by counting (the largest first), and a pass in order then
//   leaves the positions that stay, each at its place in the result.
// paged_evict_move: rows that stay, with scales and weights, to their new places.  In its own pages a row moves down or not at all, so a
//   workgroup that reads a tile of rows whole, and then writes it, has read whatever it writes over, and rows of later tiles
//   lie behind everything that it writes: one workgroup walks each (sequence, K/V head, half) from the first row on.  Into other
//   pages rows are independent, and many workgroups share them.
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

__global__ __launch_bounds__(kChoosers) void paged_evict_choose(const Evict p) {
  __shared__ uint32_t count[kChooserWaves][256];
  __shared__ uint32_t found[2];                  // the digit, and how many of it are kept
  __shared__ int waves[2][kChooserWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
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
  auto order_at = [&](int at) {
    int slot;
    const int page = table[p.g.by_page.quotient(at, slot)];
    return order_of(p.weights[(int64_t)page * p.w_sp + (int64_t)slot * p.w_ss + (int64_t)hk * p.w_sh]);
  };

  // ---- the number of the last one kept, and how many of that number are ------------------------------------------------------
  const int others = len - p.recent;             // (recent <= keep <= limit < len)
  uint32_t need = p.keep - p.recent, last = 0;
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < kChooserWaves * 256; i += kChoosers) (&count[0][0])[i] = 0;
      __syncthreads();
      for (int at = tid; at < others; at += kChoosers) {
        const uint32_t x = order_at(at);
        if (shift == 24 || (x ^ last) >> (shift + 8) == 0) atomicAdd(&count[wave][x >> shift & 255u], 1u);
      }
      __syncthreads();
      if (tid < 256) {
        uint32_t sum = 0;
        for (int v = 0; v < kChooserWaves; ++v) sum += count[v][tid];
        count[0][tid] = sum;
      }
      __syncthreads();
      if (wave == 0) {
        // lane l has the digits 255 - 4 l .. 252 - 4 l: how many are above them, and in which of them the last one kept is
        uint32_t c[4], sum = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += c[e] = count[0][255 - 4 * lane - e];
        uint32_t above = sum;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const uint32_t x = __shfl_up(above, off);
          if (lane >= off) above += x;
        }
        above -= sum;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (above < need && need <= above + c[e]) {
            found[0] = 255 - 4 * lane - e;
            found[1] = need - above;
          }
          above += c[e];
        }
      }
      __syncthreads();
      last |= found[0] << shift;
      need = found[1];
      __syncthreads();
    }
  }

  // ---- the positions in order: those above, and of those equal the first `need` ------------------------------------------------
  int above = 0, equal = 0;
  if (p.keep > p.recent) {
    for (int at0 = 0; at0 < others; at0 += kChoosers) {
      const int at = at0 + tid;
      const uint32_t x = at < others ? order_at(at) : 0;
      const bool is_above = at < others && x > last, is_equal = at < others && x == last;
      const uint64_t mask_above = __builtin_amdgcn_ballot_w64(is_above), mask_equal = __builtin_amdgcn_ballot_w64(is_equal);
      if (lane == 0) {
        waves[0][wave] = __builtin_popcountll(mask_above);
        waves[1][wave] = __builtin_popcountll(mask_equal);
      }
      __syncthreads();
      int here_above = above, here_equal = equal;
      for (int v = 0; v < kChooserWaves; ++v) {
        if (v < wave) {
          here_above += waves[0][v];
          here_equal += waves[1][v];
        }
        above += waves[0][v];
        equal += waves[1][v];
      }
      const uint64_t below = (1ull << lane) - 1;
      here_above += __builtin_popcountll(mask_above & below);
      here_equal += __builtin_popcountll(mask_equal & below);
      if (is_above || (is_equal && here_equal < (int)need)) kept[here_above + (here_equal < (int)need ? here_equal : (int)need)] = at;
      __syncthreads();
    }
  }
  for (int i = tid; i < p.limit - (p.keep - p.recent); i += kChoosers) kept[p.keep - p.recent + i] = i < p.recent ? others + i : -1;
}

constexpr int kMovers = 256;

// LANES lanes take a row, of up to 16 bytes each; a workgroup moves 256 / LANES rows at once and `DEEP` times as many with their loads in flight together.
template <int LANES, int DEEP, bool APART>
__global__ __launch_bounds__(kMovers) void paged_evict_move(const Evict p, const int tiles) {
  constexpr int kRows = kMovers / LANES, kTile = kRows * DEEP;
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
  uint8_t* rows = half ? p.v : p.k;
  float* scales = half ? p.v_scales : p.k_scales;
  const bool real = sub * 16 < p.row;

  for (int i0 = tile * kTile; i0 < count; i0 = APART ? count : i0 + kTile) {
    const int last = i0 + kTile < count ? i0 + kTile - 1 : count - 1;
    if (!APART && kept[last] == last) continue;  // (positions rise: every row of the tile is in its place)
    u32x4 x[DEEP];
    float scale[DEEP], weight[DEEP];
    int64_t to_page[DEEP];
    int to_slot[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      const int i = i0 + u * kRows + group;
      const int at = i < count ? kept[i] : -1;
      to_page[u] = -1;
      x[u] = u32x4{};
      scale[u] = weight[u] = 0.f;
      if (at >= 0) {
        int slot;
        const int64_t page = table[p.g.by_page.quotient(at, slot)];
        const int to = to_table[p.g.by_page.quotient(i, to_slot[u])];
        if ((uint32_t)to < (uint32_t)p.g.pages) to_page[u] = to;
        if (real) x[u] = *reinterpret_cast<const u32x4*>(rows + page * p.c_sp + (int64_t)slot * p.c_ss + (int64_t)hk * p.c_sh + sub * 16);
        if (sub == 0 && scales) scale[u] = scales[page * p.s_sp + (int64_t)slot * p.s_ss + (int64_t)hk * p.s_sh];
        if (sub == 0 && half == 0) weight[u] = p.weights[page * p.w_sp + (int64_t)slot * p.w_ss + (int64_t)hk * p.w_sh];
      }
    }
    if (!APART) {                                // what the tile writes over has been read by all
#pragma unroll
      for (int u = 0; u < DEEP; ++u) asm volatile("" : "+v"(x[u]), "+v"(scale[u]), "+v"(weight[u]));
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < DEEP; ++u) {
      if (to_page[u] < 0) continue;
      if (real) *reinterpret_cast<u32x4*>(rows + to_page[u] * p.c_sp + (int64_t)to_slot[u] * p.c_ss + (int64_t)hk * p.c_sh + sub * 16) = x[u];
      if (sub == 0 && scales) scales[to_page[u] * p.s_sp + (int64_t)to_slot[u] * p.s_ss + (int64_t)hk * p.s_sh] = scale[u];
      if (sub == 0 && half == 0) p.weights[to_page[u] * p.w_sp + (int64_t)to_slot[u] * p.w_ss + (int64_t)hk * p.w_sh] = weight[u];
    }
  }
}

constexpr int kDeep = 8;
int lanes_of(int row) { return row <= 64 ? 4 : row <= 128 ? 8 : 16; }
int64_t tiles_of(const Evict& p) {
  const int tile = kMovers / lanes_of(p.row) * kDeep;
  return p.out_table ? ((int64_t)p.limit + tile - 1) / tile : 1;
}
template <int LANES>
void move(const Evict& p, int64_t items, hipStream_t st) {
  const int tiles = (int)tiles_of(p);
  const dim3 grid((unsigned)(items * 2 * tiles));
  if (p.out_table) hipLaunchKernelGGL((paged_evict_move<LANES, kDeep, true>), grid, dim3(kMovers), 0, st, p, tiles);
  else hipLaunchKernelGGL((paged_evict_move<LANES, kDeep, false>), grid, dim3(kMovers), 0, st, p, tiles);
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
