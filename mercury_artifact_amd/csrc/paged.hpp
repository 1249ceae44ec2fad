// What the kernels over a paged K/V cache share: where the rows of a sequence lie.
//
// Key (value) j of sequence b lies in slot j % page of page table[b][j / page] of the cache.  A table entry outside
// [0, pages) says that the page is not here -- freed, or on another rank: its keys are seen by nobody, rows written to it
// are dropped and rows read from it are zeros.  lengths[b] counts the keys of a sequence with its new tokens, which are the
// last ones; the kernels read lengths, table and starts from device memory when they run, so a captured graph follows them,
// and take every value of them without leaving the tensors: a length counts as one from 0 to what a table row holds, a
// start as one from 0 to T.
#pragma once

#include "mhip_common.hpp"

namespace mhip {

struct PagedGeom {
  const int* table; const int* lengths; const int* starts;     // starts: NULL where every sequence has n new tokens
  int64_t t_sb;                    // entries from one sequence's table row to the next one's
  int B, n, T;                     // sequences, new tokens of each, new tokens of all
  int pages, page, width;          // pages of the cache, their rows, entries of a table row (width * page <= 2^31 - 2^16)
  Divisor by_page;
};

// New tokens of a sequence: rows start .. start + n - 1 of the packed tensors (of its own batch entry without starts), at
// positions len - n .. len - 1.
struct PagedSeq { int start, n, len; };

// A value that earlier work left in memory, through the scalar cache where the index is wavefront-uniform.
__device__ __forceinline__ int uniform_load(const int* p, int64_t i) {
  return ((__attribute__((address_space(4))) const int*)(uintptr_t)p)[i];
}
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32);
}
__device__ __forceinline__ int clamped(int x, int low, int high) { return x < low ? low : x > high ? high : x; }

template <bool UNIFORM>
__device__ __forceinline__ PagedSeq paged_seq(const PagedGeom& g, int b) {
  auto get = [&](const int* p, int64_t i) { return UNIFORM ? uniform_load(p, i) : p[i]; };
  PagedSeq s;
  s.len = clamped(get(g.lengths, b), 0, g.width * g.page);
  s.start = 0;
  s.n = g.n;
  if (g.starts) {
    s.start = clamped(get(g.starts, b), 0, g.T);
    s.n = clamped(get(g.starts, b + 1), s.start, g.T) - s.start;
  }
  return s;
}

// The sequence that packed row t belongs to: as many sequences end at or before it.  Called by whole wavefronts, each of
// whose groups of `LANES` lanes has a t of its own; B where there is none.
template <int LANES>
__device__ __forceinline__ int paged_owner(const PagedGeom& g, int t, int lane) {
  const int sub = lane % LANES, shift = lane - sub;
  const uint64_t mine = LANES == 64 ? ~0ull : ((1ull << (LANES % 64)) - 1) << shift;
  int b = 0;
  for (int at = 0; at < g.B; at += LANES) {
    const bool before = at + sub < g.B && g.starts[at + sub + 1] <= t;
    b += __builtin_popcountll(__builtin_amdgcn_ballot_w64(before) & mine);
  }
  return b;
}

// Bytes of a row of the cache, and four fp4 scales of a row, a byte each: that of 32 columns as an fp32 power of two, exact from 2^-126 on.
constexpr int row_bytes(int type, int D) { return type == MHIP_BF16 ? 2 * D : type == MHIP_E4M3 ? D : D / 2; }
__device__ __forceinline__ float e8m0(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Eight e4m3 codes as bf16, exact.
__device__ __forceinline__ bf16x8 e4m3_to_bf16(uint32_t a, uint32_t c) {
  const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false), x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true);
  const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, false), x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, true);
  return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

// Eight e2m1 codes of a dword, times a scale that is a power of two, as bf16: exact while they are normal numbers there; a scale with
// the exponent 255 makes them NaN, and one with the exponent 0 counts as 2^-127.
__device__ __forceinline__ u32x4 e2m1_to_bf16(uint32_t codes, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
}

// Rows (new tokens times query heads) of a sequence and K/V head that the kernels for few rows take, attention's and weights' alike, and the tile
// of 16, 32 or 64 that holds so many.
constexpr int kFewRows = 64;
constexpr int few_tile(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

// What the entry points ask of tables, lengths and starts, and of the cache: MHIP_OK, or the code to return.
int paged_geometry(PagedGeom& g, const int* table, const int* lengths, const int* starts, int64_t t_sb, int B, int n, int T, int pages,
                   int page, int width);
int paged_cache_fits(const void* kc, const void* vc, const void* ks, const void* vs, int pages, int Hkv, int D,
                     int64_t c_sp, int64_t c_ss, int64_t c_sh, int dtype);

}  // namespace mhip
