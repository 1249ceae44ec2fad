// Rows of a paged K/V cache written (and quantised on the way) and read back as a dense chunk.
//
// Both move each row once and compute next to nothing: bound by memory, and by the launch for a step of generation.  16
// lanes take a row, 16 bytes of bf16 each, so that a wavefront has four rows and a CU some 30 KB of them in flight.
//
// An e4m3 row x is kept as codes and one scale s = 2^e, the least power of two from 2^-126 on with max|x| <= 448 s (1 for a
// row of zeros):  code = round-to-nearest-even e4m3(x / s).  With a power of two the division and, reading back, the product
// code * s are exact (s times four bits fits bf16), and the codes' relative step of 2^-4 is the same as with max|x| / 448;
// what it costs is at most one of the 18 binades below the largest value.  A row that holds an infinity or a NaN gets
// the scale NaN and codes of 0: it reads back as NaN, and attention sees that in the rows that see the key.
//
// An e2m1 row is the same 32 columns at a time: codes of four bits, rounded to nearest even by v_cvt_scalef32_pk_fp4_f32, and a byte
// for the least power of two from 2^-126 to 2^125 with max|x| <= 6 s; beyond, 6 * 2^125 is the largest that stays finite when it is read back.
#include "paged.hpp"

namespace mhip {
namespace {

struct RowsParams {
  PagedGeom g;
  uint8_t* k_cache; uint8_t* v_cache; float* k_scales; float* v_scales;
  int64_t c_sp, c_ss, c_sh;        // of the cache, bytes
  int64_t s_sp, s_ss, s_sh;        // of the scales, elements
  const uint16_t* k; const uint16_t* v;                    // write: the new rows
  int64_t k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
  uint16_t* out;                                           // read: the chunk
  int64_t o_half, o_sb, o_ss, o_sh;
  int total, begin, D;             // total: pairs of rows to move
  Divisor by_rows, by_head, by_new;
};

// Workgroup i runs on XCD i % 8.  The scales of neighbouring keys share a line, so with them each XCD gets a run of neighbouring rows
// (32768 rows read back 153.9 us to 150.8, 16403 tokens written 27.4 to 25.7; bf16 rows as they come, 46 MB read back in 11.2 us and 11.6).
template <int TYPE>
__device__ __forceinline__ int block_here() { return TYPE != MHIP_BF16 ? (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3) : blockIdx.x; }
int64_t blocks_of(int64_t total, int each) { return ((total + each - 1) / each + 7) & ~int64_t(7); }

// Largest of the lane's group of 16, 8 or 4, in all of its lanes.
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
  auto with = [](uint32_t v, auto ctrl) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, false);
    return other > v ? other : v;
  };
  x = with(x, std::integral_constant<int, 0xb1>{});      // the other of a pair
  x = with(x, std::integral_constant<int, 0x4e>{});      // the other pair of four
  if (LANES >= 8) x = with(x, std::integral_constant<int, 0x141>{});     // the other four of eight, mirrored
  if (LANES == 16) x = with(x, std::integral_constant<int, 0x128>{});          // the other eight of sixteen
  return x;
}

// LANES = 16, or 8 where a row has 64 columns or fewer.  The key and the value of a token and head lie in the same slot, so a group of
// lanes moves both with one look-up, and asks for them before it looks up (16403 tokens H8 D128: 36.9 us to 26.3).
template <int TYPE, int LANES>
__global__ __launch_bounds__(256) void paged_write_kernel(const RowsParams p) {
  const int lane = threadIdx.x & 63, col = (threadIdx.x % LANES) * 8;
  const int id = block_here<TYPE>() * (256 / LANES) + threadIdx.x / LANES;
  // pairs of rows in the order (token, head); lanes past the last one repeat it and store nothing
  int head, i = 0, b;
  const int token = p.by_head.quotient(id < p.total ? id : p.total - 1, head);
  bool real = id < p.total && col < p.D;
  const uint16_t *k = p.k + (int64_t)head * p.k_sh + col, *v = p.v + (int64_t)head * p.v_sh + col;
  if (p.g.starts) {
    k += (int64_t)token * p.k_ss;
    v += (int64_t)token * p.v_ss;
  } else {
    b = p.by_new.quotient(token, i);
    k += (int64_t)b * p.k_sb + (int64_t)i * p.k_ss;
    v += (int64_t)b * p.v_sb + (int64_t)i * p.v_ss;
  }
  u32x4 w[2] = {};
  if (real) {
    w[0] = *reinterpret_cast<const u32x4*>(k);
    w[1] = *reinterpret_cast<const u32x4*>(v);
  }
  if (p.g.starts) b = paged_owner<LANES>(p.g, token, lane);
  real = real && b < p.g.B;
  PagedSeq s{};
  if (b < p.g.B) s = paged_seq<false>(p.g, b);
  if (p.g.starts) {
    i = token - s.start;
    real = real && i >= 0 && i < s.n;
  }
  const int position = s.len - s.n + i;
  int slot = 0, page = -1;
  if (real && position >= 0) page = p.g.table[b * p.g.t_sb + p.g.by_page.quotient(position, slot)];
  real = real && page >= 0 && page < p.g.pages;
  const int64_t at = (int64_t)page * p.c_sp + (int64_t)slot * p.c_ss + (int64_t)head * p.c_sh;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint8_t* dst = (half ? p.v_cache : p.k_cache) + at;
    if constexpr (TYPE == MHIP_BF16) {
      if (real) *reinterpret_cast<u32x4*>(dst + col * 2) = w[half];
      continue;
    }
    // |x| of non-negative floats orders like the bits, and infinities and NaNs come out on top
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = w[half][j] << 16 & 0x7fffffffu, hi = w[half][j] & 0x7fff0000u, m = lo > hi ? lo : hi;
      top = m > top ? m : top;
    }
    const int64_t s_at = (int64_t)page * p.s_sp + (int64_t)slot * p.s_ss + (int64_t)head * p.s_sh;
    if constexpr (TYPE == MHIP_E2M1) {
      // (four lanes share 32 columns) 6 = 1.5 * 2^2: the least e is t - 2, one more if 1.f > 1.5
      top = group_max<4>(top);
      int power = (int)((top + 0x3fffffu) >> 23) - 2;
      power = top == 0 ? 127 : power < 1 ? 1 : power > 252 ? 252 : power;
      const bool finite = top < 0x7f800000u;
      uint32_t codes = 0;
      if (finite) {
        const float scale = e8m0((uint32_t)power);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, bf16_lo(w[half][0]), bf16_hi(w[half][0]), scale, 0);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, bf16_lo(w[half][1]), bf16_hi(w[half][1]), scale, 1);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, bf16_lo(w[half][2]), bf16_hi(w[half][2]), scale, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, bf16_lo(w[half][3]), bf16_hi(w[half][3]), scale, 3);
      }
      if (real) {
        *reinterpret_cast<uint32_t*>(dst + col / 2) = codes;
        if (col % 32 == 0) reinterpret_cast<uint8_t*>((half ? p.v_scales : p.k_scales) + s_at)[col / 32] = (uint8_t)(finite ? power : 255);
      }
      continue;
    }
    top = group_max<LANES>(top);
    // top = 1.f * 2^t with 1 <= 1.f < 2, and 448 = 1.75 * 2^8: the least e is t - 8, one more if 1.f > 1.75
    int power = (int)((top + 0x1fffffu) >> 23) - 8;        // + 127
    power = top == 0 ? 127 : power < 1 ? 1 : power;
    const bool finite = top < 0x7f800000u;
    const float scale = finite ? __builtin_bit_cast(float, (uint32_t)power << 23) : __builtin_nanf("");
    u32x2 codes{};
    if (finite) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          x[2 * j] = __builtin_ldexpf(bf16_lo(w[half][2 * h + j]), 127 - power);
          x[2 * j + 1] = __builtin_ldexpf(bf16_hi(w[half][2 * h + j]), 127 - power);
        }
        int packed = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        codes[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], packed, true);
      }
    }
    if (real) {
      *reinterpret_cast<u32x2*>(dst + col) = codes;
      if (col == 0)
        (half ? p.v_scales : p.k_scales)[s_at] = scale;
    }
  }
}

constexpr int kReadRows = 2;       // pairs of rows of a group of lanes, so that their loads are in flight together

// ONCE: a chunk that does not fit the last-level cache (256 MB) passes it by, and so do the rows: 537 MB of e4m3 rows as bf16 take 154 us
// so and 167 otherwise, 46 MB 13.5 and 11.1.
constexpr int64_t kLastLevel = int64_t(256) << 20;

template <int TYPE, int LANES, bool ONCE>
__global__ __launch_bounds__(256) void paged_read_kernel(const RowsParams p) {
  constexpr int kGroups = 256 / LANES;
  const int col = (threadIdx.x % LANES) * 8;
  if (col >= p.D) return;
  const int first = block_here<TYPE>() * (kGroups * kReadRows) + threadIdx.x / LANES;
  // keys and values of (sequence, row, head), in the chunk's order
  int b[kReadRows], i[kReadRows], head[kReadRows], page[kReadRows], slot[kReadRows];
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    const int id = first + kGroups * u;
    b[u] = p.by_rows.quotient(p.by_head.quotient(id < p.total ? id : 0, head[u]), i[u]);
    const int position = p.begin + i[u];
    page[u] = -1;
    slot[u] = 0;
    if (id < p.total && position < clamped(p.g.lengths[b[u]], 0, p.g.width * p.g.page))
      page[u] = p.g.table[b[u] * p.g.t_sb + p.g.by_page.quotient(position, slot[u])];
  }
  u32x4 w[kReadRows][2];
  u32x2 codes[kReadRows][2];
  float scale[kReadRows][2];
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    const int64_t at = (int64_t)page[u] * p.c_sp + (int64_t)slot[u] * p.c_ss + (int64_t)head[u] * p.c_sh;
    const int64_t s = (int64_t)page[u] * p.s_sp + (int64_t)slot[u] * p.s_ss + (int64_t)head[u] * p.s_sh;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      w[u][half] = u32x4{};
      codes[u][half] = u32x2{};
      scale[u][half] = 1.f;
    }
    if (page[u] >= 0 && page[u] < p.g.pages) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint8_t* src = (half ? p.v_cache : p.k_cache) + at;
        if constexpr (TYPE == MHIP_E2M1) {
          const uint32_t* from = reinterpret_cast<const uint32_t*>(src + col / 2);
          codes[u][half][0] = ONCE ? __builtin_nontemporal_load(from) : *from;
          scale[u][half] = e8m0(reinterpret_cast<const uint8_t*>((half ? p.v_scales : p.k_scales) + s)[col / 32]);
        } else if constexpr (TYPE == MHIP_E4M3) {
          const u32x2* from = reinterpret_cast<const u32x2*>(src + col);
          codes[u][half] = ONCE ? __builtin_nontemporal_load(from) : *from;
          scale[u][half] = (half ? p.v_scales : p.k_scales)[s];
        } else {
          const u32x4* from = reinterpret_cast<const u32x4*>(src + col * 2);
          w[u][half] = ONCE ? __builtin_nontemporal_load(from) : *from;
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    if (first + kGroups * u >= p.total) break;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if constexpr (TYPE == MHIP_E2M1) w[u][half] = e2m1_to_bf16(codes[u][half][0], scale[u][half]);
      if constexpr (TYPE == MHIP_E4M3) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t c = codes[u][half][h];
          const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
          w[u][half][2 * h] = pack_bf16(lo[0] * scale[u][half], lo[1] * scale[u][half]);
          w[u][half][2 * h + 1] = pack_bf16(hi[0] * scale[u][half], hi[1] * scale[u][half]);
        }
      }
      u32x4* to = reinterpret_cast<u32x4*>(p.out + half * p.o_half + b[u] * p.o_sb + i[u] * p.o_ss + head[u] * p.o_sh + col);
      if (ONCE) __builtin_nontemporal_store(w[u][half], to);
      else *to = w[u][half];
    }
  }
}

bool mult(int64_t x, int m) { return x % m == 0; }

void take_cache(RowsParams& p, const void* kc, const void* vc, const void* ks, const void* vs, int64_t c_sp, int64_t c_ss, int64_t c_sh,
                int64_t s_sp, int64_t s_ss, int64_t s_sh, int D, int dtype) {
  const int size = dtype == MHIP_BF16 ? 2 : 1;
  p.k_cache = static_cast<uint8_t*>(const_cast<void*>(kc)); p.v_cache = static_cast<uint8_t*>(const_cast<void*>(vc));
  p.k_scales = static_cast<float*>(const_cast<void*>(ks)); p.v_scales = static_cast<float*>(const_cast<void*>(vs));
  p.c_sp = c_sp * size; p.c_ss = c_ss * size; p.c_sh = c_sh * size;
  p.s_sp = s_sp; p.s_ss = s_ss; p.s_sh = s_sh;
  p.D = D;
}

}  // namespace

int paged_cache_fits(const void* kc, const void* vc, const void* ks, const void* vs, int pages, int Hkv, int D,
                     int64_t c_sp, int64_t c_ss, int64_t c_sh, int dtype) {
  if (dtype != MHIP_BF16 && dtype != MHIP_E4M3 && dtype != MHIP_E2M1) return MHIP_EDTYPE;
  if (Hkv <= 0) return MHIP_EINVAL;
  if (D <= 0 || D > 128 || row_bytes(dtype, D) % 16 || (dtype == MHIP_E2M1 && D % 32)) return MHIP_EHEADDIM;
  const bool scaled = dtype != MHIP_BF16;
  const int size = scaled ? 1 : 2, step = 16 / size;
  if (pages > 0 && (!kc || !vc || (scaled && (!ks || !vs)))) return MHIP_EINVAL;
  if (c_ss < row_bytes(dtype, D) / size || c_ss >= (int64_t(1) << 30) / 16 / size) return MHIP_EUNSUPPORTED;
  if (!aligned16(kc) || !aligned16(vc) || !mult(c_sp, step) || !mult(c_ss, step) || !mult(c_sh, step)) return MHIP_EALIGN;
  if (scaled && ((reinterpret_cast<uintptr_t>(ks) | reinterpret_cast<uintptr_t>(vs)) & 3u)) return MHIP_EALIGN;
  return MHIP_OK;
}

int paged_geometry(PagedGeom& g, const int* table, const int* lengths, const int* starts, int64_t t_sb, int B, int n, int T, int pages,
                   int page, int width) {
  if (B < 0 || n < 0 || T < 0 || pages < 0 || width < 0 || page <= 0) return MHIP_EINVAL;
  if (page % 16 != 0 || (int64_t)width * page > 0x7fff0000) return MHIP_EUNSUPPORTED;      // (positions a few tiles past the last key are ints)
  if (B > 0 && (!lengths || (width > 0 && !table))) return MHIP_EINVAL;
  if ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(starts)) & 3u) return MHIP_EALIGN;
  g.table = table; g.lengths = lengths; g.starts = starts;
  g.t_sb = t_sb;
  g.B = B; g.n = n; g.T = T;
  g.pages = pages; g.page = page; g.width = width;
  g.by_page = Divisor(page);
  return MHIP_OK;
}

}  // namespace mhip

using namespace mhip;

extern "C" int mhip_paged_cache_write(const void* k, const void* v, void* k_cache, void* v_cache, void* k_scales, void* v_scales,
                                      const int* page_table, const int* lengths, const int* starts,
                                      int B, int n, int T, int Hkv, int D, int pages, int page_size, int table_pages, int64_t t_sb,
                                      int64_t k_sb, int64_t k_ss, int64_t k_sh, int64_t v_sb, int64_t v_ss, int64_t v_sh,
                                      int64_t c_sp, int64_t c_ss, int64_t c_sh, int64_t s_sp, int64_t s_ss, int64_t s_sh,
                                      int dtype, void* stream) {
  RowsParams p{};
  if (B < 0 || n < 0 || T < 0) return MHIP_EINVAL;
  if (!starts && (int64_t)B * n > 0x7fffffff) return MHIP_EUNSUPPORTED;
  if (!starts) T = B * n;
  if (int code = paged_geometry(p.g, page_table, lengths, starts, t_sb, B, n, T, pages, page_size, table_pages)) return code;
  if (int code = paged_cache_fits(k_cache, v_cache, k_scales, v_scales, pages, Hkv, D, c_sp, c_ss, c_sh, dtype)) return code;
  if (T == 0 || B == 0 || pages == 0 || table_pages == 0) return MHIP_OK;
  if (!k || !v) return MHIP_EINVAL;
  if (!aligned16(k) || !aligned16(v)) return MHIP_EALIGN;
  for (int64_t s : {k_sb, k_ss, k_sh, v_sb, v_ss, v_sh})
    if (!mult(s, 8)) return MHIP_EALIGN;
  const bool wide = D > 64;
  const int groups = wide ? 16 : 32;
  const int64_t blocks = blocks_of((int64_t)T * Hkv, groups);
  if (!grid_fits(blocks, 256)) return MHIP_EUNSUPPORTED;       // (so T * Hkv is an int)
  take_cache(p, k_cache, v_cache, k_scales, v_scales, c_sp, c_ss, c_sh, s_sp, s_ss, s_sh, D, dtype);
  p.k = static_cast<const uint16_t*>(k); p.v = static_cast<const uint16_t*>(v);
  p.k_sb = k_sb; p.k_ss = k_ss; p.k_sh = k_sh;
  p.v_sb = v_sb; p.v_ss = v_ss; p.v_sh = v_sh;
  p.total = T * Hkv;
  p.by_head = Divisor(Hkv); p.by_new = Divisor(n);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks), block(256);
  auto launch = [&](auto type) {
    constexpr int T = decltype(type)::value;
    if (wide) hipLaunchKernelGGL((paged_write_kernel<T, 16>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((paged_write_kernel<T, 8>), grid, block, 0, st, p);
  };
  if (dtype == MHIP_E2M1) launch(std::integral_constant<int, MHIP_E2M1>{});
  else if (dtype == MHIP_E4M3) launch(std::integral_constant<int, MHIP_E4M3>{});
  else launch(std::integral_constant<int, MHIP_BF16>{});
  return launch_status();
}

extern "C" int mhip_paged_cache_read(const void* k_cache, const void* v_cache, const void* k_scales, const void* v_scales,
                                     const int* page_table, const int* lengths, void* out,
                                     int B, int begin, int rows, int Hkv, int D, int pages, int page_size, int table_pages, int64_t t_sb,
                                     int64_t c_sp, int64_t c_ss, int64_t c_sh, int64_t s_sp, int64_t s_ss, int64_t s_sh,
                                     int64_t o_half, int64_t o_sb, int64_t o_ss, int64_t o_sh, int dtype, void* stream) {
  RowsParams p{};
  if (begin < 0 || rows < 0 || (int64_t)begin + rows > 0x7fffffff) return MHIP_EINVAL;
  if (int code = paged_geometry(p.g, page_table, lengths, nullptr, t_sb, B, 0, 0, pages, page_size, table_pages)) return code;
  if (int code = paged_cache_fits(k_cache, v_cache, k_scales, v_scales, pages, Hkv, D, c_sp, c_ss, c_sh, dtype)) return code;
  if (B == 0 || rows == 0) return MHIP_OK;
  if (!out) return MHIP_EINVAL;
  if (!aligned16(out)) return MHIP_EALIGN;
  for (int64_t s : {o_half, o_sb, o_ss, o_sh})
    if (!mult(s, 8)) return MHIP_EALIGN;
  if ((double)B * rows * 2 * Hkv >= 2147483648.0 - 256) return MHIP_EUNSUPPORTED;
  const bool wide = D > 64;
  const int groups = (wide ? 16 : 32) * kReadRows;
  const int64_t blocks = blocks_of((int64_t)B * rows * Hkv, groups);
  if (!grid_fits(blocks, 256)) return MHIP_EUNSUPPORTED;
  take_cache(p, k_cache, v_cache, k_scales, v_scales, c_sp, c_ss, c_sh, s_sp, s_ss, s_sh, D, dtype);
  p.out = static_cast<uint16_t*>(out);
  p.o_half = o_half; p.o_sb = o_sb; p.o_ss = o_ss; p.o_sh = o_sh;
  p.total = B * rows * Hkv;
  p.begin = begin;
  p.by_head = Divisor(Hkv); p.by_rows = Divisor(rows);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)blocks), block(256);
  const bool once = (int64_t)p.total * D * 4 > kLastLevel;
  auto launch = [&](auto lanes, auto past) {
    constexpr int L = decltype(lanes)::value;
    constexpr bool O = decltype(past)::value;
    if (dtype == MHIP_E2M1) hipLaunchKernelGGL((paged_read_kernel<MHIP_E2M1, L, O>), grid, block, 0, st, p);
    else if (dtype == MHIP_E4M3) hipLaunchKernelGGL((paged_read_kernel<MHIP_E4M3, L, O>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((paged_read_kernel<MHIP_BF16, L, O>), grid, block, 0, st, p);
  };
  using std::integral_constant;
  if (wide && once) launch(integral_constant<int, 16>{}, std::true_type{});
  else if (wide) launch(integral_constant<int, 16>{}, std::false_type{});
  else if (once) launch(integral_constant<int, 8>{}, std::true_type{});
  else launch(integral_constant<int, 8>{}, std::false_type{});
  return launch_status();
}
