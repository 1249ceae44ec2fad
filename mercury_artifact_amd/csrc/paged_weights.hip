// What attention each key of a paged K/V cache has had:
//     w_j <- decay * w_j + sum over the new tokens i and the query heads h of the K/V head of exp(scale * q_ih k_j - lse_ih),
// with the lse that attention left, and nothing of the old w_j for a new token's own key.
//
// paged_weights_few: bound by memory, a key's row is read once.  No softmax is left to do, so keys are independent of one another: a
// wavefront takes a run of units of 32 (bf16) or 64 keys, whose rows go from memory into registers as the B operand of S = Q K^T
// (v_mfma_f32_16x16x32_bf16) while the queries (A) stay in registers for the run.  Lane (ln, lg) then holds rows 4 lg .. +3 of key ln: their
// exponentials are added in the lane and over the four lane groups.  The units of all sequences are dealt out evenly to 16 wavefronts on
// every CU, whose loads are in flight together; no LDS, no barrier, no atomics, so that results are the same in every run.
#include "paged.hpp"

#include <math.h>

namespace mhip {
namespace {

struct Gather {
  PagedGeom g;
  const uint8_t* k; const float* k_scales;       // (e2m1: four bytes of scales in a float's place)
  int64_t c_sp, c_ss, c_sh;                      // of the cache, bytes
  int64_t s_sp, s_ss, s_sh;                      // of the scales, four bytes
  const uint16_t* q; const float* lse;
  int64_t q_sb, q_ss, q_sh, l_sb, l_sh;
  const float* old; float* out;
  int64_t w_sp, w_ss, w_sh, o_sp, o_ss, o_sh;
  int Hkv, G, D, causal;
  float scale_log2, decay;
  Divisor by_group;
};

constexpr int kWorkers = 4096;                   // wavefronts of a launch: 16 on a CU

template <int TYPE>
constexpr int kBlocksOf = TYPE == MHIP_BF16 ? 2 : 4;       // 16-key blocks of a unit

template <int UNIT>
__device__ __forceinline__ int64_t units_of(const Gather& p, const PagedSeq& s) { return (int64_t)((s.len + UNIT - 1) / UNIT) * p.Hkv; }

template <int TYPE, int COLS, int NR>
__global__ __launch_bounds__(256, 4) void paged_weights_few(const Gather p) {
  constexpr int kBlocks = kBlocksOf<TYPE>, UNIT = 16 * kBlocks, ROWS = 16 * NR;
  constexpr bool E4M3 = TYPE == MHIP_E4M3, E2M1 = TYPE == MHIP_E2M1;
  constexpr int KB = COLS / 32, KR = E2M1 ? 1 : E4M3 ? KB / 2 : KB;      // k-steps of 32 columns, loads of a key's row
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, lg = lane >> 4;

  // ---- this wavefront's share of the units: those before each lane's run of sequences, and of all ---------------------------
  const int w = ((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) * 4 + wave, workers = gridDim.x * 4;
  const int per = (p.g.B + 63) / 64;
  int64_t mine = 0;
  for (int j = 0; j < per; ++j)
    if (lane * per + j < p.g.B) mine += units_of<UNIT>(p, paged_seq<false>(p.g, lane * per + j));
  int64_t before = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t below = __shfl_up((long long)before, off);
    if (lane >= off) before += below;
  }
  const int64_t total = uniform64(__shfl((long long)before, 63)), shares = total < workers ? total : workers;
  before -= mine;
  if (w >= shares) return;
  int64_t lo = total * w / shares;
  const int64_t hi = total * (w + 1) / shares;
  const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lo >= before && lo < before + mine));
  int b = owner * per;
  int64_t pos = lo - uniform64(__shfl((long long)before, owner));        // inside sequence b
  for (int64_t u; b + 1 < p.g.B && pos >= (u = units_of<UNIT>(p, paged_seq<true>(p.g, b))); ++b) pos -= u;

  const int k_block = COLS == 128 ? lg : lg >> 1;                        // (e2m1: the 32 columns that the lane's are of)
  auto col_of = [&](int ks) { return E2M1 ? (lg * KB + ks) * 8 : E4M3 ? (ks >> 1) * 64 + lg * 16 + (ks & 1) * 8 : ks * 32 + lg * 8; };
  auto mfma = [](const bf16x8& x, const bf16x8& y, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0); };

  while (lo < hi) {
    const PagedSeq s = paged_seq<true>(p.g, b);
    const int tiles = (s.len + UNIT - 1) / UNIT, rows = s.n * p.G;
    if (tiles == 0 || pos >= (int64_t)tiles * p.Hkv) {
      pos -= (int64_t)tiles * p.Hkv;
      ++b;
      continue;
    }
    const int hk = (int)(pos / tiles), t0 = (int)(pos - (int64_t)hk * tiles);
    const int run = (int)(tiles - t0 < hi - lo ? tiles - t0 : hi - lo);
    lo += run;
    pos += run;
    const int old_keys = s.len - s.n;                                    // (below 0: more new tokens than keys)
    const bool reads_old = s.n == 0 || p.decay != 0.f;
    const float decay = s.n == 0 ? 1.f : p.decay;
    const int* table = p.g.table + b * p.g.t_sb;

    // ---- a tile of rows: A operand, and of rows 4 lg + j what is taken from their scores and how many keys they see ------------
    bf16x8 qf[NR][KB];
    float nlse[NR][4];
    int lim[NR][4];
    auto load_rows = [&](int row0) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const int row = row0 + r * 16 + ln;
        int of_group;
        const int token = p.by_group.quotient(row < rows ? row : 0, of_group);
        const uint16_t* src = p.q + b * p.q_sb + (int64_t)(s.start + token) * p.q_ss + (hk * p.G + of_group) * p.q_sh;
#pragma unroll
        for (int ks = 0; ks < KB; ++ks) {
          qf[r][ks] = bf16x8{};
          if (row < rows && col_of(ks) < p.D) qf[r][ks] = *reinterpret_cast<const bf16x8*>(src + col_of(ks));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = row0 + r * 16 + 4 * lg + j;
          int head;
          const int t = p.by_group.quotient(at < rows ? at : 0, head);
          lim[r][j] = 0;
          nlse[r][j] = 0.f;
          if (at < rows) {
            const float lse = p.lse[b * p.l_sb + (hk * p.G + head) * p.l_sh + s.start + t];
            lim[r][j] = p.causal ? clamped(old_keys + t + 1, 0, s.len) : s.len;
            nlse[r][j] = -lse * kLog2e;
            if (lse == -INFINITY) lim[r][j] = 0;                         // (a row that saw no key)
          }
        }
      }
    };
    if (rows <= ROWS) load_rows(0);

    for (int t = t0; t < t0 + run; ++t) {
      const int key0 = t * UNIT;
      u32x4 w4[kBlocks][KR];
      float mult[kBlocks];
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const int key = key0 + 16 * i;
        int slot = 0, page = -1;
        if (key < s.len) page = uniform_load(table, p.g.by_page.quotient(key, slot));
        mult[i] = p.scale_log2;
#pragma unroll
        for (int u = 0; u < KR; ++u) w4[i][u] = u32x4{};
        if ((uint32_t)page < (uint32_t)p.g.pages) {
          const uint8_t* row = p.k + (int64_t)page * p.c_sp + (int64_t)(slot + ln) * p.c_ss + (int64_t)hk * p.c_sh;
          const float* scale = p.k_scales + ((int64_t)page * p.s_sp + (int64_t)(slot + ln) * p.s_ss + (int64_t)hk * p.s_sh);
          if constexpr (E2M1) {
            if (k_block * 32 < p.D) {
              if constexpr (COLS == 128) w4[i][0] = *reinterpret_cast<const u32x4*>(row + lg * 16);
              else {
                const u32x2 x = *reinterpret_cast<const u32x2*>(row + lg * 8);
                w4[i][0][0] = x[0];
                w4[i][0][1] = x[1];
              }
              mult[i] = e8m0(reinterpret_cast<const uint8_t*>(scale)[k_block]);
            } else {
              mult[i] = 1.f;
            }
          } else {
            if constexpr (E4M3) mult[i] = *scale;
#pragma unroll
            for (int u = 0; u < KR; ++u)
              if ((u * 4 + lg) * 16 < row_bytes(TYPE, p.D)) w4[i][u] = *reinterpret_cast<const u32x4*>(row + (u * 4 + lg) * 16);
          }
        }
      }
      // the lane's own key, key0 + lane: what it had, and where it goes
      const int own = key0 + lane;
      int own_slot = 0, own_page = -1;
      if (lane < UNIT && own < s.len) own_page = table[p.g.by_page.quotient(own, own_slot)];
      const bool held = (uint32_t)own_page < (uint32_t)p.g.pages;
      float had = 0.f;
      if (held && reads_old && own < (s.n == 0 ? s.len : old_keys))
        had = decay * p.old[(int64_t)own_page * p.w_sp + (int64_t)own_slot * p.w_ss + (int64_t)hk * p.w_sh];

      float sum[kBlocks] = {};
      for (int row0 = 0; row0 < rows; row0 += ROWS) {
        const int row_end = row0 + ROWS < rows ? row0 + ROWS : rows;
        if (p.causal && key0 > old_keys + p.by_group.quotient(row_end - 1)) continue;       // nobody sees any of them
        if (rows > ROWS) load_rows(row0);
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
          f32x4 sc[NR];
#pragma unroll
          for (int ks = 0; ks < KB; ++ks) {
            bf16x8 kf;
            if constexpr (E2M1) kf = __builtin_bit_cast(bf16x8, e2m1_to_bf16(w4[i][0][ks], mult[i]));
            else if constexpr (E4M3) kf = e4m3_to_bf16(w4[i][ks >> 1][2 * (ks & 1)], w4[i][ks >> 1][2 * (ks & 1) + 1]);
            else kf = __builtin_bit_cast(bf16x8, w4[i][ks]);
#pragma unroll
            for (int r = 0; r < NR; ++r) sc[r] = mfma(qf[r][ks], kf, ks == 0 ? f32x4{} : sc[r]);
          }
          const float times = E4M3 ? p.scale_log2 * mult[i] : p.scale_log2;
          const int key = key0 + 16 * i + ln;
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float x = fast_exp2(__builtin_fmaf(sc[r][j], times, nlse[r][j]));
              sum[i] += key < lim[r][j] ? x : 0.f;
            }
        }
      }
      float all = 0.f;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const float x = quad_sum(sum[i]);
        if (lg == i) all = x;
      }
      if (held) p.out[(int64_t)own_page * p.o_sp + (int64_t)own_slot * p.o_ss + (int64_t)hk * p.o_sh] = had + all;
    }
  }
}

template <int TYPE, int COLS, int NR>
void launch_few(const Gather& p, hipStream_t st) {
  hipLaunchKernelGGL((paged_weights_few<TYPE, COLS, NR>), dim3(kWorkers / 4), dim3(256), 0, st, p);
}
template <int TYPE, int COLS>
void launch_rows(const Gather& p, int64_t rows, hipStream_t st) {
  if (rows <= 16) launch_few<TYPE, COLS, 1>(p, st);
  else launch_few<TYPE, COLS, 2>(p, st);
}
template <int TYPE>
void launch(const Gather& p, int64_t rows, hipStream_t st) {
  if (p.D <= 64) launch_rows<TYPE, 64>(p, rows, st);
  else launch_rows<TYPE, 128>(p, rows, st);
}

}  // namespace
}  // namespace mhip

using namespace mhip;

extern "C" int mhip_paged_attn_weights(const void* q, const void* k_cache, const void* k_scales, const int* page_table, const int* lengths,
                                       const int* starts, const float* lse, const float* weights, float* out,
                                       int B, int n, int T, int most_new, int Hq, int Hkv, int D, int pages, int page_size, int table_pages,
                                       int64_t t_sb, int64_t q_sb, int64_t q_ss, int64_t q_sh,
                                       int64_t c_sp, int64_t c_ss, int64_t c_sh, int64_t s_sp, int64_t s_ss, int64_t s_sh,
                                       int64_t w_sp, int64_t w_ss, int64_t w_sh, int64_t o_sp, int64_t o_ss, int64_t o_sh,
                                       float softmax_scale, float decay, int mask, int dtype, void* stream) {
  Gather p{};
  if (B < 0 || n < 0 || T < 0 || most_new < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return MHIP_EINVAL;
  if (!(softmax_scale > 0.f) || !(softmax_scale < INFINITY)) return MHIP_EINVAL;
  if (!(decay >= 0.f) || !(decay < INFINITY)) return MHIP_EINVAL;
  if (mask != MHIP_MASK_NONE && mask != MHIP_MASK_CAUSAL) return MHIP_EINVAL;
  if (!starts && (int64_t)B * n > 0x7fffffff) return MHIP_EUNSUPPORTED;
  if (!starts) { T = B * n; most_new = n; }
  if (int code = paged_geometry(p.g, page_table, lengths, starts, t_sb, B, n, T, pages, page_size, table_pages)) return code;
  if (int code = paged_cache_fits(k_cache, k_cache, k_scales, k_scales, pages, Hkv, D, c_sp, c_ss, c_sh, dtype)) return code;
  if (B == 0 || pages == 0 || table_pages == 0) return MHIP_OK;
  if (!weights || !out || (T > 0 && (!q || !lse))) return MHIP_EINVAL;
  if (!aligned16(q) || ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(out)) & 3u)) return MHIP_EALIGN;
  for (int64_t x : {q_sb, q_ss, q_sh})
    if (x % 8 != 0) return MHIP_EALIGN;
  if ((int64_t)T * Hq >= (int64_t(1) << 31) - 256) return MHIP_EUNSUPPORTED;       // (rows, up to a whole tile of them, are ints)
  const int size = dtype == MHIP_BF16 ? 2 : 1;
  p.k = static_cast<const uint8_t*>(k_cache); p.k_scales = static_cast<const float*>(k_scales);
  p.c_sp = c_sp * size; p.c_ss = c_ss * size; p.c_sh = c_sh * size;
  p.s_sp = s_sp; p.s_ss = s_ss; p.s_sh = s_sh;
  p.q = static_cast<const uint16_t*>(q); p.lse = lse;
  p.q_sb = starts ? 0 : q_sb; p.q_ss = q_ss; p.q_sh = q_sh;
  p.l_sb = starts ? 0 : (int64_t)Hq * n; p.l_sh = starts ? T : n;
  p.old = weights; p.out = out;
  p.w_sp = w_sp; p.w_ss = w_ss; p.w_sh = w_sh;
  p.o_sp = o_sp; p.o_ss = o_ss; p.o_sh = o_sh;
  p.Hkv = Hkv; p.G = Hq / Hkv; p.D = D;
  p.causal = mask == MHIP_MASK_CAUSAL;
  p.scale_log2 = softmax_scale * kLog2e;
  p.decay = decay;
  p.by_group = Divisor(p.G);
  const int64_t rows = (int64_t)most_new * p.G;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MHIP_E2M1) launch<MHIP_E2M1>(p, rows, st);
  else if (dtype == MHIP_E4M3) launch<MHIP_E4M3>(p, rows, st);
  else launch<MHIP_BF16>(p, rows, st);
  return launch_status();
}
