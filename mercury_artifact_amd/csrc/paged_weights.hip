// What attention each key of a paged K/V cache has had:
//     w_j <- decay * w_j + sum over the new tokens i and the query heads h of the K/V head of exp(scale * q_ih k_j - lse_ih),
// with the lse that attention left, and nothing of the old w_j for a new token's own key.
//
// paged_weights_few: bound by memory, a key's row is read once.  No softmax is left to do, so keys are independent of one another: a
// wavefront takes a run of units of 32 (bf16) or 64 keys, whose rows go from memory into registers as the B operand of S = Q K^T
// (v_mfma_f32_16x16x32_bf16) while the queries (A) stay in registers for the run.  Lane (ln, lg) then holds rows 4 lg .. +3 of key ln: their
// exponentials are added in the lane and over the four lane groups.  The units of all sequences are dealt out evenly to 16 (e4m3 12; 8 with
// more than 16 rows) wavefronts on every CU, and a unit's loads go out together (4 x 131072 in e2m1, waiting for each scale byte in
// turn, 93 us, 83 so); no LDS, no barrier, no atomics, so that results are the same in every run.
//
// paged_weights_many: for prompts, bound by the vector unit (an exponential, a multiply-add and an add for each 2 D operations of the matrix
// unit).  Here the keys stay: a workgroup of four wavefronts holds 256 of a (sequence, K/V head), 64 to a wavefront, as the A operand of
// S^T = K Q^T (v_mfma_f32_32x32x16_bf16), and tiles of 32 queries come through a ring in LDS, copied there without passing through
// registers; each operand read from LDS feeds two MFMAs (with 32 keys to a wavefront, four wavefronts on a SIMD, a prompt of 8192
// tokens H32/8 takes 292 us on 128 columns and 203 on 64, so 280 and 219).
// Lane (ln, lg) holds query ln, its keys' weights are added in registers, and over the lanes once in 64 tiles (which keeps the sums short: 64
// in a row, then 32 as a tree).  The exponentials of a tile stand between the MFMAs of the next one.  The tiles that see a key differ with
// the mask, so the tiles of all items are counted in closed form and dealt out evenly, in order; a workgroup whose share ends inside an
// item leaves partial sums, and paged_weights_join adds those up in their order.
//
// Measured, us: a step of 32 x 300 .. 16384 tokens H32/8 D128 in bf16 122 (4.8 TB/s of keys and weights); 64 x 100 .. 2048, five tokens each of
// H16/8, in e2m1 19; a prompt of 8192 tokens H32/8 D128 283 (970 TFLOP/s, with an exponential for each 256 operations).
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
  int most_fold;                                 // paged_weights_many: log2 of the heads that a query tile may have
  float* parts; int* shared;                     // paged_weights_many: two partial results of each workgroup; items that begin in it and end elsewhere
  int few_rows;                                  // sequences of up to so many rows are paged_weights_few's, the others paged_weights_many's
};

// Wavefronts on a SIMD: four where there are registers for them; units of e4m3 take more (us, four / three: 4 x 131072 H32/8 154 / 131,
// 64 x 100 .. 2048 32 / 20; e2m1, which has them, 83 / 86).
template <int TYPE, int NR>
constexpr int kFewWaves = NR > 1 ? 2 : TYPE == MHIP_E4M3 ? 3 : 4;

template <int TYPE, int NR>
constexpr int kBlocksOf = TYPE == MHIP_BF16 || NR == 4 ? 2 : 4;      // 16-key blocks of a unit

// Whether a sequence has few rows: asked where a call's sequences may be of both kinds, in e4m3 (see few_rows_of).
__device__ __forceinline__ bool is_few(const Gather& p, const PagedSeq& s) { return s.n * p.G <= p.few_rows; }

template <int TYPE, int UNIT>
__device__ __forceinline__ int64_t units_of(const Gather& p, const PagedSeq& s) {
  return TYPE != MHIP_E4M3 || is_few(p, s) ? (int64_t)((s.len + UNIT - 1) / UNIT) * p.Hkv : 0;
}

template <int TYPE, int COLS, int NR>
__global__ __launch_bounds__(256, (kFewWaves<TYPE, NR>)) void paged_weights_few(const Gather p) {
  constexpr int kBlocks = kBlocksOf<TYPE, NR>, UNIT = 16 * kBlocks, ROWS = 16 * NR;
  constexpr bool E4M3 = TYPE == MHIP_E4M3, E2M1 = TYPE == MHIP_E2M1;
  constexpr int KB = COLS / 32, KR = E2M1 ? 1 : E4M3 ? KB / 2 : KB;      // k-steps of 32 columns, loads of a key's row
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, lg = lane >> 4;

  // ---- this wavefront's share of the units: those before each lane's run of sequences, and of all ---------------------------
  const int w = ((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) * 4 + wave, workers = gridDim.x * 4;
  const int per = (p.g.B + 63) / 64;
  int64_t mine = 0;
  for (int j = 0; j < per; ++j)
    if (lane * per + j < p.g.B) mine += units_of<TYPE, UNIT>(p, paged_seq<false>(p.g, lane * per + j));
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
  for (int64_t u; b + 1 < p.g.B && pos >= (u = units_of<TYPE, UNIT>(p, paged_seq<true>(p.g, b))); ++b) pos -= u;

  const int k_block = COLS == 128 ? lg : lg >> 1;                        // (e2m1: the 32 columns that the lane's are of)
  auto col_of = [&](int ks) { return E2M1 ? (lg * KB + ks) * 8 : E4M3 ? (ks >> 1) * 64 + lg * 16 + (ks & 1) * 8 : ks * 32 + lg * 8; };
  auto mfma = [](const bf16x8& x, const bf16x8& y, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0); };

  while (lo < hi) {
    const PagedSeq s = paged_seq<true>(p.g, b);
    const int tiles = (s.len + UNIT - 1) / UNIT, rows = s.n * p.G;
    const bool here = !E4M3 || is_few(p, s);
    if (!here || tiles == 0 || pos >= (int64_t)tiles * p.Hkv) {
      if (here) pos -= (int64_t)tiles * p.Hkv;
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

    // where a lane's columns begin in a row (within the row there is), and its row's scales
    const int64_t row_of_lane = ln * p.c_ss + (E2M1 ? (k_block * 32 < p.D ? lg * (COLS == 128 ? 16 : 8) : 0) : lg * 16);
    const int64_t scale_of_lane = ln * p.s_ss;
    // The table's entries of a unit: the wavefront's blocks', and of the lane's own key.  They are on their way while the unit before is worked on.
    struct Entries { int page[kBlocks], own; } next;
    auto look_up = [&](int t) __attribute__((always_inline)) {
      int slot;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const int key = t * UNIT + 16 * i;
        next.page[i] = uniform_load(table, p.g.by_page.quotient(key < s.len ? key : s.len - 1, slot));
      }
      const int own = t * UNIT + lane;
      next.own = table[p.g.by_page.quotient(own < s.len ? own : s.len - 1, slot)];
    };
    look_up(t0);
    for (int t = t0; t < t0 + run; ++t) {
      const int key0 = t * UNIT;
      const Entries here = next;
      // (all loads go out before the first is waited for; a key that is not here reads one that is, and its sum goes nowhere)
      u32x4 w4[kBlocks][KR];
      float mult[kBlocks];
      uint32_t scales[kBlocks];
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        int slot;
        p.g.by_page.quotient(key0 + 16 * i, slot);
        const bool held = key0 + 16 * i < s.len && (uint32_t)here.page[i] < (uint32_t)p.g.pages;
        const int64_t page = held ? here.page[i] : 0;
        if (!held) slot = 0;
        const uint8_t* row = p.k + (page * p.c_sp + (int64_t)slot * p.c_ss + (int64_t)hk * p.c_sh) + row_of_lane;
        const float* scale = p.k_scales + (page * p.s_sp + (int64_t)slot * p.s_ss + (int64_t)hk * p.s_sh) + scale_of_lane;
        if constexpr (E2M1) {
          if constexpr (COLS == 128) w4[i][0] = *reinterpret_cast<const u32x4*>(row);
          else {
            const u32x2 x = *reinterpret_cast<const u32x2*>(row);
            w4[i][0] = u32x4{x[0], x[1], 0u, 0u};
          }
          scales[i] = *reinterpret_cast<const uint32_t*>(scale);
        } else {
          if constexpr (E4M3) scales[i] = *reinterpret_cast<const uint32_t*>(scale);
#pragma unroll
          for (int u = 0; u < KR; ++u) {
            w4[i][u] = u32x4{};
            if ((u * 4 + lg) * 16 < row_bytes(TYPE, p.D)) w4[i][u] = *reinterpret_cast<const u32x4*>(row + u * 64);
          }
        }
      }
      // the lane's own key, key0 + lane: what it had, and where it goes
      const int own = key0 + lane;
      int own_slot;
      p.g.by_page.quotient(own, own_slot);
      const int own_page = lane < UNIT && own < s.len ? here.own : -1;
      const bool held = (uint32_t)own_page < (uint32_t)p.g.pages;
      float had = 0.f;
      if (held && reads_old && own < (s.n == 0 ? s.len : old_keys))
        had = decay * p.old[(int64_t)own_page * p.w_sp + (int64_t)own_slot * p.w_ss + (int64_t)hk * p.w_sh];

      if (t + 1 < t0 + run) look_up(t + 1);
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {          // columns past the last are nothing
        mult[i] = E4M3 ? __builtin_bit_cast(float, scales[i]) : p.scale_log2;
        if constexpr (E2M1) {
          mult[i] = k_block * 32 < p.D ? e8m0(scales[i] >> (k_block * 8) & 255u) : 1.f;
          if (k_block * 32 >= p.D) w4[i][0] = u32x4{};
        }
      }
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

// ---- prompts -------------------------------------------------------------------------------------------------------------------
constexpr int kKeys = 256, kQueries = 32;        // of a workgroup's item, of a step
constexpr int kManyWaves = kKeys / 64;
constexpr int kManyWorkers = 512;                // workgroups: two on a CU
constexpr int kManyStages = 4;
constexpr int kQueryTile = kQueries * 256, kStageBytes = kQueryTile + kManyWaves * 256;     // rows of 256 bytes; each wavefront's copy of the rows' lse
// What entering an item costs, in steps, and the query tiles (eight, of one head) that cut through an item's keys cost twice.  (A prompt of
// 8192 tokens H32/8 D128 with all steps alike: workgroups end after 217 to 331 us, 229 to 315 so.)
constexpr int kPause = 4, kCut = 8;
constexpr int kFrags = 4;                        // LDS operand reads ahead of the MFMAs
constexpr int kNoColumn = 0x7fff0000;            // vector offset out of every descriptor's range (spans stay below 2^31, see kFarRows)
constexpr int64_t kFarRows = 1 << 23, kFarHeads = 1 << 24;       // elements between tokens, and between the heads of a tile, that paged_weights_many takes
constexpr int kFlush = 64;                       // steps whose weights are added up in a register

// Items of a sequence and K/V head: tiles of 256 keys.  A query tile is 32 / F tokens of F heads, F a power of two, so that short chunks of
// grouped heads fill it too; heads past the last of a K/V head are masked.  F grows while the query tiles become no more and a group of heads
// has less than four.  (us, one head to a tile / so: 8 x 4000 keys, 16 tokens of 16 heads on one 33.0 / 17.9, one token of 64 89.2 / 16.8;
// 84 x 1300, up to 16 tokens of seven heads on one 249 / 157; a prompt of 8192 tokens H32/8, which has tiles enough, 274 / 280.)  Key tile k is seen
// by the query tiles from max(0, 8 F k + z) on (all, without a mask), of each group of heads.
struct Steps {
  int tiles, queries, fold, groups, flat, z;     // key tiles, query tiles of a group, log2 F, groups; key tiles that all query tiles see
  int64_t all;                                   // of all key tiles
  __device__ __forceinline__ Steps() {}
  __device__ __forceinline__ Steps(const Gather& p, const PagedSeq& s) {
    tiles = (s.len + kKeys - 1) / kKeys;
    auto tiles_of = [&](int f) { return (int)((((int64_t)s.n << f) + kQueries - 1) / kQueries); };
    auto groups_of = [&](int f) { return (p.G + (1 << f) - 1) >> f; };
    fold = 0;
    queries = tiles_of(0);
    groups = p.G;
    while (fold < p.most_fold && (int64_t)s.n << fold < 4 * kQueries && groups > 1) {
      const int q = tiles_of(fold + 1), g = groups_of(fold + 1);
      if (q * g > queries * groups) break;       // (both below 128 or G: far below 2^31)
      queries = q;
      groups = g;
      ++fold;
    }
    z = p.causal ? (s.n - s.len) >> (5 - fold) : 0;        // (floor)
    flat = !p.causal ? tiles : z > 0 ? 0 : (-z >> (3 + fold)) + 1;
    flat = flat < tiles ? flat : tiles;
    all = before(tiles);
  }
  __device__ __forceinline__ int first(int k) const { return k < flat ? 0 : (k << (3 + fold)) + z; }
  __device__ __forceinline__ int of(int k) const { return queries > 0 ? (queries - first(k)) * groups : 0; }
  __device__ __forceinline__ int cost(int k) const { return of(k) + (queries > 0 && k >= flat ? (kCut << fold) * groups : 0); }      // behind kPause
  __device__ __forceinline__ int64_t before(int k) const {       // what the key tiles before k count for
    int64_t sum = (int64_t)k * queries;
    if (k > flat) sum -= (((int64_t)k * (k - 1) - (int64_t)flat * (flat - 1)) << (2 + fold)) + (int64_t)(z - (kCut << fold)) * (k - flat);
    return (queries > 0 ? sum * groups : 0) + (int64_t)k * kPause;
  }
};

// Sums over the 32 lanes of a half-wavefront of 32 registers each, lane ln with that of register ln: 31 exchanges instead of 160.
template <int HALF = 16>
__device__ __forceinline__ float sums_of_lanes(float (&x)[32], int ln) {
  const bool upper = ln & HALF;
#pragma unroll
  for (int i = 0; i < HALF; ++i) {
    const float keep = upper ? x[i + HALF] : x[i], give = upper ? x[i] : x[i + HALF];
    x[i] = keep + __shfl_xor(give, HALF);
  }
  if constexpr (HALF > 1) return sums_of_lanes<HALF / 2>(x, ln);
  else return x[0];
}

// Where the weight of a key lies, if its page is here.
struct Place { int page, slot; };
__device__ __forceinline__ Place place_of(const Gather& p, int b, int key, int len) {
  Place at{-1, 0};
  if (key < len) at.page = p.g.table[b * p.g.t_sb + p.g.by_page.quotient(key, at.slot)];
  if ((uint32_t)at.page >= (uint32_t)p.g.pages) at.page = -1;
  return at;
}
// What a key had of its weight that counts on.
__device__ __forceinline__ float had_before(const Gather& p, const PagedSeq& s, const Place& at, int hk, int key) {
  if (at.page < 0 || (s.n > 0 && p.decay == 0.f) || key >= (s.n == 0 ? s.len : s.len - s.n)) return 0.f;
  const float old = p.old[(int64_t)at.page * p.w_sp + (int64_t)at.slot * p.w_ss + (int64_t)hk * p.w_sh];
  return s.n == 0 ? old : p.decay * old;
}

template <int TYPE, int COLS>
__global__ __launch_bounds__(kManyWaves * 64, 2) void paged_weights_many(const Gather p) {
  constexpr int KB = COLS / 16;                  // k-steps of 16 columns
  __shared__ __attribute__((aligned(16))) unsigned char smem[kManyStages * kStageBytes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 31, lg = lane >> 5;

  // ---- this workgroup's share ------------------------------------------------------------------------------------------------
  const int w = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const int per = (p.g.B + 63) / 64;
  int64_t mine = 0;
  for (int j = 0; j < per; ++j)
    if (lane * per + j < p.g.B) {
      const PagedSeq s = paged_seq<false>(p.g, lane * per + j);
      if (TYPE != MHIP_E4M3 || !is_few(p, s)) mine += Steps(p, s).all * p.Hkv;
    }
  int64_t before = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t below = __shfl_up((long long)before, off);
    if (lane >= off) before += below;
  }
  const int64_t total = uniform64(__shfl((long long)before, 63)), shares = total < (int64_t)gridDim.x ? total : gridDim.x;
  before -= mine;
  if (threadIdx.x == 0) p.shared[w * 4] = 0;
  if (w >= shares) return;
  int64_t lo = total * w / shares;
  const int64_t hi = total * (w + 1) / shares;
  const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lo >= before && lo < before + mine));
  int b = owner * per;
  int64_t pos = lo - uniform64(__shfl((long long)before, owner));        // inside sequence b

  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  int q_a[KB];                                   // Q operand (B): lane (ln, lg) reads chunk 2 ks + lg of row ln
#pragma unroll
  for (int ks = 0; ks < KB; ++ks) q_a[ks] = (int)lds + ln * 256 + (((2 * ks + lg) ^ lds_row_swizzle(ln)) << 4);
  const int lse_a = (int)lds + kQueryTile + wave * 256 + ln * 4;
  typedef __attribute__((address_space(3))) const bf16x8* lds_bf16x8;
  typedef __attribute__((address_space(3))) const float* lds_float;
  float scale_log2 = p.scale_log2;
  asm volatile("" : "+s"(scale_log2));

  PagedSeq s{};
  Steps st;
  int heads = 0, tokens = 0, voff[2] = {}, l_off = 0;
  int hk = 0, kt = 0, from = 0;                  // the next item, and the units of it that lie in shares before this one
  for (bool enters = true; lo < hi;) {
    if (enters) {                                // sequence b, `pos` units behind its first
      s = paged_seq<true>(p.g, b);
      st = Steps(p, s);
      if (TYPE == MHIP_E4M3 && is_few(p, s)) st.all = 0;
      if (pos >= st.all * p.Hkv) {
        pos -= st.all * p.Hkv;
        ++b;
        continue;
      }
      enters = false;
      hk = kt = from = 0;
      if (pos > 0) {
        hk = (int)(pos / st.all);
        const int64_t in_head = pos - hk * st.all;
        for (int span = st.tiles; span > 1;) {   // the last key tile that begins at or before in_head
          const int half = span / 2;
          if (st.before(kt + half) <= in_head) { kt += half; span -= half; }
          else span = half;
        }
        from = (int)(in_head - st.before(kt));
      }
      // copies of a query tile, row r of which is token r / F and head r % F: four rows each, columns past the last are zeros
      heads = (1 << st.fold) - 1;
      tokens = kQueries >> st.fold;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = wave * 8 + u * 4 + (lane >> 4), chunk = (lane & 15) ^ lds_row_swizzle(r);
        voff[u] = chunk * 8 < p.D ? ((r >> st.fold) * (int)p.q_ss + (r & heads) * (int)p.q_sh) * 2 + chunk * 16 : kNoColumn;
      }
      l_off = ((ln >> st.fold) + (ln & heads) * (int)p.l_sh) * 4;
    }
    const int item_b = b, item_hk = hk, item_kt = kt;
    const int steps = st.of(kt), cost = st.cost(kt), weight = cost + kPause;
    const int take = (int)(weight - from < hi - lo ? weight - from : hi - lo);
    int first = 0, count = steps;                // steps of this share
    if (take < weight) {
      auto step_at = [&](int unit) { return unit > kPause ? (int)((int64_t)(unit - kPause) * steps / cost) : 0; };
      first = step_at(from);
      count = step_at(from + take) - first;
    }
    const int64_t start = lo - from;             // of the item
    const bool leaves_none = count == 0 && first == 0 && (steps > 0 || from > 0);        // (with steps before and behind it, it leaves sums of nothing)
    lo += take;
    from = 0;
    if (++kt == st.tiles) {
      kt = 0;
      if (++hk == p.Hkv) {
        ++b;
        pos = 0;
        enters = true;
      }
    }
    if (leaves_none) continue;
    const int key_at = item_kt * kKeys + wave * 64;          // the wavefront's first key
    // lane (ln, lg) ends with the sum of register ln: key 32 (ln / 16) + 8 (ln % 16 / 4) + 4 lg + ln % 4, which what it had is read for now
    const int own = key_at + (ln >> 4) * 32 + ((ln >> 2) & 3) * 8 + lg * 4 + (ln & 3);
    const Place own_at = place_of(p, item_b, own, s.len);
    float had = count == steps ? had_before(p, s, own_at, item_hk, own) : 0.f;

    float total_sum = 0.f;
    if (count > 0) {
      // ---- keys: A operand, lane (ln, lg) holds columns 16 ks + 8 lg .. +7 of keys ln and 32 + ln, scaled ------------------------
      // (all loads go out before the first is waited for; what is not here reads something that is, and is nothing)
      constexpr int kCodes = TYPE == MHIP_E2M1 ? 1 : TYPE == MHIP_E4M3 ? 2 : 4;          // words of eight columns
      uint32_t codes[2][KB][kCodes], scales[2] = {};
      bool here[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const Place at = place_of(p, item_b, key_at + kb * 32 + ln, s.len);
        here[kb] = at.page >= 0;
        const int64_t page = here[kb] ? at.page : 0, slot = here[kb] ? at.slot : 0;
        const uint8_t* row = p.k + (page * p.c_sp + slot * p.c_ss + (int64_t)item_hk * p.c_sh);
        if constexpr (TYPE != MHIP_BF16)
          scales[kb] = *reinterpret_cast<const uint32_t*>(p.k_scales + (page * p.s_sp + slot * p.s_ss + (int64_t)item_hk * p.s_sh));
#pragma unroll
        for (int ks = 0; ks < KB; ++ks) {
          const int col = ks * 16 + lg * 8;
          typedef __attribute__((__vector_size__(kCodes * sizeof(uint32_t)))) uint32_t Words;
          const Words w = *reinterpret_cast<const Words*>(row + (col < p.D ? col : 0) * kCodes / 2);
#pragma unroll
          for (int i = 0; i < kCodes; ++i) codes[kb][ks][i] = w[i];
        }
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int ks = 0; ks < KB; ++ks)
#pragma unroll
          for (int i = 0; i < kCodes; ++i) asm volatile("" : "+v"(codes[kb][ks][i]));
      bf16x8 kf[2][KB];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int ks = 0; ks < KB; ++ks) {
          const uint32_t (&c)[kCodes] = codes[kb][ks];
          u32x4 x;
          if constexpr (TYPE == MHIP_E2M1) {
            x = e2m1_to_bf16(c[0], e8m0(scales[kb] >> (ks / 2 * 8) & 255u));
          } else if constexpr (TYPE == MHIP_E4M3) {
            // (times the scale, rounded to bf16: exact for powers of two, and what attention takes for the sequences that come here, see few_rows_of)
            const float scale = __builtin_bit_cast(float, scales[kb]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(c[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c[h], true);
              x[2 * h] = pack_bf16(lo[0] * scale, lo[1] * scale);
              x[2 * h + 1] = pack_bf16(hi[0] * scale, hi[1] * scale);
            }
          } else {
            x = u32x4{c[0], c[1], c[2], c[3]};
          }
          const bool real = here[kb] && ks * 16 + lg * 8 < p.D;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = real ? x[i] : 0u;
          kf[kb][ks] = __builtin_bit_cast(bf16x8, x);
        }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int ks = 0; ks < KB; ++ks) asm volatile("" : "+v"(kf[kb][ks]));       // loaded before the first copy goes out
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();              // (the item before is through with the ring)
      const int qt0 = st.first(item_kt);

      // ---- query tiles: step i is tile qt of a group of heads, tiles fastest -------------------------------------------------------
      const int of_group = st.queries - qt0, group0 = first == 0 ? 0 : first / of_group;
      int copy_qt = qt0 + first - group0 * of_group, left = count;       // of the next copies, those that are left
      int qt = copy_qt;
      const int head0 = item_hk * p.G + (group0 << st.fold);
      int copy_last = p.G - 1 - (group0 << st.fold), here_last = copy_last;        // of the copies' heads, of the next step's: the last there is
      int q_tail, l_tail;                        // bytes of a copy's descriptors besides those of its tokens
      auto tails = [&]() __attribute__((always_inline)) {
        const int top = copy_last < heads ? copy_last : heads;
        q_tail = (top * (int)p.q_sh + p.D - (int)p.q_ss) * 2;
        l_tail = top * (int)p.l_sh * 4;
      };
      tails();
      const uint16_t* q_group = p.q + item_b * p.q_sb + (int64_t)s.start * p.q_ss + (int64_t)head0 * p.q_sh;
      const float* l_group = p.lse + item_b * p.l_sb + s.start + (int64_t)head0 * p.l_sh;
      // (tokens and heads past the last: zeros, or a row that there is; they are masked)
      auto copy = [&](int stage) __attribute__((always_inline)) {
        const int token0 = copy_qt * tokens, here = s.n - token0 < tokens ? s.n - token0 : tokens;
        const u32x4 rs = rsrc_words(q_group + (int64_t)token0 * p.q_ss, (uint32_t)(here * (int)p.q_ss * 2 + q_tail));
#pragma unroll
        for (int u = 0; u < 2; ++u) copy16_to_lds(rs, lds + stage * kStageBytes + (wave * 2 + u) * 1024, voff[u], 0);
        copy4_to_lds(rsrc_words(l_group + token0, (uint32_t)(here * 4 + l_tail)), lds + stage * kStageBytes + kQueryTile + wave * 256, l_off, 0);
        if (left > 1) {                          // (past the share's last tile that one again)
          --left;
          if (++copy_qt == st.queries) {
            copy_qt = qt0;
            q_group += p.q_sh << st.fold;
            l_group += p.l_sh << st.fold;
            copy_last -= heads + 1;
            tails();
          }
        }
      };
      const int old_keys = s.len - s.n;
      float sum[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) sum[e] = 0.f;
      f32x16 sc[2][2];
      float lse[2];
      bf16x8 frag[kFrags];
      // Of the tile in stage kStage: its rows' lse, and S^T with the operands kFrags reads ahead; between(m) goes behind MFMA m.
      auto product = [&](auto stage_of, f32x16 (&to)[2], float& to_lse, auto&& between) __attribute__((always_inline)) {
        constexpr int kAt = decltype(stage_of)::value * kStageBytes;
        auto read_q = [&](int ks) { return *(lds_bf16x8)(uintptr_t)(uint32_t)(q_a[ks] + kAt); };
        to_lse = *(lds_float)(uintptr_t)(uint32_t)(lse_a + kAt);
#pragma unroll
        for (int ks = 0; ks < kFrags; ++ks) frag[ks] = read_q(ks);
#pragma unroll
        for (int ks = 0; ks < KB; ++ks)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            to[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kb][ks], frag[ks % kFrags], ks == 0 ? f32x16{} : to[kb], 0, 0, 0);
            if (kb == 1 && ks + kFrags < KB) frag[ks % kFrags] = read_q(ks + kFrags);
            between(2 * ks + kb);
            __builtin_amdgcn_sched_barrier(0);
          }
      };
      copy(0);
      copy(1);
      copy(2);
      copy(3);
      asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      product(std::integral_constant<int, 0>{}, sc[0], lse[0], [](int) {});
      // Step i: the weights of tile i, and between them the product of tile i + 1 (past the share's last tile that one again), which
      // has been copied, by this wavefront and then by all; all have read tile i, whose stage tile i + 4 takes.  The loop is
      // written out four times, so that a stage is an immediate offset of the reads.
      auto step = [&](auto stage_of, int i) __attribute__((always_inline)) {
        constexpr int kStage = decltype(stage_of)::value;
        f32x16 (&now)[2] = sc[kStage & 1];
        asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        copy(kStage);
        // rows past the last, and those that saw no key, weigh nothing
        const int token0 = qt * tokens, token = token0 + (ln >> st.fold), top = here_last;
        const float mine = lse[kStage & 1];
        float minus = mine * -kLog2e;
        if (++qt == st.queries) {
          qt = qt0;
          here_last -= heads + 1;
        }
        if (p.causal && key_at > old_keys + token0 + tokens - 1) {       // nobody sees any of them
          product(std::integral_constant<int, (kStage + 1) & 3>{}, sc[(kStage + 1) & 1], lse[(kStage + 1) & 1], [](int) {});
        } else {
          if (__builtin_expect((p.causal && key_at + 63 > old_keys + token0) || token0 + tokens > s.n || top < heads ||
                               __builtin_amdgcn_ballot_w64(mine == -INFINITY) != 0, 0)) {
            asm volatile("");
            const bool counts = token < s.n && (ln & heads) <= top && mine != -INFINITY;
            // keys that the row sees, from the lane's first one
            const int seen = counts ? (p.causal ? old_keys + token + 1 : s.len) - key_at - 4 * lg : (int)0x80000000;
            // (an lse that is no number is that of the keys that the row sees, not of the others: they stay at -inf)
            const float odd = counts && !(minus < INFINITY) ? minus : 0.f;
            if (!counts || odd != 0.f) minus = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              now[e >> 4][e & 15] = (e >> 4) * 32 + 8 * (e >> 2 & 3) + (e & 3) >= seen ? -INFINITY : now[e >> 4][e & 15] + odd;
              if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
          }
          // Behind MFMA m the next weights' multiply-adds, the exponentials of those before, and the sums of those before them: none waits for another.
          constexpr int kEach = (32 + 2 * KB - 3) / (2 * KB - 2);
          auto ahead = [&](int e) __attribute__((always_inline)) {
            if (e < 32) now[e >> 4][e & 15] = __builtin_fmaf(now[e >> 4][e & 15], scale_log2, minus);
          };
          auto power = [&](int e) __attribute__((always_inline)) {
            if (e >= 0 && e < 32) now[e >> 4][e & 15] = fast_exp2(now[e >> 4][e & 15]);
          };
          auto add = [&](int e) __attribute__((always_inline)) {
            if (e >= 0 && e < 32) sum[e] += now[e >> 4][e & 15];
          };
          product(std::integral_constant<int, (kStage + 1) & 3>{}, sc[(kStage + 1) & 1], lse[(kStage + 1) & 1], [&](int m) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) power((m - 1) * kEach + e);
#pragma unroll
            for (int e = 0; e < kEach; ++e) ahead(m * kEach + e);
#pragma unroll
            for (int e = 0; e < kEach; ++e) add((m - 2) * kEach + e);
          });
#pragma unroll
          for (int e = (2 * KB - 2) * kEach; e < 32; ++e) add(e);
        }
        if (kStage == 3 && (i & (kFlush - 1)) == kFlush - 1) {
          asm volatile("");
          total_sum += sums_of_lanes(sum, ln);
#pragma unroll
          for (int e = 0; e < 32; ++e) sum[e] = 0.f;
        }
      };
      for (int i = 0; i < count; i += 4) {
        // The two workgroups of a CU take turns in going first: otherwise the older one ends long before the other, which is slow alone (a prompt of
        // 8192 tokens H32/8 D128 290 us, 280 with turns of 16 steps, 284 of four).
        if ((i >> 4 ^ blockIdx.x >> 8) & 1) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        step(std::integral_constant<int, 0>{}, i);
        if (i + 1 == count) break;
        step(std::integral_constant<int, 1>{}, i + 1);
        if (i + 2 == count) break;
        step(std::integral_constant<int, 2>{}, i + 2);
        if (i + 3 == count) break;
        step(std::integral_constant<int, 3>{}, i + 3);
      }
      __builtin_amdgcn_s_setprio(0);
      total_sum += sums_of_lanes(sum, ln);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // copies past the last step
    }
    if (count == steps) {
      if (own_at.page >= 0) p.out[(int64_t)own_at.page * p.o_sp + (int64_t)own_at.slot * p.o_ss + (int64_t)item_hk * p.o_sh] = had + total_sum;
      continue;
    }
    p.parts[(2 * (int64_t)w + (first == 0 ? 1 : 0)) * kKeys + own - item_kt * kKeys] = total_sum;
    if (first == 0 && threadIdx.x == 0) {
      const int last = (int)(((start + weight) * shares - 1) / total);           // the workgroup with its last unit
      p.shared[w * 4 + 1] = item_b;
      p.shared[w * 4 + 2] = item_hk;
      p.shared[w * 4 + 3] = item_kt;
      p.shared[w * 4] = last - w + 1;
    }
  }
}

// Items that several workgroups shared: their partial sums in order.  A workgroup for each that one may begin in, a thread for each key.
__global__ __launch_bounds__(kKeys) void paged_weights_join(const Gather p) {
  const int w = blockIdx.x, parts = uniform_load(p.shared, w * 4);
  if (parts == 0) return;
  const int b = uniform_load(p.shared, w * 4 + 1), hk = uniform_load(p.shared, w * 4 + 2), key = uniform_load(p.shared, w * 4 + 3) * kKeys + threadIdx.x;
  const PagedSeq s = paged_seq<true>(p.g, b);
  const Place at = place_of(p, b, key, s.len);
  float sum = p.parts[(2 * (int64_t)w + 1) * kKeys + threadIdx.x];
#pragma unroll 8
  for (int i = 1; i < parts; ++i) sum += p.parts[2 * (int64_t)(w + i) * kKeys + threadIdx.x];
  if (at.page >= 0) p.out[(int64_t)at.page * p.o_sp + (int64_t)at.slot * p.o_ss + (int64_t)hk * p.o_sh] = had_before(p, s, at, hk, key) + sum;
}

template <int TYPE>
void launch_many(const Gather& p, hipStream_t st) {
  if (p.D <= 64) hipLaunchKernelGGL((paged_weights_many<TYPE, 64>), dim3(kManyWorkers), dim3(kManyWaves * 64), 0, st, p);
  else if (p.D <= 96) hipLaunchKernelGGL((paged_weights_many<TYPE, 96>), dim3(kManyWorkers), dim3(kManyWaves * 64), 0, st, p);
  else hipLaunchKernelGGL((paged_weights_many<TYPE, 128>), dim3(kManyWorkers), dim3(kManyWaves * 64), 0, st, p);
  hipLaunchKernelGGL(paged_weights_join, dim3(kManyWorkers), dim3(kKeys), 0, st, p);
}

constexpr int64_t kManyBytes = (int64_t)kManyWorkers * (2 * kKeys * 4 + 16);

template <int TYPE, int COLS, int NR>
void launch_few(const Gather& p, hipStream_t st) {
  hipLaunchKernelGGL((paged_weights_few<TYPE, COLS, NR>), dim3(256 * kFewWaves<TYPE, NR>), dim3(256), 0, st, p);
}
template <int TYPE, int COLS>
void launch_rows(const Gather& p, int64_t rows, hipStream_t st) {
  if (rows <= 16) launch_few<TYPE, COLS, 1>(p, st);
  else if (rows <= 32) launch_few<TYPE, COLS, 2>(p, st);
  else launch_few<TYPE, COLS, 4>(p, st);
}

// Which sequences are paged_weights_few's: all up to kFewRows rows, else none, but of packed e4m3 those whose attention takes the keys' scales in
// fp32, so that every sequence's scores are those that its lse was made of.  (Another launch, and generating sequences in the form that reads keys
// once.  us, all with paged_weights_many / so: two short sequences 11.5 / 17.2, 16 of 600 .. 8192 keys H32/4 D96 that take 1 .. 512 tokens 122 / 110, 84 x 1300
// H112/16 up to 16 tokens 165 / 132, eight prompts of 1500 .. 2500 H32/8 210 / 214.  The other formats' keys are exact in both.)
int few_rows_of(const Gather& p, int64_t rows, int dtype, bool packed) {
  if (rows <= kFewRows || p.q_ss > kFarRows) return 0x7fffffff;
  return packed && dtype == MHIP_E4M3 && p.G <= kFewRows ? few_tile(p.G) : -1;
}
template <int TYPE>
void launch(const Gather& p, int64_t rows, hipStream_t st) {
  if (p.few_rows > 0) {
    const int64_t few = p.few_rows < rows ? p.few_rows : rows;
    if (p.D <= 64) launch_rows<TYPE, 64>(p, few, st);
    else launch_rows<TYPE, 128>(p, few, st);
  }
  if (p.few_rows < 0x7fffffff) launch_many<TYPE>(p, st);
}

}  // namespace
}  // namespace mhip

using namespace mhip;

extern "C" int64_t mhip_paged_attn_weights_workspace_bytes(int n, int T, int most_new, int packed, int Hq, int Hkv) {
  if (n < 0 || T < 0 || most_new < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return MHIP_EINVAL;
  return (int64_t)(packed ? most_new : n) * (Hq / Hkv) > kFewRows ? kManyBytes : 0;
}

extern "C" int mhip_paged_attn_weights(const void* q, const void* k_cache, const void* k_scales, const int* page_table, const int* lengths,
                                       const int* starts, const float* lse, const float* weights, float* out,
                                       int B, int n, int T, int most_new, int Hq, int Hkv, int D, int pages, int page_size, int table_pages,
                                       int64_t t_sb, int64_t q_sb, int64_t q_ss, int64_t q_sh,
                                       int64_t c_sp, int64_t c_ss, int64_t c_sh, int64_t s_sp, int64_t s_ss, int64_t s_sh,
                                       int64_t w_sp, int64_t w_ss, int64_t w_sh, int64_t o_sp, int64_t o_ss, int64_t o_sh,
                                       float softmax_scale, float decay, int mask, int dtype, void* workspace, void* stream) {
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
  p.few_rows = few_rows_of(p, rows, dtype, starts != nullptr);
  if (rows > kFewRows) {
    if (!workspace) return MHIP_EINVAL;
    if (!aligned16(workspace)) return MHIP_EALIGN;
    p.parts = static_cast<float*>(workspace);
    p.shared = reinterpret_cast<int*>(p.parts + (int64_t)kManyWorkers * 2 * kKeys);
    while (p.most_fold < 5 && (q_sh << (p.most_fold + 1)) <= kFarHeads && (p.l_sh << (p.most_fold + 1)) <= kFarHeads)
      ++p.most_fold;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MHIP_E2M1) launch<MHIP_E2M1>(p, rows, st);
  else if (dtype == MHIP_E4M3) launch<MHIP_E4M3>(p, rows, st);
  else launch<MHIP_BF16>(p, rows, st);
  return launch_status();
}
