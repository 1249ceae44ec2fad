// What the two forms of attention over a paged cache share: the arguments, and the last step of rows that several workgroups shared.
#pragma once

#include "paged.hpp"

#include <math.h>

namespace mhip {

// What the plan of a launch of long chunks leaves of a sequence: its first piece; the slot of its first partial result, where there
// are several parts; parts of an item; row tiles.
struct Record { int first, slot, parts, rts; };
// Rows (of sequence b and K/V head hk, from number row0 on; none: no item) that several workgroups shared: their partial results are in
// the slots first, second, second + step, ...
struct Shared { int b, hk, row0, rows, parts, first, second, step; };

// (Arguments are read by lines of 64 bytes: with the numbers behind the pointers a call of one token takes 9.8 us, in other orders up to 10.2.)
struct PagedAttn {
  PagedGeom g;
  const uint8_t* k; const uint8_t* v; const float* k_scales; const float* v_scales;
  uint32_t c_sp16, c_ss16;                 // strides of the cache from page to page and slot to slot, in 16 bytes,
  int64_t c_sh;                            // and from head to head, bytes
  int64_t s_sp, s_ss, s_sh;                // of the scales, elements
  const uint16_t* q; uint16_t* out; float* lse;
  int64_t q_sb, q_ss, q_sh, o_sb, o_ss, o_sh, l_sb, l_sh;
  float* part_o; f32x2* part_ml;           // partial results
  Shared* shared; Record* records; int* pieces;
  int Hkv, G, D, causal;
  float scale, scale_log2;
  Divisor by_group;
  int by_item;                             // paged_attn_few: shared items by their number, not by the workgroup they begin in
  int few_rows;                            // sequences of up to so many rows are paged_attn_few's, the others paged_attn_chunk's
};

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32);
}

// Values that are no numbers, in a tile of which some rows do not see some keys: 0 * NaN would reach rows that do not see the key.
// They are zeros in the product with P then, and a product of odd_marks with seen_marks counts for every row and column how many
// it sees of each kind: +inf in ones, -inf in 128s, NaN in 16384s (at most 64 keys; all of it exact).
__device__ __forceinline__ u32x4 finite_part(const u32x4& v, uint32_t& odd) {
  u32x4 fine;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = (v[i] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u, hi = (v[i] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
    fine[i] = v[i] & ~(lo | hi);
    odd |= lo | hi;
  }
  return fine;
}
__device__ __forceinline__ u32x4 odd_marks(const u32x4& v) {
  u32x4 marks;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    auto mark = [](uint32_t x) {       // 1, 128 and 16384 in bf16
      return (x & 0x7f80u) != 0x7f80u ? 0u : x & 0x7fu ? 0x4680u : x & 0x8000u ? 0x4300u : 0x3f80u;
    };
    marks[i] = mark(v[i] & 0xffffu) | mark(v[i] >> 16) << 16;
  }
  return marks;
}
// Of a lane's keys, four and four, of which its row sees the first left0 and left1: ones in bf16.  (By place and not by weight: a weight may
// be zero for being small.)
__device__ __forceinline__ u32x4 seen_marks(int left0, int left1) {
  u32x4 marks;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = i < 2 ? left0 : left1, j = 2 * (i & 1);
    marks[i] = (j < left ? 0x3f80u : 0u) | (j + 1 < left ? 0x3f800000u : 0u);
  }
  return marks;
}
__device__ __forceinline__ float with_odd(float o, float counts) {
  const int n = (int)counts;
  if (n >= 16384) return __builtin_nanf("");
  if (n & 127) o += INFINITY;
  if (n >> 7) o -= INFINITY;
  return o;
}

// The arguments once more, read from memory where this stands: values that only the end of a kernel needs would otherwise stay in
// (or move in and out of) scalar registers through its main loop.
__device__ __forceinline__ PagedAttn arguments_again() {
  auto at = (__attribute__((address_space(4))) const PagedAttn*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *(const PagedAttn*)at;
}

// Where row `slot` of a page begins, from the first row of the cache.
__device__ __forceinline__ int64_t row_offset(const PagedAttn& p, int page, int slot) {
  return (int64_t)(((uint64_t)(uint32_t)page * p.c_sp16 + (uint64_t)((uint32_t)slot * p.c_ss16)) << 4);
}

// The last step of items that several workgroups shared: their partial results with the weights that their maxima and sums give.  A
// wavefront does R rows at a time, two columns a lane; the weights are found by a lane each, so that the rows' loads wait for nothing.
// (The rows of an item are neighbouring workgroups, on all XCDs; the few items' own numbers are often all of one.)
template <int COLS, int ROWS, int R, int BLOCK>
__global__ __launch_bounds__(256) void paged_attn_join(const PagedAttn p) {
  static_assert(BLOCK % (4 * R) == 0, "rows of a workgroup");
  const int* record = reinterpret_cast<const int*>(p.shared + blockIdx.y);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = uniform_load(record, 3), begin = blockIdx.x * BLOCK;
  if (begin >= rows) return;
  const int b = uniform_load(record, 0), hk = uniform_load(record, 1), row0 = uniform_load(record, 2), n_parts = uniform_load(record, 4);
  const int first = uniform_load(record, 5), second = uniform_load(record, 6), step = uniform_load(record, 7);
  const PagedSeq s = paged_seq<true>(p.g, b);
  const int col = lane * 2 < COLS ? lane * 2 : 0;
  for (int row = begin + wave * R; row < begin + BLOCK && row < rows; row += 4 * R) {
    auto at = [&](int k, int r) {
      const int here = row + r < rows ? row + r : rows - 1;
      return (int64_t)(k == 0 ? first : second + (k - 1) * step) * ROWS + here;
    };
    f32x2 ml[R];
    float top[R], ref[R], sum[R], a0[R], a1[R];
    constexpr int kDeep = 8 / R;
    // The parts that are added next, on their way while the weights are found (64 tokens at 32768: 57.9 us to 56.1).
    f32x2 next[kDeep][R];
    auto request = [&](int k) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < kDeep; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r)
          next[u][r] = *reinterpret_cast<const f32x2*>(p.part_o + at(k + u < n_parts ? k + u : n_parts - 1, r) * COLS + col);
    };
#pragma unroll
    for (int r = 0; r < R; ++r) {
      ml[r] = f32x2{-INFINITY, 0.f};
      if (lane < n_parts) ml[r] = p.part_ml[at(lane, r)];
    }
    request(0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      top[r] = ml[r][0];
      sum[r] = a0[r] = a1[r] = 0.f;
      for (int k = lane + 64; k < n_parts; k += 64) top[r] = fmaxf(top[r], p.part_ml[at(k, r)][0]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) top[r] = fmaxf(top[r], __shfl_xor(top[r], off));
      ref[r] = top[r] == -INFINITY ? 0.f : top[r];
    }
    for (int k0 = 0; k0 < n_parts; k0 += 64) {
      float weight[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (n_parts > 64) ml[r] = k0 + lane < n_parts ? p.part_ml[at(k0 + lane, r)] : f32x2{-INFINITY, 0.f};
        weight[r] = fast_exp2(ml[r][0] - ref[r]);
        sum[r] += ml[r][1] * weight[r];
      }
      const int here = n_parts - k0 < 64 ? n_parts - k0 : 64;
      for (int k = 0; k < here; k += kDeep) {
        f32x2 x[kDeep][R];
#pragma unroll
        for (int u = 0; u < kDeep; ++u)
#pragma unroll
          for (int r = 0; r < R; ++r) x[u][r] = next[u][r];
        if (k0 + k + kDeep < n_parts) request(k0 + k + kDeep);
#pragma unroll
        for (int u = 0; u < kDeep; ++u)
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight[r]), k + u));
            a0[r] += k + u < here ? x[u][r][0] * w : 0.f;        // (past the last part its row again, which may hold an infinity)
            a1[r] += k + u < here ? x[u][r][1] * w : 0.f;
          }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) sum[r] += __shfl_xor(sum[r], off);
      if (row + r >= rows) continue;
      int of_group;
      const int token = s.start + p.by_group.quotient(row0 + row + r, of_group), head = hk * p.G + of_group;
      const float inv = sum[r] == 0.f ? 0.f : 1.f / sum[r];
      if (lane * 2 < p.D)
        *reinterpret_cast<uint32_t*>(p.out + b * p.o_sb + (int64_t)token * p.o_ss + head * p.o_sh + col) = pack_bf16(a0[r] * inv, a1[r] * inv);
      if (lane == 0) p.lse[b * p.l_sb + head * p.l_sh + token] = sum[r] == 0.f ? -INFINITY : (top[r] + fast_log2(sum[r])) * kLn2;
    }
  }
}

int64_t paged_attn_chunk_bytes(int64_t B, int64_t n, int64_t T, int G, int Hkv, int D, bool packed);
bool paged_attn_chunk_fits(int64_t B, int64_t n, int64_t T, int G, int Hkv, bool packed);       // into a launch
void paged_attn_chunk_launch(const PagedAttn& p, bool e4m3, hipStream_t stream);

}  // namespace mhip
