// What the two forms of attention over a paged cache share: the arguments, and the last step of rows that several workgroups shared.
#pragma once

#include "paged.hpp"

#include <math.h>

namespace mhip {

// What the plan of a launch of long chunks leaves of a sequence (its first piece; the slot of its first partial result, where there
// are several parts; parts of an item; row tiles), and of all (partial results).
struct Record { int first, slot, parts, rts; };
struct PlanOut { int slots; };

struct PagedAttn {
  PagedGeom g;
  const uint8_t* k; const uint8_t* v; const float* k_scales; const float* v_scales;
  uint32_t c_sp16, c_ss16;                 // strides of the cache from page to page and slot to slot, in 16 bytes,
  int64_t c_sh;                            // and from head to head, bytes
  int64_t s_sp, s_ss, s_sh;                // of the scales, elements
  const uint16_t* q; uint16_t* out; float* lse;
  int64_t q_sb, q_ss, q_sh, o_sb, o_ss, o_sh, l_sb, l_sh;
  int Hq, Hkv, G, D, causal;
  float scale, scale_log2;
  Divisor by_group, by_heads, by_new;
  int few_rows;                            // sequences of up to so many rows are paged_attn_few's, the others paged_attn_chunk's
  float* part_o; f32x2* part_ml;           // partial results
  PlanOut* plan; Record* records; int* pieces;
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
__device__ __forceinline__ u32x4 seen_marks(const u32x4& p) {
  u32x4 marks;
#pragma unroll
  for (int i = 0; i < 4; ++i) marks[i] = (p[i] & 0x7fffu ? 0x3f80u : 0u) | (p[i] & 0x7fff0000u ? 0x3f800000u : 0u);
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

// One row from its partial results, the slot of number k at at(k): a wavefront, two columns a lane.  The weights are found by a
// lane each, so that the rows' loads wait for nothing.
template <int COLS, class At>
__device__ __forceinline__ void join_row(const PagedAttn& p, int lane, int n_parts, At at, int b, int token, int head) {
  float top = -INFINITY;
  f32x2 ml = {-INFINITY, 0.f};
  for (int k = lane; k < n_parts; k += 64) {
    ml = p.part_ml[at(k)];
    top = fmaxf(top, ml[0]);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  const float ref = top == -INFINITY ? 0.f : top;
  const int col = lane * 2 < COLS ? lane * 2 : 0;
  float sum = 0.f, a0 = 0.f, a1 = 0.f;
  for (int k0 = 0; k0 < n_parts; k0 += 64) {
    if (n_parts > 64) ml = k0 + lane < n_parts ? p.part_ml[at(k0 + lane)] : f32x2{-INFINITY, 0.f};
    const float weight = fast_exp2(ml[0] - ref);
    sum += ml[1] * weight;
    const int here = n_parts - k0 < 64 ? n_parts - k0 : 64;
    for (int k = 0; k < here; k += 8) {
      f32x2 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        x[u] = *reinterpret_cast<const f32x2*>(p.part_o + at(k0 + (k + u < here ? k + u : here - 1)) * COLS + col);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), k + u));
        a0 += k + u < here ? x[u][0] * w : 0.f;        // (past the last part its row again, which may hold an infinity)
        a1 += k + u < here ? x[u][1] * w : 0.f;
      }
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (lane * 2 < p.D) *reinterpret_cast<uint32_t*>(p.out + b * p.o_sb + (int64_t)token * p.o_ss + head * p.o_sh + col) = pack_bf16(a0 * inv, a1 * inv);
  if (lane == 0) p.lse[b * p.l_sb + head * p.l_sh + token] = sum == 0.f ? -INFINITY : (top + fast_log2(sum)) * kLn2;
}

// Number `id` of all T * Hq rows of q, in two steps: the token (whose number is returned) and the head; the token's sequence and
// its number there, false where there is none.  row_number: the row's number among those of the sequence and K/V head.
struct RowOf { int b, i, head, hk; PagedSeq s; };
__device__ __forceinline__ int token_of(const PagedAttn& p, int id, RowOf& x) {
  const int t = __builtin_amdgcn_readfirstlane(p.by_heads.quotient(id, x.head));
  x.head = __builtin_amdgcn_readfirstlane(x.head);
  return t;
}
__device__ __forceinline__ bool seq_of(const PagedAttn& p, int t, int lane, RowOf& x) {
  int i = 0;
  if (p.g.starts) x.b = paged_owner<64>(p.g, t, lane);
  else x.b = p.by_new.quotient(t, i);
  x.b = __builtin_amdgcn_readfirstlane(x.b);
  if (x.b >= p.g.B) return false;
  x.s = paged_seq<true>(p.g, x.b);
  x.i = p.g.starts ? t - x.s.start : i;
  return x.i >= 0 && x.i < x.s.n;
}
__device__ __forceinline__ int row_number(const PagedAttn& p, RowOf& x) {
  int of_group;
  x.hk = p.by_group.quotient(x.head, of_group);
  return x.i * p.G + of_group;
}

// Rows of a wavefront of the last step: one while there are CUs without any, up to eight.
inline int join_rows(int64_t n_rows) { return n_rows <= 8192 ? 1 : n_rows >= 65536 ? 8 : (int)(n_rows / 8192); }

int64_t paged_attn_chunk_bytes(int64_t B, int64_t n, int64_t T, int G, int Hkv, int D, bool packed);
int paged_attn_chunk_launch(const PagedAttn& p, bool e4m3, hipStream_t stream);

}  // namespace mhip
