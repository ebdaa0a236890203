// The attention of 32 queries against tiles of keys, one wave's part, on v_mfma_f32_32x32x16_bf16: shared by the kernels
// over whole prompts and over the pages of a cache.
//
// The scores are computed transposed, S^T = K Q^T: lane l holds 16 scores of query l % 32 per 32 keys (keys 8b + 4h + i of
// a tile for b, i in 0..3 and h = l / 32), so the softmax needs one exchange between the halves of a wave, and the
// probabilities are the B operand of O^T = V^T P^T as they are: with the 16 keys of a product taken in the order that the
// lanes hold them, V^T's fragments are two transposing LDS reads each.
//
// Keys and values lie in LDS row by row as in memory, staged by direct-to-LDS loads, each row's 16-byte units (keys) or
// 32-byte groups (values) permuted by its number against bank repeats.
#pragma once

#include "oasis_common.h"

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;

namespace flash {

constexpr int NW = 8;  // waves of a workgroup
constexpr float LOG2E = 1.4426950408889634f;
// How far a row's scores may pass its running maximum before the sums are rescaled, as a power of two: the probabilities
// reach 2^8 then, which costs neither bf16 nor fp32 any precision.
constexpr float SLACK = 8.f;
// Scaled scores beyond this are taken as differences before scaling: there the rounding of a scaled maximum, against whose
// fixed value scores are taken below it, is no longer small against 1. (2^20, less what keeps a number and SINK below it too.)
constexpr float HUGE_SCORE = 1048512.f;

// Probabilities are taken 2^-30 times as large as their sum needs: with SLACK a row's are 2^-22 at most, so the sums of up to
// 2^22 finite values stay finite, whatever the values are (and of 2^30 values up to 2^120). A probability vanishes below 2^-96 of
// the row's largest instead of 2^-126.
constexpr float SINK = 30.f;

// The base of probabilities whose running maximum is m, as a power of two (scale: softmax scale times log2 e). Up to
// HUGE_SCORE it is the rounded sum, which is off by as much as 2^-5 there: sums taken on different bases have to be brought
// to one by these rounded values and no others. Beyond, it is m * scale + SINK exactly.
OASIS_DEV float base_of(float m, float scale) { return fmaf(m, scale, SINK); }
OASIS_DEV bool is_huge(float base) { return fabsf(base) > HUGE_SCORE; }
// A base in two: raw * scale + number, one of them taken as a product yet.
struct Base {
  float raw, number;
};
OASIS_DEV Base split_base(float m, float scale) {
  const float b = base_of(m, scale);
  return is_huge(b) ? Base{m, SINK} : Base{0.f, b};
}
// What brings sums on the base `from` to the base `to`, as a power of two. A huge base is near one that is not at HUGE_SCORE
// only, where SINK is a multiple of the other's last place. (Without branches: with them own_kernel of heads of 128 spills a
// thousand registers.)
OASIS_DEV float shift(Base from, Base to, float scale) { return fmaf(from.raw - to.raw, scale, from.number - to.number); }

OASIS_DEV f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// Where 16-byte unit u of key row r, and of value row r, lies in the row.
template <int D>
OASIS_DEV int k_unit(int r, int u) { return u ^ (r & (D / 8 - 1)); }
template <int D>
OASIS_DEV int v_unit(int r, int u) {
  const int f = D == 128 ? (r & 3) ^ ((r & 3) << 1) : ((r >> 1) & 1) * 3;
  return u ^ (f << 1);
}

template <int D>
struct Tile {
  static constexpr int ROW = D * 2;      // bytes of a staged row
  static constexpr int DS = D / 16;      // products of a score
  static constexpr int DT = D / 32;      // 32-dim tiles of the output

  bf16x8 q[DS];   // lane l: query l % 32, dims 16 s + 8 (l / 32) ..
  f32x16 o[DT];   // lane l: query l % 32, dims 32 dt + 8 b + 4 (l / 32) + i at [4 b + i]
  float m;        // running maximum of the raw scores (the lanes of a query alike)
  float l;        // sum of the probabilities of this lane's keys

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  }

  // raw scores of the 32 keys whose rows start at kb
  __device__ __forceinline__ f32x16 scores(const char* kb, int lane) const {
    const int r = lane & 31, h = lane >> 5;
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DS; ++d)
      s = mfma32(*reinterpret_cast<const bf16x8*>(kb + r * ROW + (k_unit<D>(r, 2 * d + h) << 4)), q[d], s);
    return s;
  }

  // The running maximum moves to that of N * 32 more scores (scale: softmax scale times log2 e, positive), and the output so
  // far with it, where they pass it by SLACK. Returns what to take off the scaled scores. Masked scores are -inf. Scores that
  // are huge once scaled are taken off here, before scaling: one branch for whatever is rare.
  template <int N>
  __device__ __forceinline__ float settle(f32x16* s, float scale) {
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
    mx = max_xor32(mx);
    float at = base_of(m, scale);
    const float top = base_of(mx, scale);
    if (__any(top > at + SLACK || is_huge(at))) {
      const float to = fmaxf(m, mx);
      const float alpha = to == m ? 1.f : __builtin_amdgcn_exp2f(shift(split_base(m, scale), split_base(to, scale), scale));
      m = to;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
      at = m == -INFINITY ? 0.f : base_of(m, scale);
      if (__any(is_huge(at))) {
        const float raw = is_huge(at) ? m : 0.f;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[t][i] -= raw;
        at = is_huge(at) ? SINK : at;
      }
    }
    return at;
  }
  // settled scores to probabilities
  template <int N>
  __device__ __forceinline__ void exponents(f32x16* s, float scale, float at) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], scale, -at));
        sum[i & 3] += s[t][i];
      }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }
  template <int N>
  __device__ __forceinline__ void softmax(f32x16* s, float scale) {
    const float at = settle<N>(s, scale);
    exponents<N>(s, scale, at);
  }

  // The V^T fragment of keys 16 s .. + 15 of the rows at vb, dims 32 dt ..
  __device__ __forceinline__ bf16x8 values(const char* vb, int s, int dt, int lane) const {
    typedef short i16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) i16x4* lds4;
    const int r = 16 * s + 4 * (lane >> 5) + ((lane & 15) >> 2);  // and 8 rows on: the same permutation
    const int u = 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const char* p = vb + r * ROW + (v_unit<D>(r, u) << 4) + (lane & 1) * 8;
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 8 * ROW));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }

  // the B operand of keys 16 s .. + 15 of 32. Rounded to bf16, half a step (2^-9 to 2^-8) of each probability: the matrix
  // cores take no wider type at this rate; the sum divided by is of the unrounded ones.
  static __device__ __forceinline__ bf16x8 probs(const f32x16& p, int s) {
    bf16x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = f2bf(p[8 * s + j]);
    return r;
  }

  // o += V^T P^T over the 32 keys whose rows start at vb
  __device__ __forceinline__ void weigh(const f32x16& p, const char* vb, int lane) {
    const bf16x8 pb[2] = {probs(p, 0), probs(p, 1)};
    weigh(pb, vb, lane);
  }
  __device__ __forceinline__ void weigh(const bf16x8* pb, const char* vb, int lane) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] = mfma32(values(vb, s, dt, lane), pb[s], o[dt]);
  }

  // Whether any of the wave's outputs is not finite.
  __device__ __forceinline__ bool broken() const {
    float z = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) z = fmaf(o[d][i], 0.f, z);
    return __any(z != 0.f);
  }

  // weigh() where a masked key's value may be infinite or NaN, against which a probability of 0 is NaN: the finite values
  // through the product as they are, and what is not finite by which of it the query sees. `pb` is 0 for masked keys, bit i
  // of `seen` set for the others.
  __device__ __forceinline__ void weigh_masked(const bf16x8* pb, uint32_t seen, const char* vb, int lane) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 vis;
#pragma unroll
      for (int j = 0; j < 8; ++j) vis[j] = f2bf((seen >> (8 * s + j)) & 1 ? 1.f : 0.f);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const bf16x8 v = values(vb, s, dt, lane);
        bf16x8 fin;
#pragma unroll
        for (int j = 0; j < 8; ++j) fin[j] = fabsf(bf2f(v[j])) < INFINITY ? v[j] : f2bf(0.f);
        o[dt] = mfma32(fin, pb[s], o[dt]);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          __builtin_amdgcn_sched_barrier(0);  // one at a time: interleaved they take more registers than there are
          bf16x8 kind;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = bf2f(v[j]);
            kind[j] = f2bf((k == 0 ? x == INFINITY : k == 1 ? x == -INFINITY : x != x) ? 1.f : 0.f);
          }
          f32x16 n;
#pragma unroll
          for (int i = 0; i < 16; ++i) n[i] = 0.f;
          n = mfma32(kind, vis, n);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[dt][i] += n[i] > 0.f ? (k == 0 ? INFINITY : k == 1 ? -INFINITY : NAN) : 0.f;
        }
      }
    }
  }

  // The lane's query's output, times inv, to `to` (dim 0): the two halves of a wave trade so that each stores 16 bytes.
  // Called by whole waves; `store` says whether this lane's query exists.
  __device__ __forceinline__ void store(bf16* to, float inv, bool store, int lane) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int b = 0; b < 4; b += 2) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = o[d][4 * b + i] * inv;          // dims 8 b + 4 h + i
          x[4 + i] = o[d][4 * b + 4 + i] * inv;  // dims 8 (b + 1) + 4 h + i
          swap_halves32(x[i], x[4 + i]);         // now dims 8 (b + h) + i and 8 (b + h) + 4 + i
        }
        if (store) *reinterpret_cast<bf16x8*>(to + 32 * d + 8 * (b + (lane >> 5))) = pack8(x);
      }
  }
};

// Eight waves, each with 32 queries of its own, over the same 64-key tiles n - 1, .., 0.
// issue(tile, stage) loads the wave's share of a tile to LDS at `stage`. `skip`: the wave's first tiles that it takes no part
// in (n where it takes none). A lane's query sees keys up to `last`, key 0 being tile 0's first; the wave's first tile may have
// others, whose values count for nothing whatever they are. CUT: so may the next ones, down to the tile of `least`, the wave's
// least `last`; there a value that is not finite breaks the outputs of the queries that do not see it too.
//
// A tile takes two steps with a barrier after each: the softmax of its scores, then on the matrix units the scores of the next
// tile and the products of this one with the values. The second four waves, one on each SIMD with one of the first, are a step
// behind: while one of the two has the vector units the other has the matrix units. Round r (tile n - 1 - r) is in stage
// r % 4; stage r + 2 is loaded from the first step of round r on, which is two barriers after the last read of the stage that it
// replaces, and waited for at the end of the second, two barriers before its first read.
template <int D>
struct Turns {
  typedef Tile<D> Tile;
  static constexpr int KS = 64, ROW = Tile::ROW, HALF = KS * ROW, STAGE = 2 * HALF, ST = 4, SMEM = ST * STAGE;
  static constexpr int RPB = 1024 / ROW;         // rows of a 1 KB load
  static constexpr int LPW = 2 * KS / RPB / NW;  // loads of a wave and stage: rows [16 (wave % 4), + 16) of the keys (the
                                                 // first four waves) or the values
  static_assert(LPW * RPB == 16 && SMEM <= 160 * 1024, "a wave loads 16 rows");

  template <bool CUT, typename Issue>
  static __device__ __forceinline__ void go(Tile& w, char* smem, int n, int skip, int last, int least, float scale, Issue issue) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const bool second = wave >= NW / 2;
    auto stage = [&](int r) -> char* { return smem + r % ST * STAGE; };
    f32x16 s[2];
    bf16x8 pb[2][2];
    auto scores = [&](int r) {
      s[0] = w.scores(stage(r), lane);
      s[1] = w.scores(stage(r) + 32 * ROW, lane);
    };
    auto load = [&](int r) { issue(n > r + 3 ? n - 3 - r : 0, stage(r + 2)); };  // past the last tile, the first again
    auto meet = [&]() {  // the steps are kept apart: what the compiler moves over a barrier runs beside its like
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
    };
    auto landed = [&]() {
      __builtin_amdgcn_s_waitcnt((0x7 << 4) | (0xF << 8));  // vmcnt(0)
      meet();
    };
    auto soften = [&]() {  // scores to probabilities
      const float at = w.template settle<2>(s, scale);
      w.template exponents<2>(s, scale, at);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) pb[t][x] = Tile::probs(s[t], x);
    };
    issue(n - 1, stage(0));
    issue(n > 1 ? n - 2 : 0, stage(1));
    landed();
    if (second) __builtin_amdgcn_s_barrier();
    int r = 0;
    if (skip == 0) scores(0);
    for (; r < skip; ++r) {
      load(r);
      meet();
      if (r == skip - 1 && r + 1 < n) scores(r + 1);
      landed();
    }
    if (r < n) {  // a wave's first tile: the only one that keys of no query may lie in
      load(r);
      uint32_t seen[2] = {0, 0};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool sees = (n - 1 - r) * KS + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) <= last;
          seen[t] |= (sees ? 1u : 0u) << i;
          if (!sees) s[t][i] = -INFINITY;
        }
      soften();
      meet();
      const char* vb = stage(r) + HALF;
      if (r + 1 < n) scores(r + 1);
      w.weigh(pb[0], vb, lane);
      w.weigh(pb[1], vb + 32 * ROW, lane);
      if (w.broken()) {  // by a value that is not finite, or a score: the output was zero before, so once more
#pragma unroll
        for (int d = 0; d < Tile::DT; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) w.o[d][i] = 0.f;
        w.weigh_masked(pb[0], seen[0], vb, lane);
        w.weigh_masked(pb[1], seen[1], vb + 32 * ROW, lane);
      }
      landed();
      ++r;
    }
#pragma unroll 1
    for (; r < n; ++r) {
      load(r);
      if (CUT && (n - r) * KS - 1 > least) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if ((n - 1 - r) * KS + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) > last) s[t][i] = -INFINITY;
      }
      soften();
      meet();
      const char* vb = stage(r) + HALF;
      scores(r + 1);  // past the last round, of a stage that holds some tile: not used
      w.weigh(pb[0], vb, lane);
      w.weigh(pb[1], vb + 32 * ROW, lane);
      // the matrix units' step keeps its LDS reads four ahead of the products (of two reads each for the values')
      constexpr int AHEAD = 4;
      __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
      for (int x = 0; x < 2 * Tile::DS - AHEAD; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
#pragma unroll
      for (int x = 0; x < 4 * Tile::DT; ++x) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, AHEAD, 0);
      landed();
    }
    if (!second) __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_s_waitcnt(0);  // no load into LDS outlives the workgroup
  }
};

}  // namespace flash
