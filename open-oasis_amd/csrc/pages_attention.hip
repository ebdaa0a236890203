// Attention of single query tokens against the pages of a cache, the tokens that a group of sequences shares read once for
// all of them.
//
// Shared prefixes (prefix_part): a part is a set of query columns (the heads of the group's rows, 32 R at a time), one key
// head and a run of keys. A workgroup of eight waves takes a part. For few columns (Walk, R = 1) the waves take tiles of 32
// keys in turn for the same 32 columns, and none waits for another until their sums are joined at the end. For more (Crowd,
// R = 8) all eight read the same tiles, so that a large group's prefix is a matter of the matrix cores and not of the L2.
// Every row's own tokens (own_part): 16 columns, the heads of one row that share a key head, by S waves in turn, keys from
// memory to registers and only the values through LDS, so that 16 waves of a CU have loads on their way. Up to some number of
// rows one launch does both and join_kernel joins all parts, in a fixed order; beyond it own_kernel joins the prefix's
// parts, and splits and joins its own only where few rows have long sequences. Partial sums are fp32.
//
// What bounds it: own tokens are read once, which is bandwidth (256 rows of up to 1024 tokens, 8 key heads of 128, 545 MB: 116
// us, 4.7 TB/s); a prefix of many columns the products on tiles of 256 columns (256 rows in four groups, prefixes of up to
// 16000 tokens, 32 heads of 128, 8 key heads, with their own tokens up to 1024: 180 us); few rows the latency of loads
// behind each other and of two launches (one row of 720 tokens, 16 heads of 64: 7.4 us; 32 rows behind 4608 shared ones: 15.7).
#include <algorithm>
#include <type_traits>

#include "flash_tile.h"

namespace {

typedef oasis_page_cache_t Cache;

// a static member that every caller holds inline
#define OASIS_WALK __device__ __forceinline__

struct Sum {
  float m, l;  // running maximum of the raw scores, sum of the probabilities
};
struct WaveSum {
  float m, l;
  flash::Base base;  // of the probabilities, split once for all that join it
};
// what a sum whose maximum is m is joined on: an empty one, any
OASIS_DEV flash::Base top_base(float m, float scale) { return flash::split_base(m == -INFINITY ? 0.f : m, scale); }

struct PagesArgs {
  Cache c;
  int64_t layer;
  const bf16* q;
  bf16* out;
  int64_t ld_q, ld_out;
  const int32_t *seqs, *cu, *prefix;
  int n_rows, n_groups, heads, group;  // group: query heads of a key head
  float scale_log2;
  int p_tiles, p_splits, s_tiles, s_splits;  // column tiles of all prefixes (at most), and of one row; splits of each
  int parts;  // of a row in the workspace: the prefix's, then its own where these are not joined at once
  float* o;   // [rows][heads][parts][D]
  Sum* ml;    // [rows][heads][parts]
};

using flash::NW;
constexpr int MIN_CHUNK = 256;  // keys of a part at least: a tile of 32 for every wave, two where it is a row's own

// keys of each of `splits` parts of n
OASIS_DEV int chunk_of(int n, int splits, int least) {
  const int c = (n + splits - 1) / splits;
  return max((c + least - 1) / least * least, least);
}

// An integer of the bookkeeping, which no kernel here writes: through the constant address space, so that an index known to
// be the same in every lane gives a scalar, and with it the page's address. (A vector's would make every load of a page a
// loop over the lanes' different addresses.)
OASIS_DEV int fixed(const int32_t* p) { return *(const __attribute__((address_space(4))) int32_t*)p; }

OASIS_DEV bool is_seq(const PagesArgs& a, int seq) { return seq >= 0 && seq < a.c.max_seqs; }
OASIS_DEV int len_of(const PagesArgs& a, int seq) {
  return is_seq(a, seq) ? (int)min((int64_t)max(fixed(a.c.lens + seq), 0), a.c.max_pages * a.c.page_size) : 0;
}
// first and last row of a group, kept inside the rows
OASIS_DEV int bound_of(const PagesArgs& a, int g) { return min(max(fixed(a.cu + g), 0), a.n_rows); }
// tokens that group g reads through its first row
OASIS_DEV int prefix_of(const PagesArgs& a, int g, int first_row) {
  return min(max(fixed(a.prefix + g), 0), len_of(a, fixed(a.seqs + first_row)));
}
// the group of a row, or -1: the wave's lanes look at 64 groups at a time
OASIS_DEV int group_of(const PagesArgs& a, int row, int lane) {
  for (int b = 0; b < a.n_groups; b += 64) {
    const int g = b + lane;
    const bool in = g < a.n_groups && bound_of(a, g) <= row && row < bound_of(a, g + 1);
    const uint64_t hit = __ballot(in);
    if (hit) return __builtin_amdgcn_readfirstlane(b + __builtin_ctzll(hit));
  }
  return -1;
}

// tokens of a row's sequence that its group reads for it
OASIS_DEV int shared_of(const PagesArgs& a, int row, int lane) {
  const int g = group_of(a, row, lane);
  return g < 0 ? 0 : prefix_of(a, g, bound_of(a, g));
}

// A part: columns col0 .. col0 + cols - 1 of (rows from base_row on) x (heads of kvh), keys [k0, k1) of table_seq's pages.
struct Part {
  int kvh, base_row, col0, cols, k0, k1, table_seq, part;
};

// The tiles of KS keys from `first` on, every `step`-th of them, again for a wave whose rows do not all see all of them and which a
// value that is not finite has broken: key by key, each query's sums from the keys that it sees.
template <int D, int KS>
OASIS_DEV void by_hand(flash::Tile<D>& w, const PagesArgs& a, const int32_t* table, int64_t head0, int first, int step, int k1,
                       int end) {
  const int h = (threadIdx.x & 63) >> 5, ps = (int)a.c.page_size;
  const int64_t page_size = a.c.n_kv_heads * ps * D;
  w.clear();
#pragma unroll 1
  for (int t0 = first; t0 < k1; t0 += step * KS)
#pragma unroll 1
    for (int key = t0; key < min(t0 + KS, k1); ++key) {
      const int page = fixed(table + key / ps);
      if ((uint32_t)page >= (uint32_t)a.c.n_pages) continue;  // the part is NaN
      const int64_t at = head0 + page * page_size + (key - key / ps * ps) * D;
      const bf16 *k = static_cast<const bf16*>(a.c.k) + at, *v = static_cast<const bf16*>(a.c.v) + at;
      float dot = 0.f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) dot = fmaf(bf2f(w.q[s][j]), bf2f(k[16 * s + 8 * h + j]), dot);
      dot = sum_xor32(dot);
      if (key >= end) continue;
      const float to = fmaxf(w.m, dot);
      const flash::Base base = top_base(to, a.scale_log2);  // as in settle: the joins take it to be this one
      const float alpha = to == w.m ? 1.f : __builtin_amdgcn_exp2f(flash::shift(flash::split_base(w.m, a.scale_log2), base, a.scale_log2));
      const float p = __builtin_amdgcn_exp2f(fmaf(dot - base.raw, a.scale_log2, -base.number));
      w.m = to;
      w.l = w.l * alpha + (h ? 0.f : p);  // the halves of a wave add up
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) w.o[d][i] = w.o[d][i] * alpha + p * bf2f(v[32 * d + 8 * (i >> 2) + 4 * h + (i & 3)]);
    }
}

// For 32 columns, on tiles that the waves take in turn.
template <int D>
struct Walk {
  typedef flash::Tile<D> Tile;
  static constexpr int S = NW;                       // waves that take tiles in turn
  static constexpr int KT = 32;                      // keys of a tile
  static constexpr int ROW = Tile::ROW, HALF = KT * ROW, STAGE = 2 * HALF;
  static constexpr int RPB = 1024 / ROW;             // rows of a 1 KB load
  static constexpr int LPW = 2 * KT / RPB;       // loads of a wave and stage
  static constexpr int NG = LPW * RPB / 16;          // 16-key groups of a wave's loads: a page each
  static constexpr int REGS = D / 2;                 // outputs of a lane
  static constexpr int MERGE = NW * REGS * 256;
  static constexpr int SMEM = S * STAGE > MERGE ? S * STAGE : MERGE;
  static_assert(LPW * RPB == 2 * KT && NG * 16 == LPW * RPB && LPW <= 63, "loads");

  static OASIS_WALK void go(const PagesArgs& a, const Part& pt, char* smem, WaveSum (*wml)[32], int* missing) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 31, h = lane >> 5;
    const int hk = (int)a.c.n_kv_heads, ps = (int)a.c.page_size;
    const int k0 = pt.k0, k1 = pt.k1;  // k0 is a multiple of MIN_CHUNK
    const int n = (k1 - k0 + KT - 1) / KT, rounds = (n + S - 1) / S;
    // this lane's column: its row and head, and where its sequence ends
    const int flat = pt.col0 + min(lr, pt.cols - 1), row = pt.base_row + flat / a.group,
              head = pt.kvh * a.group + flat % a.group;
    const int32_t* table = a.c.tables + (int64_t)(is_seq(a, pt.table_seq) ? pt.table_seq : 0) * a.c.max_pages;
    char* stage = smem + wave * STAGE;
    // of the layer's page 0, key head kvh; a page of all its key heads
    const int64_t head0 = (a.layer * a.c.n_pages * hk + pt.kvh) * ps * D, page_size = (int64_t)hk * ps * D;
    bool bad = false;
    int page[NG];  // of the next tile's groups: looked up a tile ahead

    // the loads are the stage's keys and then values; 16 rows of them lie in one page. Groups past the part are its last one,
    // masked below.
    auto group_key = [&](int tile, int g) {
      return min(k0 + tile * KT + g * 16 % KT, (k1 - 1) & ~15);
    };
    auto look = [&](int tile) {
#pragma unroll
      for (int g = 0; g < NG; ++g) page[g] = fixed(table + group_key(tile, g) / ps);
    };
    auto issue = [&](int tile) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int key = group_key(tile, g), slot = key - key / ps * ps;
        const bool out = (uint32_t)page[g] >= (uint32_t)a.c.n_pages;
        bad |= out;
        const int64_t at = head0 + (out ? 0 : page[g]) * page_size + slot * D;
        const int first = g * 16;  // of the stage's rows
        const bool isv = first >= KT;
        const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(static_cast<const bf16*>(isv ? a.c.v : a.c.k) + at);
#pragma unroll
        for (int u = 0; u < 16 / RPB; ++u) {
          const int r = u * RPB + lane / (ROW / 16), x = lane % (ROW / 16), rr = first % KT + r;
          const uint32_t off = r * ROW + (isv ? flash::v_unit<D>(rr, x) : flash::k_unit<D>(rr, x)) * 16;
          char* to = stage + (first / RPB + u) * 1024;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)to, 16, off, 0, 0, 0);
        }
      }
    };

    if (wave < n) {
      look(wave);
      issue(wave);
      if (wave + S < n) look(wave + S);
    }
    Tile w;
    w.clear();
    const int end = len_of(a, fixed(a.seqs + row));
    {
      const bf16* qp = a.q + (int64_t)row * a.ld_q + head * D + 8 * h;
#pragma unroll
      for (int s = 0; s < Tile::DS; ++s) w.q[s] = *reinterpret_cast<const bf16x8*>(qp + 16 * s);
    }
    auto leave = [&](int it) {
      const int t = it * S + wave;
      if (t + S < n) {
        __builtin_amdgcn_s_waitcnt(0xF | (3 << 14) | (0x7 << 4));  // the stage is read before it is loaded again
        issue(t + S);
        if (t + 2 * S < n) look(t + 2 * S);
      }
    };
    auto careful = [&](int it) {
      const int t = it * S + wave, key0 = k0 + t * KT;
      __builtin_amdgcn_s_waitcnt(0);
      const char* kb = stage;
      char* vb = stage + HALF;
      if (key0 + KT > k1 && t < n)  // keys outside the part: what their slots hold must not count
        for (int x = lane; x < HALF / 16; x += 64) {
          const int key = key0 + x / (ROW / 16);
          if (key >= k1) *reinterpret_cast<f32x4*>(vb + x * 16) = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      if (t < n) {
        f32x16 s = w.scores(kb, lane);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + 8 * (i >> 2) + 4 * h + (i & 3) >= min(k1, end)) s[i] = -INFINITY;
        w.template softmax<1>(&s, a.scale_log2);
        w.weigh(s, vb, lane);
      }
      leave(it);
    };
    // The last round has the part's end, and from some round on a row may have ended; before them tiles without masks, in a
    // loop without the registers that masks take.
    int least = end;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) least = min(least, __shfl_xor(least, o, 64));
    least = __builtin_amdgcn_readfirstlane(least);
    const int whole = max(least - k0 - wave * KT, 0) / KT;  // tiles from the wave's first on that every column sees whole
    const int plain = min(rounds - 1, (whole + S - 1) / S);
    int it = 0;
#pragma unroll 1
    while (it < plain) {
      __builtin_amdgcn_s_waitcnt(0);
      const char *kb = stage, *vb = stage + HALF;
      f32x16 s = w.scores(kb, lane);
      w.template softmax<1>(&s, a.scale_log2);
      w.weigh(s, vb, lane);
      leave(it++);
    }
#pragma unroll 1
    while (it < rounds) careful(it++);
    if (least < k1 && w.broken()) by_hand<D, KT>(w, a, table, head0, k0 + wave * KT, S, k1, end);
    __builtin_amdgcn_s_waitcnt(0);

    // The waves' sums. Lane l of every wave holds the same column's outputs; each wave joins its share.
    const int keys = max(min(k1, end) - k0, 0);  // that this lane's column sees
    // the column's row and head once more: kept over the loops they go to scratch (32 branches 15.9 us, 15.6 this way)
    int again = lr;
    asm volatile("" : "+v"(again));
    const int flat2 = pt.col0 + min(again, pt.cols - 1), row2 = pt.base_row + flat2 / a.group, head2 = pt.kvh * a.group + flat2 % a.group;
    if (bad) *missing = 1;
    __syncthreads();  // every wave is done with its stage, and has said whether it met a page that is not there
    const float lsum = *missing ? NAN : sum_xor32(w.l);
    constexpr int SHARE = REGS / S;
    float m = w.m, l = lsum, y[SHARE];
    {
      f32x4* mine = reinterpret_cast<f32x4*>(smem) + wave * REGS / 4 * 64 + lane;
#pragma unroll
      for (int r = 0; r < REGS; r += 4)
        mine[r / 4 * 64] = f32x4{w.o[r / 16][r % 16], w.o[r / 16][r % 16 + 1], w.o[r / 16][r % 16 + 2], w.o[r / 16][r % 16 + 3]};
      if (h == 0) wml[wave][lr] = WaveSum{w.m, lsum, flash::split_base(w.m, a.scale_log2)};
      __syncthreads();
#pragma unroll
      for (int i = 0; i < S; ++i) m = fmaxf(m, wml[i][lr].m);
      l = 0.f;
#pragma unroll
      for (int r = 0; r < SHARE; ++r) y[r] = 0.f;
      const flash::Base base = top_base(m, a.scale_log2);
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const WaveSum x = wml[i][lr];
        const float f = __builtin_amdgcn_exp2f(flash::shift(x.base, base, a.scale_log2));
        l += f * x.l;
        const f32x4* from = reinterpret_cast<const f32x4*>(smem) + i * REGS / 4 * 64 + lane;
#pragma unroll
        for (int r = 0; r < SHARE; r += 4) {
          const f32x4 z = from[(wave * SHARE + r) / 4 * 64];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[r + j] += f * z[j];
        }
      }
    }
    if (lr >= pt.cols) return;
    if (m == -INFINITY && l == 0.f && keys > 0) l = -1.f;  // no probability is a number, which is not an empty row
    const int64_t slot = ((int64_t)row2 * a.heads + head2) * a.parts + pt.part;
#pragma unroll
    for (int r = 0; r < SHARE; r += 4) {
      const int g = wave * SHARE + r;  // dims 32 dt + 8 b + 4 h
      *reinterpret_cast<f32x4*>(a.o + slot * D + g / 16 * 32 + g % 16 * 2 + 4 * h) = f32x4{y[r], y[r + 1], y[r + 2], y[r + 3]};
    }
    if (wave == 0 && h == 0) a.ml[slot] = Sum{m, l};
  }
};

// The same for 256 columns, 32 to each wave, on tiles that all eight read.
template <int D>
struct Crowd {
  typedef flash::Tile<D> Tile;
  typedef flash::Turns<D> Turns;
  static constexpr int ROW = Tile::ROW, RPB = Turns::RPB, KS = Turns::KS, SMEM = Turns::SMEM;

  static OASIS_WALK void go(const PagesArgs& a, const Part& pt, char* smem, int* missing) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 31, h = lane >> 5;
    const int hk = (int)a.c.n_kv_heads, ps = (int)a.c.page_size;
    const int k0 = pt.k0, k1 = pt.k1, n = (k1 - k0 + KS - 1) / KS;  // k0 is a multiple of MIN_CHUNK
    const int flat = pt.col0 + min(wave * 32 + lr, pt.cols - 1), row = pt.base_row + flat / a.group,
              head = pt.kvh * a.group + flat % a.group;
    const int32_t* table = a.c.tables + (int64_t)(is_seq(a, pt.table_seq) ? pt.table_seq : 0) * a.c.max_pages;
    const int64_t head0 = (a.layer * a.c.n_pages * hk + pt.kvh) * ps * D, page_size = (int64_t)hk * ps * D;
    // this wave loads 16 rows, which lie in one page, of every tile's keys or values: looked up a tile ahead. Rows past the
    // part are its last 16, masked.
    const bool isv = wave >= NW / 2;
    const bf16* pool = static_cast<const bf16*>(isv ? a.c.v : a.c.k) + head0;
    auto key_of = [&](int tile) { return min(k0 + tile * KS + wave % 4 * 16, (k1 - 1) & ~15); };
    bool bad = false;
    int page = fixed(table + key_of(n - 1) / ps);
    auto issue = [&](int tile, char* to) {
      const int key = key_of(tile), slot = key - key / ps * ps;
      const bool out = (uint32_t)page >= (uint32_t)a.c.n_pages;
      bad |= out;
      const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(pool + (out ? 0 : page) * page_size + slot * D);
#pragma unroll
      for (int u = 0; u < Turns::LPW; ++u) {
        const int r = u * RPB + lane / (ROW / 16), x = lane % (ROW / 16), rr = wave % 4 * 16 + r;
        const uint32_t off = r * ROW + (isv ? flash::v_unit<D>(rr, x) : flash::k_unit<D>(rr, x)) * 16;
        char* at = to + (wave * Turns::LPW + u) * 1024;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)at, 16, off, 0, 0, 0);
      }
      page = fixed(table + key_of(tile > 0 ? tile - 1 : 0) / ps);
    };
    Tile w;
    w.clear();
    const int end = len_of(a, fixed(a.seqs + row)), last = min(k1, end) - 1 - k0;  // the last key that this lane's column sees
    {
      const bf16* qp = a.q + (int64_t)row * a.ld_q + head * D + 8 * h;
#pragma unroll
      for (int s = 0; s < Tile::DS; ++s) w.q[s] = *reinterpret_cast<const bf16x8*>(qp + 16 * s);
    }
    int least = last;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) least = min(least, __shfl_xor(least, o, 64));
    least = __builtin_amdgcn_readfirstlane(least);
    Turns::template go<true>(w, smem, n, wave * 32 < pt.cols ? 0 : n, last, least, a.scale_log2, issue);
    if (least < k1 - 1 - k0 && w.broken()) by_hand<D, KS>(w, a, table, head0, k0, 1, k1, end);
    if (bad) *missing = 1;
    __syncthreads();
    float l = *missing ? NAN : sum_xor32(w.l);
    if (wave * 32 + lr >= pt.cols) return;
    if (w.m == -INFINITY && l == 0.f && last >= 0) l = -1.f;  // no probability is a number, which is not an empty row
    const int64_t slot = ((int64_t)row * a.heads + head) * a.parts + pt.part;
#pragma unroll
    for (int d = 0; d < Tile::DT; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *reinterpret_cast<f32x4*>(a.o + slot * D + 32 * d + 8 * b + 4 * h) =
            f32x4{w.o[d][4 * b], w.o[d][4 * b + 1], w.o[d][4 * b + 2], w.o[d][4 * b + 3]};
    if (h == 0) a.ml[slot] = Sum{w.m, l};
  }
};

// Part `id` of the prefixes.
template <int D, int R>
using Kind = typename std::conditional<R == 8, Crowd<D>, Walk<D>>::type;
template <int D, int R>
OASIS_DEV void prefix_part(const PagesArgs& a, int id, char* smem, WaveSum (*wml)[32], int* missing) {
  const int lane = threadIdx.x & 63, hk = (int)a.c.n_kv_heads;
  Part p;
  constexpr int COLS = 32 * R;
  const int per = hk * a.p_splits;  // the tiles of one run of keys on one XCD, where `per` is a multiple of 8
  int tile = id / per, rest = id - tile * per, g = -1, b0 = 0, b1 = 0;
  p.part = rest / hk;
  p.kvh = rest - p.part * hk;
  for (int b = 0; b < a.n_groups; b += 64) {  // the group that has the tile
    const int i = b + lane;
    int lo = 0, hi = 0;
    if (i < a.n_groups) {
      lo = bound_of(a, i);
      hi = max(bound_of(a, i + 1), lo);
    }
    int x = ((hi - lo) * a.group + COLS - 1) / COLS;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    const uint64_t hit = __ballot(x > tile);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      g = b + src;
      b0 = __shfl(lo, src, 64);
      b1 = __shfl(hi, src, 64);
      tile -= __shfl(x, src, 64) - ((b1 - b0) * a.group + COLS - 1) / COLS;
      break;
    }
    tile -= __shfl(x, 63, 64);
  }
  if (g < 0) return;
  g = __builtin_amdgcn_readfirstlane(g);
  b0 = __builtin_amdgcn_readfirstlane(b0);
  const int n = prefix_of(a, g, b0), chunk = chunk_of(n, a.p_splits, MIN_CHUNK);
  p.k0 = __builtin_amdgcn_readfirstlane(min(n, p.part * chunk));
  p.k1 = __builtin_amdgcn_readfirstlane(min(n, p.part * chunk + chunk));
  p.base_row = __builtin_amdgcn_readfirstlane(b0);
  p.col0 = __builtin_amdgcn_readfirstlane(tile * COLS);
  p.cols = __builtin_amdgcn_readfirstlane(min(COLS, (b1 - b0) * a.group - tile * COLS));
  p.table_seq = fixed(a.seqs + p.base_row);
  if (p.k0 < p.k1) {
    if constexpr (R == 8)
      Kind<D, R>::go(a, p, smem, missing);
    else
      Kind<D, R>::go(a, p, smem, wml, missing);
  } else if ((int)threadIdx.x < p.cols) {
    const int flat = p.col0 + (int)threadIdx.x, row = p.base_row + flat / a.group, head = p.kvh * a.group + flat % a.group;
    a.ml[((int64_t)row * a.heads + head) * a.parts + p.part] = Sum{-INFINITY, 0.f};
  }
}

// Where 16-byte unit u of value row r lies in the row, for the 16-row reads of own_kernel.
template <int D>
OASIS_DEV int v16_unit(int r, int u) { return u ^ ((D == 128 ? r & 7 : (r >> 1) & 3) << 1); }
// The dim of output register r of lane group g there.
OASIS_DEV int dim_of(int r, int g) { return r / 4 * 16 + 4 * g + r % 4; }

// A row's own tokens: 16 columns, the heads [16 ct, ..) of the row that share a key head, on v_mfma_f32_16x16x32_bf16 (scores
// transposed as in flash::Tile: lane l has column l % 16, keys 4 (l / 16) + i of 16). S waves of the workgroup's eight take
// tiles of 32 keys in turn. A wave's keys go to registers, one tile ahead; its values through LDS, where they are transposed
// on the read.
template <int D, int S>
OASIS_DEV void own_part(const PagesArgs& a, int block, char* smem, WaveSum (*wml)[32]) {
  constexpr int KT = 32, ROW = D * 2, STAGE = KT * ROW, RPB = 1024 / ROW, DS = D / 32, DT = D / 16, REGS = D / 4, SHARE = REGS / S;
  static_assert(REGS * 256 <= STAGE && SHARE * S == REGS, "the sums fit where the values were");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sg = wave % S, lr = lane & 15, g = lane >> 4;
  const int hk = (int)a.c.n_kv_heads, ps = (int)a.c.page_size;
  // the item: (row, key head, 16 columns, split)
  const int per = a.s_splits * a.s_tiles, items = a.n_rows * hk * per;
  const int id = block * (NW / S) + wave / S;
  const bool there = id < items;
  const int rh = (there ? id : 0) / per, rest = (there ? id : 0) - rh * per;
  const int row = rh / hk, kvh = rh - row * hk, part = rest / a.s_tiles, col0 = (rest - part * a.s_tiles) * 16;
  const int cols = min(16, a.group - col0), head = kvh * a.group + col0 + min(lr, cols - 1);
  const int seq = fixed(a.seqs + row);
  const int shared = shared_of(a, row, lane), len = len_of(a, seq), own = there ? max(len - shared, 0) : 0;
  const int chunk = chunk_of(own, a.s_splits, 2 * MIN_CHUNK);
  const int k0 = __builtin_amdgcn_readfirstlane(shared + min(own, part * chunk)),
            k1 = __builtin_amdgcn_readfirstlane(shared + min(own, part * chunk + chunk));
  const int base = k0 & ~15, n = k0 < k1 ? (k1 - base + KT - 1) / KT : 0;
  const int32_t* table = a.c.tables + (int64_t)(is_seq(a, seq) ? seq : 0) * a.c.max_pages;
  const int64_t head0 = (a.layer * a.c.n_pages * hk + kvh) * ps * D, page_size = (int64_t)hk * ps * D;
  char* vb = smem + wave * STAGE;
  bool bad = false;
  int64_t at[KT / 16];  // of the 16-key groups of the tile that is looked up
  auto look = [&](int tile) {  // groups past the part are its last one, masked below
#pragma unroll
    for (int x = 0; x < KT / 16; ++x) {
      const int key = min(base + tile * KT + x * 16, (k1 - 1) & ~15), j = key / ps, page = fixed(table + j);
      const bool out = (uint32_t)page >= (uint32_t)a.c.n_pages;
      bad |= out;
      at[x] = head0 + (out ? 0 : page) * page_size + (key - j * ps) * D;
    }
  };
  bf16x8 kf[KT / 16][DS];
  auto load_k = [&]() {
#pragma unroll
    for (int x = 0; x < KT / 16; ++x) {
      const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(static_cast<const bf16*>(a.c.k) + at[x]);
#pragma unroll
      for (int d = 0; d < DS; ++d)
        kf[x][d] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, lr * ROW + g * 16, d * 64, 0));
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int x = 0; x < KT / 16; ++x) {
      const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(static_cast<const bf16*>(a.c.v) + at[x]);
#pragma unroll
      for (int u = 0; u < 16 / RPB; ++u) {
        const int r = u * RPB + lane / (ROW / 16), unit = lane % (ROW / 16);
        const uint32_t off = r * ROW + v16_unit<D>(r, unit) * 16;
        char* to = vb + (x * 16 / RPB + u) * 1024;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)to, 16, off, 0, 0, 0);
      }
    }
  };

  bf16x8 q[DS];
  f32x4 o[DT];
  float m = -INFINITY, l = 0.f;
  flash::Base was{-INFINITY, 0.f};
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 s[2];
  auto scores = [&](int t) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      s[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < DS; ++d) s[x] = mfma16(kf[x][d], q[d], s[x]);
    }
    const int key0 = base + t * KT;
    if (key0 < k0 || key0 + KT > k1) {  // keys outside the part: what their slots hold must not count
      __builtin_amdgcn_s_waitcnt((0x7 << 4) | (0xF << 8));  // vmcnt(0): the values are there
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 16 * x + 4 * g + i;
          if (key < k0 || key >= k1) s[x][i] = -INFINITY;
        }
#pragma unroll 1
      for (int x = lane; x < STAGE / 16; x += 64) {
        const int key = key0 + x / (ROW / 16);
        if (key < k0 || key >= k1) *reinterpret_cast<f32x4*>(vb + x * 16) = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  };
  // the softmax of flash::Tile::settle and exponents on 8 scores a lane, and the products with the values once all loads but
  // the next keys' have landed (vmcnt of MORE)
  auto weigh = [&](auto more) {
    float mx = s[0][0];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[x][i]);
    mx = max_xor32(max_xor16(mx));
    const float to = fmaxf(m, mx);
    const flash::Base base = top_base(to, a.scale_log2);
    const float alpha = __builtin_amdgcn_exp2f(flash::shift(was, base, a.scale_log2));
    was = flash::Base{to == -INFINITY ? to : base.raw, base.number};  // nothing is taken on a base yet where no score is a number
    m = to;
    // Rounded for the product, as flash::Tile::probs. Here the matrix units have time, but not the registers: with a second
    // product for what the rounding leaves, 256 rows of up to 1000 tokens of 8 key heads of 128 take 126 us for 102 (16 key
    // heads of 64, up to 180 tokens: 23.9 for 23.7), and the prefixes' parts of a row are rounded like this anyway.
    bf16x8 pb;
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[x][i] - base.raw, a.scale_log2, -base.number));
        sum += p;
        pb[4 * x + i] = f2bf(p);
      }
    l = l * alpha + sum;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[d][i] *= alpha;
    __builtin_amdgcn_s_waitcnt((decltype(more)::value ? KT / 16 * DS : 0) | (0x7 << 4) | (0xF << 8));
    // O^T += V^T P^T: k-slot j of lane group g is key 4g + j (j < 4), 16 + 4g + j - 4
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      typedef short i16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) i16x4* lds4;
      const int r = 4 * g + (lr >> 2);  // and 16 rows on: the same permutation
      const char* vr = vb + r * ROW + (v16_unit<D>(r, 2 * d + ((lr & 3) >> 1)) << 4) + (lr & 1) * 8;
      const i16x4 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)vr);
      const i16x4 t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vr + 16 * ROW));
      o[d] = mfma16(__builtin_bit_cast(bf16x8, __builtin_shufflevector(t0, t1, 0, 1, 2, 3, 4, 5, 6, 7)), pb, o[d]);
    }
  };
  if (sg < n) {
    // Queries, keys, values in this order, and the last tile apart from the loop: where the compiler cannot tell what was
    // loaded after the keys, it has their products wait for the values too.
    const bf16* qp = a.q + (int64_t)row * a.ld_q + head * D + 8 * g;
#pragma unroll
    for (int d = 0; d < DS; ++d) q[d] = *reinterpret_cast<const bf16x8*>(qp + 32 * d);
    look(sg);
    __builtin_amdgcn_sched_barrier(0);
    load_k();
    load_v();
    int t = sg;
#pragma unroll 1
    for (; t + S < n; t += S) {
      scores(t);
      look(t + S);
      load_k();
      // weigh's wait counts these loads as the last before it: none may sink past it (nor rise past this tile's values, which
      // were loaded in the round before); what is not a load from memory may
      __builtin_amdgcn_sched_barrier(0x38F);
      weigh(std::true_type());
      __builtin_amdgcn_s_waitcnt(0xF | (3 << 14) | (0x7 << 4));  // lgkmcnt(0): the values are read before they are loaded over
      load_v();
    }
    scores(t);
    weigh(std::false_type());
  }
  __builtin_amdgcn_s_waitcnt(0);

  l = sum_xor32(sum_xor16(l));
  if (bad || !is_seq(a, seq)) l = NAN;
  float y[SHARE];
  if constexpr (S > 1) {
    float* mine = reinterpret_cast<float*>(smem + wave * STAGE) + lane;
#pragma unroll
    for (int r = 0; r < REGS; ++r) mine[r * 64] = o[r / 4][r % 4];
    if (g == 0) wml[wave][lr] = WaveSum{m, l, flash::split_base(m, a.scale_log2)};
    __syncthreads();
    const int w0 = wave - sg;
#pragma unroll
    for (int i = 0; i < S; ++i) m = fmaxf(m, wml[w0 + i][lr].m);
    l = 0.f;
#pragma unroll
    for (int r = 0; r < SHARE; ++r) y[r] = 0.f;
    const flash::Base base = top_base(m, a.scale_log2);
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const WaveSum x = wml[w0 + i][lr];
      const float f = __builtin_amdgcn_exp2f(flash::shift(x.base, base, a.scale_log2));
      l += f * x.l;
      const float* from = reinterpret_cast<const float*>(smem + (w0 + i) * STAGE) + lane;
#pragma unroll
      for (int r = 0; r < SHARE; ++r) y[r] += f * from[(sg * SHARE + r) * 64];
    }
  } else {
#pragma unroll
    for (int r = 0; r < SHARE; ++r) y[r] = o[r / 4][r % 4];
  }
  if (!there || lr >= cols) return;
  if (m == -INFINITY && l == 0.f && k1 > k0) l = -1.f;  // no probability is a number, which is not an empty row
  const int64_t slot = ((int64_t)row * a.heads + head) * a.parts;
  constexpr int V = SHARE < 4 ? SHARE : 4;  // dims side by side
  if (a.parts > a.p_splits) {
    float* to = a.o + (slot + a.p_splits + part) * D;
#pragma unroll
    for (int r = 0; r < SHARE; ++r) to[dim_of(sg * SHARE + r, g)] = y[r];
    if (sg == 0 && g == 0) a.ml[slot + a.p_splits + part] = Sum{m, l};
    return;
  }
  if (shared > 0) {  // all of the row's own: the prefix's parts join here
    const Sum* ml = a.ml + slot;
    float top = m;
#pragma unroll 8
    for (int p = 0; p < a.p_splits; ++p) top = fmaxf(top, ml[p].m);
    const flash::Base base = top_base(top, a.scale_log2);
    const float f = __builtin_amdgcn_exp2f(flash::shift(flash::split_base(m, a.scale_log2), base, a.scale_log2));
    bool none = l == 0.f;
    l *= f;
#pragma unroll
    for (int r = 0; r < SHARE; ++r) y[r] *= f;
    // without branches, so that the loads go out together: what an empty part's outputs hold is dropped
#pragma unroll 4
    for (int p = 0; p < a.p_splits; ++p) {
      const Sum x = ml[p];
      const bool some = x.m != -INFINITY || x.l != 0.f;
      none = none && !some;
      const float e = __builtin_amdgcn_exp2f(flash::shift(flash::split_base(x.m, a.scale_log2), base, a.scale_log2));
      l += some ? e * x.l : 0.f;
      const float* from = a.o + (slot + p) * D;
#pragma unroll
      for (int r = 0; r < SHARE; ++r) {
        const float z = from[dim_of(sg * SHARE + r, g)];
        y[r] += some ? e * z : 0.f;
      }
    }
    if (!none && top == -INFINITY) l = NAN;
  }
  const float inv = l < 0.f ? NAN : l == 0.f ? 0.f : 1.0f / l;
  bf16* to = a.out + (int64_t)row * a.ld_out + head * D;
#pragma unroll
  for (int r = 0; r < SHARE; r += V) {
    const int d = dim_of(sg * SHARE + r, g);
    if constexpr (V == 4) {
      *reinterpret_cast<bf16x4*>(to + d) = bf16x4{f2bf(y[r] * inv), f2bf(y[r + 1] * inv), f2bf(y[r + 2] * inv), f2bf(y[r + 3] * inv)};
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) to[d + j] = f2bf(y[r + j] * inv);
    }
  }
}

constexpr int OWN_SMEM(int D) { return NW * 64 * D; }  // NW * STAGE of own_part

// A workgroup to NW / S items of rows' own tokens.
template <int D, int S>
__global__ __launch_bounds__(NW * 64, 4) void own_kernel(PagesArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[OWN_SMEM(D)];
  __shared__ WaveSum wml[NW][32];
  own_part<D, S>(a, blockIdx.x, smem, wml);
}

template <int D, int R>
__global__ __launch_bounds__(NW * 64, D == 64 && R < 8 ? 4 : 2) void prefix_kernel(PagesArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[Kind<D, R>::SMEM];
  __shared__ WaveSum wml[NW][32];
  __shared__ int missing;
  if (threadIdx.x == 0) missing = 0;
  __syncthreads();
  prefix_part<D, R>(a, blockIdx.x, smem, wml, &missing);
}

// Both kinds of part in one launch: the products of the one beside the loads of the other.
template <int D, int R>
__global__ __launch_bounds__(NW * 64, D == 64 && R < 8 ? 4 : 2) void both_kernel(PagesArgs a, int prefixes) {
  constexpr int SMEM = Kind<D, R>::SMEM > OWN_SMEM(D) ? Kind<D, R>::SMEM : OWN_SMEM(D);
  __shared__ __attribute__((aligned(1024))) char smem[SMEM];
  __shared__ WaveSum wml[NW][32];
  __shared__ int missing;
  if ((int)blockIdx.x < prefixes) {
    if (threadIdx.x == 0) missing = 0;
    __syncthreads();
    prefix_part<D, R>(a, blockIdx.x, smem, wml, &missing);
  } else {
    own_part<D, 8>(a, blockIdx.x - prefixes, smem, wml);
  }
}

// Joins the parts of a row's head by W waves that take parts in turn. A wave's lanes look at 64 parts' sums at once, so the
// outputs' loads wait for nothing but these. Parts without keys have a maximum of -inf and a sum of 0.
template <int D, int W>
__global__ __launch_bounds__(256) void join_kernel(PagesArgs a) {
  constexpr int V = D / 64;
  __shared__ float ys[W > 1 ? W : 1][W > 1 ? D : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int turn = wave % W, rh = blockIdx.x * (4 / W) + wave / W;
  if (rh >= a.n_rows * a.heads) return;  // whole workgroups where W > 1
  const int row = rh / a.heads, head = rh - row * a.heads;
  const Sum* ml = a.ml + (int64_t)rh * a.parts;
  const float* o = a.o + (int64_t)rh * a.parts * D + lane * V;
  // at most 128 parts; a row of no group has none in a prefix
  Sum x[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) x[j] = lane + 64 * j < a.parts ? ml[lane + 64 * j] : Sum{-INFINITY, 0.f};
  const int p0 = a.p_splits > 0 && group_of(a, row, lane) < 0 ? a.p_splits : 0;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (lane + 64 * j < p0) x[j] = Sum{-INFINITY, 0.f};
  const float m = wave_max(fmaxf(x[0].m, x[1].m));
  const flash::Base base = top_base(m, a.scale_log2);
  float y[V] = {}, f[2];
  bool used[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    f[j] = __builtin_amdgcn_exp2f(flash::shift(flash::split_base(x[j].m, a.scale_log2), base, a.scale_log2));
    used[j] = !(x[j].m == -INFINITY && x[j].l == 0.f);
  }
  const uint64_t mask[2] = {__ballot(used[0]), __ballot(used[1])};
  const float l = wave_sum((used[0] ? f[0] * x[0].l : 0.f) + (used[1] ? f[1] * x[1].l : 0.f));
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll 4
    for (int i = turn; i < min(64, a.parts - 64 * j); i += W) {
      if (!(mask[j] >> i & 1)) continue;
      const float e = __shfl(f[j], i, 64);
#pragma unroll
      for (int d = 0; d < V; ++d) y[d] += e * o[(int64_t)(i + 64 * j) * D + d];
    }
  if constexpr (W > 1) {
#pragma unroll
    for (int d = 0; d < V; ++d) ys[turn][lane * V + d] = y[d];
    __syncthreads();
    if (turn) return;
#pragma unroll
    for (int d = 0; d < V; ++d) {
      y[d] = ys[0][lane * V + d];
#pragma unroll
      for (int w = 1; w < W; ++w) y[d] += ys[w][lane * V + d];
    }
  }
  const float inv = !is_seq(a, fixed(a.seqs + row)) ? NAN : (mask[0] | mask[1]) == 0 ? 0.f : m == -INFINITY ? NAN : 1.0f / l;
  bf16* to = a.out + (int64_t)row * a.ld_out + head * D + lane * V;
#pragma unroll
  for (int d = 0; d < V; ++d) to[d] = f2bf(y[d] * inv);
}

// How a call of these sizes is split: the same for the workspace and the launch.
struct Plan {
  int64_t p_waves, p_tiles, p_splits;  // p_waves: R
  int64_t s_waves, s_tiles, s_splits;  // s_waves: S
  bool at_once;                        // prefixes and own tokens in one launch
  int64_t parts() const { return p_splits + (at_once || s_splits > 1 ? s_splits : 0); }
};
Plan plan_of(int64_t n_rows, int64_t n_groups, int64_t max_len, int64_t group, int64_t hk, int64_t D) {
  Plan p;
  auto clamp = [](int64_t x, int64_t most) { return std::max<int64_t>(1, std::min<int64_t>(x, most)); };
  // Nothing is shared, or hardly anything: 128 to 512 rows, each a group with no prefix, of up to 600 tokens, 8 key heads of
  // 128, take 40, 74 and 150 us this way and 58, 108 and 212 in parts.
  if (n_groups >= n_rows) n_groups = 0;
  const int64_t cols = n_groups ? n_rows * group / n_groups : 0;  // of a group, on the average
  // Few columns or many. One group of 8 key heads, us with R = 1 and with 8:
  //   columns of 128    2000 tokens shared   16000         40000
  //    80               15.2, 20.7           26.9, 30.1    54.6, 51.2
  //   240               25.0, 28.1           43.3, 46.3    94.2, 71.7
  //   480               34.8, 29.4           71.4, 67.1   153.6, 108.0
  //   columns of 64
  //    80               12.0, 16.7           18.1, 24.4    27.0, 34.9
  //   132               12.8, 20.9           21.6, 31.8    36.7, 45.8
  //   240               17.2, 22.7           27.2, 34.8    52.1, 50.3
  //   480               21.2, 24.6           41.5, 52.3    92.6, 81.5
  // The border is that of long prefixes; behind shorter ones R = 8 is taken too early, by up to 11 us. (R = 2 was between the two
  // or behind both.)
  p.p_waves = cols * D > 8192 ? 8 : 1;
  p.p_tiles = n_groups ? n_rows * group / (32 * p.p_waves) + n_groups : 0;
  // A part to each CU: the four groups of the kernels' comment take 181 us, 198 with 128 parts, 192 with 384, 200 with 512.
  p.p_splits = n_groups ? clamp(256 / (p.p_tiles * hk), std::min<int64_t>(64, (max_len + 2 * MIN_CHUNK - 1) / (2 * MIN_CHUNK))) : 0;
  p.s_tiles = (group + 15) / 16;
  const int64_t items = n_rows * hk * p.s_tiles;
  // One launch for both. 8 key heads of 128, four groups behind up to 8000 tokens, up to 600 own ones: 2048 items take 112 us
  // and 132 apart, 8192 take 372 and 429; 16384 of 16 key heads 597 and 556. 16 key heads of 64, eight groups behind up to 4000,
  // up to 300 own ones: 4096 items take 64.6 and 66.4, 8192 take 115 and 101. (With own tokens up to 30 it loses earlier: 4096
  // items of 128 take 103 and 81. The host does not know their number.)
  p.at_once = n_groups && items <= 64 * D;
  // Waves of an item, from three tiles of 32 keys a wave: 2048 items of 60 tokens take 11.0 us with one wave and 19.0 with
  // eight, of 130 tokens 17.8 with two and 22.5 with eight, of 260 tokens 33.5 with four and 36.2 with one, of 600 tokens 60.1
  // with eight and 72.1 with one. From 4096 items on eight gain 6 % at most (131 us with four, 123 with eight) and lose 1.5
  // times where max_len is far above the sequences (60 tokens: 25 and 37). Behind prefixes the own tokens may be anything.
  p.s_waves = p.at_once || items < 1024       ? 8
              : n_groups || max_len <= 192    ? (!n_groups && max_len <= 64 ? 1 : 2)
              : max_len <= 384 || items >= 4096 ? 4
                                              : 8;
  // Two workgroups to a CU, one beside prefixes: 32 rows of up to 9000 tokens, 8 key heads of 128, take 115 us, 125 with half
  // as many; 4 rows of 30000 behind 2000 take 64, 98 with half as many.
  p.s_splits = clamp((n_groups ? 256 : 512) / items, std::min<int64_t>(64, max_len / (2 * MIN_CHUNK)));
  return p;
}

int64_t workspace_of(const Plan& p, int64_t n_rows, int64_t heads, int64_t D) { return n_rows * heads * p.parts() * (D + 2) * 4; }

bool sizes_ok(int64_t n_rows, int64_t n_groups, int64_t max_len, int64_t heads, int64_t hk, int64_t D) {
  return n_rows >= 0 && n_rows <= 65536 && n_groups >= 0 && n_groups <= 65536 && max_len > 0 && max_len < (1ll << 30) &&
         hk > 0 && heads > 0 && heads <= 4096 && heads % hk == 0 && (D == 64 || D == 128);
}

template <int D>
int pages_go(const PagesArgs& a, const Plan& p, hipStream_t s) {
  const int64_t hk = a.c.n_kv_heads, prefixes = p.p_tiles * hk * p.p_splits, per = NW / p.s_waves,
                owns = (a.n_rows * hk * p.s_tiles * p.s_splits + per - 1) / per;
  OASIS_REQUIRE((prefixes + owns) * NW * 64 < (1ll << 32), OASIS_ERR_SHAPE, "pages_attention: too many parts");  // one launch's threads
  if (p.at_once) {
    const auto fn = p.p_waves == 8 ? &both_kernel<D, 8> : &both_kernel<D, 1>;
    hipLaunchKernelGGL(fn, dim3((unsigned)(prefixes + owns)), dim3(NW * 64), 0, s, a, (int)prefixes);
  } else {
    if (prefixes) {
      const auto fn = p.p_waves == 8 ? &prefix_kernel<D, 8> : &prefix_kernel<D, 1>;
      hipLaunchKernelGGL(fn, dim3((unsigned)prefixes), dim3(NW * 64), 0, s, a);
      if (const int rc = oasis::check_launch("pages_attention")) return rc;
    }
    const auto fn = p.s_waves == 8   ? &own_kernel<D, 8>
                    : p.s_waves == 4 ? &own_kernel<D, 4>
                    : p.s_waves == 2 ? &own_kernel<D, 2>
                                     : &own_kernel<D, 1>;
    hipLaunchKernelGGL(fn, dim3((unsigned)owns), dim3(NW * 64), 0, s, a);
  }
  if (const int rc = oasis::check_launch("pages_attention")) return rc;
  if (p.parts() == p.p_splits) return OASIS_OK;
  // a wave to each row's head where that fills the chip: 8192 of them take 178 us with the rest of the call, 185 with four to
  // each; 512 take 16.7 and 15.4
  const int64_t rhs = (int64_t)a.n_rows * a.heads;
  if (rhs >= 2048)
    hipLaunchKernelGGL((join_kernel<D, 1>), dim3((unsigned)((rhs + 3) / 4)), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((join_kernel<D, 4>), dim3((unsigned)rhs), dim3(256), 0, s, a);
  return oasis::check_launch("pages_attention");
}

}  // namespace

extern "C" int64_t oasis_pages_attention_workspace(int64_t n_rows, int64_t n_groups, int64_t max_len, int64_t n_heads,
                                                   int64_t n_kv_heads, int64_t head_dim) {
  OASIS_REQUIRE(sizes_ok(n_rows, n_groups, max_len, n_heads, n_kv_heads, head_dim), OASIS_ERR_SHAPE,
                "pages_attention_workspace: bad shape");
  // Of any smaller counts too, whose rows may be split further: of a number of rows in groups one group is split furthest, as
  // more of them are more tiles.
  int64_t most = 0;
  for (int64_t r = 1; r <= n_rows; ++r)
    for (int64_t g = 0; g <= std::min<int64_t>(n_groups, 1); ++g)
      most = std::max(most, workspace_of(plan_of(r, g, max_len, n_heads / n_kv_heads, n_kv_heads, head_dim), r, n_heads, head_dim));
  return most;
}

extern "C" int oasis_pages_attention(const oasis_page_cache_t* cache, int64_t layer, const void* q, int64_t ld_q, void* out,
                                     int64_t ld_out, const int32_t* seqs, int64_t n_rows, const int32_t* cu_groups,
                                     const int32_t* prefix_lens, int64_t n_groups, int64_t max_len, int64_t n_heads,
                                     float scale, void* workspace, int64_t workspace_bytes, oasis_stream_t stream) {
  if (const int rc = oasis::check_page_cache(cache, "pages_attention")) return rc;
  const int64_t hk = cache->n_kv_heads, D = cache->head_dim;
  OASIS_REQUIRE(sizes_ok(n_rows, n_groups, max_len, n_heads, hk, D), OASIS_ERR_SHAPE, "pages_attention: bad shape");
  OASIS_REQUIRE(layer >= 0 && layer < cache->n_layers, OASIS_ERR_SHAPE, "pages_attention: layer %lld of %lld",
                (long long)layer, (long long)cache->n_layers);
  OASIS_REQUIRE(scale > 0 && scale * flash::LOG2E < INFINITY, OASIS_ERR_ARG,
                "pages_attention: the scale must be positive and finite");
  if (n_rows == 0) return OASIS_OK;
  OASIS_REQUIRE(q && out && seqs && (n_groups == 0 || (cu_groups && prefix_lens)), OASIS_ERR_NULL,
                "pages_attention: null pointer");
  OASIS_REQUIRE(oasis_aligned(16, q, out, workspace) && (ld_q | ld_out) % 8 == 0, OASIS_ERR_ARG,
                "pages_attention: rows and workspace must be 16-byte aligned");
  OASIS_REQUIRE(ld_q >= n_heads * D && ld_out >= n_heads * D, OASIS_ERR_SHAPE,
                "pages_attention: leading dimensions below a token's heads");
  const Plan p = plan_of(n_rows, n_groups, max_len, n_heads / hk, hk, D);
  const int64_t need = workspace_of(p, n_rows, n_heads, D);
  OASIS_REQUIRE(need == 0 || workspace, OASIS_ERR_NULL, "pages_attention: null workspace");
  OASIS_REQUIRE(workspace_bytes >= need, OASIS_ERR_SHAPE, "pages_attention: workspace of %lld bytes, the call needs %lld",
                (long long)workspace_bytes, (long long)need);
  PagesArgs a;
  a.c = *cache;
  a.layer = layer;
  a.q = static_cast<const bf16*>(q);
  a.out = static_cast<bf16*>(out);
  a.ld_q = ld_q;
  a.ld_out = ld_out;
  a.seqs = seqs;
  a.cu = cu_groups;
  a.prefix = prefix_lens;
  a.n_rows = (int)n_rows;
  a.n_groups = p.p_splits ? (int)n_groups : 0;
  a.heads = (int)n_heads;
  a.group = (int)(n_heads / hk);
  a.scale_log2 = scale * flash::LOG2E;
  a.p_tiles = (int)p.p_tiles;
  a.p_splits = (int)p.p_splits;
  a.s_tiles = (int)p.s_tiles;
  a.s_splits = (int)p.s_splits;
  a.parts = (int)p.parts();
  a.o = static_cast<float*>(workspace);
  a.ml = reinterpret_cast<Sum*>(a.o + n_rows * n_heads * p.parts() * D);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return D == 128 ? pages_go<128>(a, p, s) : pages_go<64>(a, p, s);
}
