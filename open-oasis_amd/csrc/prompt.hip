// Causal attention over packed prompts of different lengths, grouped heads.
//
// A workgroup of NW waves serves a run of query tokens and hg heads that share a key head, 32 tokens of one head to a
// wave, and walks the keys in tiles of 64 from its last token's down to the first: a wave's first tile is then the one
// with the diagonal, the only one with masked keys, while its output is still zero. Tiles are staged in a ring that all
// waves share.
//
// What bounds it: the softmax of a tile takes the vector units about as long as its products take the matrix units (D = 128:
// 190 vector instructions and 32 products of 32 cycles to a wave and tile; D = 64: the same and 16), so the waves of a SIMD
// take turns at them, kept in step by barriers. 8192 tokens, 32 heads of 128, 8 key heads: 470 to 494 us over runs, 1.11 to
// 1.17 PFLOP/s (a library product of 8192^3 reaches 1.21); before the waves took turns 533. 8192 tokens, 16 heads of 64: 160
// us, 0.86 PFLOP/s.
#include <algorithm>

#include "flash_tile.h"

namespace {

using flash::NW;

struct PromptArgs {
  const bf16 *q, *k, *v;
  bf16* out;
  int64_t ld_q, ld_k, ld_v, ld_out;
  const int32_t* cu;
  int n, total;        // sequences, rows of the buffers
  int hblocks, group;  // blocks of HG query heads, query heads of a key head
  float scale_log2;
};

// The query tile `want` of the packed sequences (tiles of `span` tokens): its sequence's first row and length and its first
// token, or len = 0 past the last tile. Called by whole waves; every bound is kept inside the buffers. Of up to 64 sequences
// the tiles with the most keys come first, whichever sequence's they are: 24 of up to 2304 tokens, 16 heads of 64, take 89
// us, 92 sequence by sequence, whose last long tiles ran alone.
OASIS_DEV void find_tile(const int32_t* cu, int n, int total, int span, int want, int lane, int* row0, int* len, int* first) {
  if (n > 1 && n <= 64) {
    int a = 0, e = 0;
    if (lane < n) {
      a = min(max(cu[lane], 0), total);
      e = min(max(cu[lane + 1], a), total);
    }
    const int tiles = (e - a + span - 1) / span;
    // tiles that are their sequence's i-th or a later one (below 2^24, so a sum of floats)
    const auto from = [&](int i) { return (int)wave_sum((float)max(tiles - i, 0)); };
    *len = 0;
    if (want >= from(0)) return;
    int lo = 0, hi = (int)wave_max((float)tiles);  // from(lo) > want >= from(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (from(mid) > want)
        lo = mid;
      else
        hi = mid;
    }
    const uint64_t has = __ballot(tiles > lo);
    const int rank = want - from(lo + 1);
    const int src = __builtin_ctzll(__ballot((has >> lane & 1) && __popcll(has & ((1ull << lane) - 1)) == rank));
    *row0 = __shfl(a, src, 64);
    *len = __shfl(e, src, 64) - *row0;
    *first = lo * span;
    return;
  }
  int before = 0;
  *len = 0;
  for (int b = 0; b < n; b += 64) {
    const int i = b + lane;
    int a = 0, e = 0;
    if (i < n) {
      a = min(max(cu[i], 0), total);
      e = min(max(cu[i + 1], a), total);
    }
    const int tiles = (e - a + span - 1) / span;
    int x = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    const uint64_t hit = __ballot(before + x > want);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      *row0 = __shfl(a, src, 64);
      *len = __shfl(e, src, 64) - *row0;
      // a sequence's longest tile first
      *first = (__shfl(before + x, src, 64) - 1 - want) * span;
      return;
    }
    before += __shfl(x, 63, 64);
  }
}

template <int D>
__global__ __launch_bounds__(NW * 64) void prompt_kernel(PromptArgs a, int hg) {
  typedef flash::Tile<D> Tile;
  typedef flash::Turns<D> Turns;
  constexpr int KS = Turns::KS, ROW = Tile::ROW, RPB = Turns::RPB;
  __shared__ __attribute__((aligned(1024))) char smem[Turns::SMEM];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hb = blockIdx.x % a.hblocks, want = blockIdx.x / a.hblocks;
  const int span = 32 * NW / hg;
  int row0, len, first;
  find_tile(a.cu, a.n, a.total, span, want, lane, &row0, &len, &first);
  if (len == 0) return;
  row0 = __builtin_amdgcn_readfirstlane(row0);
  len = __builtin_amdgcn_readfirstlane(len);
  first = __builtin_amdgcn_readfirstlane(first);
  const int head = hb * hg + wave % hg, t0 = first + wave / hg * 32;  // this wave's head and first token
  const int kvh = hb * hg / a.group;
  const bf16* kbase = a.k + (int64_t)row0 * a.ld_k + kvh * D;
  const bf16* vbase = a.v + (int64_t)row0 * a.ld_v + kvh * D;

  // this wave loads 16 rows of every tile's keys or values; past the sequence its last row: masked, as it lies past every query
  const bool isv = wave >= NW / 2;
  const int64_t ld = isv ? a.ld_v : a.ld_k;
  const bf16* from = isv ? vbase : kbase;
  auto issue = [&](int tile, char* to) {
    const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(from + (int64_t)tile * KS * ld);
    const int most = len - 1 - tile * KS;
#pragma unroll
    for (int u = 0; u < Turns::LPW; ++u) {
      const int r = wave % 4 * 16 + u * RPB + lane / (ROW / 16), x = lane % (ROW / 16);
      const uint32_t off = (uint32_t)min(r, most) * (uint32_t)ld * 2u + (isv ? flash::v_unit<D>(r, x) : flash::k_unit<D>(r, x)) * 16;
      char* at = to + (wave * Turns::LPW + u) * 1024;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)at, 16, off, 0, 0, 0);
    }
  };

  Tile w;
  w.clear();
  const int lr = lane & 31, h = lane >> 5, my_t = t0 + lr;
  {
    const bf16* qp = a.q + (int64_t)(row0 + min(my_t, len - 1)) * a.ld_q + head * D + 8 * h;
#pragma unroll
    for (int s = 0; s < Tile::DS; ++s) w.q[s] = *reinterpret_cast<const bf16x8*>(qp + 16 * s);
  }
  const int n = (min(first + span, len) + KS - 1) / KS;          // the workgroup's tiles
  const int mine = t0 < len ? min(t0 + 31, len - 1) / KS : -1;  // this wave's last tile
  Turns::template go<false>(w, smem, n, n - 1 - mine, my_t, 0, a.scale_log2, issue);
  if (mine < 0) return;
  const float inv = 1.0f / sum_xor32(w.l);
  w.store(a.out + (int64_t)(row0 + min(my_t, len - 1)) * a.ld_out + head * D, inv, my_t < len, lane);
}

template <int D>
int prompt_go(PromptArgs a, int64_t heads, int hg, hipStream_t s) {
  a.hblocks = (int)(heads / hg);
  const int64_t span = 32 * NW / hg, tiles = a.total / span + std::min<int64_t>(a.n, a.total);
  OASIS_REQUIRE(tiles * a.hblocks * NW * 64 < (1ll << 32), OASIS_ERR_SHAPE, "prompt_attention: too many query tiles");
  hipLaunchKernelGGL((prompt_kernel<D>), dim3((unsigned)(tiles * a.hblocks)), dim3(NW * 64), 0, s, a, hg);
  return oasis::check_launch("prompt_attention");
}

}  // namespace

extern "C" int oasis_prompt_attention(const void* q, int64_t ld_q, const void* k, int64_t ld_k, const void* v, int64_t ld_v,
                                      void* out, int64_t ld_out, const int32_t* cu, int64_t n, int64_t total, int64_t n_heads,
                                      int64_t n_kv_heads, int64_t head_dim, float scale, oasis_stream_t stream) {
  OASIS_REQUIRE(head_dim == 64 || head_dim == 128, OASIS_ERR_SHAPE, "prompt_attention: head_dim must be 64 or 128");
  OASIS_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads <= 4096 && n_heads % n_kv_heads == 0, OASIS_ERR_SHAPE,
                "prompt_attention: n_heads must be a multiple of n_kv_heads, up to 4096");
  OASIS_REQUIRE(n >= 0 && total >= 0 && n <= 65536 && total < (1ll << 30), OASIS_ERR_SHAPE,
                "prompt_attention: bad sequence or token count");
  OASIS_REQUIRE(scale > 0 && scale * flash::LOG2E < INFINITY, OASIS_ERR_ARG,
                "prompt_attention: the scale must be positive and finite");
  if (n == 0 || total == 0) return OASIS_OK;
  OASIS_REQUIRE(q && k && v && out && cu, OASIS_ERR_NULL, "prompt_attention: null pointer");
  OASIS_REQUIRE(ld_q >= n_heads * head_dim && ld_out >= n_heads * head_dim && ld_k >= n_kv_heads * head_dim &&
                    ld_v >= n_kv_heads * head_dim && ld_k < (1 << 24) && ld_v < (1 << 24),
                OASIS_ERR_SHAPE, "prompt_attention: leading dimensions below a token's heads, or too large");
  OASIS_REQUIRE(oasis_aligned(16, q, k, v, out) && (ld_q | ld_k | ld_v | ld_out) % 8 == 0, OASIS_ERR_ARG,
                "prompt_attention: rows must be 16-byte aligned");
  PromptArgs a;
  a.q = static_cast<const bf16*>(q);
  a.k = static_cast<const bf16*>(k);
  a.v = static_cast<const bf16*>(v);
  a.out = static_cast<bf16*>(out);
  a.ld_q = ld_q;
  a.ld_k = ld_k;
  a.ld_v = ld_v;
  a.ld_out = ld_out;
  a.cu = cu;
  a.n = (int)n;
  a.total = (int)total;
  a.group = (int)(n_heads / n_kv_heads);
  a.scale_log2 = scale * flash::LOG2E;
  // Heads of a workgroup read their keys once: 24 prompts of up to 500 tokens, 32 heads of 128, 8 key heads, take 30.6 us with
  // four, 34.9 with two and 39.6 with one; eight gain 3 % at most. A single prompt of 144 tokens takes 11.3 us with four or eight and
  // 10.5 with one or two.
  const int hg = a.group % 4 == 0 ? 4 : a.group % 2 == 0 ? 2 : 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return head_dim == 128 ? prompt_go<128>(a, n_heads, hg, s) : prompt_go<64>(a, n_heads, hg, s);
}
