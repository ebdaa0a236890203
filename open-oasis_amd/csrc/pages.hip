// The pages of a K/V cache: reserving, writing, forking, cutting and compacting, on bookkeeping in device memory.
//
// Every sequence's tokens lie in pages of page_size tokens, which its row of `tables` names in order; `refs` counts the
// sequences on each page, and a page with none is free. Free pages are handed out lowest number first, in the order of the
// call's sequences, so the same calls give the same tables. Reserving, forking and compacting are planned by one workgroup
// (prefix sums over the sequences, then over the pages' references), which checks the call's sequences, lengths and need of
// pages before it changes anything; what it plans (page copies, table entries) is carried out by launches over the whole chip.
// Cutting sequences and writing tokens need no plan. A table entry that names no page is met where the table is walked: a
// fork passes it on, a cut drops it, a write skips it, and attention gives NaN.
//
// What bounds them: a plan is a few dependent passes over some thousand integers, so latency (37 sequences of one token 6.4
// us, 16 prompts of up to 2304 tokens 9.2; forks 4.4 to 5.5 with 3.8 to 4.7 to carry them out, compactions 5.1 to 5.4, cuts 3.0
// to 4.8); the copies and writes read every byte once and write it once.
#include <algorithm>

#include "oasis_common.h"

namespace {

typedef oasis_page_cache_t Cache;

// scratch (cache.work): the copies planned, whether a fork goes ahead, then lists
constexpr int W_COPIES = 0, W_OK = 1, W_LIVE = 2, W_LISTS = 16;
OASIS_DEV int32_t* w_list(const Cache& c) { return c.work + W_LISTS; }                       // [n_pages] pages handed out
OASIS_DEV int32_t* w_src(const Cache& c) { return c.work + W_LISTS + c.n_pages; }            // [n_pages] copies: from
OASIS_DEV int32_t* w_dst(const Cache& c) { return c.work + W_LISTS + 2 * c.n_pages; }        // [n_pages] copies: to
OASIS_DEV int32_t* w_off(const Cache& c) { return c.work + W_LISTS + 3 * c.n_pages; }        // [max_seqs] first page handed out
OASIS_DEV int32_t* w_cow(const Cache& c) { return w_off(c) + c.max_seqs; }                   // [max_seqs] copy's number or -1

constexpr int REFUSED = OASIS_PAGES_FULL | OASIS_PAGES_BAD_CALL;  // these stop every planned call until they are cleared

constexpr int PT = 1024;  // threads of a planning workgroup
constexpr int MAX_SEQS = 65536;

constexpr int NEAR = 2048;  // sequences of a call whose offsets are kept in LDS: a search there takes a tenth of one in memory

struct PlanShared {
  uint32_t claim[MAX_SEQS / 32];  // sequences named by the call
  uint64_t wsum[PT / 64];
  int32_t off[NEAR], cow[NEAR];
  int bad;
};

// Exclusive prefix sum of v over the workgroup; *total gets the sum. Two barriers; sh.wsum is free again after the next one.
template <typename T>
OASIS_DEV T block_scan(T v, PlanShared& sh, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the last call's readers are done
  if (lane == 63) sh.wsum[wave] = x;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < PT / 64; ++w) {
    const T s = (T)sh.wsum[w];
    before += w < wave ? s : 0;
    all += s;
  }
  *total = all;
  return before + x - v;
}

OASIS_DEV int64_t pages_of(int64_t tokens, int64_t page) { return (tokens + page - 1) / page; }

// a sequence's tokens as its length says, or -1 where that is no possible length
OASIS_DEV int64_t tokens_of(const Cache& c, int64_t seq) {
  const int64_t n = c.lens[seq];
  return n >= 0 && n <= c.max_pages * c.page_size ? n : -1;
}

OASIS_DEV void clear_claims(const Cache& c, PlanShared& sh) {
  for (int i = threadIdx.x; i < (int)((c.max_seqs + 31) / 32); i += PT) sh.claim[i] = 0;
  if (threadIdx.x == 0) sh.bad = 0;
  __syncthreads();
}
// names a sequence; false if the call named it before
OASIS_DEV bool claim(PlanShared& sh, int seq) {
  const uint32_t bit = 1u << (seq & 31);
  return !(atomicOr(&sh.claim[seq >> 5], bit) & bit);
}

// The four references from 4q on, those past the pool as if taken.
OASIS_DEV i32x4 refs4(const Cache& c, int64_t q) {
  if (4 * q + 3 < c.n_pages) return *reinterpret_cast<const i32x4*>(c.refs + 4 * q);
  i32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = 4 * q + j < c.n_pages ? c.refs[4 * q + j] : 1;
  return r;
}

// The references of the pool's first 4 PT pages, four to a thread.
OASIS_DEV i32x4 first_refs(const Cache& c) {
  return 4 * (int64_t)threadIdx.x < c.n_pages ? refs4(c, threadIdx.x) : i32x4{1, 1, 1, 1};
}

// Hands the `want` lowest free pages out in order: use(number, page). Returns whether there were as many (the same in every
// thread); if not, none is handed out. Where the first 4 PT pages have them that is one scan of `r0`, their references, loaded
// at the kernel's start; else two passes over the references, of which the second finds them in the caches.
template <typename Use>
OASIS_DEV bool take_free(const Cache& c, int64_t want, PlanShared& sh, const i32x4& r0, Use use) {
  if (want == 0) return true;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t got = 0;
    for (int64_t b = 0; b * 4 < c.n_pages && got < want; b += PT) {
      const int64_t q = b + threadIdx.x;
      const i32x4 r = b == 0 ? r0 : q * 4 < c.n_pages ? refs4(c, q) : i32x4{1, 1, 1, 1};
      uint32_t total;
      int64_t at = got + block_scan<uint32_t>((r[0] == 0) + (r[1] == 0) + (r[2] == 0) + (r[3] == 0), sh, &total);
      if (b == 0 && total >= want) pass = 1;  // the first of them have enough: nothing to look for
      if (pass)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r[j] == 0 && at < want) use(at++, (int)(4 * q + j));
      got += total;
    }
    if (got < want) return false;
  }
  return true;
}

// the largest i of [0, n) with off[i] <= p (off[0] = 0; of equal ones the last)
OASIS_DEV int find_last(const int32_t* off, int n, int64_t p) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (off[mid] <= p)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__global__ __launch_bounds__(PT) void reserve_plan_kernel(Cache c, const int32_t* __restrict__ seqs,
                                                          const int32_t* __restrict__ cu, int n) {
  __shared__ PlanShared sh;
  if (threadIdx.x == 0) c.work[W_COPIES] = 0;
  const i32x4 r0 = first_refs(c);
  if (*c.status & REFUSED) return;
  clear_claims(c, sh);
  // pages that each sequence needs: those past its last, and one in place of a part-filled last page that others share
  uint64_t sum = 0;  // pages in the low 40 bits, copies above
  for (int b = 0; b < n; b += PT) {
    const int i = b + threadIdx.x;
    uint64_t need = 0;
    bool cow = false;
    if (i < n) {
      const int seq = seqs[i];
      const int64_t more = (int64_t)cu[i + 1] - cu[i];
      bool ok = seq >= 0 && seq < c.max_seqs && more >= 0;
      ok = ok && claim(sh, seq);
      const int64_t old = ok ? tokens_of(c, seq) : -1;
      ok = ok && old >= 0 && old + more <= c.max_pages * c.page_size;
      if (ok) {
        const int64_t have = pages_of(old, c.page_size);
        if (more > 0 && old % c.page_size) {
          const int last = c.tables[seq * c.max_pages + have - 1];
          ok = last >= 0 && last < c.n_pages;
          cow = ok && c.refs[last] > 1;
        }
        need = pages_of(old + more, c.page_size) - have + cow;
      }
      if (!ok) sh.bad = 1;
    }
    uint64_t total;
    const uint64_t at = sum + block_scan(need + ((uint64_t)cow << 40), sh, &total);
    if (i < n) {
      const int32_t first = (int32_t)std::min<uint64_t>(at & ((1ull << 40) - 1), 0x7fffffff), copy = cow ? (int32_t)(at >> 40) : -1;
      if (n <= NEAR) {
        sh.off[i] = first;
        sh.cow[i] = copy;
      } else {
        w_off(c)[i] = first;
        w_cow(c)[i] = copy;
      }
    }
    sum += total;
  }
  __syncthreads();
  const int64_t want = (int64_t)(sum & ((1ull << 40) - 1));
  const int32_t* offs = n <= NEAR ? sh.off : w_off(c);
  const int32_t* cows = n <= NEAR ? sh.cow : w_cow(c);
  const auto use = [&](int64_t p, int id) {
    const int i = find_last(offs, n, p), seq = seqs[i], copy = cows[i];
    const int64_t j = p - offs[i], have = pages_of(c.lens[seq], c.page_size);
    int32_t* entry = c.tables + seq * c.max_pages + have - (copy >= 0) + j;
    if (copy >= 0 && j == 0) {
      const int from = *entry;
      w_src(c)[copy] = from;
      w_dst(c)[copy] = id;
    }
    *entry = id;
    c.refs[id] = 1;
  };
  if (sh.bad || !take_free(c, want, sh, r0, use)) {
    if (threadIdx.x == 0) atomicOr(c.status, sh.bad ? OASIS_PAGES_BAD_CALL : OASIS_PAGES_FULL);
    return;
  }
  __syncthreads();  // every length and reference is read
  for (int i = threadIdx.x; i < n; i += PT) c.lens[seqs[i]] += cu[i + 1] - cu[i];
  // the shared pages that were copied, which become free where nobody is left on them
  for (int i = threadIdx.x; i < (int)(sum >> 40); i += PT) atomicSub(c.refs + w_src(c)[i], 1);
  if (threadIdx.x == 0) c.work[W_COPIES] = (int32_t)(sum >> 40);
}

__global__ __launch_bounds__(PT) void fork_plan_kernel(Cache c, const int32_t* __restrict__ parents,
                                                       const int32_t* __restrict__ children, int n, int copy) {
  __shared__ PlanShared sh;
  if (threadIdx.x == 0) c.work[W_COPIES] = c.work[W_OK] = 0;
  const i32x4 r0 = first_refs(c);
  if (*c.status & REFUSED) return;
  clear_claims(c, sh);
  for (int i = threadIdx.x; i < n; i += PT) {
    const int a = parents[i], b = children[i];
    if (a < 0 || a >= c.max_seqs || b < 0 || b >= c.max_seqs || !claim(sh, b) || c.lens[b] != 0 || tokens_of(c, a) < 0)
      sh.bad = 1;
  }
  __syncthreads();
  uint64_t sum = 0;
  if (!sh.bad)  // uniform: written before the barrier only
    for (int b = 0; b < n; b += PT) {
      const int i = b + threadIdx.x;
      uint64_t need = 0;
      if (i < n) need = copy ? pages_of(c.lens[parents[i]], c.page_size) : 0;
      uint64_t total;
      const uint64_t at = sum + block_scan(need, sh, &total);
      if (i < n) w_off(c)[i] = (int32_t)std::min<uint64_t>(at, 0x7fffffff);
      sum += total;
    }
  __syncthreads();
  // a parent that is one of the children has no length to go by
  if (!sh.bad)
    for (int i = threadIdx.x; i < n; i += PT)
      if (sh.claim[parents[i] >> 5] >> (parents[i] & 31) & 1) sh.bad = 2;
  __syncthreads();
  if (sh.bad || !take_free(c, (int64_t)sum, sh, r0, [&](int64_t p, int id) { w_list(c)[p] = id; })) {
    if (threadIdx.x == 0) atomicOr(c.status, sh.bad ? OASIS_PAGES_BAD_CALL : OASIS_PAGES_FULL);
    return;
  }
  if (threadIdx.x == 0) {
    c.work[W_COPIES] = (int32_t)sum;
    c.work[W_OK] = 1;
  }
}

// one workgroup to a child: its table row, the references, and the copies' list
__global__ __launch_bounds__(256) void fork_apply_kernel(Cache c, const int32_t* __restrict__ parents,
                                                         const int32_t* __restrict__ children, int copy) {
  if (!c.work[W_OK]) return;
  const int i = blockIdx.x, a = parents[i], b = children[i];
  const int64_t n = pages_of(c.lens[a], c.page_size);
  const int32_t* from = c.tables + a * c.max_pages;
  int32_t* to = c.tables + b * c.max_pages;
  for (int64_t t = threadIdx.x; t < n; t += 256) {
    const int p = from[t];
    const bool in = p >= 0 && p < c.n_pages;
    if (copy) {  // the page for an entry that names none stays free: copied onto itself
      const int at = w_off(c)[i] + (int)t, id = w_list(c)[at];
      w_src(c)[at] = in ? p : id;
      w_dst(c)[at] = id;
      if (in) c.refs[id] = 1;
      to[t] = in ? id : p;
    } else {
      if (in) atomicAdd(c.refs + p, 1);
      to[t] = p;
    }
    if (!in) atomicOr(c.status, OASIS_PAGES_BAD_ENTRY);
  }
  if (threadIdx.x == 0) c.lens[b] = c.lens[a];
}

// One workgroup to an entry of the call. The minimum taken atomically hands each page of a sequence that is named twice
// to one of the two, whichever comes first, so the result does not depend on their order.
__global__ __launch_bounds__(256) void truncate_kernel(Cache c, const int32_t* __restrict__ seqs,
                                                       const int32_t* __restrict__ keep) {
  __shared__ int was;
  const int seq = seqs[blockIdx.x], left = keep ? keep[blockIdx.x] : 0;
  if (seq < 0 || seq >= c.max_seqs || left < 0) {
    if (threadIdx.x == 0) atomicOr(c.status, OASIS_PAGES_BAD_ENTRY);
    return;
  }
  if (threadIdx.x == 0) was = atomicMin(c.lens + seq, left);
  __syncthreads();
  const int64_t end = std::min<int64_t>(pages_of(was, c.page_size), c.max_pages);
  int32_t* row = c.tables + seq * c.max_pages;
  for (int64_t t = pages_of(left, c.page_size) + threadIdx.x; t < end; t += 256) {
    const int p = row[t];
    row[t] = -1;
    if (p < 0 || p >= c.n_pages || atomicSub(c.refs + p, 1) <= 0) {
      if (p >= 0 && p < c.n_pages) atomicAdd(c.refs + p, 1);
      atomicOr(c.status, OASIS_PAGES_BAD_ENTRY);
    }
  }
}

// Pages in use from the number of pages in use on move, in order, into the gaps below it: sources and destinations are
// apart, and no other plan moves fewer pages.
__global__ __launch_bounds__(PT) void compact_plan_kernel(Cache c) {
  __shared__ PlanShared sh;
  if (threadIdx.x == 0) c.work[W_COPIES] = c.work[W_LIVE] = 0;
  if (*c.status & REFUSED) return;
  const int64_t quads = (c.n_pages + 3) / 4;
  int mine = 0;
  for (int64_t q = threadIdx.x; q < quads; q += PT) {
    const i32x4 r = refs4(c, q);
#pragma unroll
    for (int j = 0; j < 4; ++j) mine += 4 * q + j < c.n_pages && r[j] != 0;
  }
  uint64_t live;
  block_scan<uint64_t>(mine, sh, &live);
  uint64_t sum = 0;  // gaps in the low half, pages to move above
  for (int64_t b = 0; b < quads; b += PT) {
    const int64_t q = b + threadIdx.x;
    const i32x4 r = q < quads ? refs4(c, q) : i32x4{1, 1, 1, 1};
    uint64_t mark[4], total, count = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t p = 4 * q + j;
      mark[j] = p >= (uint64_t)c.n_pages ? 0 : p < live ? (uint64_t)(r[j] == 0) : (uint64_t)(r[j] != 0) << 32;
      count += mark[j];
    }
    uint64_t at = sum + block_scan(count, sh, &total);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = (int)(4 * q + j);
      if (mark[j] == 1) w_dst(c)[at & 0xffffffff] = p;
      if (mark[j] > 1) w_src(c)[at >> 32] = p;
      if (mark[j] == 0 && p < c.n_pages) w_list(c)[p] = p;  // stays where it is
      at += mark[j];
    }
    sum += total;
  }
  __syncthreads();
  const int moves = (int)(sum >> 32);  // as many as gaps
  for (int i = threadIdx.x; i < moves; i += PT) {
    const int from = w_src(c)[i], to = w_dst(c)[i];
    w_list(c)[from] = to;
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
  }
  if (threadIdx.x == 0) {
    c.work[W_COPIES] = moves;
    c.work[W_LIVE] = (int32_t)live;
  }
}

OASIS_DEV void compact_tables(const Cache& c, int block, int blocks) {
  const int live = c.work[W_LIVE];
  for (int64_t seq = block; seq < c.max_seqs; seq += blocks) {
    const int64_t n = pages_of(std::max<int64_t>(0, tokens_of(c, seq)), c.page_size);
    int32_t* row = c.tables + seq * c.max_pages;
    for (int64_t t = threadIdx.x; t < n; t += 256) {
      const int p = row[t];
      if (p >= live && p < c.n_pages) row[t] = w_list(c)[p];
    }
  }
}

// The planned copies, every layer's keys and values: pieces of 16 KB at most, in page order: bandwidth (5.2 TB/s read and
// written where a compaction moves 0.8 GB, 5.3 in a fork with copies of as much). The first `tables` workgroups
// let the tables follow a compaction.
constexpr int PIECE = 1024;  // 16-byte vectors
__global__ __launch_bounds__(256) void copy_pages_kernel(Cache c, int64_t vecs, int tables) {
  if (!c.work[W_COPIES]) return;
  if ((int)blockIdx.x < tables) {
    compact_tables(c, blockIdx.x, tables);
    return;
  }
  const int64_t pieces = (vecs + PIECE - 1) / PIECE, per_copy = pieces * c.n_layers * 2;
  const int64_t n = (int64_t)c.work[W_COPIES] * per_copy;
  for (int64_t u = blockIdx.x - tables; u < n; u += gridDim.x - tables) {
    const int64_t copy = u / per_copy, rest = u - copy * per_copy, plane = rest / pieces, piece = rest - plane * pieces;
    f32x4* base = static_cast<f32x4*>((plane & 1) ? c.v : c.k) + (plane >> 1) * c.n_pages * vecs + piece * PIECE;
    const f32x4* src = base + w_src(c)[copy] * vecs;
    f32x4* dst = base + w_dst(c)[copy] * vecs;
    const int m = (int)std::min<int64_t>(PIECE, vecs - piece * PIECE);
    f32x4 x[PIECE / 256];
#pragma unroll
    for (int j = 0; j < PIECE / 256; ++j)
      if ((int)threadIdx.x + j * 256 < m) x[j] = ld_stream(src + threadIdx.x + j * 256);
#pragma unroll
    for (int j = 0; j < PIECE / 256; ++j)
      if ((int)threadIdx.x + j * 256 < m) st_stream(dst + threadIdx.x + j * 256, x[j]);
  }
}

// Four consecutive tokens to a workgroup. Their places are looked up once, by one thread each, while their rows (up to PRE
// vectors of keys and of values to a thread) are on their way. Bound by the bytes, each read and written once, and for few
// tokens by the lookup's chain of loads. With the reserve and cut around it, 8 layers of 8 x 128: 4800 tokens 94 us, 117 with
// 16 tokens to a workgroup and nothing ahead, 105 with 2 or 8; 9700 tokens 157, 177, 168 and 166. Four layers of 19400 tokens
// take 148, and 144 with PRE = 1, which has 9700 in 165.
constexpr int WT = 4;
__global__ __launch_bounds__(256) void write_kernel(Cache c, int64_t layer, const bf16* __restrict__ k, int64_t ld_k,
                                                    const bf16* __restrict__ v, int64_t ld_v,
                                                    const int32_t* __restrict__ seqs, const int32_t* __restrict__ cu, int n,
                                                    int64_t total) {
  constexpr int PRE = 2, FEW = 1024;
  __shared__ int64_t place[WT];  // element offset of (page, head 0, slot, dim 0), or -1
  __shared__ int32_t near[FEW];
  const int64_t t0 = (int64_t)blockIdx.x * WT;
  const int tid = threadIdx.x, vph = (int)c.head_dim / 8, vpt = vph * (int)c.n_kv_heads;  // 16-byte vectors of a head, a token
  const int rows = (int)std::min<int64_t>(WT, total - t0), all = rows * vpt;
  const bool refused = *c.status & REFUSED;
  if (n < FEW)
    for (int i = tid; i <= n; i += 256) near[i] = cu[i];
  f32x4 a[PRE], b[PRE];
  auto load = [&](int e, f32x4* x, f32x4* y) {
    const int r = e / vpt;
    *x = ld_stream(reinterpret_cast<const f32x4*>(k + (t0 + r) * ld_k + (e - r * vpt) * 8));
    *y = ld_stream(reinterpret_cast<const f32x4*>(v + (t0 + r) * ld_v + (e - r * vpt) * 8));
  };
  auto store = [&](int e, const f32x4& x, const f32x4& y) {
    const int r = e / vpt, u = e - r * vpt, h = u / vph;
    if (place[r] < 0) return;
    const int64_t to = place[r] + h * c.page_size * c.head_dim + (u - h * vph) * 8;
    *reinterpret_cast<f32x4*>(static_cast<bf16*>(c.k) + to) = x;
    *reinterpret_cast<f32x4*>(static_cast<bf16*>(c.v) + to) = y;
  };
  const int64_t lo = cu[0], hi = cu[n];  // rows of no sequence are not read
  auto in = [&](int e) { return e < all && t0 + e / vpt >= lo && t0 + e / vpt < hi; };
#pragma unroll
  for (int j = 0; j < PRE; ++j)
    if (in(tid + j * 256)) load(tid + j * 256, &a[j], &b[j]);
  __syncthreads();
  if (refused) return;
  if (blockIdx.x == 0 && tid == 0 && (lo < 0 || hi > total)) atomicOr(c.status, OASIS_PAGES_BAD_ENTRY);  // tokens without rows
  const int32_t* cus = n < FEW ? near : cu;
  if (tid < rows) {
    const int64_t t = t0 + tid;
    int64_t at = -1;
    if (t >= lo && t < hi) {
      const int i = find_last(cus, n, t), seq = seqs[i];
      bool ok = seq >= 0 && seq < c.max_seqs && t >= cus[i] && t < cus[i + 1];
      const int64_t len = ok ? tokens_of(c, seq) : -1, pos = len - cus[i + 1] + t;
      ok = ok && len >= 0 && pos >= 0 && pos < len;
      if (ok) {
        const int page = (int)c.page_size, j = (int)pos / page;
        const int p = c.tables[seq * c.max_pages + j];
        ok = p >= 0 && p < c.n_pages;
        at = ok ? ((layer * c.n_pages + p) * c.n_kv_heads * c.page_size + ((int)pos - j * page)) * c.head_dim : -1;
      }
      if (!ok) atomicOr(c.status, OASIS_PAGES_BAD_ENTRY);
    }
    place[tid] = at;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PRE; ++j)
    if (in(tid + j * 256)) store(tid + j * 256, a[j], b[j]);
  for (int e = tid + PRE * 256; e < all; e += 256)
    if (in(e)) {
      f32x4 x, y;
      load(e, &x, &y);
      store(e, x, y);
    }
}

}  // namespace

int oasis::check_page_cache(const Cache* c, const char* what) {
  OASIS_REQUIRE(c, OASIS_ERR_NULL, "%s: null cache", what);
  OASIS_REQUIRE(c->k && c->v && c->refs && c->tables && c->lens && c->status && c->work, OASIS_ERR_NULL,
                "%s: null pointer in the cache", what);
  OASIS_REQUIRE(oasis_aligned(16, c->k, c->v, c->refs) && oasis_aligned(4, c->tables, c->lens, c->status, c->work),
                OASIS_ERR_ARG, "%s: the cache's keys, values and references must be 16-byte aligned", what);
  OASIS_REQUIRE(c->head_dim == 64 || c->head_dim == 128, OASIS_ERR_SHAPE, "%s: head_dim must be 64 or 128", what);
  OASIS_REQUIRE(c->page_size >= 16 && c->page_size <= 1024 && c->page_size % 16 == 0, OASIS_ERR_SHAPE,
                "%s: page_size must be a multiple of 16 up to 1024", what);
  OASIS_REQUIRE(c->n_layers > 0 && c->n_layers <= 65535 && c->n_kv_heads > 0 && c->n_kv_heads <= 1024 && c->n_pages > 0 &&
                    c->n_pages < (1 << 28) && c->max_seqs > 0 && c->max_seqs <= MAX_SEQS && c->max_pages > 0 &&
                    c->max_pages * c->page_size < (1ll << 30),
                OASIS_ERR_SHAPE, "%s: bad cache shape", what);
  return OASIS_OK;
}

namespace {

int check_list(const Cache* c, const void* seqs, int64_t n, const char* what) {
  OASIS_REQUIRE(n >= 0 && n <= c->max_seqs, OASIS_ERR_SHAPE, "%s: %lld sequences, the cache holds %lld", what, (long long)n,
                (long long)c->max_seqs);
  OASIS_REQUIRE(n == 0 || seqs, OASIS_ERR_NULL, "%s: null sequence list", what);
  return OASIS_OK;
}

// the copies of a plan that holds `most` of them at most
int copy_pages(const Cache& c, int64_t most, int tables, hipStream_t s, const char* what) {
  const int64_t vecs = c.n_kv_heads * c.page_size * c.head_dim / 8;
  const int64_t pieces = std::min(most, c.n_pages) * c.n_layers * 2 * ((vecs + PIECE - 1) / PIECE);
  // Four workgroups to a CU: 1.6 GB copied by a compaction take 328 us, 334 with two and 336 with eight to a CU. A plan without
  // copies is a launch of as many that end at once.
  hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)std::min<int64_t>(pieces, 1024) + tables), dim3(256), 0, s, c, vecs, tables);
  return oasis::check_launch(what);
}

}  // namespace

extern "C" int64_t oasis_pages_work(int64_t n_pages, int64_t max_seqs) {
  OASIS_REQUIRE(n_pages > 0 && max_seqs > 0, OASIS_ERR_SHAPE, "pages_work: %lld pages and %lld sequences", (long long)n_pages,
                (long long)max_seqs);
  return W_LISTS + 3 * n_pages + 2 * max_seqs;
}

extern "C" int oasis_pages_reserve(const oasis_page_cache_t* cache, const int32_t* seqs, const int32_t* cu, int64_t n,
                                   oasis_stream_t stream) {
  if (const int rc = oasis::check_page_cache(cache, "pages_reserve")) return rc;
  if (const int rc = check_list(cache, seqs, n, "pages_reserve")) return rc;
  if (n == 0) return OASIS_OK;
  OASIS_REQUIRE(cu, OASIS_ERR_NULL, "pages_reserve: null cu");
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(reserve_plan_kernel, dim3(1), dim3(PT), 0, s, *cache, seqs, cu, (int)n);
  if (const int rc = oasis::check_launch("pages_reserve")) return rc;
  return copy_pages(*cache, n, 0, s, "pages_reserve");
}

extern "C" int oasis_pages_write(const oasis_page_cache_t* cache, int64_t layer, const void* k, int64_t ld_k, const void* v,
                                 int64_t ld_v, const int32_t* seqs, const int32_t* cu, int64_t n, int64_t total,
                                 oasis_stream_t stream) {
  if (const int rc = oasis::check_page_cache(cache, "pages_write")) return rc;
  if (const int rc = check_list(cache, seqs, n, "pages_write")) return rc;
  OASIS_REQUIRE(layer >= 0 && layer < cache->n_layers, OASIS_ERR_SHAPE, "pages_write: layer %lld of %lld", (long long)layer,
                (long long)cache->n_layers);
  OASIS_REQUIRE(total >= 0 && total < (1ll << 26), OASIS_ERR_SHAPE, "pages_write: bad token count");
  if (n == 0 || total == 0) return OASIS_OK;
  OASIS_REQUIRE(k && v && cu, OASIS_ERR_NULL, "pages_write: null pointer");
  const int64_t row = cache->n_kv_heads * cache->head_dim;
  OASIS_REQUIRE(oasis_aligned(16, k, v) && ld_k % 8 == 0 && ld_v % 8 == 0, OASIS_ERR_ARG,
                "pages_write: rows must be 16-byte aligned");
  OASIS_REQUIRE(ld_k >= row && ld_v >= row, OASIS_ERR_SHAPE, "pages_write: leading dimensions below n_kv_heads * head_dim");
  hipLaunchKernelGGL(write_kernel, dim3((unsigned)((total + WT - 1) / WT)), dim3(256), 0, static_cast<hipStream_t>(stream), *cache,
                     layer, static_cast<const bf16*>(k), ld_k, static_cast<const bf16*>(v), ld_v, seqs, cu, (int)n, total);
  return oasis::check_launch("pages_write");
}

extern "C" int oasis_pages_fork(const oasis_page_cache_t* cache, const int32_t* parents, const int32_t* children, int64_t n,
                                int copy, oasis_stream_t stream) {
  if (const int rc = oasis::check_page_cache(cache, "pages_fork")) return rc;
  if (const int rc = check_list(cache, parents, n, "pages_fork")) return rc;
  if (n == 0) return OASIS_OK;
  OASIS_REQUIRE(children, OASIS_ERR_NULL, "pages_fork: null sequence list");
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(PT), 0, s, *cache, parents, children, (int)n, copy != 0);
  if (const int rc = oasis::check_launch("pages_fork")) return rc;
  hipLaunchKernelGGL(fork_apply_kernel, dim3((unsigned)n), dim3(256), 0, s, *cache, parents, children, copy != 0);
  if (const int rc = oasis::check_launch("pages_fork")) return rc;
  return copy ? copy_pages(*cache, n * cache->max_pages, 0, s, "pages_fork") : OASIS_OK;
}

extern "C" int oasis_pages_truncate(const oasis_page_cache_t* cache, const int32_t* seqs, const int32_t* keep, int64_t n,
                                    oasis_stream_t stream) {
  if (const int rc = oasis::check_page_cache(cache, "pages_truncate")) return rc;
  if (const int rc = check_list(cache, seqs, n, "pages_truncate")) return rc;
  if (n == 0) return OASIS_OK;
  hipLaunchKernelGGL(truncate_kernel, dim3((unsigned)n), dim3(256), 0, static_cast<hipStream_t>(stream), *cache, seqs, keep);
  return oasis::check_launch("pages_truncate");
}

extern "C" int oasis_pages_compact(const oasis_page_cache_t* cache, oasis_stream_t stream) {
  if (const int rc = oasis::check_page_cache(cache, "pages_compact")) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(PT), 0, s, *cache);
  if (const int rc = oasis::check_launch("pages_compact")) return rc;
  return copy_pages(*cache, cache->n_pages, (int)std::min<int64_t>(cache->max_seqs, 256), s, "pages_compact");
}
