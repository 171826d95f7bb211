// prefix.cu -- dense attention over the paged latent cache for a batch whose
// requests share one prefix: token t attends to the prefix's rows and then to
// the first token_lens[t] rows of its request's own pages,
//   o = sum_k p_k ckv_k / sum_k p_k,  p_k = exp(sm_scale (q_nope.ckv_k + q_pe.kpe_k)),
//   lse = log2 sum_k p_k.
//
// Every token reads the same prefix rows, so the (token, head) rows of the whole
// batch are stacked and a row block of 128 of them (8 tokens of 16 heads, or one
// of 128) meets each cache row once: 2 * 128 * 1088 operations a cache row of 1152
// bytes, work for the 5th-generation tensor cores.  An accumulator of 128 rows x
// 512 values alone fills a CTA's tensor memory, so a PAIR of CTAs shares a row
// block (tcgen05 cta_group::2, M = 128): each holds 64 of its rows, O takes 256
// TMEM columns and two buffers of scores 64 each.  A tile is two cache pages
// (128 rows): CTA c stages page c for Q.K^T (N = 128 from the pair) and its 256
// of the 512 values of both pages for P.V (N = 256 from the pair).
//
// The pages of a row block form one list -- the prefix, then the own pages of its
// tokens one after the other -- and the lists of all row blocks are dealt out over
// the pairs (one persistent cluster per two SMs); a row block that several pairs
// share is joined by a merge grid.  A token's own page is masked for the
// other tokens of the block twice: their weights are not counted, and the MMA
// leaves their TMEM lanes alone, so a request whose rows hold NaN or infinities
// cannot touch another's output.  Rows behind a length are never read: a partly
// filled page is loaded from a row coordinate below zero, which moves its rows to
// the end of the tile and has the TMA write zeros before them.
//
// Bound by the MMA: 2196 cycles a tile alone (36 at N = 128 of 32.4, 16 at N = 256
// of 64.4), 2510-2800 here.  128 tokens of 128 heads behind 16384 rows: 440-470 us,
// 1.25-1.34 PFLOP/s at the clock that the power limit leaves (91% or more of what a
// cuBLAS product sustains); 64 tokens of 16 heads behind 32768 rows: 66-80 us, 20 of
// them the plan, the first loads, partials and merge.
#include <cuda.h>

#include <mutex>

#include "../../../include/dsa_b200.h"
#include "pair.cuh"

namespace dsa {
namespace {

constexpr int kRows = 64;                      // (token, head) rows per CTA
constexpr int kGroups = 8;                     // 16-head groups per row block
constexpr int kPanel = 64 * 128;               // 64 rows x 64 values, 128-byte swizzle
constexpr int kKChunk = 3 * kPanel;            // a third of the 576 key values of a page
constexpr int kVChunk = 4 * kPanel;            // 128 values of both pages
constexpr int kThreads = 12 * 32;
constexpr int kSoftmaxThreads = 256;
constexpr uint32_t kTmemS = 256;               // TMEM columns: O 0-255, scores 256 and 320
constexpr int kSlotFloats = 2 * kRows * 512 + 4 * kRows;  // partial: O, m, l of 128 rows
constexpr int kCutTiles = 3;  // what a second row block costs a pair: queries, a refill and a partial, in tiles
// Pages of 73728 bytes that stay in the 126 MB of L2 beside the rest: where row blocks
// walk the prefix in step or not makes no difference up to 80000 rows (141.8 and 141.7
// us for 8 tokens of 128 heads); beyond, in step is sooner done (90000 rows 156 against
// 165 us, 131072 218 against 234, 180000 297 against 331).
constexpr int kL2Pages = 1300;
constexpr int kSoloBlocks = 64;  // row blocks that a warp plans alone: 2 a lane
constexpr int kWholeTiles = 3;
constexpr float kLazy = 8.f;  // the running maximum follows only a rise of more than 2^8

struct PrefixParams {
  const int32_t *prefix_pages, *prefix_len, *block_table, *token_request, *token_lens;
  int64_t bt_stride;
  int max_prefix, batch, max_own, num_pages;  // max_own: rows that a row of the block table has room for
  int groups, blocks, group_per_token, max_pairs;
  int share;  // pairs that each row block can have of its own
  int whole;  // one pair each, whatever the plan says: no merge grid follows
  int q_boxes;  // query loads of 64 rows
  float scale_log2;  // above zero
  int negate;        // sm_scale is below zero
  __nv_bfloat16* out;
  int64_t out_st, out_sh;
  float* lse;
  int64_t lse_st, lse_sh;
  int* err;
  // for the merge grid: tiles before each row block [blocks + 1] and the pairs
  // that each has of its own, if so; the row block in which each pair begins
  long long* cum;
  int* begins;
  // partials, two a pair: of the stretch's first row block and, where that is
  // another one, of its last; those between are the pair's alone
  float* parts;
};

__device__ __forceinline__ int prefix_rows(const PrefixParams& p) {
  return p.prefix_len ? min(p.max_prefix, max(*p.prefix_len, 0)) : p.max_prefix;
}
// Row of the block table of token t, and its own rows: what does not fit the
// table is cut off.
__device__ __forceinline__ int request_of(const PrefixParams& p, int t) { return p.token_request ? p.token_request[t] : t; }
__device__ __forceinline__ bool bad_rows(const PrefixParams& p, int request, int len) {
  return len > 0 && (request < 0 || request >= p.batch || len > p.max_own);
}
__device__ __forceinline__ int own_rows(const PrefixParams& p, int request, int len) {
  return request >= 0 && request < p.batch ? min(max(len, 0), p.max_own) : 0;
}
__device__ __forceinline__ int first_token(const PrefixParams& p, int block) {
  return (unsigned)block * kGroups / (unsigned)p.group_per_token;
}
__device__ __forceinline__ int tokens_of(const PrefixParams& p, int block) {
  const unsigned last = min((unsigned)(block + 1) * kGroups, (unsigned)p.groups) - 1;
  return (int)(last / (unsigned)p.group_per_token) - first_token(p, block) + 1;
}
// The tiles of all row blocks in one line are dealt out in stretches of `each`,
// one more for the first `more` pairs; with fewer tiles than pairs some stay idle.
struct Deal {
  long long each;
  int more, pairs;
  __device__ __forceinline__ Deal(const PrefixParams& p, long long tiles) {
    pairs = (int)min((long long)p.max_pairs, tiles);
    each = tiles < (1LL << 31) ? (long long)((unsigned)tiles / (unsigned)pairs) : tiles / pairs;
    more = (int)(tiles - each * pairs);
  }
  __device__ __forceinline__ long long start(int pair) const { return each * pair + min(pair, more); }
  __device__ __forceinline__ int pair_of(long long tile) const {
    const long long longer = (each + 1) * more;
    return tile < longer ? (int)(tile / (each + 1)) : more + (int)((tile - longer) / each);
  }
};

// Tiles of a row block's page list: the prefix, then for every run of tokens of
// the same request the pages that all of them see whole, once, and for every
// token the pages that are left.  Tokens without own rows (padded rows are of
// request 0) are of no request here: in a run they would leave it nothing to share.
__device__ int tiles_of(const PrefixParams& p, int block, int pre_pages) {
  const int t0 = first_token(p, block), nt = tokens_of(p, block);
  int request[kGroups], len[kGroups];  // all loads first: they are in flight together
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    request[i] = i < nt ? request_of(p, t0 + i) : -1;
    len[i] = i < nt ? p.token_lens[t0 + i] : 0;
  }
  int pages = pre_pages, least = 0, more = 0;  // more: tokens of the run behind its first
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int own = own_rows(p, request[i], len[i]);
    if (own == 0) request[i] = -1;
    if (i > 0 && i < nt && request[i] == request[i - 1]) {
      least = min(least, own);
      ++more;
    } else {
      pages -= more * (least >> 6);
      least = own;
      more = 0;
    }
    pages += (int)(((unsigned)own + 63) >> 6);
  }
  pages -= more * (least >> 6);
  return max((pages + 1) >> 1, 1);  // one at least: an empty row block still writes its rows
}

// ------------------------------------------------------------ attention
// One pair's stretch of a row block's pages.  Span 2 i: the pages that the run of
// tokens beginning with token i shares, span 2 i + 1: the other pages of token i.
struct Segment {
  int block, tile0, count, whole, slot;  // whole: no other pair works on the row block; slot of the partial otherwise
  int pre_pages, pre_rows, pages;
  int end[2 * kGroups], from[2 * kGroups];      // last page + 1 in the list, first page of the request
  int request[2 * kGroups], rows[2 * kGroups];  // rows of the request that the span's tokens see
  uint8_t sees[2 * kGroups];                    // its 16-head groups of the block
};

struct PairSmem {
  uint8_t q[9][kPanel];
  uint8_t k[3][kKChunk];
  uint8_t v[2][kVChunk];
  uint8_t p[2][kPanel];
  float red[2][4][kRows];
  Segment seg[2];
  int valid[4][2];  // rows of the two pages of the last tiles
  uint64_t q_full, q_empty, k_full[3], k_empty[3], v_full[2], v_empty[2], s_full[2], p_full, pv_done;
  uint64_t seg_full[2], seg_empty[2], valid_full[4];
  long long start, u0, u1;  // tiles before this pair's first row block; its stretch
  long long sums[kThreads / 32];
  int most[kThreads / 32], block;
  uint32_t tmem;
};
static_assert(sizeof(PairSmem) <= 232448, "shared memory of a CTA");

// Span of page k >= pre_pages of the segment's list, searched from `span` on.
__device__ __forceinline__ int span_of(const Segment& g, int k, int span) {
  while (span < 2 * kGroups - 1 && k >= g.end[span]) ++span;
  return span;
}
// TMEM lanes (rows 0-31 and 32-63 of each CTA) of the groups that do not see the page.
__device__ __forceinline__ uint32_t lanes_off(uint32_t sees, int word) {
  const uint32_t two = ~sees >> (2 * word);
  return (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
}

// Where this pair begins and ends, by kWidth threads (a warp or the CTA) that take
// a stretch of the row blocks each: every CTA adds up all the tiles by itself,
// which is cheaper than a grid that plans.
template <int kWidth>
__device__ __forceinline__ void make_plan(const PrefixParams& p, PairSmem& S, int pair, int idx) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pre_pages = (int)(((unsigned)prefix_rows(p) + 63) >> 6);
  const int stretch = (p.blocks + kWidth - 1) / kWidth;
  const int b0 = min(idx * stretch, p.blocks), b1 = min(b0 + stretch, p.blocks);
  long long mine = 0;
  int most = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = tiles_of(p, b, pre_pages);
    mine += n;
    most = max(most, n);
  }
  long long before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += a;
  }
  most = __reduce_max_sync(0xffffffffu, most);
  long long tiles = __shfl_sync(0xffffffffu, before, 31);
  before -= mine;
  if (kWidth > 32) {
    if (lane == 0) {
      S.sums[warp] = tiles;
      S.most[warp] = most;
    }
    __syncthreads();
    tiles = 0;
#pragma unroll
    for (int w = 0; w < kWidth / 32; ++w) {
      if (w < warp) before += S.sums[w];
      tiles += S.sums[w];
      most = max(most, S.most[w]);
    }
  }
  // Either every row block has `share` pairs of its own, or the line of all
  // tiles is cut evenly, and then most pairs work on two row blocks: whichever
  // leaves the last pair less.  Pairs of their own also walk the prefix in step,
  // so that a page comes from HBM once for all row blocks; where the prefix does
  // not fit L2 that is worth an eighth (8 tokens of 128 heads behind 131072 rows,
  // at the clock that the power limit leaves: 251 against 294 us).
  const Deal deal(p, tiles);
  long long even = deal.each + (deal.more > 0) + kCutTiles;
  if (pre_pages > kL2Pages) even += even >> 3;
  const int share = p.whole || most <= even * p.share ? p.share : 0;
  const int own_block = share > 0 ? pair / share : -1;
  const long long at = share > 0 ? -1 : pair < deal.pairs ? deal.start(pair) : tiles;
  if (idx == 0 && (own_block >= p.blocks || at == tiles)) S.u0 = S.u1 = S.block = 0;  // nothing for this pair
  if (blockIdx.x == 0 || (b0 <= own_block && own_block < b1) || (before <= at && at < before + mine)) {
    long long c = before;
    for (int b = b0; b < b1; ++b) {
      const int n = stretch == 1 ? (int)mine : tiles_of(p, b, pre_pages);
      if (blockIdx.x == 0) p.cum[b] = c;
      if (b == own_block) {
        const int parts = min(share, n), part = pair - b * share, each = n / parts, more = n - each * parts;
        S.block = b;
        S.start = c;
        S.u0 = c + (part < parts ? each * part + min(part, more) : n);
        S.u1 = c + (part < parts ? each * (part + 1) + min(part + 1, more) : n);
      } else if (c <= at && at < c + n) {
        S.block = b;
        S.start = c;
        S.u0 = at;
        S.u1 = deal.start(pair + 1);
      }
      c += n;
    }
    if (blockIdx.x == 0 && idx == 0) {
      p.cum[p.blocks] = tiles;
      p.cum[p.blocks + 1] = share;
    }
  }
  if (kWidth > 32)
    __syncthreads();
  else
    __syncwarp();
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    dsa_prefix_attention_kernel(const __grid_constant__ CUtensorMap map_qn, const __grid_constant__ CUtensorMap map_qp,
                                const __grid_constant__ CUtensorMap map_ckv3, const __grid_constant__ CUtensorMap map_ckv2,
                                const __grid_constant__ CUtensorMap map_kpe, const __grid_constant__ PrefixParams p) {
  extern __shared__ __align__(1024) uint8_t raw[];
  PairSmem& S = *reinterpret_cast<PairSmem*>(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank(), pair = blockIdx.x >> 1;

  if (threadIdx.x == 32)
    for (const CUtensorMap* m : {&map_qn, &map_qp, &map_ckv3, &map_ckv2, &map_kpe})
      asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
  if (threadIdx.x == 0) {
    mbar_init(&S.q_full, 2);
    mbar_init(&S.q_empty, 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&S.k_full[i], 2);
      mbar_init(&S.k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.v_full[i], 2);
      mbar_init(&S.v_empty[i], 1);
      mbar_init(&S.s_full[i], 1);
      mbar_init(&S.seg_full[i], 1);
      mbar_init(&S.seg_empty[i], 8 + 2 + (rank == 0));
    }
    for (int i = 0; i < 4; ++i) mbar_init(&S.valid_full[i], 1);
    mbar_init(&S.p_full, 2 * kSoftmaxThreads / 32);
    mbar_init(&S.pv_done, 1);
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc_pair(&S.tmem, 512);
  tc_fence_before();
  __syncthreads();
  cluster_arrive();
  // few row blocks: the warp that cuts segments plans alone, while the pair meets
  const bool alone = p.blocks <= kSoloBlocks;
  if (alone && warp == 11) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // what ran before is done
    make_plan<32>(p, S, pair, lane);
  }
  cluster_wait();  // both CTAs' barriers and TMEM are there
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!alone) make_plan<kThreads>(p, S, pair, threadIdx.x);

  if (warp == 11) {
    // ------------------------------------------------------------- segments
    const int pre = prefix_rows(p), pre_pages = (int)(((unsigned)pre + 63) >> 6);
    const long long u1 = S.u1;
    int block = S.block;
    long long u = S.u0, c0 = S.start;
    if (rank == 0 && lane == 0 && u < u1) p.begins[pair] = block;
    for (int n = 0;; ++n) {
      const int s = n & 1;
      if (!mbar_wait_warp(&S.seg_empty[s], ((n >> 1) & 1) ^ 1)) {
        set_error(p.err, kErrTimeout);
        break;
      }
      Segment& g = S.seg[s];
      if (u >= u1) {  // no more: an empty segment ends the other roles
        if (lane == 0) {
          g.count = 0;
          mbar_arrive(&S.seg_full[s]);
        }
        break;
      }
      const int nt = tokens_of(p, block), t0 = first_token(p, block);
      int len = 0, request = -1;
      if (lane < nt) {
        request = request_of(p, t0 + lane);
        len = p.token_lens[t0 + lane];
      }
      if (bad_rows(p, request, len)) set_error(p.err, kErrBadIndex);
      len = own_rows(p, request, len);
      if (len == 0) request = -1;  // as in tiles_of
      // groups of the block that are this token's; those behind the last one
      // are nobody's and their lanes may be written
      const int g0 = (t0 + lane) * p.group_per_token - block * kGroups;
      const uint32_t sees = lane < nt ? (0xffu << max(g0, 0)) & (0xffu >> max(kGroups - g0 - p.group_per_token, 0)) : 0u;
      const int behind = p.groups - block * kGroups;
      const uint32_t nobody = behind < kGroups ? 0xffu << behind & 0xffu : 0u;
      const int left = __shfl_up_sync(0xffffffffu, request, 1);
      const bool first = lane < nt && (lane == 0 || left != request);
      const uint32_t firsts = __ballot_sync(0xffffffffu, first);
      const int run = __popc(firsts & (0xffffffffu >> (31 - lane)));
      int least = len;
      uint32_t run_sees = sees;
      for (int i = 0; i < kGroups && __popc(firsts) < nt; ++i) {  // some run is longer than one token
        const int r = __shfl_sync(0xffffffffu, run, i), l = __shfl_sync(0xffffffffu, len, i);
        const uint32_t m = __shfl_sync(0xffffffffu, sees, i);
        if (i < nt && r == run) {
          least = min(least, l);
          run_sees |= m;
        }
      }
      const int shared = least >> 6, own = (int)(((unsigned)len + 63) >> 6) - shared, both = (first ? shared : 0) + own;
      int end = lane < nt ? both : 0;
#pragma unroll
      for (int o = 1; o < kGroups; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += a;
      }
      end += pre_pages;
      if (lane < kGroups) {
        const int own_pages = lane < nt ? own : 0;
        g.end[2 * lane] = end - own_pages;
        g.end[2 * lane + 1] = end;
        g.from[2 * lane] = 0;
        g.from[2 * lane + 1] = shared;
        g.request[2 * lane] = g.request[2 * lane + 1] = request;
        g.rows[2 * lane] = shared * 64;
        g.rows[2 * lane + 1] = len;
        g.sees[2 * lane] = (uint8_t)(run_sees | nobody);
        g.sees[2 * lane + 1] = (uint8_t)(sees | nobody);
      }
      const int pages = __shfl_sync(0xffffffffu, end, kGroups - 1);
      const long long c1 = c0 + max((pages + 1) >> 1, 1);
      if (lane == 0) {
        g.block = block;
        g.tile0 = (int)(u - c0);
        g.count = (int)(min(u1, c1) - u);
        g.pre_pages = pre_pages;
        g.pre_rows = pre;
        g.pages = pages;
        g.whole = u == c0 && c1 <= u1;
        g.slot = 2 * pair + (n > 0);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.seg_full[s]);
      u = c0 = min(u1, c1);
      ++block;
    }
  } else if (warp == 8 || warp == 10) {
    // ------------------------------------------------- loads: Q and K, or V
    // Lane i looks up page i of the next 16 tiles, a round ahead, so that no
    // tile waits for its page ids.
    const uint32_t q_bar = cluster_map(smem_u32(&S.q_full), 0);
    const uint32_t k_bar = cluster_map(smem_u32(&S.k_full[0]), 0), v_bar = cluster_map(smem_u32(&S.v_full[0]), 0);
    const bool keys = warp == 8;
    bool ok = true;
    int it = 0;
    for (int n = 0; ok; ++n) {
      const Segment& g = S.seg[n & 1];
      if (!mbar_wait_warp(&S.seg_full[n & 1], (n >> 1) & 1)) {
        ok = false;
        break;
      }
      const int count = __shfl_sync(0xffffffffu, g.count, 0);
      if (count <= 0) break;
      auto look_up = [&](int first, int* id, int* rows) {  // page `lane` from tile `first` on
        const int k = 2 * (g.tile0 + first) + lane;
        *id = 0;
        *rows = 0;
        if (first + (lane >> 1) >= count || k >= g.pages) return;
        if (k < g.pre_pages) {
          *id = p.prefix_pages[k];
          *rows = min(64, g.pre_rows - k * 64);
        } else {
          const int i = span_of(g, k, 0), at = k - (i ? g.end[i - 1] : g.pre_pages) + g.from[i];
          *id = p.block_table[g.request[i] * p.bt_stride + at];
          *rows = min(64, g.rows[i] - at * 64);
        }
      };
      int next_id, next_rows, id = 0, rows = 0;
      look_up(0, &next_id, &next_rows);
      // queries: of the first segment by the warp that waits longest for its own
      // loads, later by the one that sees the queries' last use first
      if (keys == (n > 0)) {
        if (!mbar_wait_warp(&S.q_empty, (n & 1) ^ 1)) {
          ok = false;
          break;
        }
        // boxes of whole tokens or of whole quarters of the 64 rows; what lies
        // behind the last token is filled with zeros
        if (elect_one()) {
          mbar_arrive_expect_tx_at(q_bar, 9 * kPanel);
          for (int i = 0; i < p.q_boxes; ++i) {
            const unsigned group = g.block * kGroups + rank * 4 + i * (4 / p.q_boxes);
            const int t = group / (unsigned)p.group_per_token, h = (group - t * p.group_per_token) * 16;
            if (p.q_boxes == 1) {
              tma_load_4d_pair(smem_u32(S.q[0]), &map_qn, 0, h, t, 0, q_bar);
            } else {
              for (int j = 0; j < 8; ++j)
                tma_load_4d_pair(smem_u32(S.q[j]) + i * (kPanel / p.q_boxes), &map_qn, 0, h, t, j, q_bar);
            }
            tma_load_4d_pair(smem_u32(S.q[8]) + i * (kPanel / p.q_boxes), &map_qp, 0, h, t, 0, q_bar);
          }
        }
        __syncwarp();
      }
      for (int i = 0; i < count && ok; ++i, ++it) {
        if ((i & 15) == 0) {
          id = next_id;
          rows = next_rows;
          if (rows > 0 && (id < 0 || id >= p.num_pages)) {
            if (keys) set_error(p.err, kErrBadIndex);
            rows = 0;
          }
          if (rows == 0) id = 0;
          look_up(i + 16, &next_id, &next_rows);
        }
        int page[2], row[2], valid[2];  // row: the coordinate that puts the valid rows at the tile's end
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          page[b] = __shfl_sync(0xffffffffu, id, 2 * (i & 15) + b);
          valid[b] = __shfl_sync(0xffffffffu, rows, 2 * (i & 15) + b);
          row[b] = valid[b] ? valid[b] - 64 : 64;  // 64: nothing of the page, all zeros
        }
        const uint32_t parity = (it & 1) ^ 1;
        if (keys) {
          const int my_page = rank ? page[1] : page[0], my_row = rank ? row[1] : row[0];
#pragma unroll
          for (int c = 0; c < 3; ++c) {
            if (!mbar_wait_warp(&S.k_empty[c], parity)) {
              ok = false;
              break;
            }
            if (elect_one()) {
              if (c == 0) {
                S.valid[it & 3][0] = valid[0];
                S.valid[it & 3][1] = valid[1];
                mbar_arrive(&S.valid_full[it & 3]);
              }
              mbar_arrive_expect_tx_at(k_bar + 8 * c, kKChunk);
              tma_load_4d_pair(smem_u32(S.k[c]), c < 2 ? &map_ckv3 : &map_ckv2, 0, my_row, 3 * c, my_page, k_bar + 8 * c);
              if (c == 2) tma_load_4d_pair(smem_u32(S.k[2]) + 2 * kPanel, &map_kpe, 0, my_row, 0, my_page, k_bar + 16);
            }
            __syncwarp();
          }
        } else {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (!mbar_wait_warp(&S.v_empty[c], parity)) {
              ok = false;
              break;
            }
            if (elect_one()) {
              mbar_arrive_expect_tx_at(v_bar + 8 * c, kVChunk);
#pragma unroll
              for (int b = 0; b < 2; ++b)  // this CTA's 128 of 256 columns, as two panels a page
                tma_load_4d_pair(smem_u32(S.v[c]) + b * 2 * kPanel, &map_ckv2, 0, row[b], c * 4 + rank * 2, page[b],
                                 v_bar + 8 * c);
            }
            __syncwarp();
          }
        }
      }
      if (lane == 0) mbar_arrive(&S.seg_empty[n & 1]);
    }
    if (!ok) set_error(p.err, kErrTimeout);
  } else if (warp == 9) {
    // ----------------------------------------------------------- MMA issue
    // The warp stays together and one elected lane issues: the operands are
    // then the same for all lanes and need no detour through lane registers.
    if (rank == 0) {
      constexpr uint32_t id_qk = umma_idesc(1, 1, 0, 0, 128, 128);
      constexpr uint32_t id_pv = umma_idesc(1, 1, 0, 1, 128, 256);
      const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t q_desc = umma_desc(smem_u32(S.q[0]), 16, 1024, kSwizzle128B);
      const uint64_t k_desc = umma_desc(smem_u32(S.k[0]), 16, 1024, kSwizzle128B);
      const uint64_t p_desc = umma_desc(smem_u32(S.p[0]), 16, 1024, kSwizzle128B);
      const uint64_t v_desc = umma_desc(smem_u32(S.v[0]), kPanel, 1024, kSwizzle128B);
      bool ok = true;
      int it = 0;          // tiles whose scores are issued
      uint32_t off[2][4];  // lanes left alone by the two pages of the tile before
      bool masked = false;
      auto weigh = [&](int i) -> bool {  // O += P V of tile i
        if (!mbar_wait_cluster_warp(&S.p_full, i & 1)) return false;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (!mbar_wait_cluster_warp(&S.v_full[c], i & 1)) return false;
          tc_fence_after();
          if (elect_one()) {
            if (masked) {
#pragma unroll
              for (int ks = 0; ks < 8; ++ks)
                umma_f16_pair_masked(base + c * 128, p_desc + (((ks >> 2) * kPanel + (ks & 3) * 32) >> 4),
                                     v_desc + ((c * kVChunk + (ks >> 2) * 2 * kPanel + (ks & 3) * 2048) >> 4), id_pv,
                                     off[ks >> 2]);
            } else {
#pragma unroll
              for (int ks = 0; ks < 8; ++ks)
                umma_f16_pair(base + c * 128, p_desc + (((ks >> 2) * kPanel + (ks & 3) * 32) >> 4),
                              v_desc + ((c * kVChunk + (ks >> 2) * 2 * kPanel + (ks & 3) * 2048) >> 4), id_pv, 1u);
            }
            umma_commit_pair(&S.v_empty[c]);
            if (c == 1) umma_commit_pair(&S.pv_done);
          }
          __syncwarp();
        }
        return true;
      };
      for (int n = 0; ok; ++n) {
        const Segment& g = S.seg[n & 1];
        if (!mbar_wait_warp(&S.seg_full[n & 1], (n >> 1) & 1)) {
          ok = false;
          break;
        }
        // a segment's last P.V does not wait for the next one's queries
        if (it > 0 && !weigh(it - 1)) {
          ok = false;
          break;
        }
        const int count = __shfl_sync(0xffffffffu, g.count, 0);
        if (count <= 0) break;
        int span = 0;
        if (!mbar_wait_cluster_warp(&S.q_full, n & 1)) {
          ok = false;
          break;
        }
        for (int i = 0; i < count && ok; ++i, ++it) {
          const uint32_t scores = base + kTmemS + 64 * (it & 1);
#pragma unroll
          for (int c = 0; c < 3; ++c) {
            if (!mbar_wait_cluster_warp(&S.k_full[c], it & 1)) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < 12; ++j)
                umma_f16_pair(scores, q_desc + (((3 * c + (j >> 2)) * kPanel + (j & 3) * 32) >> 4),
                              k_desc + ((c * kKChunk + (j >> 2) * kPanel + (j & 3) * 32) >> 4), id_qk,
                              (c > 0 || j > 0) ? 1u : 0u);
              umma_commit_pair(&S.k_empty[c]);
              if (c == 2) {
                umma_commit_pair(&S.s_full[it & 1]);
                if (i + 1 == count) umma_commit_pair(&S.q_empty);
              }
            }
            __syncwarp();
          }
          if (!ok) break;
          if (i > 0 && !weigh(it - 1)) {
            ok = false;
            break;
          }
          uint32_t any = 0;
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int k = 2 * (g.tile0 + i) + b;
            uint32_t sees = 0xff;
            if (k >= g.pre_pages && k < g.pages) {
              span = span_of(g, k, span);
              sees = g.sees[span];
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              off[b][w] = __shfl_sync(0xffffffffu, lanes_off(sees, w), 0);
              any |= off[b][w];
            }
          }
          masked = any != 0;
        }
        if (lane == 0) mbar_arrive(&S.seg_empty[n & 1]);
      }
      if (!ok) set_error(p.err, kErrTimeout);
    }
  } else {
    // --------------------------------------------------- softmax, epilogue
    // Lane quarter q of TMEM: rows 32 (q & 1) + lane against page q >> 1; the
    // two warps of a quarter take 32 columns (and 128 columns of O) each.
    const int quarter = warp & 3, half = warp >> 2, page = quarter >> 1;
    const int row = (quarter & 1) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t p_bar = cluster_map(smem_u32(&S.p_full), 0);
    // a wait that gave up in one warp takes all eight out at their next barrier, and
    // nowhere else: a warp that left alone would keep the others waiting there
    bool ok = true, left = false;
    int it = 0;
    for (int n = 0;; ++n) {
      const Segment& g = S.seg[n & 1];
      ok = mbar_wait_warp(&S.seg_full[n & 1], (n >> 1) & 1);
      if (!named_bar_all(1, kSoftmaxThreads, ok)) break;
      const int count = g.count;
      if (count <= 0) break;
      const int group = g.block * kGroups + rank * 4 + (row >> 4);
      const bool live = group < p.groups;
      const int token = live ? (unsigned)group / (unsigned)p.group_per_token : 0;
      const int my_bit = rank * 4 + (row >> 4);
      float m = -INFINITY;
      float2 sums = make_float2(0.f, 0.f);
      int span = 0;
      for (int i = 0; i < count; ++i, ++it) {
        const int k = 2 * (g.tile0 + i) + page;
        // ok is the same in all lanes of a warp: the votes of the waits are taken by all or none
        ok = ok && mbar_wait_warp(&S.valid_full[it & 3], (it >> 2) & 1) && mbar_wait_cluster_warp(&S.s_full[it & 1], (it >> 1) & 1);
        tc_fence_after();
        bool sees = true;  // rows behind the last token see all: their queries are zeros and nobody reads them
        if (k >= g.pre_pages && k < g.pages) {
          span = span_of(g, k, span);
          sees = (g.sees[span] >> my_bit) & 1;
        }
        // the page's rows are at the end of its 64 columns
        const int from = sees ? 64 - S.valid[it & 3][page] - 32 * half : 32;
        float2 x[16];
        tmem_ld32(lanes + kTmemS + 64 * (it & 1) + 32 * half, reinterpret_cast<float*>(x));
        if (p.negate) {
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] = make_float2(-x[j].x, -x[j].y);
        }
        if (!__all_sync(0xffffffffu, from <= 0)) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (2 * j < from) x[j].x = -INFINITY;
            if (2 * j + 1 < from) x[j].y = -INFINITY;
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, fmaxf(x[j].x, x[j].y));
        S.red[it & 1][page * 2 + half][row] = top;
        if ((left = !named_bar_all(1, kSoftmaxThreads, ok))) break;
        top = p.scale_log2 * fmaxf(fmaxf(S.red[it & 1][0][row], S.red[it & 1][1][row]),
                                   fmaxf(S.red[it & 1][2][row], S.red[it & 1][3][row]));
        // the maximum moves on a rise of more than 2^kLazy only (weights up to
        // 2^8 lose nothing in 32 bits), so O is rescaled on few tiles
        float alpha = 1.f;
        if (top > m + kLazy || m == -INFINITY) {
          alpha = m == -INFINITY ? 1.f : ex2_approx(m - top);
          m = top;
          sums = make_float2(sums.x * alpha, sums.y * alpha);
        }
        const float sub = m == -INFINITY ? 0.f : -m;
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          // Weights are rounded to bf16 for the matrix product, whose two operands are of
          // one type (in two parts they would cost 47% more MMA); the sum takes them as
          // they are.  Each is off by at most 2^-8 of itself, independently of the others:
          // a bf16 output's error against 64 bits grows from 1.7e-3 of its norm, the
          // output's own rounding, to 1.7e-3 (32768 rows) - 2.1e-3 (1000 rows).
          float2 e = fma2(x[j], make_float2(p.scale_log2, p.scale_log2), make_float2(sub, sub));
          e = make_float2(ex2_approx(e.x), ex2_approx(e.y));
          sums = add2(sums, e);
          w[j] = pack_bf16(e.x, e.y);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) asm volatile("" : "+r"(w[j]));  // done before the wait, not behind it
        if (it > 0) ok = mbar_wait_cluster_warp(&S.pv_done, (it - 1) & 1);  // P is read, O settled
        __syncwarp();  // of one mind for the accesses to TMEM, whichever way the lanes came
        tc_fence_after();
        if (i == 0) {
          float z[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) z[j] = 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_st32(lanes + half * 128 + c * 32, z);
          tmem_wait_st();
        } else if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float o[32];
            tmem_ld32(lanes + half * 128 + c * 32, o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] *= alpha;
            tmem_st32(lanes + half * 128 + c * 32, o);
          }
          tmem_wait_st();
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<uint4*>(S.p[page] + row * 128 + (((half * 4 + c) ^ (row & 7)) << 4)) =
              make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(p_bar);
      }
      if (left) {
        ok = false;
        break;
      }
      // the four threads of a row add up their sums; O is complete
      float l = sums.x + sums.y;
      S.red[it & 1][page * 2 + half][row] = l;
      ok = ok && mbar_wait_cluster_warp(&S.pv_done, (it - 1) & 1);
      if (!(ok = named_bar_all(1, kSoftmaxThreads, ok))) break;
      tc_fence_after();
      l = S.red[it & 1][0][row] + S.red[it & 1][1][row] + S.red[it & 1][2][row] + S.red[it & 1][3][row];
      __syncwarp();
      named_bar_sync(1, kSoftmaxThreads);  // red is written again by the next tile
      const int head = live ? (group - token * p.group_per_token) * 16 + (row & 15) : 0;
      const int dv = half * 256 + page * 128;  // the 128 columns of O in these lanes
      if (g.whole) {
        // A lane holds a row, and 32 rows of 16 bytes are 32 lines a store: the warp
        // turns 32 x 32 values over in its part of the idle weight buffer, so that
        // four lanes store 64 bytes of a row (4 stores of 8 lines instead of 32).
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint8_t* stage = S.p[0] + warp * 2048;
        const int chunk = lane & 3;
        __nv_bfloat16* dst[2];  // of the two 16-head groups of the warp's rows
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int its = g.block * kGroups + rank * 4 + (quarter & 1) * 2 + i;
          const int t = (unsigned)its / (unsigned)p.group_per_token, h = (its - t * p.group_per_token) * 16;
          dst[i] = its < p.groups ? p.out + t * p.out_st + (h + (lane >> 2)) * p.out_sh + dv + chunk * 8 : nullptr;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float o[32];
          __syncwarp();
          tmem_ld32(lanes + half * 128 + c * 32, o);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((j ^ (lane >> 1 & 3)) << 4)) =
                make_uint4(pack_bf16(o[8 * j] * inv, o[8 * j + 1] * inv), pack_bf16(o[8 * j + 2] * inv, o[8 * j + 3] * inv),
                           pack_bf16(o[8 * j + 4] * inv, o[8 * j + 5] * inv), pack_bf16(o[8 * j + 6] * inv, o[8 * j + 7] * inv));
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // rows 8 k + lane / 4
            const int r = 8 * k + (lane >> 2);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 64 + ((chunk ^ (r >> 1 & 3)) << 4));
            if (dst[k >> 1]) *reinterpret_cast<uint4*>(dst[k >> 1] + (k & 1) * 8 * p.out_sh + c * 32) = v;
          }
        }
        if (live && half == 0 && page == 0)
          p.lse[token * p.lse_st + head * p.lse_sh] = l == 0.f ? -INFINITY : m + log2f(l);
      } else {
        // partials lie as [512 / 4][128 rows][4]: the lanes of a warp store side by side
        float* part = p.parts + (int64_t)g.slot * kSlotFloats;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float o[32];
          __syncwarp();
          tmem_ld32(lanes + half * 128 + c * 32, o);
          if (!live) continue;
          float4* dst = reinterpret_cast<float4*>(part) + (dv + c * 32) / 4 * (2 * kRows) + rank * kRows + row;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            __stcg(dst + j * (2 * kRows), make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]));
        }
        if (live && half == 0 && page == 0) {
          __stcg(part + 2 * kRows * 512 + rank * kRows + row, m);
          __stcg(part + 2 * kRows * 512 + 2 * kRows + rank * kRows + row, l);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.seg_empty[n & 1]);
    }
    if (!ok) set_error(p.err, kErrTimeout);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the pair's MMAs or arrivals may reach it
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
  // here and not at the start: 13.4 against 14.6 us for the smallest call, no
  // difference beyond 1% for the others
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ----------------------------------------------------------------- merge
// Rows whose block several pairs share: with partials (O_k, m_k, l_k),
//   o = sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k.
// A CTA takes 8 rows of a row block and kMergeColumns / kStreams x kQuads of its
// 128 column quads: thread i the row i % 8, so that 8 rows of a quad are read as
// one line, and one partial of kStreams.  The grid has a slice for every row block
// or, where those are more, for every boundary between pairs: then the row block
// whose first cut the boundary is.
constexpr int kMergeRows = 8, kMergeColumns = 32;

template <int kQuads, int kAhead, int kStreams>  // kAhead: partials whose loads are in flight together
__global__ void __launch_bounds__(kMergeRows * kMergeColumns)
    dsa_prefix_merge_kernel(const PrefixParams p, const int by_cut) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long tiles = p.cum[p.blocks];
  const int cut = blockIdx.y + 1;
  int lo = blockIdx.y;
  if (by_cut) lo = p.begins[cut];  // tiles >= blocks >= pairs here: every pair works
  const long long c0 = p.cum[lo], c1 = p.cum[lo + 1];
  const int share = (int)p.cum[p.blocks + 1];
  int first, last;
  bool began_before = false;
  if (share > 0) {
    first = lo * share;
    last = first + (int)min((long long)share, c1 - c0) - 1;
  } else {
    const Deal deal(p, tiles);
    // a cut on the block's edge is none, and a block is joined once, at its first
    if (by_cut && (deal.start(cut) == c0 || deal.start(cut - 1) > c0)) return;
    first = deal.pair_of(c0);
    last = deal.pair_of(c1 - 1);
    began_before = deal.start(first) < c0;
  }
  if (first == last) return;  // one pair had it all and wrote the results
  constexpr int kWide = kMergeColumns / kStreams, kParts = 128 / (kWide * kQuads);
  const int column = threadIdx.x / kMergeRows, stream = column / kWide;
  const int row = blockIdx.x / kParts * kMergeRows + threadIdx.x % kMergeRows;
  const int quad = blockIdx.x % kParts * (kWide * kQuads) + column % kWide;
  const int group = lo * kGroups + (row >> 4);
  if (group >= p.groups) return;
  float m = -INFINITY, l = 0.f;
  float4 o[kQuads];
#pragma unroll
  for (int j = 0; j < kQuads; ++j) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = first + stream; k0 <= last; k0 += kAhead * kStreams) {
    float mk[kAhead], lk[kAhead];
    float4 v[kAhead][kQuads];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      mk[i] = -INFINITY;
      lk[i] = 0.f;
#pragma unroll
      for (int j = 0; j < kQuads; ++j) v[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
      const int k = k0 + i * kStreams;
      if (k <= last) {
        // a pair that began before the block has it as its last, any other as its first
        const int slot = 2 * k + (k == first && began_before);
        const float* part = p.parts + (int64_t)slot * kSlotFloats;
        mk[i] = __ldcg(part + 2 * kRows * 512 + row);
        lk[i] = __ldcg(part + 2 * kRows * 512 + 2 * kRows + row);
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
          v[i][j] = __ldcg(reinterpret_cast<const float4*>(part) + (quad + kWide * j) * (2 * kRows) + row);
      }
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) top = fmaxf(top, mk[i]);
    const float a = m == -INFINITY ? 0.f : exp2f(m - top);
    m = top;
    l *= a;
#pragma unroll
    for (int j = 0; j < kQuads; ++j) o[j] = make_float4(o[j].x * a, o[j].y * a, o[j].z * a, o[j].w * a);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float b = mk[i] == -INFINITY ? 0.f : exp2f(mk[i] - top);
      l += lk[i] * b;
#pragma unroll
      for (int j = 0; j < kQuads; ++j) {
        o[j].x += v[i][j].x * b;
        o[j].y += v[i][j].y * b;
        o[j].z += v[i][j].z * b;
        o[j].w += v[i][j].w * b;
      }
    }
  }
  if (kStreams > 1) {  // rows of a CTA are of one group: all its threads are here
    __shared__ float4 all_o[kStreams > 1 ? kMergeRows * kMergeColumns : 1];
    __shared__ float2 all_ml[kStreams > 1 ? kMergeRows * kMergeColumns : 1];
    all_o[threadIdx.x] = o[0];
    all_ml[threadIdx.x] = make_float2(m, l);
    __syncthreads();
    if (stream > 0) return;
    for (int s = 1; s < kStreams; ++s) {
      const int at = threadIdx.x + s * kWide * kMergeRows;
      const float2 ml = all_ml[at];
      const float top = fmaxf(m, ml.x);
      const float a = m == -INFINITY ? 0.f : exp2f(m - top), b = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
      m = top;
      l = l * a + ml.y * b;
      o[0] = make_float4(o[0].x * a + all_o[at].x * b, o[0].y * a + all_o[at].y * b, o[0].z * a + all_o[at].z * b,
                         o[0].w * a + all_o[at].w * b);
    }
  }
  const int token = (unsigned)group / (unsigned)p.group_per_token;
  const int head = (group - token * p.group_per_token) * 16 + (row & 15);
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < kQuads; ++j)
    *reinterpret_cast<uint2*>(p.out + token * p.out_st + head * p.out_sh + (quad + kWide * j) * 4) =
        make_uint2(pack_bf16(o[j].x * inv, o[j].y * inv), pack_bf16(o[j].z * inv, o[j].w * inv));
  if (quad == 0) p.lse[token * p.lse_st + head * p.lse_sh] = l == 0.f ? -INFINITY : m + log2f(l);
}

// ------------------------------------------------------------------ host
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(f);
  });
  return fn;
}

// bf16 rows of 64 values: dimensions 1 to 3 with their strides in elements, and
// the box of them that one load takes.
bool encode(CUtensorMap* map, const void* base, int64_t n1, int64_t s1, int b1, int64_t n2, int64_t s2, int b2, int64_t n3,
            int64_t s3, int b3) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[4] = {64, (cuuint64_t)n1, (cuuint64_t)n2, (cuuint64_t)n3};
  const cuuint64_t strides[3] = {(cuuint64_t)s1 * 2, (cuuint64_t)s2 * 2, (cuuint64_t)s3 * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)b1, (cuuint32_t)b2, (cuuint32_t)b3}, step[4] = {1, 1, 1, 1};
  auto attempt = [&] {
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  return attempt() || (bind_context() && attempt());
}

// Pairs of CTAs that fit on the current device at once (cached), 0 on an error.
int resident_pairs() {
  static std::mutex mu;
  static int cached[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> lock(mu);
  if (cached[dev] == 0) {
    int sms = 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (cudaFuncSetAttribute(dsa_prefix_attention_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)sizeof(PairSmem)) != cudaSuccess)
      return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sms / 2 * 2));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(PairSmem);
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, dsa_prefix_attention_kernel, &cfg) != cudaSuccess || n < 1) return 0;
    cached[dev] = n < sms / 2 ? n : sms / 2;
  }
  return cached[dev];
}

struct Layout {
  int64_t blocks, cum, begins, parts;
  size_t bytes;
};
Layout workspace_layout(int64_t tokens, int64_t heads, int pairs) {
  Layout w;
  w.blocks = (tokens * (heads / 16) + kGroups - 1) / kGroups;
  w.cum = 256;
  w.begins = w.cum + (w.blocks + 2) * 8;
  w.parts = (w.begins + pairs * 4 + 255) / 256 * 256;
  w.bytes = (size_t)(w.parts + 2 * pairs * (int64_t)kSlotFloats * 4);
  return w;
}

// Launch with programmatic dependence on the grid before it.
template <typename... Params, typename... Args>
cudaError_t launch_after(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream,
                         Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_shared_prefix_attention_workspace_size(int64_t num_tokens, int64_t num_heads, size_t* bytes) {
  if (!bytes) return report_error(DSA_ERR_INVALID_ARG, "NULL pointer argument");
  if (num_tokens < 0) return report_error(DSA_ERR_INVALID_ARG, "negative size");
  if (num_heads <= 0 || num_heads % 16) return report_error(DSA_ERR_INVALID_ARG, "heads must be a positive multiple of 16");
  if (num_tokens * (num_heads / 16) > (1 << 30))
    return report_error(DSA_ERR_UNSUPPORTED, "too many tokens");
  const int pairs = resident_pairs();
  if (pairs < 1) return report_error(DSA_ERR_CUDA, "cannot query how many CTA pairs fit on the device");
  *bytes = workspace_layout(num_tokens, num_heads, pairs).bytes;
  return DSA_OK;
}

extern "C" int dsa_shared_prefix_attention_scratch(
    const void* q_nope, int64_t q_nope_stride_token, int64_t q_nope_stride_head, const void* q_pe,
    int64_t q_pe_stride_token, int64_t q_pe_stride_head, const void* ckv_cache, int64_t ckv_stride_page,
    int64_t ckv_stride_row, const void* kpe_cache, int64_t kpe_stride_page, int64_t kpe_stride_row,
    const int32_t* prefix_pages, int64_t max_prefix_len, const int32_t* prefix_len, const int32_t* block_table,
    int64_t block_table_stride, int64_t batch, int64_t max_pages, const int32_t* token_request,
    const int32_t* token_lens, int64_t num_tokens, int64_t num_heads, int64_t num_pages, float sm_scale,
    void* output, int64_t out_stride_token, int64_t out_stride_head, float* lse, int64_t lse_stride_token,
    int64_t lse_stride_head, void* workspace, size_t workspace_bytes, int* device_error, void* stream) {
  if (num_tokens < 0 || max_prefix_len < 0 || batch < 0 || max_pages < 0 || num_pages < 0)
    return report_error(DSA_ERR_INVALID_ARG, "negative size");
  if (num_heads <= 0 || num_heads % 16)
    return report_error(DSA_ERR_INVALID_ARG, "heads must be a positive multiple of 16");
  if (num_heads > 65536) return report_error(DSA_ERR_UNSUPPORTED, "at most 65536 heads");
  if (num_tokens == 0) return DSA_OK;
  if (num_tokens * (num_heads / 16) > (1 << 30) || max_prefix_len > INT32_MAX || num_pages > INT32_MAX)
    return report_error(DSA_ERR_UNSUPPORTED, "tokens, rows and pages are counted in 32 bits");
  if (!q_nope || !q_pe || !ckv_cache || !kpe_cache || !token_lens || !output || !lse || !workspace ||
      (max_prefix_len > 0 && !prefix_pages) || (batch > 0 && max_pages > 0 && !block_table))
    return report_error(DSA_ERR_INVALID_ARG, "NULL pointer argument");
  if (num_pages == 0) return report_error(DSA_ERR_UNSUPPORTED, "the cache has no pages");
  if (!token_request && batch < num_tokens)
    return report_error(DSA_ERR_INVALID_ARG, "without token_request the block table needs a row for every token");
  for (const void* q : {q_nope, q_pe, ckv_cache, kpe_cache, (const void*)output})
    if (reinterpret_cast<uintptr_t>(q) & 15)
      return report_error(DSA_ERR_INVALID_ARG, "queries, caches and output must be 16-byte aligned");
  if (out_stride_token % 8 || out_stride_head % 8)
    return report_error(DSA_ERR_INVALID_ARG, "output strides must be multiples of 8 elements");
  // a stride over a single token or page is never used: any value will do
  if (num_tokens == 1) {
    q_nope_stride_token = num_heads * q_nope_stride_head;
    q_pe_stride_token = num_heads * q_pe_stride_head;
  }
  if (num_pages == 1) {
    ckv_stride_page = 64 * ckv_stride_row;
    kpe_stride_page = 64 * kpe_stride_row;
  }
  const int64_t inner[4] = {q_nope_stride_head, q_pe_stride_head, ckv_stride_row, kpe_stride_row};
  const int64_t outer[4] = {q_nope_stride_token, q_pe_stride_token, ckv_stride_page, kpe_stride_page};
  for (int i = 0; i < 4; ++i) {
    const int64_t width = i & 1 ? 64 : 512;
    if (inner[i] < width || inner[i] % 8 || outer[i] < inner[i] || outer[i] % 8 || outer[i] >= (1LL << 39))
      return report_error(DSA_ERR_INVALID_ARG,
                          "heads and cache rows must be 16-byte aligned and must not overlap");
  }
  const int fit = resident_pairs();
  if (fit < 1) return report_error(DSA_ERR_CUDA, "cannot query how many CTA pairs fit on the device");
  const Layout w = workspace_layout(num_tokens, num_heads, fit);
  if (workspace_bytes < w.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return report_error(DSA_ERR_WORKSPACE, "workspace too small or not 256-byte aligned");
  // What the host knows of the work: the longest list a row block can have.  No
  // more pairs than tiles are launched, and up to kWholeTiles tiles are left to
  // one pair a row block: one launch less for the host (20 against 22 us a call),
  // and on the GPU as soon done as a split and its merge grid.  Two tiles 11.5 us
  // either way for a token, 12.7 against 14.6 for 16 row blocks; three 12.9 against
  // 11.5 and 14.3 against 15.8; four 11.5 for the split against 14.2 whole.
  const int64_t per = num_heads / 16;  // 16-head groups of a token
  const int64_t block_tokens = kGroups % per == 0 ? kGroups / per : per % kGroups == 0 ? 1 : (kGroups + per - 1) / per + 1;
  const int64_t block_pages = (max_prefix_len + 63) / 64 + (block_tokens < num_tokens ? block_tokens : num_tokens) * max_pages;
  const int64_t block_tiles = block_pages < 2 ? 1 : (block_pages + 1) / 2;
  const int pairs = (int)(w.blocks >= fit || block_tiles >= fit || w.blocks * block_tiles >= fit ? fit : w.blocks * block_tiles);
  const bool whole = w.blocks <= pairs && block_tiles <= kWholeTiles;
  // a query box holds whole tokens (of at most 64 heads), 64 heads of one, or 32 or 16
  const int gpt = (int)per;
  const int box_groups = gpt % 4 == 0 ? 4 : gpt % 2 == 0 ? 2 : 1, box_tokens = box_groups == gpt ? 4 / gpt : 1;
  const int q_boxes = 4 / (box_groups * box_tokens);
  CUtensorMap map_qn, map_qp, map_ckv3, map_ckv2, map_kpe;
  if (!encode(&map_qn, q_nope, num_heads, q_nope_stride_head, 16 * box_groups, num_tokens, q_nope_stride_token, box_tokens, 8,
              64, q_boxes == 1 ? 8 : 1) ||
      !encode(&map_qp, q_pe, num_heads, q_pe_stride_head, 16 * box_groups, num_tokens, q_pe_stride_token, box_tokens, 1, 64, 1) ||
      !encode(&map_ckv3, ckv_cache, 64, ckv_stride_row, 64, 8, 64, 3, num_pages, ckv_stride_page, 1) ||
      !encode(&map_ckv2, ckv_cache, 64, ckv_stride_row, 64, 8, 64, 2, num_pages, ckv_stride_page, 1) ||
      !encode(&map_kpe, kpe_cache, 64, kpe_stride_row, 64, 1, 64, 1, num_pages, kpe_stride_page, 1))
    return report_error(DSA_ERR_CUDA, "cannot encode a tensor map");
  PrefixParams p;
  p.prefix_pages = prefix_pages;
  p.prefix_len = prefix_len;
  p.block_table = block_table;
  p.token_request = token_request;
  p.token_lens = token_lens;
  p.max_prefix = (int)max_prefix_len;
  p.bt_stride = block_table_stride;
  p.batch = (int)(batch < INT32_MAX ? batch : INT32_MAX);
  p.max_own = (int)(max_pages < INT32_MAX / 64 ? max_pages * 64 : INT32_MAX);
  p.num_pages = (int)num_pages;
  p.group_per_token = gpt;
  p.groups = (int)(num_tokens * gpt);
  p.blocks = (int)w.blocks;
  p.max_pairs = pairs;
  p.share = whole ? 1 : pairs / p.blocks;
  p.whole = whole;
  p.q_boxes = q_boxes;
  // scores are scaled after the maximum is taken: a scale below zero turns them
  // over first, and zero becomes a scale that makes every score nothing
  const float scale = sm_scale * 1.44269504088896340736f;
  p.negate = scale < 0.f;
  p.scale_log2 = scale == 0.f ? 1e-30f : p.negate ? -scale : scale;
  p.out = static_cast<__nv_bfloat16*>(output);
  p.out_st = out_stride_token;
  p.out_sh = out_stride_head;
  p.lse = lse;
  p.lse_st = lse_stride_token;
  p.lse_sh = lse_stride_head;
  p.err = device_error;
  p.cum = reinterpret_cast<long long*>(static_cast<char*>(workspace) + w.cum);
  p.begins = reinterpret_cast<int*>(static_cast<char*>(workspace) + w.begins);
  p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.parts);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_after(dsa_prefix_attention_kernel, dim3(2 * (whole ? p.blocks : pairs)), kThreads, sizeof(PairSmem), s, map_qn, map_qp,
                               map_ckv3, map_ckv2, map_kpe, p);
  if (e == cudaSuccess && pairs > 1 && !whole) {
    const int rows = (p.groups < kGroups ? p.groups : kGroups) * 16, by_cut = p.blocks >= pairs;
    const unsigned x = rows / kMergeRows, y = (unsigned)(by_cut ? pairs - 1 : p.blocks), threads = kMergeRows * kMergeColumns;
    // few row blocks have many partials each: more of them in flight, and over 24
    // dealt out to 8 threads.  With one, two, three, four row blocks of 128 rows
    // behind 20000 rows (74 to 18 partials) 8 threads take 19.7, 23.7, 29.0, 33.1 us
    // a call, one thread 25.6, 24.2, 26.9, 29.3.  One thread with 10 partials in
    // flight against four column quads a thread with 2: 16 row blocks of 4 partials
    // 74.4 against 71.8 us, 5 of 14 34.9 against 39.1.
    if (pairs / p.blocks > 24)
      e = launch_after(dsa_prefix_merge_kernel<1, 5, 8>, dim3(32 * x, y), threads, 0, s, p, by_cut);
    else if (x * y <= 148)
      e = launch_after(dsa_prefix_merge_kernel<1, 10, 1>, dim3(4 * x, y), threads, 0, s, p, by_cut);
    else
      e = launch_after(dsa_prefix_merge_kernel<4, 2, 1>, dim3(x, y), threads, 0, s, p, by_cut);
  }
  if (e != cudaSuccess) return report_error(DSA_ERR_CUDA, cudaGetErrorString(e));
  return DSA_OK;
}

extern "C" int dsa_shared_prefix_attention(
    const void* q_nope, int64_t q_nope_stride_token, int64_t q_nope_stride_head, const void* q_pe,
    int64_t q_pe_stride_token, int64_t q_pe_stride_head, const void* ckv_cache, int64_t ckv_stride_page,
    int64_t ckv_stride_row, const void* kpe_cache, int64_t kpe_stride_page, int64_t kpe_stride_row,
    const int32_t* prefix_pages, int64_t max_prefix_len, const int32_t* prefix_len, const int32_t* block_table,
    int64_t block_table_stride, int64_t batch, int64_t max_pages, const int32_t* token_request,
    const int32_t* token_lens, int64_t num_tokens, int64_t num_heads, int64_t num_pages, float sm_scale,
    void* output, int64_t out_stride_token, int64_t out_stride_head, float* lse, int64_t lse_stride_token,
    int64_t lse_stride_head, void* workspace, size_t workspace_bytes, void* stream) {
  return dsa_shared_prefix_attention_scratch(
      q_nope, q_nope_stride_token, q_nope_stride_head, q_pe, q_pe_stride_token, q_pe_stride_head, ckv_cache,
      ckv_stride_page, ckv_stride_row, kpe_cache, kpe_stride_page, kpe_stride_row, prefix_pages, max_prefix_len,
      prefix_len, block_table, block_table_stride, batch, max_pages, token_request, token_lens, num_tokens, num_heads,
      num_pages, sm_scale, output, out_stride_token, out_stride_head, lse, lse_stride_token, lse_stride_head, workspace,
      workspace_bytes, static_cast<int*>(workspace), stream);
}
