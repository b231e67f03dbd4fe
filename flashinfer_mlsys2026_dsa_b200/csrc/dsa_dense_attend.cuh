// Dense attention over the latent cache on pairs of CTAs.
//
// Work.  A unit is up to 128 query rows (row = token x heads + head of T = 128 / heads
// consecutive tokens) against the positions that they see, in tiles of 192 keys.  A pair of CTAs
// takes a unit's tiles: 64 rows in each CTA, every tensor-core instruction spanning both
// (cta_group::2, M = 128):
//   S[128 x 192] = Q K^T         36 instructions, N = 192; each CTA holds 96 of the keys
//   O[128 x 512] += P V     2 x 12 instructions, N = 256; each CTA holds 256 of the value columns
// O (fp32) fills half of each CTA's tensor memory, which no smaller group could: one CTA with
// 128 rows would need all of it, and 64 rows in one CTA run the tensor cores at half rate.  In
// this form S needs no exchange between the CTAs, Q and P stay with their rows, and a key passes
// each CTA's shared memory 1.9 times (as K: its own half of the keys; as V: its half of the
// columns), 63 bytes a cycle at the tensor cores' full rate, which L2 delivers.
// Measured instruction costs (cycles): N = 64 .. 128 45, N = 192 48, N = 256 64; so 192 keys a
// tile is the smallest at full rate, 17 cycles a key.
//
// The units of all rows form one line of tiles, cut into equal parts, one for each pair.  A unit
// that is cut leaves partial results (O, maximum, sum) that combine kernels join.
//
// Warps of a CTA:  0 loads keys and values, 1 issues the tensor-core work (rank 0 alone), 2 loads
// queries, 3 walks the units, 4-11 softmax and output: a thread is a row and a quarter of a
// tile's keys (its lane quadrant holds half of them, two warps share a quadrant).
#pragma once

namespace dsa {
namespace dense {

constexpr int kChunk = 32;                 // positions that are looked up and masked together
constexpr int kTileChunks = 6;
constexpr int kTile = kChunk * kTileChunks;
constexpr int kSlots = 5;                  // ring of 24 KB: [96 keys x 128 columns]
constexpr int kBlkB = 96 * 128;            // [96 keys x 64 columns], 128-byte swizzle
constexpr int kSlotB = 2 * kBlkB;
constexpr int kQBlk = 64 * 128;            // [64 rows x 64 columns]
constexpr int kThreads = 384;
constexpr int kLoadWarp = 0, kMmaWarp = 1, kQWarp = 2, kWalkWarp = 3, kSm0 = 4, kSmWarps = 8;
constexpr int kSegs = 4;                   // units that the walker is ahead
constexpr float kTau = 8.f;                // a maximum that grows by less leaves O as it is

constexpr int OFF_Q = 0;
constexpr int OFF_P = OFF_Q + 9 * kQBlk;   // [64 rows x 192 keys] bf16: three blocks
constexpr int OFF_KV = OFF_P + 3 * kQBlk;
constexpr int OFF_BAR = OFF_KV + kSlots * kSlotB;
constexpr int OFF_SEG = OFF_BAR + 512;
constexpr int OFF_MASK = OFF_SEG + kSegs * 64;   // [4 tiles][8] visible positions of a chunk
constexpr int OFF_POS = OFF_MASK + 4 * 8 * 4;    // [4 tiles][8] a chunk's first position
constexpr int OFF_MAX = OFF_POS + 4 * 8 * 4;     // [2][4][64] row maxima of the quarters
constexpr int OFF_SUM = OFF_MAX + 2 * 4 * 64 * 4;  // [4][64] row sums of the quarters
constexpr int OFF_SCAN = OFF_SUM + 4 * 64 * 4;   // the start's scan: 12 x (tiles, units), result
constexpr int OFF_MISC = OFF_SCAN + 256;
constexpr int SMEM_BYTES = OFF_MISC + 64 + 1024;
static_assert(OFF_P % 1024 == 0 && OFF_KV % 1024 == 0 && kBlkB % 1024 == 0, "swizzle atoms");
static_assert(SMEM_BYTES <= 232448, "shared memory budget");
constexpr int S_COL = 0, O_COL = 256;      // S [2 x 96 columns], O [256]

enum : int {
  B_FULL = 0,                   // [slot] landed in both CTAs (rank 0's)
  B_EMPTY = B_FULL + kSlots,    // [slot] read by the tensor cores
  B_QF = B_EMPTY + kSlots,      // queries landed in both CTAs (rank 0's)
  B_QE,                         // ... read
  B_SF,                         // [2] S written
  B_PF = B_SF + 2,              // P written by both CTAs (rank 0's)
  B_PD,                         // P V done
  B_OE,                         // O read by both CTAs (rank 0's)
  B_MF,                         // [4] masks of a tile written
  B_ME = B_MF + 4,              // [4] ... read
  B_GF = B_ME + 4,              // [kSegs] unit written
  B_GE = B_GF + kSegs,          // [kSegs] ... read
  B_RX = B_GE + kSegs,          // [2] the warps that share rows have written maxima or sums
  B_COUNT = B_RX + 2
};
static_assert(B_COUNT * 8 <= 512, "barrier block");

// A part of a unit, as the walker hands it to the other warps.
struct Seg {
  int tok0, ntok;    // tokens
  int row, own;      // row of the page table; own positions (tokens differ in what they see) or a prefix
  int p_lo;          // the first token's position (a prefix: its last one, for all tokens)
  int t0, t1, nt;    // tiles of nt
  int chunks, cs;    // chunks: the first cs from position 0 on, the others from `base` on
  int base;
  int slot;          // partial result's first row, -1: the unit is whole
  int pad[4];
};
static_assert(sizeof(Seg) == 64, "ring entry");

__device__ __forceinline__ int chunk_pos(const Seg& s, int k) {
  return kChunk * (k < s.cs ? k : s.base + k - s.cs);
}
__device__ __forceinline__ int seg_chunk(const Seg& s, int t) {  // first chunk of tile t
  return (int)((int64_t)s.chunks * t / s.nt);
}

// Bits 0 .. x.
__device__ __forceinline__ uint32_t bits_to(int x) {
  return x < 0 ? 0u : (x >= 31 ? 0xFFFFFFFFu : (2u << x) - 1u);
}
// Positions pos .. pos + 31 that a token at p (tokens p_lo .. p together) sees.
__device__ __forceinline__ uint32_t visible(const Params& p, int pos, int p_lo, int p_hi) {
  const uint32_t near = p.window == 0 ? 0u : ~bits_to(p_lo - p.window - pos);
  return bits_to(p_hi - pos) & (near | bits_to(p.sinks - 1 - pos));
}

// ------------------------------------------------------------------- the line of units
// Entries: the groups' prefixes, then the rows.  Every unit has at least one tile.
struct Entry {
  int tok0, tok1, len, own;
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

__device__ __forceinline__ int row_token(const Params& p, int r) {
  return p.row_offsets == nullptr ? r : clampi(p.row_offsets[r], 0, p.tokens);
}
__device__ __forceinline__ Entry load_entry(const Params& p, int e) {
  Entry x;
  x.own = e >= p.groups;
  if (x.own) {
    const int r = e - p.groups;
    x.tok0 = row_token(p, r);
    x.tok1 = max(x.tok0, row_token(p, r + 1));
    x.len = max(0, p.lengths[r]);
  } else {
    int r0 = 0, r1 = p.rows;
    if (p.group_offsets != nullptr) {
      r0 = clampi(p.group_offsets[e], 0, p.rows);
      r1 = clampi(p.group_offsets[e + 1], r0, p.rows);
    }
    x.tok0 = row_token(p, r0);
    x.tok1 = max(x.tok0, row_token(p, r1));
    x.len = max(0, p.pre_lengths[e]);
  }
  return x;
}
__device__ __forceinline__ int entry_units(const Params& p, const Entry& x) {
  return (x.tok1 - x.tok0 + p.tpu - 1) / p.tpu;
}
__device__ __forceinline__ int cap_of(const Params& p, int own) {
  return (own ? p.own.cols : p.pre.cols) << p.page_shift;
}
// Tiles of units 0 .. x - 1 of a sequence whose unit i ends at position (i + 1) T: ceil((i + 1) / D)
// each (D = 192 / T units a tile), `most` at most.
__device__ __forceinline__ int64_t tiles_to(int64_t x, int d, int64_t most) {
  const int64_t y = min(x, most * (int64_t)d), q = y / d, r = y % d;
  return d * (q * (q + 1) / 2) + r * (q + 1) + (x - y) * most;
}
// Tiles of the first j units of an entry.
__device__ __forceinline__ int64_t entry_tiles(const Params& p, const Entry& x, int j) {
  const int cap = cap_of(p, x.own);
  if (!x.own) return (int64_t)j * max(1, (min(x.len, cap) + kTile - 1) / kTile);
  const int64_t most = min(p.unit_tiles, (int64_t)max(1, (cap + kTile - 1) / kTile));
  const int d = kTile / p.tpu;
  const int64_t a = ((int64_t)max(0, x.len - (x.tok1 - x.tok0)) + p.tpu - 1) / p.tpu;
  return tiles_to(a + j, d, most) - tiles_to(a, d, most);
}

__device__ __forceinline__ int64_t cut_at(int64_t tiles, int pairs, int64_t c) {
  return tiles * c / pairs;
}
// The pair whose part holds tile x.
__device__ __forceinline__ int pair_of(int64_t tiles, int pairs, int64_t x) {
  return (int)(((x + 1) * pairs - 1) / tiles);
}

// Where a partial result's values and (maximum, sum) lie: blocks of 16 rows, so that a warp's
// threads (rows) write and read whole sectors.
__device__ __forceinline__ int64_t part_at(int64_t row, int d) {
  return (row >> 4) * (16 * kDCkv) + (d >> 2) * 64 + (row & 15) * 4;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    attend_kernel(const __grid_constant__ CUtensorMap m_ckv, const __grid_constant__ CUtensorMap m_kpe,
                  const __grid_constant__ CUtensorMap m_ckv1,
                  const __grid_constant__ CUtensorMap m_kpe1,
                  const __grid_constant__ CUtensorMap m_qn, const __grid_constant__ CUtensorMap m_qp,
                  const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const int pair = blockIdx.x >> 1;
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(sgen + OFF_MISC);
  const uint32_t bar0 = sbase + OFF_BAR;
#define bar(k) (bar0 + 8u * (uint32_t)(k))

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      ptx::mbar_init(bar(B_FULL + s), 2);
      ptx::mbar_init(bar(B_EMPTY + s), 1);
    }
    ptx::mbar_init(bar(B_QF), 2);
    ptx::mbar_init(bar(B_QE), 1);
    ptx::mbar_init(bar(B_SF), 1);
    ptx::mbar_init(bar(B_SF + 1), 1);
    ptx::mbar_init(bar(B_PF), 2 * kSmWarps);
    ptx::mbar_init(bar(B_PD), 1);
    ptx::mbar_init(bar(B_OE), 2 * kSmWarps);
    for (int i = 0; i < 4; ++i) {
      ptx::mbar_init(bar(B_MF + i), 1);
      ptx::mbar_init(bar(B_ME + i), kSmWarps);
    }
    for (int i = 0; i < kSegs; ++i) {
      ptx::mbar_init(bar(B_GF + i), 1);
      // loader, query loader, softmax warps and, in rank 0, the issuer
      ptx::mbar_init(bar(B_GE + i), 2 + kSmWarps + (rank == 0 ? 1 : 0));
    }
    ptx::mbar_init(bar(B_RX), 4);
    ptx::mbar_init(bar(B_RX + 1), 4);
    misc[1] = 0;
    misc[2] = 0;
    misc[3] = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    ptx::pair_tmem_alloc(sbase + OFF_MISC, 512);
    ptx::pair_tmem_relinquish();
  }
  if (warp == kLoadWarp && lane < 6)
    ptx::prefetch_tmap(lane == 0 ? &m_ckv : lane == 1 ? &m_kpe : lane == 2 ? &m_ckv1
                       : lane == 3 ? &m_kpe1 : lane == 4 ? &m_qn : &m_qp);
  ptx::tc_fence_before();
  ptx::cluster_sync();
  ptx::tc_fence_after();
  const uint32_t tmem = misc[0];
  ptx::grid_dep_wait();
  ptx::launch_dependents();

  // ---------------------------------------------------------------- this pair's tiles
  const int entries = p.groups + p.rows;
  int64_t* scan = reinterpret_cast<int64_t*>(sgen + OFF_SCAN);
  if (p.whole) {
    // a pair for each row's one unit
    if (threadIdx.x == 0) {
      const Entry x = load_entry(p, pair);
      scan[24] = pair;
      scan[25] = scan[26] = 0;
      scan[27] = entry_tiles(p, x, entry_units(p, x));
    }
    __syncthreads();
  } else {
    const int per = (entries + kThreads - 1) / kThreads;
    const int e0 = min(entries, (int)threadIdx.x * per), e1 = min(entries, e0 + per);
    int64_t mine = 0;
    int units = 0;
    for (int e = e0; e < e1; ++e) {
      const Entry x = load_entry(p, e);
      const int n = entry_units(p, x);
      mine += entry_tiles(p, x, n);
      units += n;
    }
    int64_t run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
      units += __shfl_xor_sync(0xffffffffu, units, o);
    }
    if (lane == 31) scan[warp] = run;
    if (lane == 0) scan[12 + warp] = units;
    __syncthreads();
    int64_t tiles = 0, before = run - mine;
    int all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += scan[w];
      tiles += scan[w];
      all += (int)scan[12 + w];
    }
    // A window's units cost about the same: whole ones, or equal parts of each, while they fit.
    int pairs = (int)(gridDim.x >> 1);
    if (p.groups == 0 && all <= pairs && all > 0) pairs = all * (pairs / all);
    pairs = (int)min((int64_t)pairs, tiles);
    const int64_t lo = pair < pairs ? cut_at(tiles, pairs, pair) : tiles;
    const int64_t hi = pair < pairs ? cut_at(tiles, pairs, pair + 1) : tiles;
    if (lo < hi && lo >= before && lo < before + mine) {
      int e = e0;
      for (;; ++e) {
        const Entry x = load_entry(p, e);
        const int64_t n = entry_tiles(p, x, entry_units(p, x));
        if (lo < before + n) break;
        before += n;
      }
      scan[24] = e;
      scan[25] = before;
    }
    if (threadIdx.x == 0) {
      scan[26] = lo;
      scan[27] = hi;
      scan[28] = tiles;
      scan[29] = pairs;
    }
    __syncthreads();
  }
  const Waiter wait{misc + 2, p.err, p.wait_cycles};
  // One unit record after another; false at the line's end or when a wait gave up.
  auto next_seg = [&](Seg& s, int n) -> bool {
    const bool ok = wait(bar(B_GF + (n % kSegs)), (uint32_t)((n / kSegs) & 1));
    s = *reinterpret_cast<const Seg*>(sgen + OFF_SEG + 64 * (n % kSegs));
    __syncwarp();
    return __all_sync(0xffffffffu, ok) && s.t0 < s.t1;
  };
  auto seg_read = [&](int n) {
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar(B_GE + (n % kSegs)));
  };

  if (warp == kWalkWarp) {
    // ------------------------------------------------------------------ units
    if (lane == 0) {
      int64_t x = scan[26];
      const int64_t hi = scan[27];
      if (rank == 0 && pair == 0 && !p.whole) {
        p.head[0] = scan[28];
        p.head[1] = scan[29];
      }
      int n = 0;
      bool ok = true;
      auto put = [&](const Seg& s) {
        if (n >= kSegs) ok = wait(bar(B_GE + (n % kSegs)), (uint32_t)(((n / kSegs) - 1) & 1));
        if (!ok) return;
        *reinterpret_cast<Seg*>(sgen + OFF_SEG + 64 * (n % kSegs)) = s;
        ptx::mbar_arrive(bar(B_GF + (n % kSegs)));
        ++n;
      };
      int e = x < hi ? (int)scan[24] : 0;
      int64_t ebase = x < hi ? scan[25] : 0;
      const int heads = p.heads;
      while (ok && x < hi) {
        const Entry en = load_entry(p, e);
        const int units = entry_units(p, en);
        const int64_t etiles = entry_tiles(p, en, units);
        if (x >= ebase + etiles) {
          ebase += etiles;
          ++e;
          continue;
        }
        // the unit that holds tile x
        int j = 0, top = units;
        while (top - j > 1) {
          const int mid = (j + top) >> 1;
          if (ebase + entry_tiles(p, en, mid) <= x) j = mid;
          else top = mid;
        }
        const int cap = cap_of(p, en.own);
        for (; ok && j < units && x < hi; ++j) {
          Seg s = {};
          const int64_t ubase = ebase + entry_tiles(p, en, j);
          s.nt = (int)(ebase + entry_tiles(p, en, j + 1) - ubase);
          s.tok0 = en.tok0 + j * p.tpu;
          s.ntok = min(p.tpu, en.tok1 - s.tok0);
          s.own = en.own;
          s.row = en.own ? e - p.groups : e;
          s.t0 = (int)(x - ubase);
          s.t1 = (int)min((int64_t)s.nt, hi - ubase);
          if (en.own) {
            s.p_lo = en.len - (en.tok1 - en.tok0) + j * p.tpu;
            const int p_hi = s.p_lo + s.ntok - 1, last = min(p_hi, cap - 1);
            const int lo = max(0, s.p_lo - p.window + 1);
            const int all = last < 0 ? 0 : last / kChunk + 1;
            const int base = lo / kChunk, sink = (p.sinks + kChunk - 1) / kChunk;
            const int near = last >= lo ? last / kChunk - base + 1 : 0;
            s.chunks = min(all, sink + near);
            s.cs = all <= sink + near ? all : sink;
            s.base = base;
            if (p_hi >= cap) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
          } else {
            s.p_lo = min(en.len, cap) - 1;
            s.chunks = s.cs = (min(en.len, cap) + kChunk - 1) / kChunk;
            if (en.len > cap) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
          }
          const bool whole = s.t0 == 0 && s.t1 == s.nt;
          if (p.groups == 0) {
            // two partial results of a pair at most: its line's first unit and its last
            s.slot = whole ? -1 : 128 * (2 * pair + (s.t0 == 0 ? 1 : 0));
            if (rank == 0 && x == scan[26] && !p.whole) {
              int64_t* m = p.cuts + 4 * pair;
              m[0] = ubase;
              m[1] = ubase + s.nt;
              m[2] = s.tok0;
              m[3] = s.ntok;
            }
          } else {
            s.slot = heads * (s.tok0 + (en.own ? p.tokens : 0)) + 128 * pair;
            if (rank == 0 && s.t0 == 0)
              for (int i = 0; i < s.ntok; ++i) {
                int64_t* m = p.cuts + 3 * (2 * (int64_t)(s.tok0 + i) + en.own);
                m[0] = ubase;
                m[1] = ubase + s.nt;
                m[2] = s.tok0;
              }
          }
          put(s);
          x = ubase + s.t1;
        }
      }
      if (ok) put(Seg{});
    }
    __syncwarp();
  } else if (warp == kQWarp) {
    // ------------------------------------------------------------------ queries
    const uint32_t qf = ptx::mapa(bar(B_QF), 0);
    Seg s;
    for (int n = 0; next_seg(s, n); ++n) {
      seg_read(n);
      if (lane == 0) {
        if (n > 0 && !wait(bar(B_QE), (uint32_t)((n - 1) & 1))) break;
        ptx::mbar_arrive_expect_tx_cluster(qf, 9 * kQBlk);
        const int hb = min(64, p.heads);
        const int tok = s.tok0 + (p.heads == 128 ? 0 : (int)rank * (64 / hb));
        const int head = p.heads == 128 ? 64 * (int)rank : 0;
        for (int b = 0; b < 8; ++b)
          ptx::pair_load_3d(sbase + OFF_Q + b * kQBlk, &m_qn, 64 * b, head, tok, qf);
        ptx::pair_load_3d(sbase + OFF_Q + 8 * kQBlk, &m_qp, 0, head, tok, qf);
      }
      __syncwarp();
    }
    __syncwarp();
  } else if (warp == kLoadWarp) {
    // ------------------------------------------------------------------ keys and values
    // A tile's keys are looked up once; K and V slots then follow in the order in which the
    // issuer reads them: K of tile i + 1 before V of tile i.
    const int hbs = min(5, p.page_shift);      // log2 of a box's rows
    const bool by_row = p.page_shift < 3;      // pages too small for boxes: four rows at a time
    const int nbs = by_row ? 0 : 5 - hbs;      // log2 of the boxes in a chunk
    const int none = (int)p.num_slots;         // a row outside the pool: reads as zeros
    const int64_t num_pages = p.num_slots >> p.page_shift;
    volatile uint32_t* masks = reinterpret_cast<volatile uint32_t*>(sgen + OFF_MASK);
    volatile int* poss = reinterpret_cast<volatile int*>(sgen + OFF_POS);
    struct Keys {
      int nc;                        // chunks
      int box;                       // lane: the slot of box `lane` (chunk lane >> nbs)
      uint32_t w[kTileChunks];       // visible positions of each chunk
      int rows[kTileChunks];         // by_row: lane: the slot of row `lane` of each chunk
    };
    int cnt = 0, tile = 0;
    bool ok = true;

    auto look_up = [&](const Seg& s, int t, Keys& k) {
      const Table& tab = s.own ? p.own : p.pre;
      const int32_t* pages = tab.pt + (int64_t)s.row * tab.sb;
      const int c0 = seg_chunk(s, t);
      k.nc = seg_chunk(s, t + 1) - c0;
      const int p_hi = s.own ? s.p_lo + s.ntok - 1 : s.p_lo;
      auto slot_of = [&](int pos) -> int {
        const int pg = pos >> p.page_shift;
        const int id = pg < tab.cols ? pages[pg] : -1;
        return id >= 0 && id < num_pages ? (id << p.page_shift) + (pos & ((1 << p.page_shift) - 1))
                                         : none;
      };
      bool bad = false;
      k.box = none;
      uint32_t absent = 0;  // boxes without a page
      if (!by_row) {
        const int c = lane >> nbs;
        if (c < k.nc) k.box = slot_of(chunk_pos(s, c0 + c) + ((lane & ((1 << nbs) - 1)) << hbs));
        absent = __ballot_sync(0xffffffffu, c < k.nc && k.box == none);
      }
#pragma unroll
      for (int c = 0; c < kTileChunks; ++c) {
        k.w[c] = 0;
        if (c >= k.nc) continue;
        const int pos = chunk_pos(s, c0 + c);
        uint32_t w = s.own ? visible(p, pos, s.p_lo, p_hi) : bits_to(p_hi - pos);
        if (by_row) {
          k.rows[c] = (w >> lane) & 1u ? slot_of(pos + lane) : none;
          const uint32_t have = __ballot_sync(0xffffffffu, k.rows[c] != none);
          bad |= (have != w);
          w = have;
        } else if (absent) {
          uint32_t gone = 0;
          for (int b = 0; b < (1 << nbs); ++b)
            if ((absent >> ((c << nbs) + b)) & 1u)
              gone |= (hbs == 5 ? 0xFFFFFFFFu : ((1u << (1 << hbs)) - 1u)) << (b << hbs);
          bad |= (w & gone) != 0u;
          w &= ~gone;
        }
        k.w[c] = w;
        if (lane == c) {
          masks[(tile & 3) * 8 + c] = w;
          poss[(tile & 3) * 8 + c] = pos;
        }
      }
      if (bad && lane == 0) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
      if (lane >= k.nc && lane < kTileChunks) masks[(tile & 3) * 8 + lane] = 0;
    };

    // Fills the next slot: chunks c3 .. c3 + 2 (3 x `hi`), columns col .. of 64 x blocks.
    auto fill = [&](const Keys& k, bool hi, const CUtensorMap* map, const CUtensorMap* map1,
                    int col, int blocks_shift, bool values) {
      const int slot = cnt % kSlots;
      if (cnt >= kSlots) ok = ok && wait(bar(B_EMPTY + slot), (uint32_t)((cnt / kSlots - 1) & 1));
      ok = __all_sync(0xffffffffu, ok);
      ++cnt;
      if (!ok) return;
      const uint32_t full = ptx::mapa(bar(B_FULL + slot), 0);
      const int c3 = hi ? 3 : 0;
      const int n = min(3, max(0, k.nc - c3));
      if (lane == 0) {
        if (n) ptx::mbar_arrive_expect_tx_cluster(full, (uint32_t)(n * kChunk * 128) << blocks_shift);
        else ptx::mbar_arrive_cluster(full);
      }
      __syncwarp();
      const uint32_t dst = sbase + OFF_KV + slot * kSlotB;
      const int blk = lane & ((1 << blocks_shift) - 1);
      const int bx = lane >> blocks_shift;
      if (!by_row) {
        const int row = __shfl_sync(0xffffffffu, k.box, ((c3 << nbs) + bx) & 31);
        const int c = bx >> nbs;
        bool mine = bx < (n << nbs);
        // values of a chunk that is not seen whole: row by row below, zeros for the rest
        if (values && mine) {
          const uint32_t w = c == 0 ? (hi ? k.w[3] : k.w[0])
                             : c == 1 ? (hi ? k.w[4] : k.w[1]) : (hi ? k.w[5] : k.w[2]);
          mine = w == 0xFFFFFFFFu;
        }
        if (mine)
          ptx::pair_load_2d(dst + blk * kBlkB + (bx << hbs) * 128, map, col + 64 * blk, row, full);
      }
      if (by_row || values) {
#pragma unroll
        for (int c = 0; c < 3; ++c) {
          const uint32_t w = hi ? k.w[3 + c] : k.w[c];
          if (c >= n || (!by_row && w == 0xFFFFFFFFu)) continue;
          int row;
          if (by_row) row = hi ? k.rows[3 + c] : k.rows[c];
          else {
            const int b = __shfl_sync(0xffffffffu, k.box, ((c3 + c) << nbs) + (lane >> hbs));
            row = (w >> lane) & 1u ? b + (lane & ((1 << hbs) - 1)) : none;
          }
          const int g = bx & 7;
          int4 r;
          r.x = __shfl_sync(0xffffffffu, row, 4 * g);
          r.y = __shfl_sync(0xffffffffu, row, 4 * g + 1);
          r.z = __shfl_sync(0xffffffffu, row, 4 * g + 2);
          r.w = __shfl_sync(0xffffffffu, row, 4 * g + 3);
          if (bx < 8)
            ptx::pair_gather4(dst + blk * kBlkB + (c * kChunk + 4 * g) * 128, map1, col + 64 * blk, r,
                              full);
        }
      }
      __syncwarp();
    };
    auto load_k = [&](const Keys& k) {
      if (k.nc == 0) return;
#pragma unroll 1
      for (int b = 0; b < 4; ++b) fill(k, rank == 1, &m_ckv, &m_ckv1, 128 * b, 1, false);
      fill(k, rank == 1, &m_kpe, &m_kpe1, 0, 0, false);
    };
    auto load_v = [&](const Keys& k) {
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        if (k.nc <= 3 * h) break;
#pragma unroll 1
        for (int d = 0; d < 2; ++d)
          fill(k, h == 1, &m_ckv, &m_ckv1, 256 * (int)rank + 128 * d, 1, true);
      }
    };

    Seg s;
    for (int n = 0; ok && next_seg(s, n); ++n) {
      seg_read(n);
      Keys prev, now;
      for (int t = s.t0; ok && t < s.t1; ++t, ++tile) {
        if (tile >= 4)
          ok = __all_sync(0xffffffffu, wait(bar(B_ME + (tile & 3)), (uint32_t)(((tile >> 2) - 1) & 1)));
        if (!ok) break;
        look_up(s, t, now);
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(B_MF + (tile & 3)));
        load_k(now);
        if (t > s.t0) load_v(prev);
        prev = now;
      }
      if (ok) load_v(prev);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------------ tensor cores
    if (rank == 0) {
      const Waiter pwait{misc + 2, p.err, p.wait_cycles, true};
      constexpr uint32_t kIdS = idesc_bf16(128, kTile, false), kIdO = idesc_bf16(128, 256, false, true);
      const uint64_t dq = desc(sbase + OFF_Q, 16, 1024, kSw128);
      const uint64_t dp = desc(sbase + OFF_P, 16, 1024, kSw128);
      const uint64_t dk = desc(sbase + OFF_KV, 16, 1024, kSw128);
      const uint64_t dv = desc(sbase + OFF_KV, kBlkB, 1024, kSw128);
      int cnt = 0, i = 0;  // slots and tiles so far
      bool ok = true;
      Seg s;
      for (int n = 0; ok && next_seg(s, n); ++n) {
        seg_read(n);
        if (lane == 0) {
          bool o_init = false;
          auto scores = [&](int nc) {
            const uint32_t d = tmem + S_COL + 96 * (i & 1);
            if (nc > 0) {
#pragma unroll 1
              for (int b = 0; b < 5 && ok; ++b, ++cnt) {
                const int slot = cnt % kSlots;
                ok = pwait(bar(B_FULL + slot), (uint32_t)((cnt / kSlots) & 1));
                if (!ok) return;
                ptx::tc_fence_after();
                const uint64_t ko = (uint64_t)((slot * kSlotB) >> 4);
                const uint64_t qo = (uint64_t)((2 * b * kQBlk) >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  ptx::pair_umma_bf16(d, dq + qo + (uint64_t)((k * 32) >> 4),
                                      dk + ko + (uint64_t)((k * 32) >> 4), kIdS, (b | k) ? 1u : 0u);
                if (b < 4) {
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    ptx::pair_umma_bf16(d, dq + qo + (uint64_t)((kQBlk + k * 32) >> 4),
                                        dk + ko + (uint64_t)((kBlkB + k * 32) >> 4), kIdS, 1u);
                }
                ptx::pair_commit(bar(B_EMPTY + slot));
              }
            }
            ptx::pair_commit(bar(B_SF + (i & 1)));
          };
          auto values = [&](int tile, int nc, bool first) {
            ok = ok && pwait(bar(B_PF), (uint32_t)(tile & 1));
            if (ok && first && n > 0) ok = pwait(bar(B_OE), (uint32_t)((n - 1) & 1));
            if (!ok) return;
            ptx::tc_fence_after();
#pragma unroll 1
            for (int h = 0; h < 2 && nc > 3 * h; ++h) {
              const int steps = 2 * min(3, nc - 3 * h);
#pragma unroll 1
              for (int dd = 0; dd < 2; ++dd, ++cnt) {
                const int slot = cnt % kSlots;
                ok = pwait(bar(B_FULL + slot), (uint32_t)((cnt / kSlots) & 1));
                if (!ok) return;
                ptx::tc_fence_after();
                const uint64_t vo = (uint64_t)((slot * kSlotB) >> 4);
#pragma unroll
                for (int k = 0; k < 6; ++k) {
                  if (k < steps) {
                    const int kk = 6 * h + k;
                    ptx::pair_umma_bf16(tmem + O_COL + 128 * dd,
                                        dp + (uint64_t)(((kk >> 2) * kQBlk + (kk & 3) * 32) >> 4),
                                        dv + vo + (uint64_t)((k * 2048) >> 4), kIdO,
                                        (o_init || kk > 0) ? 1u : 0u);
                  }
                }
                ptx::pair_commit(bar(B_EMPTY + slot));
              }
            }
            if (nc > 0) o_init = true;
            ptx::pair_commit(bar(B_PD));
          };
          ok = pwait(bar(B_QF), (uint32_t)(n & 1));
          int before = 0;
          for (int t = s.t0; ok && t < s.t1; ++t, ++i) {
            const int nc = seg_chunk(s, t + 1) - seg_chunk(s, t);
            scores(nc);
            if (!ok) break;
            if (t == s.t1 - 1) ptx::pair_commit(bar(B_QE));
            if (t > s.t0) values(i - 1, before, t - 1 == s.t0);
            before = nc;
          }
          if (ok) values(i - 1, before, s.t1 - s.t0 == 1);
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        i = __shfl_sync(0xffffffffu, i, 0);
        cnt = __shfl_sync(0xffffffffu, cnt, 0);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax and output
    const int quad = warp & 3, ch = (warp - kSm0) >> 2;  // lanes 32 quad ..; which half of their keys
    const int half = quad >> 1, row = (quad & 1) * 32 + lane;
    const uint32_t lanes = (uint32_t)(32 * quad) << 16;
    const uint32_t pf = ptx::mapa(bar(B_PF), 0), oe = ptx::mapa(bar(B_OE), 0);
    volatile uint32_t* masks = reinterpret_cast<volatile uint32_t*>(sgen + OFF_MASK);
    volatile int* poss = reinterpret_cast<volatile int*>(sgen + OFF_POS);
    float* maxes = reinterpret_cast<float*>(sgen + OFF_MAX);
    float* sums = reinterpret_cast<float*>(sgen + OFF_SUM);
    const int part = 2 * half + ch;
    int i = 0, shared = 0;
    bool ok = true;
    // The four warps that share these rows have written what they exchange.
    auto exchange = [&]() -> bool {
      const uint32_t b = bar(B_RX + (quad & 1));
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(b);
      const bool done = wait(b, (uint32_t)(shared & 1));
      ++shared;
      return __all_sync(0xffffffffu, done);
    };
    Seg s;
    for (int n = 0; ok && next_seg(s, n); ++n) {
      seg_read(n);
      const int r = 64 * (int)rank + row;  // row of the unit: token r >> head_shift
      const bool live = 64 * (int)rank + 32 * (quad & 1) < (s.ntok << p.head_shift);
      const int pos = s.own ? s.p_lo + (r >> p.head_shift) : s.p_lo;
      const bool differ = s.own && s.ntok > 1;
      float m = -INFINITY, l = 0.f;
      bool o_valid = false;
      for (int t = s.t0; t < s.t1; ++t, ++i) {
        ok = wait(bar(B_MF + (i & 3)), (uint32_t)((i >> 2) & 1));
        // keys: chunk 3 half + 2 ch whole (A), and 16 positions of chunk 3 half + 1 (B)
        const int ca = 3 * half + 2 * ch, cb = 3 * half + 1;
        uint32_t wa = masks[(i & 3) * 8 + ca], wb = masks[(i & 3) * 8 + cb];
        if (differ) {
          if (wa) wa &= visible(p, poss[(i & 3) * 8 + ca], pos, pos);
          if (wb) wb &= visible(p, poss[(i & 3) * 8 + cb], pos, pos);
        }
        wb = (wb >> (16 * ch)) & 0xFFFFu;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(B_ME + (i & 3)));
        ok = ok && wait(bar(B_SF + (i & 1)), (uint32_t)((i >> 1) & 1));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int nc = seg_chunk(s, t + 1) - seg_chunk(s, t);
        if (live) {
          ptx::tc_fence_after();
          uint32_t a[32], b[16];
          const uint32_t sc = tmem + lanes + S_COL + 96 * (i & 1);
          ptx::tmem_ld32(sc + 64 * ch, a);
          ptx::tmem_ld16(sc + 32 + 16 * ch, b);
          ptx::tmem_wait_ld();
          float mt = -INFINITY;
          if (__all_sync(0xffffffffu, wa == 0xFFFFFFFFu && wb == 0xFFFFu)) {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float x = __uint_as_float(a[k]) * p.scale_log2;
              a[k] = __float_as_uint(x);
              mt = fmaxf(mt, x);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float x = __uint_as_float(b[k]) * p.scale_log2;
              b[k] = __float_as_uint(x);
              mt = fmaxf(mt, x);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float x = (wa >> k) & 1u ? __uint_as_float(a[k]) * p.scale_log2 : -INFINITY;
              a[k] = __float_as_uint(x);
              mt = fmaxf(mt, x);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float x = (wb >> k) & 1u ? __uint_as_float(b[k]) * p.scale_log2 : -INFINITY;
              b[k] = __float_as_uint(x);
              mt = fmaxf(mt, x);
            }
          }
          // the row's maximum over the four threads that share it
          float* mx = maxes + (i & 1) * 256;
          mx[part * 64 + row] = mt;
          ok = exchange();
          if (!ok) break;
          mt = fmaxf(fmaxf(mx[row], mx[64 + row]), fmaxf(mx[128 + row], mx[192 + row]));
          float alpha = 1.f;
          const bool need = mt > m + kTau;
          if (need) {
            alpha = m == -INFINITY ? 0.f : ptx::ex2(m - mt);
            l *= alpha;
            m = mt;
          }
          const float me = m == -INFINITY ? 0.f : m;
          float l0 = 0.f, l1 = 0.f;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float x = ptx::ex2(__uint_as_float(a[2 * k]) - me);
            const float y = ptx::ex2(__uint_as_float(a[2 * k + 1]) - me);
            l0 += x;
            l1 += y;
            // P is rounded to bf16 (2^-9 of a value on average less, the values' own type): a
            // second term would double the tensor cores' work on it
            a[k] = pack2(x, y);
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float x = ptx::ex2(__uint_as_float(b[2 * k]) - me);
            const float y = ptx::ex2(__uint_as_float(b[2 * k + 1]) - me);
            l0 += x;
            l1 += y;
            b[k] = pack2(x, y);
          }
          l += l0 + l1;
          // P V of the tile before has read P and written O
          if (i > 0) ok = __all_sync(0xffffffffu, wait(bar(B_PD), (uint32_t)((i - 1) & 1)));
          if (!ok) break;
          if (__any_sync(0xffffffffu, need) && o_valid) {
            ptx::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              const uint32_t ta = tmem + lanes + O_COL + 128 * ch + 32 * c;
              uint32_t o[32];
              ptx::tmem_ld32(ta, o);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              ptx::tmem_st32(ta, o);
            }
            ptx::tmem_wait_st();
          }
          uint8_t* pr = sgen + OFF_P + row * 128;
          auto put = [&](int key, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
            const int kc = key >> 3;
            *reinterpret_cast<uint4*>(pr + (kc >> 3) * kQBlk + (((kc & 7) ^ (row & 7)) << 4)) =
                make_uint4(x, y, z, w);
          };
#pragma unroll
          for (int k = 0; k < 4; ++k)
            put(96 * half + 64 * ch + 8 * k, a[4 * k], a[4 * k + 1], a[4 * k + 2], a[4 * k + 3]);
#pragma unroll
          for (int k = 0; k < 2; ++k)
            put(96 * half + 32 + 16 * ch + 8 * k, b[4 * k], b[4 * k + 1], b[4 * k + 2], b[4 * k + 3]);
          ptx::fence_proxy_async_smem();
          ptx::tc_fence_before();
        } else if (i > 0) {
          ok = __all_sync(0xffffffffu, wait(bar(B_PD), (uint32_t)((i - 1) & 1)));
          if (!ok) break;
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(pf);
        o_valid = o_valid || nc > 0;
      }
      if (!ok) break;
      // the unit's (or its part's) output
      ok = __all_sync(0xffffffffu, wait(bar(B_PD), (uint32_t)((i - 1) & 1)));
      if (!ok) break;
      if (live) {
        ptx::tc_fence_after();
        sums[part * 64 + row] = l;
        ok = exchange();
        if (!ok) break;
        l = sums[row] + sums[64 + row] + sums[128 + row] + sums[192 + row];
        const bool mine = r < (s.ntok << p.head_shift);
        const int64_t tok = s.tok0 + (r >> p.head_shift);
        const int head = r & (p.heads - 1);
        const int d0 = 256 * half + 128 * ch;
        const bool empty = l == 0.f;  // nothing was visible; NaN is not empty
        if (s.slot < 0) {
          const float inv = 1.f / l;
          __nv_bfloat16* out = p.out + tok * p.out_sb + head * p.out_sh + d0;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            ptx::tmem_ld32(tmem + lanes + O_COL + 128 * ch + 32 * c, o);
            ptx::tmem_wait_ld();
            if (mine) {
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  w[k] = empty ? 0u : pack2(__uint_as_float(o[8 * v + 2 * k]) * inv,
                                            __uint_as_float(o[8 * v + 2 * k + 1]) * inv);
                *reinterpret_cast<uint4*>(out + 32 * c + 8 * v) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
          }
          if (mine && part == 0)
            p.lse[tok * p.lse_sb + head * p.lse_sh] =
                empty ? -INFINITY : (m == -INFINITY ? 0.f : m) + ptx::lg2(l);
        } else {
          const int64_t at = (int64_t)s.slot + r;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            ptx::tmem_ld32(tmem + lanes + O_COL + 128 * ch + 32 * c, o);
            ptx::tmem_wait_ld();
            if (mine) {
#pragma unroll
              for (int v = 0; v < 8; ++v)
                *reinterpret_cast<uint4*>(p.part + part_at(at, d0 + 32 * c + 4 * v)) =
                    make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
            }
          }
          if (mine && part == 0)
            p.sums[at] = make_float2(m == -INFINITY ? 0.f : m, l);
        }
        ptx::tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(oe);
    }
  }

  // Neither CTA leaves while the other, or a copy in flight, may still reach its memory: where a
  // wait gave up in either, both first let what is in flight land.
  ptx::tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0)
    ptx::st_cluster_u32(ptx::mapa(sbase + OFF_MISC + 4 * 3, rank ^ 1u), misc[2]);
  ptx::cluster_sync();
  if (misc[2] | misc[3]) {
    if (threadIdx.x == 0) {
      const uint64_t t0 = ptx::cycles();
      while (ptx::cycles() - t0 < 200000ull) __nanosleep(256);
    }
    __syncthreads();
    ptx::cluster_sync();
  }
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::pair_tmem_dealloc(tmem, 512);
  }
#undef bar
}

// ------------------------------------------------------------------- partial results joined
// Rows 16 at a time, a thread a row and kCols consecutive columns: the parts' maxima and sums
// first, then sum_i 2^(m_i - M) O_i over 2^(m_i - M) l_i.

template <int kCols, typename Rows>
__device__ __forceinline__ void join_rows(const Params& p, int64_t tok, int head, int d0,
                                          const Rows& each) {
  float m = -INFINITY;
  each([&](int64_t at) {
    const float2 z = p.sums[at];
    if (z.y != 0.f) m = fmaxf(m, z.x);
  });
  const float base = m == -INFINITY ? 0.f : m;
  float o[kCols] = {}, l = 0.f;
  each([&](int64_t at) {
    const float2 z = p.sums[at];
    if (z.y == 0.f) return;
    const float w = ptx::ex2(z.x - base);
    l += w * z.y;
#pragma unroll
    for (int k = 0; k < kCols / 4; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(p.part + part_at(at, d0 + 4 * k));
      o[4 * k] += w * v.x;
      o[4 * k + 1] += w * v.y;
      o[4 * k + 2] += w * v.z;
      o[4 * k + 3] += w * v.w;
    }
  });
  const float inv = 1.f / l;
  const bool empty = l == 0.f;
  __nv_bfloat16* out = p.out + tok * p.out_sb + head * p.out_sh + d0;
#pragma unroll
  for (int k = 0; k < kCols / 8; ++k) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = empty ? 0u : pack2(o[8 * k + 2 * j] * inv, o[8 * k + 2 * j + 1] * inv);
    *reinterpret_cast<uint4*>(out + 8 * k) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (d0 == 0) p.lse[tok * p.lse_sb + head * p.lse_sh] = empty ? -INFINITY : base + ptx::lg2(l);
}

// Window calls: the units that a cut goes through.  Block (c, rows 16 y ..): the unit that pair c
// goes on with, if pair c - 1 began it.
__global__ void __launch_bounds__(256) join_cuts_kernel(const Params p) {
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  const int64_t tiles = p.head[0];
  const int pairs = (int)p.head[1], c = (int)blockIdx.x + 1;
  if (c >= pairs) return;
  const int64_t *m = p.cuts + 4 * (int64_t)c, lo = m[0], hi = m[1];
  const int first = pair_of(tiles, pairs, lo), last = pair_of(tiles, pairs, hi - 1);
  if (first != c - 1 || cut_at(tiles, pairs, c) == lo) return;
  const int r = 16 * (int)blockIdx.y + ((int)threadIdx.x & 15);
  if (r >= (int)m[3] << p.head_shift) return;
  join_rows<32>(p, m[2] + (r >> p.head_shift), r & (p.heads - 1), 32 * ((int)threadIdx.x >> 4),
                [&](auto&& f) {
                  f((int64_t)128 * (2 * first + 1) + r);
                  for (int k = first + 1; k <= last; ++k) f((int64_t)256 * k + r);
                });
}

// Shared calls: every token, its prefix's parts and its own.  Block (16 rows, 128 columns).
__global__ void __launch_bounds__(128) join_tokens_kernel(const Params p) {
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  const int64_t tiles = p.head[0];
  const int pairs = (int)p.head[1];
  const int64_t r = 16 * (int64_t)blockIdx.x + (threadIdx.x & 15);
  const int tok = (int)(r >> p.head_shift);
  if (tok < row_token(p, 0) || tok >= row_token(p, p.rows)) return;
  int r0 = 0, r1 = p.rows;  // rows with a prefix
  if (p.group_offsets != nullptr) {
    r0 = clampi(p.group_offsets[0], 0, p.rows);
    r1 = clampi(p.group_offsets[p.groups], r0, p.rows);
  }
  const bool prefixed = tok >= row_token(p, r0) && tok < row_token(p, r1);
  const int64_t* rec = p.cuts + 6 * (int64_t)tok;
  int64_t at[2];
  int first[2], last[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    first[k] = 0;
    last[k] = -1;
    if (k == 0 && !prefixed) continue;
    const int64_t lo = rec[3 * k], hi = rec[3 * k + 1];
    first[k] = max(0, pair_of(tiles, pairs, lo));
    last[k] = min(pairs - 1, pair_of(tiles, pairs, hi - 1));
    at[k] = r + (k ? (int64_t)p.tokens * p.heads : 0);
  }
  join_rows<16>(p, tok, (int)(r & (p.heads - 1)), 128 * blockIdx.y + 16 * (threadIdx.x >> 4),
                [&](auto&& f) {
#pragma unroll
                  for (int k = 0; k < 2; ++k)
                    for (int c = first[k]; c <= last[k]; ++c) f(at[k] + 128 * (int64_t)c);
                });
}

}  // namespace dense
}  // namespace dsa
