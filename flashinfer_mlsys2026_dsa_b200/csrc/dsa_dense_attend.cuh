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
// this form S needs no exchange between the CTAs, Q and P stay with their rows, and each CTA takes
// 1,088 of a key's 1,152 bytes into its shared memory (as K: its own half of the keys; as V: its half
// of the columns), 63 bytes a cycle at the tensor cores' full rate, which L2 delivers.
// Measured instruction costs (cycles): N = 64 .. 128 45, N = 192 48, N = 256 64; so 192 keys a
// tile is the smallest at full rate, 17 cycles a key.
//
// The units of all rows form one line of tiles, cut into equal parts, one for each pair (window
// calls with no more units than pairs: for as many pairs as are a multiple of the units; with a token
// a row and more than half as many rows as pairs, a pair for each row and no cut).  A unit that is cut
// leaves partial results (O, maximum, sum) that combine kernels join, and so does every unit of a
// shared call.
//
// Warps of a CTA:  0 and 12 load keys, 13 and 14 values (64 columns each of a slot's 128), 1 and 15
// issue the tensor-core work for S and for O (rank 0 alone), 2 loads queries, 3 walks the units,
// 4-11 softmax and output: a thread is a row and a quarter of a tile's keys (its lane quadrant
// holds half of them, two warps share a quadrant).
#pragma once

namespace dsa {
namespace dense {

constexpr int kChunk = 32;                 // positions that are looked up and masked together
constexpr int kTileChunks = 6;
constexpr int kTile = kChunk * kTileChunks;
constexpr int kSlots = 5;                  // ring of 24 KB: [96 keys x 128 columns]
constexpr int kTurns = 2 * kSlots;         // two barriers a slot, for its fillings in turn
constexpr int kBlkB = 96 * 128;            // [96 keys x 64 columns], 128-byte swizzle
constexpr int kSlotB = 2 * kBlkB;
constexpr int kQBlk = 64 * 128;            // [64 rows x 64 columns]
constexpr int kThreads = 512;
constexpr int kLoadWarp = 0, kMmaWarp = 1, kQWarp = 2, kWalkWarp = 3, kSm0 = 4, kSmWarps = 8,
              kLoadWarp2 = 12,  // and the two behind it
              kPvWarp = 15;
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
constexpr int OFF_SCAN = OFF_SUM + 4 * 64 * 4;   // the start's scan: 16 x (tiles, units); Part
constexpr int OFF_ROWS = OFF_SCAN + 320;         // 6 x [32 + 192] slots, for the loaders
constexpr int OFF_MISC = OFF_ROWS + 6 * 224 * 4;
constexpr int SMEM_BYTES = OFF_MISC + 64 + 1024;
static_assert(OFF_P % 1024 == 0 && OFF_KV % 1024 == 0 && kBlkB % 1024 == 0, "swizzle atoms");
static_assert(SMEM_BYTES <= 232448, "shared memory budget");
constexpr int S_COL = 0, O_COL = 256;      // S [2 x 96 columns], O [256]

enum : int {
  B_FULL = 0,                   // [turn] landed in both CTAs (rank 0's)
  B_EMPTY = B_FULL + kTurns,    // [turn] read by the tensor cores
  B_QF = B_EMPTY + kTurns,      // queries landed in both CTAs (rank 0's)
  B_QE,                         // ... read
  B_SF,                         // [2] S written
  B_PF = B_SF + 2,              // [2] P written by both CTAs (rank 0's)
  B_PD = B_PF + 2,              // P V done
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
  int per, rem;      // chunks of a tile; so many tiles have one more
  int cs, base;      // the first cs chunks are from position 0 on, the others from chunk `base` on
  int slot;          // partial result's first row, -1: the unit is whole
  int pad[3];
};
static_assert(sizeof(Seg) == 64, "ring entry");

__device__ __forceinline__ int chunk_pos(const Seg& s, int k) {
  return kChunk * (k < s.cs ? k : s.base + k - s.cs);
}
__device__ __forceinline__ int seg_chunk(const Seg& s, int t) {  // first chunk of tile t
  return s.per * t + min(t, s.rem);
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
__device__ __forceinline__ int cap_of(const Params& p, int own) {
  return (own ? p.own.cols : p.pre.cols) << p.page_shift;
}
// Tiles of units 0 .. x - 1 of a sequence whose unit i ends at position (i + 1) T: ceil((i + 1) / D)
// each (D = 192 / T = 3 x 2^shift units a tile), `most` at most.  The host refuses calls whose line
// could pass 2^30 places.
__device__ __forceinline__ int tiles_to(uint32_t x, int shift, uint32_t most) {
  const uint32_t whole = min((x >> shift) / 3u, most);  // units that fill their last tile, in D
  const uint32_t y = (3u * whole) << shift;
  return (int)((y >> 1) * (whole + 1) + (x - y) * min(whole + 1, most));
}
// An entry with what its units' tiles follow from.
struct Line {
  int units;
  uint32_t a, most;  // own: units that would fit before the first token; tiles of a unit, at most
  int own, shift;
};
__device__ __forceinline__ Line line_of(const Params& p, const Entry& x) {
  Line y;
  const int tpu_shift = 7 - p.head_shift, cap = cap_of(p, x.own), n = x.tok1 - x.tok0;
  y.units = (n + p.tpu - 1) >> tpu_shift;
  y.own = x.own;
  y.shift = p.head_shift - 1;
  if (x.own) {
    y.a = ((uint32_t)max(0, x.len - n) + p.tpu - 1) >> tpu_shift;
    y.most = (uint32_t)min(p.unit_tiles, max(1, (cap + kTile - 1) / kTile));
  } else {
    y.a = 0;
    y.most = (uint32_t)max(1, (min(x.len, cap) + kTile - 1) / kTile);
  }
  return y;
}
// Places of its first j units: their tiles, and kExtra for what a unit takes besides (its queries,
// its output, the first softmax before there is a P).
constexpr int kExtra = 2;
__device__ __forceinline__ int line_tiles(const Line& y, int j) {
  if (!y.own) return j * (int)(y.most + kExtra);
  return tiles_to(y.a + j, y.shift, y.most) - tiles_to(y.a, y.shift, y.most) + j * kExtra;
}
// Tiles of unit j.
__device__ __forceinline__ int unit_tiles(const Line& y, int j) {
  return y.own ? (int)min(y.most, ((y.a + j) >> y.shift) / 3u + 1u) : (int)y.most;
}

// Places of entries e0 .. e1 - 1, and their units.
__device__ __noinline__ int2 count_entries(const Params& p, int e0, int e1) {
  int2 n = make_int2(0, 0);
#pragma unroll 1
  for (int e = e0; e < e1; ++e) {
    const Line y = line_of(p, load_entry(p, e));
    n.x += line_tiles(y, y.units);
    n.y += y.units;
  }
  return n;
}

// Where part c of `pairs` equal ones begins, and the part that place x lies in.
__device__ __forceinline__ int cut_at(int tiles, int pairs, int c) {
  const uint32_t q = (uint32_t)tiles / (uint32_t)pairs, r = (uint32_t)tiles - q * pairs;
  return (int)(q * c + r * c / (uint32_t)pairs);
}
__device__ __forceinline__ int pair_of(int tiles, int pairs, int x) {
  int c = min(pairs - 1, (int)((float)x * (float)pairs / (float)tiles));  // one off at most
  if (cut_at(tiles, pairs, c) > x) --c;
  else if (c + 1 < pairs && cut_at(tiles, pairs, c + 1) <= x) ++c;
  return c;
}

// Where a partial result's values and (maximum, sum) lie: blocks of 16 rows, so that a warp's
// threads (rows) write and read whole sectors.
__device__ __forceinline__ int64_t part_at(int64_t row, int d) {
  return (row >> 4) * (16 * kDCkv) + (d >> 2) * 64 + (row & 15) * 4;
}

__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
        "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// A pair's part of the line, as the walker found it.
struct Part {
  int start, end;     // places
  int entry, before;  // the entry that holds the first, and the places before that entry
};

// What a pair that gave up leaves: NaN in all query rows of its part, in output and lse where no
// other pair works on their unit, and as the statistics of its partial results, which every join of
// their rows meets.
__device__ __noinline__ void spoil(const Params& p, const Part& x, int pair) {
  const int entries = x.start < x.end ? p.groups + p.rows : 0;
  int ubase = x.before;
#pragma unroll 1
  for (int e = x.entry; e < entries && ubase < x.end; ++e) {
    const Entry en = load_entry(p, e);
    const Line y = line_of(p, en);
#pragma unroll 1
    for (int j = 0; j < y.units && ubase < x.end; ++j) {
      const int nt = unit_tiles(y, j), t0 = max(0, x.start - ubase), t1 = min(nt, x.end - ubase);
      const int tok0 = en.tok0 + j * p.tpu, ntok = min(p.tpu, en.tok1 - tok0);
      const int rows = t0 < t1 ? ntok << p.head_shift : 0;
      const int nan = 0x7fffffff;  // two of bf16 also
      if (p.groups == 0 && t0 == 0 && t1 == nt) {
#pragma unroll 1
        for (int i = threadIdx.x; i < rows * (kDCkv / 8); i += kThreads) {
          const int r = i / (kDCkv / 8), tok = tok0 + (r >> p.head_shift), h = r & (p.heads - 1);
          *reinterpret_cast<int4*>(p.out + (int64_t)tok * p.out_sb + (int64_t)h * p.out_sh +
                                   8 * (i % (kDCkv / 8))) = make_int4(nan, nan, nan, nan);
          if (i % (kDCkv / 8) == 0)
            p.lse[(int64_t)tok * p.lse_sb + (int64_t)h * p.lse_sh] = __int_as_float(nan);
        }
      } else {
        const int64_t slot = p.groups > 0 ? p.heads * (tok0 + (en.own ? p.tokens : 0)) + 128 * pair
                                          : 128 * (2 * pair + (t0 == 0 ? 1 : 0));
#pragma unroll 1
        for (int r = threadIdx.x; r < rows; r += kThreads)
          p.sums[slot + r] = make_float2(__int_as_float(nan), __int_as_float(nan));
        if (p.groups > 0 && t0 == 0 && (int)threadIdx.x < ntok && rows > 0)
          reinterpret_cast<int2*>(p.cuts)[2 * (int64_t)(tok0 + threadIdx.x) + en.own] =
              make_int2(pair, pair);
      }
      ubase += nt + kExtra;
    }
  }
}

// Bounded wait on an mbarrier.  The kernel's roles run side by side, and their code has to fit the
// instruction caches together: 256 rows behind 32768 shared positions took 345 us with 109 KB of it and
// 317 with 85 KB.  So what follows a first look that fails is out of line, but for the walker, whose
// loops are 25 KB longer with a call in them.
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag,
                                     uint32_t* err, uint64_t limit) {
  const uint64_t t0 = ptx::cycles();
#pragma unroll 1
  for (uint32_t it = 1;; ++it) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 0) {
      if (*abort_flag) return false;
      if (ptx::cycles() - t0 > limit) {
        *abort_flag = 1;
        atomicOr(err, (uint32_t)DSA_DEVERR_TIMEOUT);
        return false;
      }
    }
  }
}
struct Wait {
  volatile uint32_t* abort_flag;
  uint32_t* err;
  uint64_t limit;
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
    return ptx::mbar_try_wait(bar, parity) || wait_on(bar, parity, abort_flag, err, limit);
  }
  __device__ __forceinline__ bool here(uint32_t bar, uint32_t parity) const {
    const uint64_t t0 = ptx::cycles();
#pragma unroll 1
    while (!ptx::mbar_try_wait(bar, parity)) {
      if (*abort_flag) return false;
      if (ptx::cycles() - t0 > limit) {
        *abort_flag = 1;
        atomicOr(err, (uint32_t)DSA_DEVERR_TIMEOUT);
        return false;
      }
    }
    return true;
  }
};

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
  // What a warp's lanes hold alike is taken from lane 0 where it comes out of memory or the thread's
  // number: only then does the compiler keep it, and the loops and operands that follow from it,
  // in uniform registers, where copies and tensor-core instructions want them.
  const int warp = uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const int pair = blockIdx.x >> 1;
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(sgen + OFF_MISC);
  const uint32_t bar0 = sbase + OFF_BAR;
#define bar(k) (bar0 + 8u * (uint32_t)(k))

  if (threadIdx.x == 0) {
    for (int s = 0; s < kTurns; ++s) {
      ptx::mbar_init(bar(B_FULL + s), 4);
      ptx::mbar_init(bar(B_EMPTY + s), 1);
    }
    ptx::mbar_init(bar(B_QF), 2);
    ptx::mbar_init(bar(B_QE), 1);
    ptx::mbar_init(bar(B_SF), 1);
    ptx::mbar_init(bar(B_SF + 1), 1);
    ptx::mbar_init(bar(B_PF), 2 * kSmWarps);
    ptx::mbar_init(bar(B_PF + 1), 2 * kSmWarps);
    ptx::mbar_init(bar(B_PD), 1);
    ptx::mbar_init(bar(B_OE), 2 * kSmWarps);
    for (int i = 0; i < 4; ++i) {
      ptx::mbar_init(bar(B_MF + i), 1);
      ptx::mbar_init(bar(B_ME + i), kSmWarps);
    }
    for (int i = 0; i < kSegs; ++i) {
      ptx::mbar_init(bar(B_GF + i), 1);
      // loaders, query loader, softmax warps and, in rank 0, the issuers
      ptx::mbar_init(bar(B_GE + i), 5 + kSmWarps + (rank == 0 ? 2 : 0));
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
  const uint32_t tmem = (uint32_t)uniform((int)misc[0]);
  ptx::grid_dep_wait();
  ptx::launch_dependents();

  // ---------------------------------------------------------------- the line's length
  // Up to 32 entries are counted by the walker itself, more by all warps, for the walker.
  const int entries = p.groups + p.rows, per = (entries + kThreads - 1) / kThreads;
  int2* scan = reinterpret_cast<int2*>(sgen + OFF_SCAN);
  if (entries > 32 && !p.whole) {
    const int e0 = min(entries, (int)threadIdx.x * per), e1 = min(entries, e0 + per);
    const int2 n = count_entries(p, e0, e1);
    const int places = __reduce_add_sync(0xffffffffu, n.x), units = __reduce_add_sync(0xffffffffu, n.y);
    if (lane == 0) scan[warp] = make_int2(places, units);
    __syncthreads();
  }
  const Wait wait{misc + 2, p.err, p.wait_cycles};
  // One unit record after another; false at the line's end or when a wait gave up.
  auto next_seg = [&](Seg& s, int n) -> bool {
    const bool ok = wait(bar(B_GF + (n % kSegs)), (uint32_t)((n / kSegs) & 1));
    const int v = reinterpret_cast<const int*>(sgen + OFF_SEG + 64 * (n % kSegs))[lane & 15];
    int w[sizeof(Seg) / 4];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Seg) / 4); ++i) w[i] = __shfl_sync(0xffffffffu, v, i);
    s = *reinterpret_cast<const Seg*>(w);
    return __all_sync(0xffffffffu, ok) && s.t0 < s.t1;
  };
  auto seg_read = [&](int n) {
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar(B_GE + (n % kSegs)));
  };

  if (warp == kWalkWarp) {
    // ------------------------------------------------------------------ units
    // This pair's part of the line, and the entry where that begins.
    int tiles = 0, pairs = 1, start = 0, hi = 0, e = pair, ebase = 0;
    if (p.whole) {
      hi = count_entries(p, e, e + 1).x;  // a pair for each row's one unit
    } else {
      auto up = [&](int x) {  // sums of the lanes up to this one
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        return x;
      };
      const bool alone = entries <= 32;
      const int step = alone ? 1 : per;
      int2 mine = make_int2(0, 0);
      if (!alone) {
        if (lane < kThreads / 32) mine = scan[lane];
      } else if (lane < entries) {
        mine = count_entries(p, lane, lane + 1);
      }
      tiles = __reduce_add_sync(0xffffffffu, mine.x);
      const int units = __reduce_add_sync(0xffffffffu, mine.y);
      // Windows that the rows fill cost about the same, and as many parts of each unit as of the
      // others cut each of them the same number of times.  (Units of unequal length are cut where
      // the line's equal parts end; up to half of the pairs have none.)
      pairs = p.pairs;
      if (p.groups == 0 && units <= pairs && units > 0) pairs = units * (pairs / units);
      pairs = min(pairs, tiles);
      start = pair < pairs ? cut_at(tiles, pairs, pair) : tiles;
      hi = pair < pairs ? cut_at(tiles, pairs, pair + 1) : tiles;
      e = 0;
#pragma unroll 1
      for (int level = alone ? 1 : 0; level < 2; ++level) {
        // the warp's entries that hold `start`, then the lane's
        const int from = ebase + up(mine.x) - mine.x;
        const uint32_t here = __ballot_sync(0xffffffffu, start >= from && start < from + mine.x);
        const int at = max(0, __ffs(here) - 1);
        ebase = __shfl_sync(0xffffffffu, from, at);
        e += at * (level ? step : 32 * step);
        if (level == 0) {
          const int e0 = min(entries, e + lane * step);
          mine = count_entries(p, e0, min(entries, e0 + step));
        }
      }
    }
    if (lane == 0) {
      *reinterpret_cast<Part*>(scan + 16) = {start, hi, e, ebase};
      int x = start;
      int4 cut = make_int4(0, 0, 0, 0);
      int n = 0;
      bool ok = true;
      auto put = [&](const Seg& s) {
        ok = wait.here(bar(B_GE + (n % kSegs)), (uint32_t)((n / kSegs + 1) & 1));
        if (!ok) return;
        *reinterpret_cast<Seg*>(sgen + OFF_SEG + 64 * (n % kSegs)) = s;
        ptx::mbar_arrive(bar(B_GF + (n % kSegs)));
        ++n;
      };
      const int heads = p.heads;
#pragma unroll 1
      for (; ok && x < hi && e < entries; ++e) {
        const Entry en = load_entry(p, e);
        const Line y = line_of(p, en);
        if (x >= ebase + line_tiles(y, y.units)) {  // an entry before the one sought, or empty
          ebase += line_tiles(y, y.units);
          continue;
        }
        int j = 0, ubase = ebase;
        if (x > ebase) {  // the first entry: the unit that holds place x
          int top = y.units;
#pragma unroll 1
          while (top - j > 1) {
            const int mid = (j + top) >> 1;
            if (ebase + line_tiles(y, mid) <= x) j = mid;
            else top = mid;
          }
          ubase = ebase + line_tiles(y, j);
        }
        const int cap = cap_of(p, en.own);
#pragma unroll 1
        for (; ok && j < y.units && x < hi; ++j) {
          Seg s = {};
          s.nt = unit_tiles(y, j);
          const int next = ubase + s.nt + kExtra;
          if (x - ubase >= s.nt) {  // a cut behind its last tile
            x = ubase = next;
            continue;
          }
          s.tok0 = en.tok0 + j * p.tpu;
          s.ntok = min(p.tpu, en.tok1 - s.tok0);
          s.own = en.own;
          s.row = en.own ? e - p.groups : e;
          s.t0 = x - ubase;
          s.t1 = min(s.nt, hi - ubase);
          int chunks;
          if (en.own) {
            s.p_lo = en.len - (en.tok1 - en.tok0) + j * p.tpu;
            const int p_hi = s.p_lo + s.ntok - 1, last = min(p_hi, cap - 1);
            const int lo = max(0, s.p_lo - p.window + 1);
            const int all = last < 0 ? 0 : last / kChunk + 1;
            const int base = lo / kChunk, sink = (p.sinks + kChunk - 1) / kChunk;
            const int near = last >= lo ? last / kChunk - base + 1 : 0;
            chunks = min(all, sink + near);
            s.cs = all <= sink + near ? all : sink;
            s.base = base;
            if (p_hi >= cap) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
          } else {
            s.p_lo = min(en.len, cap) - 1;
            chunks = s.cs = (min(en.len, cap) + kChunk - 1) / kChunk;
            if (en.len > cap) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
          }
          // Every tile has a chunk: where there are too few, further ones of which nothing is seen.
          if (s.cs == chunks) s.base = s.cs;
          chunks = max(chunks, s.nt);
          s.per = chunks / s.nt;
          s.rem = chunks - s.per * s.nt;
          // a window's pair leaves two partial results at most: its part's first unit and its last
          s.slot = p.groups > 0 ? heads * (s.tok0 + (en.own ? p.tokens : 0)) + 128 * pair
                   : s.t0 == 0 && s.t1 == s.nt ? -1 : 128 * (2 * pair + (s.t0 == 0 ? 1 : 0));
          put(s);
          // where the joins find the unit's parts
          if (rank == 0 && (p.groups > 0 ? s.t0 == 0 : s.t0 > 0)) {
            const int first = pair_of(tiles, pairs, ubase), last = pair_of(tiles, pairs, ubase + s.nt - 1);
            if (p.groups > 0)
              for (int i = 0; i < s.ntok; ++i)
                reinterpret_cast<int2*>(p.cuts)[2 * (int64_t)(s.tok0 + i) + en.own] = make_int2(first, last);
            else if (first == pair - 1)  // at its first cut
              cut = make_int4(first, last, s.tok0, s.ntok);
          }
          x = min(hi, next);
          ubase = next;
        }
        ebase = ubase;
      }
      if (p.groups == 0 && rank == 0 && !p.whole) p.cuts[pair] = cut;
      if (ok) put(Seg{});
    }
    __syncwarp();
  } else if (warp == kQWarp) {
    // ------------------------------------------------------------------ queries
    const uint32_t qf = ptx::mapa(bar(B_QF), 0);
    Seg s;
    bool ok = true;
    for (int n = 0; ok && next_seg(s, n); ++n) {
      seg_read(n);
      if (n > 0) ok = __all_sync(0xffffffffu, wait(bar(B_QE), (uint32_t)((n - 1) & 1)));
      if (ok && lane == 0) {
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
  } else if (warp == kLoadWarp || (warp >= kLoadWarp2 && warp != kPvWarp)) {
    // ------------------------------------------------------------------ keys and values
    // The ring holds, in the order in which the issuer reads them, K of tile i + 1 (this CTA's half
    // of the keys; slots of 128 latent columns, the rope keys third of five), then V of tile i (four
    // slots: half of the keys, half of this CTA's columns; two where it has up to 96 keys).  Two
    // warps load the latent keys, two the rope keys and V: one chain of wait, arrive and copy is too
    // long for every slot.  A warp passes the others' slots without a look, and the two issuers do
    // not read in one order, so a slot has two pairs of barriers in turn: a wait tells a barrier's
    // fillings apart by their parity, and with ten slots' fillings between two of one barrier the
    // one before is always over (with five it need not be: a model of the five warps and the
    // issuers in random steps finds both).
    const bool vals = warp > kLoadWarp2;
    const int blk = vals ? warp - kLoadWarp2 - 1 : warp == kLoadWarp2, me = vals ? 2 + blk : blk;
    const bool el = ptx::elect_one();  // warp-uniform loops around one issuing thread
    const int hbs = min(5, p.page_shift);      // log2 of a box's rows
    const bool by_row = p.page_shift < 3;      // pages too small for boxes: four rows at a time
    const int nbs = by_row ? 0 : 5 - hbs;      // log2 of the boxes in a chunk
    const int none = (int)p.num_slots;         // a row outside the pool: reads as zeros
    const int64_t num_pages = p.num_slots >> p.page_shift;
    volatile uint32_t* masks = reinterpret_cast<volatile uint32_t*>(sgen + OFF_MASK);
    volatile int* poss = reinterpret_cast<volatile int*>(sgen + OFF_POS);
    // Of a tile's keys, for this warp: the slots of its boxes, and of its rows where a chunk goes
    // row by row (a value warp holds two tiles).
    struct Keys {
      int nc;          // chunks
      uint32_t whole;  // chunks seen whole (bits)
      int* boxes;
      int row[6];      // pages of 32 and more: the chunks' slots
    };
    int at = 0, tile = 0;  // the ring's turn, 0 .. 9; tiles so far
    uint32_t round = 0;    // rounds of ten, as a parity
    bool ok = true;
    const uint32_t full0 = ptx::mapa(bar(B_FULL), 0);
    const uint32_t ring0 = sbase + OFF_KV + blk * kBlkB;

    // The page of this lane's box of tile t (-1: no box, or none in the table).
    auto page_of = [&](const Seg& s, int t) -> int {
      const Table& tab = s.own ? p.own : p.pre;
      const int c0 = seg_chunk(s, t), c = lane >> nbs;
      if (by_row || c >= seg_chunk(s, t + 1) - c0) return -1;
      const int pg = (chunk_pos(s, c0 + c) + ((lane & ((1 << nbs) - 1)) << hbs)) >> p.page_shift;
      return pg < tab.cols ? tab.pt[(int64_t)s.row * tab.sb + pg] : -1;
    };
    auto look_up = [&](const Seg& s, int t, int page, Keys& k) {
      const int c0 = seg_chunk(s, t);
      k.nc = seg_chunk(s, t + 1) - c0;
      const int p_hi = s.own ? s.p_lo + s.ntok - 1 : s.p_lo;
      const int in_page = (1 << p.page_shift) - 1;
      int* boxes = reinterpret_cast<int*>(sgen + OFF_ROWS) +
                   224 * (vals ? 2 + 2 * blk + (tile & 1) : blk);
      k.boxes = boxes;
      __syncwarp();
      int box = none;
      if (page >= 0 && page < num_pages)
        box = (page << p.page_shift) +
              ((chunk_pos(s, c0 + (lane >> nbs)) + ((lane & ((1 << nbs) - 1)) << hbs)) & in_page);
      boxes[lane] = box;
#pragma unroll
      for (int c = 0; c < kTileChunks; ++c) k.row[c] = __shfl_sync(0xffffffffu, box, c);
      // lane c: chunk c's first position and what of it is seen
      const int pos = chunk_pos(s, c0 + min(lane, kTileChunks - 1));
      const uint32_t want = lane >= k.nc ? 0u : s.own ? visible(p, pos, s.p_lo, p_hi) : bits_to(p_hi - pos);
      uint32_t w = want;
      if (nbs == 0 && !by_row) {
        if (box == none) w = 0;
      } else if (!by_row) {
        const uint32_t have = __ballot_sync(0xffffffffu, box != none);
        for (int b = 0; b < (1 << nbs); ++b)
          if (!((have >> ((min(lane, kTileChunks - 1) << nbs) + b)) & 1u)) w &= ~(((1u << (1 << hbs)) - 1u) << (b << hbs));
        if (lane >= k.nc) w = 0;
      }
      k.whole = __ballot_sync(0xffffffffu, w == 0xFFFFFFFFu);
      if (by_row) k.whole = 0;
      // the rows of the chunks that are not seen whole
      if (vals || by_row) {
        uint32_t todo = ((1u << k.nc) - 1u) & ~k.whole;
        while (todo) {
          const int c = __ffs(todo) - 1;
          todo &= todo - 1;
          const uint32_t wc = __shfl_sync(0xffffffffu, w, c);
          const int pc = __shfl_sync(0xffffffffu, pos, c) + lane;
          int row = none;
          if (by_row) {
            const Table& tab = s.own ? p.own : p.pre;
            const int pg = pc >> p.page_shift;
            const int id = ((wc >> lane) & 1u) && pg < tab.cols ? tab.pt[(int64_t)s.row * tab.sb + pg] : -1;
            if (id >= 0 && id < num_pages) row = (id << p.page_shift) + (pc & in_page);
            const uint32_t have = __ballot_sync(0xffffffffu, row != none);
            if (lane == c) w = have;
          } else {
            const int b = __shfl_sync(0xffffffffu, box, (c << nbs) + (lane >> hbs));
            if ((wc >> lane) & 1u) row = b + (lane & ((1 << hbs) - 1));
          }
          boxes[32 + kChunk * c + lane] = row;
        }
      }
      if (me == 0) {
        if (lane < kTileChunks) {
          masks[(tile & 3) * 8 + lane] = w;
          poss[(tile & 3) * 8 + lane] = pos;
        }
        // a position that should be there has no page
        if (w != want) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
      }
      __syncwarp();
    };

    // The next slot, free again (its filling before, five turns ago, has been read); n chunks will
    // land in this warp's block of it.
    uint32_t dst0 = 0;
    auto claim = [&](int n) -> uint32_t {
      const bool wrapped = at >= kSlots;
      const uint32_t full = full0 + 8u * (uint32_t)at;
      dst0 = ring0 + (uint32_t)((wrapped ? at - kSlots : at) * kSlotB);
      ok = __all_sync(0xffffffffu, wait(bar(B_EMPTY) + 8u * (uint32_t)(wrapped ? at - kSlots : at + kSlots),
                                        wrapped ? round : round ^ 1u));
      if (el && ok) {
        if (n > 0) ptx::mbar_arrive_expect_tx_cluster(full, (uint32_t)(n * kChunk * 128));
        else ptx::mbar_arrive_relaxed_cluster(full);
      }
      return full;
    };
    auto skip = [&](int n) {
      at += n;
      if (at >= kTurns) {
        at -= kTurns;
        round ^= 1u;
      }
    };
    // Three chunks of which n are there, a box each.
    auto fill = [&](int n, int r0, int r1, int r2, const CUtensorMap* map, int col) {
      const uint32_t full = claim(n);
      if (el && ok) {
        const uint32_t dst = dst0;
        if (n > 0) ptx::pair_load_2d(dst, map, col, r0, full);
        if (n > 1) ptx::pair_load_2d(dst + kChunk * 128, map, col, r1, full);
        if (n > 2) ptx::pair_load_2d(dst + 2 * kChunk * 128, map, col, r2, full);
      }
      skip(1);
    };
    // The same for chunks c3 .. of smaller pages, or with values that are not seen whole: those
    // row by row, zeros where there is nothing to see.
    auto fill_parts = [&](const Keys& k, int c3, int n, bool rope, int col, bool values) {
      const uint32_t full = claim(n);
      const uint32_t all = ((1u << n) - 1u) << c3;
      uint32_t dst = dst0;
      if (ok && !by_row && nbs > 0 && (!values || (k.whole & all) == all)) {
        const CUtensorMap* map = rope ? &m_kpe : &m_ckv;
        const int2* b = reinterpret_cast<const int2*>(k.boxes + (c3 << nbs));
#pragma unroll 2
        for (int j = 0; j < (n << nbs) / 2; ++j, dst += 256 << hbs) {
          const int2 row = b[j];
          if (el) {
            ptx::pair_load_2d(dst, map, col, row.x, full);
            ptx::pair_load_2d(dst + (128 << hbs), map, col, row.y, full);
          }
        }
      } else if (ok) {
#pragma unroll 1
        for (int c = c3; c < c3 + n; ++c, dst += kChunk * 128) {
          if (!by_row && (!values || ((k.whole >> c) & 1u))) {
            const CUtensorMap* map = rope ? &m_kpe : &m_ckv;
            const int* b = k.boxes + (c << nbs);
#pragma unroll 1
            for (int j = 0; j < (1 << nbs); ++j) {
              const int row = b[j];
              if (el) ptx::pair_load_2d(dst + ((j << hbs) * 128), map, col, row, full);
            }
          } else {
            const CUtensorMap* map = rope ? &m_kpe1 : &m_ckv1;
            const int4* rows = reinterpret_cast<const int4*>(k.boxes + 32 + kChunk * c);
#pragma unroll 2
            for (int g = 0; g < 8; ++g) {
              const int4 r = rows[g];
              if (el) ptx::pair_gather4(dst + 512 * g, map, col, r, full);
            }
          }
        }
      }
      skip(1);
    };
    const bool by_box = nbs == 0 && !by_row;  // a box is a chunk
    // 64 columns of this CTA's keys.
    auto load_keys = [&](const Keys& k, bool rope, int col) {
      const int c3 = 3 * (int)rank, n = rope && blk ? 0 : min(3, max(0, k.nc - c3));
      if (by_box)
        fill(n, rank ? k.row[3] : k.row[0], rank ? k.row[4] : k.row[1], rank ? k.row[5] : k.row[2],
             rope ? &m_kpe : &m_ckv, col);
      else
        fill_parts(k, c3, n, rope, col, false);
    };
    auto load_values = [&](const Keys& k) {
      const int col = 256 * (int)rank + 64 * blk;
#pragma unroll 1
      for (int h = 0; ok && h < 2; ++h) {
        const int n = min(3, k.nc - 3 * h);
        if (n <= 0) break;
        const uint32_t all = (1u << n) - 1u;
        const bool whole = by_box && ((k.whole >> (3 * h)) & all) == all;
#pragma unroll 1
        for (int d = 0; ok && d < 2; ++d) {
          if (whole)
            fill(n, h ? k.row[3] : k.row[0], h ? k.row[4] : k.row[1], h ? k.row[5] : k.row[2], &m_ckv,
                 col + 128 * d);
          else
            fill_parts(k, 3 * h, n, false, col + 128 * d, true);
        }
      }
    };

    Seg s;
    for (int n = 0; ok && next_seg(s, n); ++n) {
      seg_read(n);
      Keys k, prev;
      prev.nc = 0;
      int page = page_of(s, s.t0);
      for (int t = s.t0; ok && t <= s.t1; ++t) {
        if (t < s.t1) {
          if (tile >= 4 && me == 0)
            ok = __all_sync(0xffffffffu, wait(bar(B_ME + (tile & 3)), (uint32_t)(((tile >> 2) - 1) & 1)));
          if (!ok) break;
          const int here = page;
          page = t + 1 < s.t1 ? page_of(s, t + 1) : -1;  // on its way meanwhile
          look_up(s, t, here, k);
          if (me == 0 && lane == 0) ptx::mbar_arrive(bar(B_MF + (tile & 3)));
          ++tile;
          if (vals) {
            skip(2);
            load_keys(k, true, 0);
            skip(2);
          } else {
#pragma unroll 1
            for (int b = 0; ok && b < 4; ++b) {
              if (b == 2) skip(1);
              load_keys(k, false, 128 * b + 64 * blk);
            }
          }
        }
        if (t > s.t0) {
          if (vals) load_values(prev);
          else skip(prev.nc > 3 ? 4 : 2);
        }
        prev = k;
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp || warp == kPvWarp) {
    // ------------------------------------------------------------------ tensor cores
    // One warp issues S = Q K^T, the other O += P V.  The tensor cores' queue is short, so what an
    // issuer does between two slots' instructions would leave them idle if it were alone (one
    // issuer: 5,100 cycles a tile of 3,270), and the scores of the next unit start behind the last
    // ones of this.  Each looks at its next slot amid a slot's instructions, so that the answer is
    // there when they are issued.
    if (rank == 0) {
      const bool el = ptx::elect_one();  // warp-uniform loops around one issuing thread
      int at = 0, i = 0;                 // the ring's turn, tiles so far
      uint32_t round = 0;
      bool ok = true, ready = false;
      auto landed = [&]() {
        if (!ready) ok = __all_sync(0xffffffffu, wait(bar(B_FULL) + 8u * (uint32_t)at, round));
        ready = false;
      };
      auto look_ahead = [&]() {
        const bool wrap = at + 1 == kTurns;
        ready = __all_sync(0xffffffffu,
                           ptx::mbar_test_wait(bar(B_FULL) + 8u * (uint32_t)(wrap ? 0 : at + 1),
                                               round ^ (wrap ? 1u : 0u)));
      };
      auto skip = [&](int n) {
        at += n;
        if (at >= kTurns) {
          at -= kTurns;
          round ^= 1u;
        }
      };
      // The wait that also acquires at cluster scope: P and what the softmax warps of rank 1 read.
      auto pair_wait = [&](uint32_t b, uint32_t parity) {
        return wait(b, parity) && ptx::mbar_test_wait_cluster(b, parity);
      };
      auto slot_at = [&]() -> uint64_t {
        return (uint64_t)(((at >= kSlots ? at - kSlots : at) * kSlotB) >> 4);
      };
      Seg s;
      if (warp == kMmaWarp) {
        constexpr uint32_t kIdS = idesc_bf16(128, kTile, false);
        const uint64_t dq = desc(sbase + OFF_Q, 16, 1024, kSw128);
        const uint64_t dk = desc(sbase + OFF_KV, 16, 1024, kSw128);
        for (int n = 0; ok && next_seg(s, n); ++n) {
          seg_read(n);
          ok = __all_sync(0xffffffffu, wait(bar(B_QF), (uint32_t)(n & 1)));
          for (int t = s.t0; ok && t < s.t1; ++t, ++i) {
            // P of two tiles before is written, so its S has been read
            if (i >= 2) {
              ok = __all_sync(0xffffffffu, pair_wait(bar(B_PF + (i & 1)), (uint32_t)(((i - 2) >> 1) & 1)));
              ptx::tc_fence_after();
            }
            const uint32_t d = tmem + S_COL + 96 * (i & 1);
#pragma unroll 1
            for (int b = 0; ok && b < 5; ++b) {
              landed();
              if (!ok) break;
              const uint64_t ko = dk + slot_at();
              const uint64_t qo = dq + (uint64_t)(((b < 2 ? 2 * b : b == 2 ? 8 : 2 * b - 2) * kQBlk) >> 4);
              if (el) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  ptx::pair_umma_bf16(d, qo + (uint64_t)((k * 32) >> 4), ko + (uint64_t)((k * 32) >> 4),
                                      kIdS, (b | k) ? 1u : 0u);
              }
              if (b < 4) look_ahead();
              if (el) {
                if (b != 2) {
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    ptx::pair_umma_bf16(d, qo + (uint64_t)((kQBlk + k * 32) >> 4),
                                        ko + (uint64_t)((kBlkB + k * 32) >> 4), kIdS, 1u);
                }
                ptx::pair_commit(bar(B_EMPTY) + 8u * (uint32_t)at);
              }
              skip(1);
            }
            if (ok && el) {
              ptx::pair_commit(bar(B_SF + (i & 1)));
              if (t == s.t1 - 1) ptx::pair_commit(bar(B_QE));
            }
            // V of the tile before, at the end of the unit of the last one too
            if (t > s.t0) skip(seg_chunk(s, t) - seg_chunk(s, t - 1) > 3 ? 4 : 2);
            if (t == s.t1 - 1) skip(seg_chunk(s, t + 1) - seg_chunk(s, t) > 3 ? 4 : 2);
          }
        }
      } else {
        constexpr uint32_t kIdO = idesc_bf16(128, 256, false, true);
        const uint64_t dp = desc(sbase + OFF_P, 16, 1024, kSw128);
        const uint64_t dv = desc(sbase + OFF_KV, kBlkB, 1024, kSw128);
        for (int n = 0; ok && next_seg(s, n); ++n) {
          seg_read(n);
          for (int t = s.t0; ok && t < s.t1; ++t, ++i) {
            skip(t == s.t0 ? 5 : 0);            // K of this tile
            skip(t + 1 < s.t1 ? 5 : 0);         // and of the next
            ok = __all_sync(0xffffffffu, pair_wait(bar(B_PF + (i & 1)), (uint32_t)((i >> 1) & 1)));
            // the last unit's output has been read
            if (ok && t == s.t0 && n > 0)
              ok = __all_sync(0xffffffffu, pair_wait(bar(B_OE), (uint32_t)((n - 1) & 1)));
            if (!ok) break;
            // S was read and O rescaled through tensor memory
            ptx::tc_fence_after();
            const int nc = seg_chunk(s, t + 1) - seg_chunk(s, t);
#pragma unroll 1
            for (int hd = 0; ok && hd < (nc > 3 ? 4 : 2); ++hd) {
              const int h = hd >> 1, dd = hd & 1, steps = 2 * min(3, nc - 3 * h);
              landed();
              if (!ok) break;
              const uint64_t vo = dv + slot_at();
              // P's 16 keys 6 h + k lie in block (6 h + k) / 4 of 64 keys
              const uint64_t po = dp + (uint64_t)((h * (kQBlk + 64)) >> 4);
              const uint32_t o = tmem + O_COL + 128 * dd;
              const bool add = t > s.t0 || h > 0;
              auto two = [&](int k0) {
#pragma unroll
                for (int k = k0; k < k0 + 2; ++k) {
                  // blocks of the two halves break at other places: 0-3, 4-5 and 6-7, 8-11
                  const uint64_t in = h ? (k < 2 ? k * 32 : kQBlk - 64 + (k - 2) * 32)
                                        : (k >> 2) * kQBlk + (k & 3) * 32;
                  ptx::pair_umma_bf16(o, po + (in >> 4), vo + (uint64_t)((k * 2048) >> 4), kIdO,
                                      (add || k) ? 1u : 0u);
                }
              };
              if (el) two(0);
              if (hd < 3) look_ahead();
              if (el && steps > 2) two(2);
              if (el && steps > 4) two(4);
              if (el) ptx::pair_commit(bar(B_EMPTY) + 8u * (uint32_t)at);
              skip(1);
            }
            ready = false;
            if (ok && el) ptx::pair_commit(bar(B_PD));
          }
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax and output
    const int quad = warp & 3, ch = (warp - kSm0) >> 2;  // lanes 32 quad ..; which half of their keys
    const int half = quad >> 1, row = (quad & 1) * 32 + lane;
    const uint32_t lanes = (uint32_t)(32 * quad) << 16;
    const uint32_t pf0 = ptx::mapa(bar(B_PF), 0), oe = ptx::mapa(bar(B_OE), 0);
    volatile uint32_t* masks = reinterpret_cast<volatile uint32_t*>(sgen + OFF_MASK);
    volatile int* poss = reinterpret_cast<volatile int*>(sgen + OFF_POS);
    float* maxes = reinterpret_cast<float*>(sgen + OFF_MAX);
    float* sums = reinterpret_cast<float*>(sgen + OFF_SUM);
    const int part = 2 * half + ch;
    const float size = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
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
    // A unit's (or a part's) output, written when the next unit's first P has been: its scores and
    // softmax run while the last P V of this one does, and P V of the next waits for this alone.
    struct Last {
      int tok0, rows, slot;
      bool live, open;
      float m, l;
    } last = {};
    auto finish = [&]() {
      last.open = false;
      if (last.live) {
        ptx::tc_fence_after();
        sums[part * 64 + row] = last.l;
        ok = exchange();
        if (!ok) return;
        const float l = sums[row] + sums[64 + row] + sums[128 + row] + sums[192 + row], m = last.m;
        const int r = 64 * (int)rank + row;
        const bool mine = r < last.rows;
        const int d0 = 256 * half + 128 * ch;
        const bool empty = l == 0.f;  // nothing was visible; NaN is not empty
        const uint32_t oc = tmem + lanes + O_COL + 128 * ch;
        uint32_t o[2][32];
        ptx::tmem_ld32(oc, o[0]);
        if (last.slot < 0) {
          const float inv = empty ? 0.f : 1.f / l;
          const int q = lane & 3;
          __nv_bfloat16* out[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int rr = 64 * (int)rank + 32 * (quad & 1) + (lane & 28) + (q ^ k);
            out[k] = p.out + (int64_t)(last.tok0 + (rr >> p.head_shift)) * p.out_sb +
                     (int64_t)(rr & (p.heads - 1)) * p.out_sh + d0 + 8 * q;
            if (rr >= last.rows) out[k] = nullptr;
          }
          // All of O first, so that the next unit's P V need not wait for the writes (5,800 cycles a
          // unit of a prompt, when all pairs write at once).
          uint32_t w[4][16];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            ptx::tmem_wait_ld();
            if (c < 3) ptx::tmem_ld32(oc + 32 * (c + 1), o[(c + 1) & 1]);
#pragma unroll
            for (int k = 0; k < 16; ++k)
              w[c][k] = empty ? 0u : pack2(__uint_as_float(o[c & 1][2 * k]) * inv,
                                           __uint_as_float(o[c & 1][2 * k + 1]) * inv);
          }
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_relaxed_cluster(oe);
          // Four lanes swap pieces of 16 bytes, so that they write 64 consecutive bytes of each of
          // their rows in turn instead of 16 bytes of four: lane q gets piece q of row q ^ k from its
          // holder, which sends piece (its own q) ^ k.
#pragma unroll
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t x[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const bool b0 = ((q ^ k) & 1) != 0, b1 = ((q ^ k) & 2) != 0;
                const uint32_t lo = b0 ? w[c][4 + j] : w[c][j], hi = b0 ? w[c][12 + j] : w[c][8 + j];
                x[j] = __shfl_xor_sync(0xffffffffu, b1 ? hi : lo, k);
              }
              if (out[k] != nullptr)
                *reinterpret_cast<uint4*>(out[k] + 32 * c) = make_uint4(x[0], x[1], x[2], x[3]);
            }
          }
          if (mine && part == 0)
            p.lse[(int64_t)(last.tok0 + (r >> p.head_shift)) * p.lse_sb +
                  (int64_t)(r & (p.heads - 1)) * p.lse_sh] =
                empty ? -INFINITY : (m == -INFINITY ? 0.f : m) + ptx::lg2(l);
          return;
        } else {
          const int64_t at = (int64_t)last.slot + r;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            ptx::tmem_wait_ld();
            if (c < 3) ptx::tmem_ld32(oc + 32 * (c + 1), o[(c + 1) & 1]);
            if (mine) {
              float* to = p.part + part_at(at, d0 + 32 * c);
#pragma unroll
              for (int v = 0; v < 8; ++v)
                *reinterpret_cast<uint4*>(to + 64 * v) =
                    make_uint4(o[c & 1][4 * v], o[c & 1][4 * v + 1], o[c & 1][4 * v + 2],
                               o[c & 1][4 * v + 3]);
            }
          }
          if (mine && part == 0)
            p.sums[at] = make_float2(m == -INFINITY ? 0.f : m, l);
        }
        ptx::tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_relaxed_cluster(oe);
    };
    Seg s = {};
    int n = 0, t = 0, pos = 0;
    bool live = false, differ = false;
    float m = -INFINITY, l = 0.f;
    auto open_unit = [&]() -> bool {
      if (!next_seg(s, n)) return false;
      seg_read(n);
      ++n;
      const int r = 64 * (int)rank + row;  // row of the unit: token r >> head_shift
      live = 64 * (int)rank + 32 * (quad & 1) < (s.ntok << p.head_shift);
      pos = s.own ? s.p_lo + (r >> p.head_shift) : s.p_lo;
      differ = s.own && s.ntok > 1;
      t = s.t0;
      m = -INFINITY;
      l = 0.f;
      return true;
    };
#pragma unroll 1
    for (bool more = true;; ++i, ++t) {
      if (t == s.t1) {  // at the start too: both are 0
        if (i > 0) last = {s.tok0, s.ntok << p.head_shift, s.slot, live, true, m, l};
        more = open_unit();
      }
      if (more) {
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
        if (live) {
          ptx::tc_fence_after();
          uint32_t a[32], b[16];
          const uint32_t sc = tmem + lanes + S_COL + 96 * (i & 1);
          ptx::tmem_ld32(sc + 64 * ch, a);
          ptx::tmem_ld16(sc + 32 + 16 * ch, b);
          ptx::tmem_wait_ld();
          // Values of the row's largest score are taken before the scale; a scale below zero turns
          // the scores round first, zero makes them all alike.
          if (p.scale_log2 <= 0.f) {
            const float turn = p.scale_log2 < 0.f ? -1.f : 0.f;
#pragma unroll
            for (int k = 0; k < 32; ++k) a[k] = __float_as_uint(__uint_as_float(a[k]) * turn);
#pragma unroll
            for (int k = 0; k < 16; ++k) b[k] = __float_as_uint(__uint_as_float(b[k]) * turn);
          }
          if (!__all_sync(0xffffffffu, wa == 0xFFFFFFFFu && wb == 0xFFFFu)) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!((wa >> k) & 1u)) a[k] = 0xFF800000u;  // -inf
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (!((wb >> k) & 1u)) b[k] = 0xFF800000u;
          }
          float mp[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int k = 0; k < 32; k += 8)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              mp[j] = fmaxf(mp[j], fmaxf(__uint_as_float(a[k + j]), __uint_as_float(a[k + j + 4])));
#pragma unroll
          for (int k = 0; k < 16; k += 8)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              mp[j] = fmaxf(mp[j], fmaxf(__uint_as_float(b[k + j]), __uint_as_float(b[k + j + 4])));
          float mt = fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3]));
          // the row's maximum over the four threads that share it
          float* mx = maxes + (i & 1) * 256;
          mx[part * 64 + row] = mt;
          ok = exchange();
          if (!ok) break;
          mt = fmaxf(fmaxf(mx[row], mx[64 + row]), fmaxf(mx[128 + row], mx[192 + row])) * size;
          float alpha = 1.f;
          const bool need = mt > m + kTau;
          if (need) {
            alpha = m == -INFINITY ? 0.f : ptx::ex2(m - mt);
            l *= alpha;
            m = mt;
          }
          const float me = m == -INFINITY ? 0.f : m;
          const float2 size2 = make_float2(size, size), me2 = make_float2(-me, -me);
          float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          auto numerator = [&](uint32_t u, uint32_t v, int j) -> uint32_t {
            const float2 x = fma2(make_float2(__uint_as_float(u), __uint_as_float(v)), size2, me2);
            const float2 e = make_float2(ptx::ex2(x.x), ptx::ex2(x.y));
            l2[j & 1] = add2(l2[j & 1], e);
            // P is rounded to bf16, as the values are (2^-8 of each at most, independent of one
            // another); a second term would double the tensor cores' work on it
            return pack2(e.x, e.y);
          };
#pragma unroll
          for (int k = 0; k < 16; ++k) a[k] = numerator(a[2 * k], a[2 * k + 1], k);
#pragma unroll
          for (int k = 0; k < 8; ++k) b[k] = numerator(b[2 * k], b[2 * k + 1], k);
          l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
          // P V of the tile before has read P and written O
          if (i > 0) ok = __all_sync(0xffffffffu, wait(bar(B_PD), (uint32_t)((i - 1) & 1)));
          if (!ok) break;
          if (__any_sync(0xffffffffu, need) && t > s.t0) {
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
        if (lane == 0) {
          ptx::fence_release_smem_cluster();  // P of all lanes
          ptx::mbar_arrive_relaxed_cluster(pf0 + 8u * (uint32_t)(i & 1));
        }
      } else {
        if (!last.open) break;
        ok = __all_sync(0xffffffffu, wait(bar(B_PD), (uint32_t)((i - 1) & 1)));
        if (!ok) break;
      }
      if (last.open) {  // P V of its last tile is done: P was written behind it
        finish();
        if (!ok) break;
      }
      if (!more) break;
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
    if (rank == 0) spoil(p, *reinterpret_cast<const Part*>(scan + 16), pair);
  }
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::pair_tmem_dealloc(tmem, 512);
  }
#undef bar
}

// ------------------------------------------------------------------- partial results joined
// Rows 16 at a time, a thread a row and kCols consecutive columns, with the running maximum and
// sum, so that a part's values are on their way together with its maximum.
template <int kCols>
struct Joined {
  float o[kCols] = {};
  float m = -INFINITY, l = 0.f;

  __device__ __forceinline__ void add(const Params& p, int64_t at, int d0) {
    const float2 z = p.sums[at];
    float4 v[kCols / 4];
#pragma unroll
    for (int k = 0; k < kCols / 4; ++k)
      v[k] = *reinterpret_cast<const float4*>(p.part + part_at(at, d0 + 4 * k));
    if (z.y == 0.f) return;  // nothing was visible: its values are none
    const float top = fmaxf(m, z.x), a = m == -INFINITY ? 0.f : ptx::ex2(m - top),
                w = ptx::ex2(z.x - top);
    m = top;
    l = l * a + w * z.y;
#pragma unroll
    for (int k = 0; k < kCols / 4; ++k) {
      o[4 * k] = o[4 * k] * a + w * v[k].x;
      o[4 * k + 1] = o[4 * k + 1] * a + w * v[k].y;
      o[4 * k + 2] = o[4 * k + 2] * a + w * v[k].z;
      o[4 * k + 3] = o[4 * k + 3] * a + w * v[k].w;
    }
  }
  __device__ __forceinline__ void write(const Params& p, int64_t tok, int head, int d0) const {
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
    if (d0 == 0) p.lse[tok * p.lse_sb + head * p.lse_sh] = empty ? -INFINITY : m + ptx::lg2(l);
  }
};

// Window calls: the units that a cut goes through.  Block (c, rows 16 y ..): the unit that pair
// c + 1 goes on with, if pair c began it.
__global__ void __launch_bounds__(256) join_cuts_kernel(const Params p) {
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  const int4 cut = p.cuts[blockIdx.x + 1];  // first and last pair, first token, tokens
  const int r = 16 * (int)blockIdx.y + ((int)threadIdx.x & 15);
  if (r >= cut.w << p.head_shift) return;
  const int d0 = 32 * ((int)threadIdx.x >> 4);
  Joined<32> x;
  x.add(p, (int64_t)128 * (2 * cut.x + 1) + r, d0);
#pragma unroll 2
  for (int k = cut.x + 1; k <= cut.y; ++k) x.add(p, (int64_t)256 * k + r, d0);
  x.write(p, cut.z + (r >> p.head_shift), r & (p.heads - 1), d0);
}

// Shared calls: every token, its prefix's parts and its own.  Block (16 rows, 128 columns).
__global__ void __launch_bounds__(128) join_tokens_kernel(const Params p) {
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  const int64_t r = 16 * (int64_t)blockIdx.x + (threadIdx.x & 15);
  const int tok = (int)(r >> p.head_shift), d0 = 128 * blockIdx.y + 16 * (threadIdx.x >> 4);
  const int2* where = reinterpret_cast<const int2*>(p.cuts) + 2 * (int64_t)tok;
  const int2 pre = where[0], own = where[1];  // first and last pair of each
  if (tok < row_token(p, 0) || tok >= row_token(p, p.rows)) return;
  int r0 = 0, r1 = p.rows;  // rows with a prefix
  if (p.group_offsets != nullptr) {
    r0 = clampi(p.group_offsets[0], 0, p.rows);
    r1 = clampi(p.group_offsets[p.groups], r0, p.rows);
  }
  Joined<16> x;
  if (tok >= row_token(p, r0) && tok < row_token(p, r1))
#pragma unroll 2
    for (int c = max(pre.x, 0); c <= min(pre.y, p.pairs - 1); ++c) x.add(p, r + 128 * (int64_t)c, d0);
  const int64_t mine = r + (int64_t)p.tokens * p.heads;
#pragma unroll 2
  for (int c = max(own.x, 0); c <= min(own.y, p.pairs - 1); ++c) x.add(p, mine + 128 * (int64_t)c, d0);
  x.write(p, tok, (int)(r & (p.heads - 1)), d0);
}

}  // namespace dense
}  // namespace dsa
