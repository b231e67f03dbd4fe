// Sparse-MLA decode over the 8-bit latent cache.  For row b, head h and the selected slots k:
//     v[k]     = float(ckv_q8[k]) * ckv_scale[k / block]
//     z[h,k]   = sm_scale * (q_nope[b,h] . v[k] + q_pe[b,h] . kpe[k])
//     lse[b,h] = log2(sum_k exp(z[h,k]))
//     out[b,h] = bf16(sum_k softmax(z)[h,k] v[k])
//     weights[b,k] = sum_h softmax(z)[h,k]          (optional)
//
// The e4m3 rows go to the tensor cores as they lie in memory (tcgen05 kind::f8f6f4, exact
// products, fp32 accumulation), so nothing is converted on the way:
//   * a slot's scale is constant along its row, so it factors out of the score and moves from
//     the value into the probability: out = sum_k (p[k] scale[k]) ckv_q8[k];
//   * a query row times a power of two (its largest value then lies in [128, 256)) is split into
//     two e4m3 terms, q = hi + lo / 16: a bf16 value has 8 significant bits and a term holds 4,
//     so the split is exact down to 2^-14 of the row's largest value and off by at most
//     2^-21 of that below;
//   * p scale / u is split into three terms, P = t0 + t1 / 16 + t2 / 256, where u, the unit, is
//     the largest scale of the first tile, but 2^-100 at least (a tile of zero tokens has 2^-126),
//     raised when a later one passes it 16-fold.  P is 3.5 2^(x + log2(scale / u) - m) with a
//     running maximum m of x + log2(scale / u) that a value may pass by 2^7 before m is raised, so
//     that P stays within e4m3's 448 and O is hardly ever rescaled; a unit that rises lowers m by
//     as much.  Three terms round to 12 significant bits, and the third's smallest step is
//     2^-18.8 of a weight at m.  (Two terms, which allow 2^3, rescaled O in about half of the
//     tiles.)  The sum l of 2^(x - m) has no scale in it: m stays so high that no score passes it by
//     more than 2^96.  That costs bits only where a head's weight lies on scales below 2^-88 of the
//     unit, and then l is 2^88 or more, so that the third term's step is under 2^-106 u of the output.
//     Scales up to 2^100 are within range (q . ckv_q8, up to 2^26, is multiplied by the scale
//     before the query's unit).
// The terms are extra columns of the same MMA (N = 2 NH and 3 NH): an M = 128 MMA costs about
// the same from N = 16 to N = 64, so they are nearly free.
//
// A CTA takes one group of NH heads (16, or 32 for rows of more) of one row, or a 1/S share of
// that group's tiles.  A tile is 96 slots in three stages of 96 x (512 + 128) bytes for 16 heads
// (64-slot tiles were slower: a tile's fixed latencies are paid more often), and 128 slots in
// two stages for 32 heads, whose queries and probabilities leave no room for a third; its slots
// are the rows of the score MMA and a multiple of the PV's K = 32, gathered whole by TMA (the
// bf16 pools need two CTAs for a row).  Where a call has fewer units (rows x groups) than SMs,
// the S x G CTAs of a row form a cluster of up to eight: splits are merged through distributed
// shared memory, so that no partial result touches global memory, calls share no state and the
// sums have one order.  Otherwise at most one CTA per SM takes unit after unit, the gathers of
// the next one under the last one's end.
//
// What bounds it.  A tile of 16 heads needs 61 kB: 1.40 us a tile at 6.5 TB/s over 148 SMs, and
// 120 copies of ~20 cycles of the SM's TMA unit, 1.2 us.  Measured: 1.34 us a tile for a row
// alone on its SMs, 1.50 us, 6.0 TB/s, with 148 SMs at work (32 heads: 2.35 and 2.71 us).  Fixed
// cost: about 6 us a call, 2 us for each further unit of a CTA.  64 rows of 16 heads and 2048
// slots: 26.8 us (3.2 TB/s of the 87 MB that they need; the bf16 kernel 42.5); 256 ragged rows: 76.7
// us (44 tiles on the busiest SM, 28 on average); 32 rows of 128 heads: 49.9 us (each slot is
// gathered by four groups, three of them from L2; the bf16 kernel 58.4); one row in eight splits:
// 12.8 us.
//
// Per CTA (512 threads):
//   warps 0-4    gather producers, one per 128-byte column block of the slots
//   warp 5       score issuer: S^T[96 or 128 slots x (hi, lo, pe)], 16 f8 + 4 bf16 MMAs
//   warp 6       PV issuer: O^T[512 x 3 terms] += V^T P^T, 12 f8 MMAs (16 for 128 slots; V^T read
//                in place)
//   warp 7       keeper: the slots of every tile with a valid entry, their scales and validity, and
//                where the row's padding begins.  (Gatherers that each looked the slots up for
//                themselves: 256 ragged rows 90.5 us, 64 rows 28.1, 32 rows of 128 heads 54.8.)
//   warps 8-15   softmax: warp w reads TMEM lanes 32 (w % 4) .. (slots) and half of the heads
#pragma once

namespace dsa {
namespace q8 {

struct AttendParams {
  const __nv_bfloat16* qn;
  int64_t qn_sb, qn_sh;
  const __nv_bfloat16* qp;
  int64_t qp_sb, qp_sh;
  Cache cache;
  const int32_t* idx;
  int64_t idx_sb;
  PageTable table;  // pt == nullptr: idx holds slot ids
  __nv_bfloat16* out;
  int64_t out_sb, out_sh;
  float* lse;
  int64_t lse_sb, lse_sh;
  float* weights;
  int64_t w_sb;
  float* scores;    // weights only: every tile's scores, [place][tile][NH][kTS]; a unit's place is
                    // its number if clustered, else its CTA's
  int32_t* tiles;   // weights only: the tiles a CTA ran, in the places of its scores
  int32_t topk;
  int32_t ntiles;
  int64_t units;    // rows x G
  int32_t splits;   // S
  int32_t groups;   // G, a power of two
  int32_t clustered;  // one unit per CTA, the S G CTAs of a row in a cluster; else CTA c takes
                      // the units c, c + grid, ...
  bool out8;        // output rows are 8-byte aligned
  float scale_log2;
  uint32_t* err;
  uint64_t wait_cycles;
};

constexpr int kBlocks = 5;            // 128-byte column blocks of a slot: four of ckv, one of kpe
constexpr int kMaxStages = 3;
constexpr int kLists = 4;             // tiles whose slots the keeper may hand out ahead
enum : int { kTile, kUnitEnd, kDone };  // what a list stands for
constexpr int kThreads = 512;
constexpr int kProdWarps = 5;
constexpr int kScore = 5, kPv = 6, kKeeper = 7, kSm0 = 8;
constexpr int kSmWarps = 8, kSmThreads = 256;
constexpr uint32_t kSmBar = 1;  // all softmax warps; + 2 + half: those of a half of the heads
constexpr float kTauQ8 = 7.f;         // log2: how far a weighted score may pass the running maximum
constexpr float kTauL = 96.f;         // the same for a score alone: the sum of 2^31 stays finite
constexpr float kTauU = 16.f;         // how far a scale may pass the unit
constexpr float kUnitMin = 7.888609e-31f;  // 2^-100, the smallest unit: its inverse is finite, and u / L
                                           // of a sum L up to 2^24 keeps its bits
constexpr float kNone = -3e38f;       // running maximum before the first score
constexpr float kPScale = 3.5f;       // P <= 3.5 * 2^7 = 448, the largest e4m3 value
constexpr int kMaxCluster = 8;
constexpr uint32_t kRise = 1u, kFailed = 2u;  // vote words
constexpr uint32_t kSw32 = 6;         // UMMA descriptor layout type: 32-byte swizzle

template <int NH>
struct Cfg {
  static_assert(NH == 16 || NH == 32, "head group width");
  static constexpr int kTS = NH == 16 ? 96 : 128;  // slots per tile
  static constexpr int kStages = NH == 16 ? 3 : 2;
  static constexpr int kQuads = kTS / 32;          // TMEM lane quadrants that hold slots
  static constexpr int kRB = kTS * 128;            // one block's region of a stage
  static constexpr int kStageB = kBlocks * kRB;
  static constexpr int kHT = NH / 2;               // heads per softmax thread
  static constexpr int kPBufs = 2;
  static constexpr int kQBlk = 2 * NH * 128;       // one 128-wide block of Q, hi rows then lo rows
  static constexpr int kPK = 3 * NH * 32;          // P^T, 32 slots of it: rows of 32 bytes
  static constexpr int kPB = kTS / 32 * kPK;
  static constexpr int OFF_Q = kStages * kStageB;
  static constexpr int OFF_QP = OFF_Q + 4 * kQBlk;
  static constexpr int OFF_P = OFF_QP + NH * 128;
  static constexpr int OFF_BAR = OFF_P + kPBufs * kPB;
  static constexpr int OFF_MISC = OFF_BAR + 256;   // [0] TMEM base, [2] abort, [3] drain, [4..7] what
                                                   // the lists of slots stand for
  static constexpr int OFF_CMD = OFF_MISC + 32;    // [stage][8]: validity words; [4] the tile (-1: end)
  static constexpr int OFF_SMAX = OFF_CMD + kStages * 32;  // [stage] largest scale of the tile
  static constexpr int OFF_QS = OFF_SMAX + 16;     // [NH] score units per query row
  static constexpr int OFF_SC = OFF_QS + NH * 4;   // [stage][kTS] scales; at the end kMl floats
  static constexpr int kMl = 2 * NH + 1;           // a CTA's m, L and u, for the merge
  static constexpr int OFF_RED = OFF_SC + kStages * kTS * 4;  // [half][2 buffers][4 warps] votes
  static constexpr int OFF_LSE = OFF_RED + 16 * 4;  // [NH], for the weights
  static constexpr int OFF_LIST = OFF_LSE + NH * 4;  // [kLists][kTS] the slots to gather
  static constexpr int SMEM_BYTES = OFF_LIST + kLists * kTS * 4;
  static_assert(OFF_LIST % 16 == 0, "slots are read four at a time");
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
  static_assert(kMl <= kStages * kTS, "m, L and u in the scales' place");
  // after the last tile, in the stages' place: this CTA's O, then the merge's table
  static constexpr int OFF_O = 0;
  static constexpr int OFF_COEF = NH * kDCkv * 4;  // [split][NH], then lse [NH]
  static_assert(OFF_COEF + (kMaxCluster + 1) * NH * 4 <= kStages * kStageB, "merge table");
  static constexpr int kSCols = 3 * NH;            // a score buffer: hi, lo, pe
  static constexpr int kSBufs = NH == 16 ? 2 : 1;  // as many as fit beside O
  static constexpr int O_COL = kSBufs * kSCols;    // four 128-row tiles of O^T, 3 NH columns each
  static constexpr int TMEM_COLS = 512;
  static_assert(O_COL + 12 * NH <= TMEM_COLS, "tensor memory");
};

enum : int {
  B_KVF = 0,                 // [stage] slots landed, scales, validity and tile number written
  B_KVE = B_KVF + kMaxStages,   // [stage] free again: PV done, and its words read by score and softmax
  B_SF = B_KVE + kMaxStages,    // [2] score written
  B_SE = B_SF + 2,           // [2] score read
  B_PF = B_SE + 2,           // [2] P written (and O rescaled)
  B_PD = B_PF + 2,           // [2] PV done
  B_QF = B_PD + 2,           // a unit's queries staged
  B_LF = B_QF + 1,           // [kLists] slots listed
  B_LE = B_LF + kLists,      // [kLists] list read by all gatherers
  B_DRAIN = B_LE + kLists,   // [2] used only when an issuer stops early
  B_COUNT = B_DRAIN + 2
};
static_assert(B_COUNT * 8 <= 256, "barrier block");

// Byte b of row r of an operand with 32-byte rows and the 32-byte swizzle.
__device__ __forceinline__ uint32_t sw32_byte(int r, int b) {
  return (uint32_t)(r * 32 + ((((b >> 4) ^ (r >> 2)) & 1) << 4) + (b & 15));
}

// Instruction descriptor, kind::f8f6f4: e4m3 A and B, fp32 D.
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N, bool a_mn_major) {
  return (1u << 4) | ((a_mn_major ? 1u : 0u) << 15) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// Read-only loads that are issued where they stand (the compiler sinks plain ones past the
// gathers, to where the value is used).
__device__ __forceinline__ int ldg_now(const int* p) {
  int v;
  asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float ldg_now(const float* p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}

// Byte b of row r of an operand with 128-byte rows and the 128-byte swizzle.
__device__ __forceinline__ uint32_t sw128_byte(int r, int b) {
  return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + (((b >> 4) ^ (r & 7)) << 4) + (b & 15));
}

// The units, (row, head group) pairs, of this CTA.
struct Units {
  int64_t first, step;
  int shift;  // log2(G)
  __device__ __forceinline__ explicit Units(const AttendParams& p) {
    shift = __ffs(p.groups) - 1;
    const unsigned per = (unsigned)(p.splits * p.groups);
    first = p.clustered ? (int64_t)(blockIdx.x / per) * p.groups + blockIdx.x % per / (unsigned)p.splits
                        : (int64_t)blockIdx.x;
    step = p.clustered ? p.units : (int64_t)gridDim.x;
  }
};

// ---------------------------------------------------------------- index entries
//
// The slots that a lane's kN entries of a tile name, fetched ahead: entries three tiles, pages (of
// a paged call) two.  -1: padding, -2: names no slot.
template <int kN, int kTS>
struct Entries {
  const AttendParams& p;
  const int32_t* ir;
  int64_t row;
  const int first, step;  // this lane: entries first + step e of a tile
  int pos2[kN], slot1[kN], slot0[kN];

  __device__ __forceinline__ void load(int64_t t, int (&pos)[kN], bool has) const {
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const int64_t k = t * kTS + first + step * e;
      pos[e] = has && k < p.topk ? ldg_now(ir + k) : -1;
    }
  }
  __device__ __forceinline__ void translate(const int (&pos)[kN], int (&slot)[kN]) const {
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      if (pos[e] == -1) slot[e] = -1;
      else if (p.table.pt != nullptr) slot[e] = slot_at(p.table, row, pos[e], p.cache.num_slots);
      else slot[e] = pos[e] >= 0 && pos[e] < p.cache.num_slots ? pos[e] : -1;
      if (slot[e] < 0 && pos[e] != -1) slot[e] = -2;
    }
  }
  __device__ __forceinline__ Entries(const AttendParams& prm, int f, int s)
      : p(prm), ir(nullptr), row(0), first(f), step(s) {}
  __device__ __forceinline__ void start(int64_t r, int64_t t, bool has) {
    row = r;
    ir = p.idx + r * p.idx_sb;
    int a[kN], b[kN];
    load(t, a, has);
    load(t + p.splits, b, has);
    load(t + 2 * p.splits, pos2, has);
    translate(a, slot0);
    translate(b, slot1);
  }
  // What tile t + 2 S and t + 3 S need, to be in slot0 two and three advances from now.
  int slot2[kN], pos3[kN];
  __device__ __forceinline__ void prefetch(int64_t t, bool has) {
    translate(pos2, slot2);
    load(t + 3 * p.splits, pos3, has);
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      slot0[e] = slot1[e];
      slot1[e] = slot2[e];
      pos2[e] = pos3[e];
    }
  }
};

// ---------------------------------------------------------------- gather producers
//
// Warp j < 5 gathers column block j of every slot of a tile, four slots a copy, from the list that
// the keeper (warp 7) hands out for every tile with a valid entry.  One elected thread issues the
// copies of a warp-uniform loop: 1,650 cycles a tile for the five warps, against 2,200 when
// each lane issues its own (and 8,000 from one warp), so that HBM and not the issue is the limit.
template <int NH>
__device__ __forceinline__ void produce(const AttendParams& p, const CUtensorMap* map, int blk,
                                        uint32_t sbase, uint8_t* sgen, const Waiter& wait) {
  using C = Cfg<NH>;
  constexpr int kTS = C::kTS, kStages = C::kStages, kRB = C::kRB, kStageB = C::kStageB;
  const uint32_t bar0 = sbase + (uint32_t)C::OFF_BAR;
  auto bar = [&](int k) { return bar0 + 8u * (uint32_t)k; };
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(sgen + C::OFF_MISC);
  const int col = blk < 4 ? 128 * blk : 0;
  const bool el = ptx::elect_one();
  const uint64_t policy = ptx::policy_evict_first();
  bool ok = true;
  int64_t n = 0;  // stages filled, lists read
  int st = 0;
  uint32_t phase = 0;
  for (;; ++n) {
    const int l = (int)(n % kLists);
    ok = __all_sync(0xffffffffu, wait(bar(B_LF + l), (uint32_t)((n / kLists) & 1)));
    if (!ok) break;
    const int what = (int)misc[4 + l];
    if (what == kDone) break;
    ok = __all_sync(0xffffffffu, wait(bar(B_KVE + st), phase ^ 1u));
    if (!ok) break;
    const uint32_t full = bar(B_KVF + st);
    if (what == kTile) {
      const int4* slots = reinterpret_cast<const int4*>(sgen + C::OFF_LIST) + l * (kTS / 4);
      const uint32_t dst = sbase + (uint32_t)(st * kStageB + blk * kRB);
      if (el) ptx::mbar_arrive_expect_tx(full, (uint32_t)kRB);
      // a slot that is none lies outside the tensor map: the copy fills its row with zeros, so
      // that PV reads 0 * 0 there
#pragma unroll
      for (int g = 0; g < kTS / 4; ++g) {
        const int4 s = slots[g];
        if (el) ptx::tma_gather4(dst + (uint32_t)(g * 512), map, col, s, full, policy);
      }
    } else if (el) {
      ptx::mbar_arrive(full);  // the unit's end: a stage without slots
    }
    __syncwarp();
    if (el) ptx::mbar_arrive(bar(B_LE + l));
    if (++st == kStages) {
      st = 0;
      phase ^= 1u;
    }
  }
  if (!ok && el) {
    // this warp's copies land before the CTA leaves
    const Waiter drain{misc + 3, p.err, p.wait_cycles};
    for (int64_t i = n - 1; i >= 0 && i >= n - kStages; --i)
      drain(bar(B_KVF + (int)(i % kStages)), (uint32_t)((i / kStages) & 1));
  }
  __syncwarp();
}

// Where a row's padding begins: behind its last entry that is not -1.  The last 512 entries
// are fetched ahead of their use; a row that is padding there is searched towards its front,
// 2048 entries a step.
struct Tail {
  const int topk, lane;
  int last[16];
  __device__ __forceinline__ Tail(const AttendParams& p, int l) : topk(p.topk), lane(l) {}
  __device__ __forceinline__ void load(const int32_t* ir) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int k = topk - 512 + 32 * i + lane;
      last[i] = k >= 0 ? ldg_now(ir + k) : -1;
    }
  }
  __device__ __forceinline__ int end(const int32_t* ir) const {
    int e = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (last[i] != -1) e = topk - 512 + 32 * i + lane + 1;
    e = __reduce_max_sync(0xffffffffu, e);
    for (int hi = topk - 512; hi > 0 && e == 0; hi -= 2048) {
#pragma unroll 32
      for (int i = 0; i < 64; ++i) {
        const int k = hi - 2048 + 32 * i + lane;
        if (k >= 0 && __ldg(ir + k) != -1) e = k + 1;
      }
      e = __reduce_max_sync(0xffffffffu, e);
    }
    return e;
  }
};

// The keeper (warp 7).  Tile by tile, lane l the entries l, l + 32, ...: the slots for the gatherers,
// scales, validity and the tile's number; tiles without a valid entry are passed over, and at
// a unit's first of them it looks where the row's padding begins, so that a short row's
// padding is not walked.
template <int NH>
__device__ __forceinline__ void keep_books(const AttendParams& p, const Units& units, int split,
                                           int lane, uint32_t sbase, uint8_t* sgen,
                                           const Waiter& wait) {
  using C = Cfg<NH>;
  constexpr int kTS = C::kTS, kStages = C::kStages, kE = C::kQuads;
  const uint32_t bar0 = sbase + (uint32_t)C::OFF_BAR;
  auto bar = [&](int k) { return bar0 + 8u * (uint32_t)k; };
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(sgen + C::OFF_MISC);
  volatile int* cmd = reinterpret_cast<volatile int*>(sgen + C::OFF_CMD);
  volatile float* smax = reinterpret_cast<volatile float*>(sgen + C::OFF_SMAX);
  float* sc = reinterpret_cast<float*>(sgen + C::OFF_SC);
  bool ok = true;
  int st = 0;
  uint32_t phase = 0;
  int64_t lists = 0;  // handed out
  Entries<kE, kTS> in(p, lane, 32);
  Tail tail(p, lane);
  auto hand_out = [&](int what) {
    const int l = (int)(lists % kLists);
    ok = __all_sync(0xffffffffu, wait(bar(B_LE + l), (uint32_t)(((lists / kLists) & 1) ^ 1)));
    if (!ok) return;
    if (what == kTile) {
      int* slots = reinterpret_cast<int*>(sgen + C::OFF_LIST) + l * kTS;
#pragma unroll
      for (int e = 0; e < kE; ++e) slots[32 * e + lane] = in.slot0[e];
    }
    if (lane == 0) misc[4 + l] = (uint32_t)what;
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar(B_LF + l));
    ++lists;
  };
  in.start(units.first >> units.shift, split, true);
  for (int64_t un = units.first; ok && un < p.units; un += units.step) {
    int end = p.ntiles;
    bool scanned = false;
    for (int64_t t = split; t < end; t += p.splits) {
      uint32_t w[kE], any = 0;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        w[e] = __ballot_sync(0xffffffffu, in.slot0[e] >= 0);
        any |= w[e];
      }
      if (any != 0u) {
        hand_out(kTile);
        if (!ok) break;
      }
      // not before the call's first list; a later unit's are on the way before its first tile
      if (un == units.first && t == split) tail.load(in.ir);
      float scale[kE], big = 0.f;
      bool bad = false;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const int slot = in.slot0[e];
        bad |= slot == -2;
        scale[e] = slot >= 0 ? ldg_now(p.cache.scale + (slot >> p.cache.block_shift)) : 0.f;
      }
      if (bad) atomicOr(p.err, (uint32_t)DSA_DEVERR_BAD_INDEX);
      in.prefetch(t, true);
      if (any != 0u) {
        ok = __all_sync(0xffffffffu, wait(bar(B_KVE + st), phase ^ 1u));
        if (!ok) break;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          sc[st * kTS + 32 * e + lane] = scale[e];
          big = fmaxf(big, fabsf(scale[e]));
        }
        big = ptx::warp_max(big);
        if (lane == 0) {
#pragma unroll
          for (int e = 0; e < kE; ++e) cmd[8 * st + e] = (int)w[e];
          cmd[8 * st + 4] = (int)t;
          smax[st] = big;
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(B_KVF + st));
        if (++st == kStages) {
          st = 0;
          phase ^= 1u;
        }
      }
      if (any == 0u && !scanned) {
        scanned = true;
        end = (tail.end(in.ir) + kTS - 1) / kTS;
      }
      in.advance();
    }
    if (!ok) break;
    if (un + units.step < p.units) {
      in.start((un + units.step) >> units.shift, split, true);
      tail.load(in.ir);
    }
    hand_out(kUnitEnd);
    if (!ok) break;
    ok = __all_sync(0xffffffffu, wait(bar(B_KVE + st), phase ^ 1u));
    if (ok && lane == 0) {
      cmd[8 * st + 4] = -1;
      ptx::mbar_arrive(bar(B_KVF + st));
    }
    if (++st == kStages) {
      st = 0;
      phase ^= 1u;
    }
  }
  if (ok) hand_out(kDone);
  __syncwarp();
}

// One query head into shared memory: hi and lo rows of q_nope in e4m3, the q_pe row in bf16.
// Returns the head's score unit: (hi + lo / 16) * unit is in log2 units.  A row with an
// infinity or a NaN has the unit NaN, which reaches every one of its scores.
struct Query {
  uint4 nope[2], pe;  // this lane's sixteen values, and eight (lanes 0 .. 7)
  __device__ __forceinline__ void load(const AttendParams& p, int64_t row, int head, int lane) {
    const uint4* src = reinterpret_cast<const uint4*>(p.qn + row * p.qn_sb + head * p.qn_sh) + 2 * lane;
    nope[0] = __ldg(src);
    nope[1] = __ldg(src + 1);
    pe = make_uint4(0u, 0u, 0u, 0u);
    if (lane < 8) pe = __ldg(reinterpret_cast<const uint4*>(p.qp + row * p.qp_sb + head * p.qp_sh) + lane);
  }
};
template <int NH>
__device__ __forceinline__ float stage_query(const Query& in, float scale_log2, int h, int lane,
                                             uint8_t* sgen) {
  using C = Cfg<NH>;
  const uint4 (&raw)[2] = in.nope;
  const uint4 pe = in.pe;
  float f[16], g[8];
  unpack8(raw[0], *reinterpret_cast<float(*)[8]>(f));
  unpack8(raw[1], *reinterpret_cast<float(*)[8]>(f + 8));
  unpack8(pe, g);
  float big = 0.f;
  bool fine = true;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    big = fmaxf(big, fabsf(f[i]));
    fine = fine && fabsf(f[i]) <= 3.402823466e38f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) fine = fine && fabsf(g[i]) <= 3.402823466e38f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  fine = __all_sync(0xffffffffu, fine);
  // 2^e <= big < 2^(e + 1); times 2^(7 - e), with e kept where both powers are normal
  int e = (int)(__float_as_uint(big) >> 23) - 127;
  e = e < -118 ? -118 : e;
  const float mul = __uint_as_float((uint32_t)(127 + 7 - e) << 23);
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi[i] = lo[i] = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float a = f[4 * i + 2 * k] * mul, b = f[4 * i + 2 * k + 1] * mul;
      const uint32_t t = to_e4m3x2(a, b);
      const float2 back = from_e4m3x2(t);
      hi[i] |= t << (16 * k);
      lo[i] |= to_e4m3x2((a - back.x) * 16.f, (b - back.y) * 16.f) << (16 * k);
    }
  }
  uint8_t* q = sgen + C::OFF_Q + (lane >> 3) * C::kQBlk;
  *reinterpret_cast<uint4*>(q + sw128_byte(h, 16 * (lane & 7))) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  *reinterpret_cast<uint4*>(q + sw128_byte(NH + h, 16 * (lane & 7))) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  if (lane < 8) *reinterpret_cast<uint4*>(sgen + C::OFF_QP + sw128_byte(h, 16 * lane)) = pe;
  return fine ? __uint_as_float((uint32_t)(127 + e - 7) << 23) * scale_log2 : NAN;
}

template <int kN>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t* r) {
#pragma unroll
  for (int c = 0; c < kN; c += 8) ptx::tmem_ld8(addr + (uint32_t)c, r + c);
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
        "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 pair(const uint32_t* r, int i) {
  return make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
}
__device__ __forceinline__ float2 lds2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// log2(a / b) of positive normal numbers, also where the quotient is not one; a whole number for
// powers of two.
__device__ __forceinline__ float log2_ratio(float a, float b) {
  const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
  const float ma = __uint_as_float((ua & 0x7FFFFFu) | 0x3F800000u);
  const float mb = __uint_as_float((ub & 0x7FFFFFu) | 0x3F800000u);
  return (float)((int)(ua >> 23) - (int)(ub >> 23)) + (ptx::lg2(ma) - ptx::lg2(mb));
}

// An entry's probability summed over the heads, from its scores (kTS apart) and their lse.
template <int NH>
__device__ __forceinline__ float head_sum(const float* scores, const float* lse) {
  constexpr int kB = 16;  // scores on the way at a time
  float w = 0.f;
#pragma unroll
  for (int h0 = 0; h0 < NH; h0 += kB) {
    float x[kB];
#pragma unroll
    for (int h = 0; h < kB; ++h) x[h] = __ldcg(scores + (h0 + h) * Cfg<NH>::kTS);
#pragma unroll
    for (int h = 0; h < kB; ++h) w += x[h] == -INFINITY ? 0.f : ptx::ex2(x[h] - lse[h0 + h]);
  }
  return w;
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <int NH>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(const __grid_constant__ CUtensorMap tm_ckv,
                  const __grid_constant__ CUtensorMap tm_kpe, const __grid_constant__ AttendParams p) {
  using C = Cfg<NH>;
  constexpr int kHT = C::kHT, kQuads = C::kQuads;
  constexpr int kTS = C::kTS, kStages = C::kStages, kRB = C::kRB, kStageB = C::kStageB;
  extern __shared__ __align__(1024) uint8_t smem_raw[];  // swizzle atoms are 1024 bytes
  const uint32_t sbase = ptx::smem_u32(smem_raw);
  uint8_t* sgen = smem_raw;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(sgen + C::OFF_MISC);
  volatile int* cmd = reinterpret_cast<volatile int*>(sgen + C::OFF_CMD);
  const uint32_t bar0 = sbase + (uint32_t)C::OFF_BAR;
  auto bar = [&](int k) { return bar0 + 8u * (uint32_t)k; };

  const int S = p.splits, G = p.groups;
  const Units units(p);
  const int split = p.clustered ? (int)(blockIdx.x % (unsigned)S) : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(bar(B_KVF + s), kProdWarps + 1);  // the gatherers (with their bytes) and the keeper
      ptx::mbar_init(bar(B_KVE + s), 3);  // PV, score issuer, softmax
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(bar(B_SF + b), 1);
      ptx::mbar_init(bar(B_SE + b), kSmWarps);  // one arrive per softmax warp
      ptx::mbar_init(bar(B_PF + b), kSmWarps);
      ptx::mbar_init(bar(B_PD + b), 1);
      ptx::mbar_init(bar(B_DRAIN + b), 1);
    }
    misc[2] = 0;
    misc[3] = 0;
    ptx::mbar_init(bar(B_QF), kSmWarps);
    for (int l = 0; l < kLists; ++l) {
      ptx::mbar_init(bar(B_LF + l), 1);
      ptx::mbar_init(bar(B_LE + l), kProdWarps);
    }
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tm_ckv);
    ptx::prefetch_tmap(&tm_kpe);
  }
  if (warp == kScore) {
    ptx::tmem_alloc(sbase + (uint32_t)C::OFF_MISC, (uint32_t)C::TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = misc[0];
  ptx::grid_dep_wait();
  ptx::launch_dependents();
  const Waiter wait{misc + 2, p.err, p.wait_cycles};
  const Waiter spin{misc + 2, p.err, p.wait_cycles, true};

  // softmax state, kept past the loop for the merge of a clustered call's single unit
  const int qd = warp & 3;                   // TMEM lane quadrant: slots 32 qd .. 32 qd + 31
  const int hh = (warp - kSm0) >> 2;         // heads kHT hh .. kHT hh + kHT - 1 of the group
  const uint32_t lane_base = (uint32_t)(32 * qd) << 16;
  float2 m_neg[kHT / 2], l_part[kHT / 2];    // per head: minus the running maximum, and its sum
  float u = 0.f;                             // the unit of the scales
  int64_t row = 0;
  int group = 0;
  int live = 0;                              // the unit's tiles
  float* ml = reinterpret_cast<float*>(sgen + C::OFF_SC);
  bool aborted = false;

  if (warp < kProdWarps)
    produce<NH>(p, warp < 4 ? &tm_ckv : &tm_kpe, warp, sbase, sgen, wait);
  else if (warp == kKeeper)
    keep_books<NH>(p, units, split, lane, sbase, sgen, wait);
  if (warp == kScore) {
    // ------------------------------------------------------------------ score issuer
    constexpr uint32_t kId = idesc_e4m3(128, 2 * NH, false), kIdPe = idesc_bf16(128, NH, false);
    const uint64_t dk = desc(sbase, 16, 1024, kSw128);
    const uint64_t dq = desc(sbase + (uint32_t)C::OFF_Q, 16, 1024, kSw128);
    const uint64_t dqp = desc(sbase + (uint32_t)C::OFF_QP, 16, 1024, kSw128);
    const bool el = ptx::elect_one();  // warp-uniform loops around one issuing thread
    bool ok = true;
    int64_t c = 0, i = 0;  // stages, tiles
    for (int64_t un = units.first, k = 0; ok && un < p.units; un += units.step, ++k) {
      ok = __all_sync(0xffffffffu, spin(bar(B_QF), (uint32_t)(k & 1)));
      for (; ok; ++i) {
        const int st = (int)(c % kStages), sb = (int)(i % C::kSBufs);
        ok = __all_sync(0xffffffffu, wait(bar(B_KVF + st), (uint32_t)((c / kStages) & 1)));
        if (!ok) break;
        const bool end = __any_sync(0xffffffffu, cmd[8 * st + 4] < 0);
        if (el) ptx::mbar_arrive(bar(B_KVE + st));
        ++c;
        if (end) break;
        ok = __all_sync(0xffffffffu, spin(bar(B_SE + sb), (uint32_t)(((i / C::kSBufs) & 1) ^ 1)));
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(C::kSCols * sb);
        const uint64_t ko = (uint64_t)((st * kStageB) >> 4);
        if (el) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              ptx::umma_f8(d, dk + ko + (uint64_t)((j * kRB + ks * 32) >> 4),
                           dq + (uint64_t)((j * C::kQBlk + ks * 32) >> 4), kId, (j | ks) ? 1u : 0u);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            ptx::umma_bf16(d + 2 * NH, dk + ko + (uint64_t)((4 * kRB + ks * 32) >> 4),
                           dqp + (uint64_t)((ks * 32) >> 4), kIdPe, ks ? 1u : 0u);
          ptx::umma_commit(bar(B_SF + sb));
        }
        __syncwarp();
      }
    }
    if (!ok && el) {
      const Waiter drain{misc + 3, p.err, p.wait_cycles};
      ptx::umma_commit(bar(B_DRAIN));
      drain(bar(B_DRAIN), 0);
    }
    __syncwarp();
  } else if (warp == kPv) {
    // ------------------------------------------------------------------ PV issuer
    constexpr uint32_t kId = idesc_e4m3(128, 3 * NH, true);
    const uint64_t dv = desc(sbase, kRB, 1024, kSw128);
    const uint64_t dp = desc(sbase + (uint32_t)C::OFF_P, 16, 256, kSw32);
    const bool el = ptx::elect_one();
    bool ok = true;
    int64_t c = 0, i = 0;  // stages, tiles
    for (int64_t un = units.first; ok && un < p.units; un += units.step) {
      for (bool first = true; ok; ++i, first = false) {
        const int st = (int)(c % kStages), pb = (int)(i & 1);
        ok = __all_sync(0xffffffffu, spin(bar(B_KVF + st), (uint32_t)((c / kStages) & 1)));
        if (!ok) break;
        ++c;
        if (__any_sync(0xffffffffu, cmd[8 * st + 4] < 0)) {
          if (el) ptx::mbar_arrive(bar(B_KVE + st));
          break;
        }
        ok = __all_sync(0xffffffffu, spin(bar(B_PF + pb), (uint32_t)((i >> 1) & 1)));
        if (!ok) break;
        ptx::tc_fence_after();
        const uint64_t vo = (uint64_t)((st * kStageB) >> 4);
        const uint64_t po = (uint64_t)(((int)(i % C::kPBufs) * C::kPB) >> 4);
        if (el) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int ks = 0; ks < kTS / 32; ++ks)
              ptx::umma_f8(tmem + (uint32_t)(C::O_COL + 3 * NH * j),
                           dv + vo + (uint64_t)((j * kRB + ks * 4096) >> 4),
                           dp + po + (uint64_t)((ks * C::kPK) >> 4), kId, (!first || ks > 0) ? 1u : 0u);
          ptx::umma_commit(bar(B_KVE + st));
          ptx::umma_commit(bar(B_PD + pb));
        }
        __syncwarp();
      }
    }
    if (!ok && el) {
      const Waiter drain{misc + 3, p.err, p.wait_cycles};
      ptx::umma_commit(bar(B_DRAIN + 1));
      drain(bar(B_DRAIN + 1), 0);
    }
    __syncwarp();
  } else if (warp >= kSm0) {
    // ------------------------------------------------------------------ softmax
    const int slot = 32 * qd + lane;
    const bool slot_ok = slot < kTS;  // the other quadrants' lanes are only rows of O
    const float* sc = reinterpret_cast<const float*>(sgen + C::OFF_SC);
    const volatile float* smax = reinterpret_cast<const volatile float*>(sgen + C::OFF_SMAX);
    const int sm_tid = (int)threadIdx.x - 32 * kSm0;
    int64_t c = 0, n = 0;  // stages, tiles
    for (int64_t un = units.first; un < p.units; un += units.step) {
      row = un >> units.shift;
      group = (int)(un & (G - 1));
      const int h0 = group * NH;  // first head of the group
      // The score issuer has passed the unit before (also one without tiles, whose queries it
      // never used) once the end's stage is free.
      bool go = !aborted;
      if (go && c > 0) go = wait(bar(B_KVE + (int)((c - 1) % kStages)), (uint32_t)(((c - 1) / kStages) & 1));
      // The queries, into a buffer whose last reader, the previous unit's last score, is done.
      float* units_s = reinterpret_cast<float*>(sgen + C::OFF_QS);
      constexpr int kQH = NH / kSmWarps;
      Query query[kQH];
#pragma unroll
      for (int j = 0; j < kQH; ++j) query[j].load(p, row, h0 + warp - kSm0 + j * kSmWarps, lane);
#pragma unroll
      for (int j = 0; j < kQH; ++j) {
        const int h = warp - kSm0 + j * kSmWarps;
        const float unit = stage_query<NH>(query[j], p.scale_log2, h, lane, sgen);
        if (lane == 0) units_s[h] = unit;
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(B_QF));
      aborted = ptx::bar_red_or(kSmBar, kSmThreads, !go);
      // entries of tiles that turn out to hold nothing get no other weight (of a clustered row,
      // group g's CTA writes the tiles with (tile / S) % G == g, here and at the end)
      if (p.weights != nullptr)
        for (int64_t t = p.clustered ? split + S * group : 0; t < p.ntiles; t += p.clustered ? S * G : 1) {
          const int64_t at = t * kTS + sm_tid;
          if (sm_tid < kTS && at < p.topk) p.weights[row * p.w_sb + at] = 0.f;
        }
      // the heads' score units: in registers, or (32 heads) read from shared memory tile by tile
      const uint32_t qs_s = sbase + (uint32_t)(C::OFF_QS + 4 * kHT * hh);
      float2 qs[kHT / 2];
#pragma unroll
      for (int j = 0; j < kHT / 2; ++j) {
        m_neg[j] = both(-kNone);
        l_part[j] = both(0.f);
        if (NH == 16) qs[j] = lds2(qs_s + 8u * (uint32_t)j);
      }
      float u_inv = 0.f;
      u = 0.f;
      bool failed = false;  // a wait of this warp ran out: the next vote ends the loop for every thread
      for (live = 0; !aborted; ++live, ++n) {
        const int st = (int)(c % kStages), sb = (int)(n % C::kSBufs), pb = (int)(n & 1);
        bool ok = wait(bar(B_KVF + st), (uint32_t)((c / kStages) & 1));
        const int tile = cmd[8 * st + 4];
        const bool end = ok && tile < 0;
        if (!end) ok = ok && wait(bar(B_SF + sb), (uint32_t)((n / C::kSBufs) & 1));
        ++c;
        // The unit of the scales, the same in every thread: the first tile's largest scale, or a
        // later one's that passes it kTauU-fold.  It rises before a scale is divided by it, so that no
        // ratio passes kTauU (a scale of 2^30 over a unit of 2^-100 would not be finite).
        const float largest = smax[st];
        float grow = 0.f;  // log2(old unit / new unit)
        if (live == 0) {
          u = fmaxf(largest, kUnitMin);
          u_inv = 1.f / u;
        } else if (!end && largest > kTauU * u) {
          grow = log2_ratio(u, largest);
          u = largest;
          u_inv = 1.f / u;
        }
        float2 x[kHT / 2], d[kHT / 2];  // scores, and over the running maximum
        float ratio = 0.f;  // scale in units, lr its log2
        float lr = -INFINITY;
        bool valid = false;
        if (slot_ok && __all_sync(0xffffffffu, ok && !end)) {  // warp-uniform
          ptx::tc_fence_after();
          uint32_t hi[kHT], lo[kHT], pe[kHT];
          const uint32_t ta = tmem + lane_base + (uint32_t)(C::kSCols * sb + kHT * hh);
          tmem_ld<kHT>(ta, hi);
          tmem_ld<kHT>(ta + NH, lo);
          tmem_ld<kHT>(ta + 2 * NH, pe);
          const float scale = sc[st * kTS + slot];
          valid = ((uint32_t)cmd[8 * st + qd] >> lane) & 1u;
          ratio = scale * u_inv;
          lr = ptx::lg2(fabsf(ratio));
          ptx::tmem_wait_ld();
          ptx::tc_fence_before();
#pragma unroll
          for (int j = 0; j < kHT / 2; ++j) {
            const float2 q = fma2(pair(lo, j), both(0.0625f), pair(hi, j));
            x[j] = fma2(mul2(q, both(scale)), NH == 16 ? qs[j] : lds2(qs_s + 8u * (uint32_t)j),
                        mul2(pair(pe, j), both(p.scale_log2)));
          }
          if (!valid) {
#pragma unroll
            for (int j = 0; j < kHT / 2; ++j) x[j] = both(-INFINITY);
          }
        } else {
#pragma unroll
          for (int j = 0; j < kHT / 2; ++j) x[j] = both(-INFINITY);
        }
        __syncwarp();
        if (lane == 0 && !end) ptx::mbar_arrive(bar(B_SE + sb));
        // Whether a running maximum or the unit has to rise, or a wait failed, through one barrier
        // of the four warps that share the heads.  Their decisions are the same, as they read
        // the same words; the words are written again two tiles later, behind the next tile's
        // barrier.
        const float tau = fminf(kTauQ8 - lr, kTauL);  // P = 2^(x + lr - m) and l's 2^(x - m) in range
        float top = kNone;
#pragma unroll
        for (int j = 0; j < kHT / 2; ++j) {
          d[j] = add2(x[j], m_neg[j]);
          top = fmaxf(top, fmaxf(d[j].x, d[j].y));
        }
        uint32_t vote = __reduce_or_sync(0xffffffffu, (ok && !failed ? 0u : kFailed) | (top > tau ? kRise : 0u));
        uint32_t* words = reinterpret_cast<uint32_t*>(sgen + C::OFF_RED) + (hh * 2 + pb) * 4;
        if (lane == 0) words[qd] = vote;
        ptx::bar_sync(kSmBar + 2 + hh, kSmThreads / 2);
        {
          const uint4 v = *reinterpret_cast<const uint4*>(words);
          vote = v.x | v.y | v.z | v.w;
        }
        if (vote & kFailed) {
          aborted = true;
          break;
        }
        if (end) break;
        if (vote != 0u || grow != 0.f) {
          // Rare past the first tile: raise the maxima to this tile's, the unit to its largest
          // scale, and bring l and O to them.
          if (live > 0) {
            const bool wok = wait(bar(B_PD + (int)((n - 1) & 1)), (uint32_t)(((n - 1) >> 1) & 1));
            if (!__all_sync(0xffffffffu, wok)) failed = true;
            ptx::tc_fence_after();
          }
          // the maxima go through this tile's P buffer, whose last reader (PV) is done
          // (in the first term's rows of these heads, which only these warps write)
          float* tops = reinterpret_cast<float*>(sgen + C::OFF_P + (int)(n % C::kPBufs) * C::kPB + hh * kHT * 32);
          // A maximum is one of x + log2(scale / u): it falls with a unit that rises, unless that
          // would take l past 2^(kTauL - 8).
          const float over = fmaxf(lr, 8.f - kTauL);
#pragma unroll
          for (int h = 0; h < kHT; ++h) {
            float v = ((h & 1) ? x[h / 2].y : x[h / 2].x) + over;
            if (grow != 0.f) {
              const float l = (h & 1) ? l_part[h / 2].y : l_part[h / 2].x;
              v = fmaxf(v, ptx::lg2(l) - ((h & 1) ? m_neg[h / 2].y : m_neg[h / 2].x) + (8.f - kTauL));
            }
            v = ptx::warp_max(v);
            if (slot_ok && lane == 0) tops[qd * kHT + h] = v;
          }
          ptx::bar_sync(kSmBar + 2 + hh, kSmThreads / 2);
          float2 alpha[kHT / 2];
#pragma unroll
          for (int j = 0; j < kHT / 2; ++j) {
            const float2* t2 = reinterpret_cast<const float2*>(tops) + j;
            float2 mn = make_float2(grow - m_neg[j].x, grow - m_neg[j].y);
#pragma unroll
            for (int q = 0; q < kQuads; ++q) {
              const float2 t = t2[q * kHT / 2];
              mn = make_float2(fmaxf(mn.x, t.x), fmaxf(mn.y, t.y));
            }
            // l's factor is 2^(kTauL - 4) at most; O, in old units, takes the unit's growth beside it in
            // the exponent, where neither can overflow
            const float2 fall = make_float2(-m_neg[j].x - mn.x, -m_neg[j].y - mn.y);
            l_part[j] = mul2(l_part[j], make_float2(ptx::ex2(fall.x), ptx::ex2(fall.y)));
            alpha[j] = make_float2(ptx::ex2(fall.x + grow), ptx::ex2(fall.y + grow));
            m_neg[j] = make_float2(-mn.x, -mn.y);
            d[j] = add2(x[j], m_neg[j]);
          }
          ptx::bar_sync(kSmBar + 2 + hh, kSmThreads / 2);  // the buffer is P's again
          if (live > 0 && !failed) {
            // four tiles of O, three terms: kC loads in flight at a time
            constexpr int kC = NH == 16 ? 4 : 2;
#pragma unroll 1
            for (int c = 0; c < 12; c += kC) {
              const uint32_t ta = tmem + lane_base + (uint32_t)(C::O_COL + NH * c + kHT * hh);
              uint32_t r[kC][kHT];
#pragma unroll
              for (int b = 0; b < kC; ++b) tmem_ld<kHT>(ta + (uint32_t)(NH * b), r[b]);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int b = 0; b < kC; ++b) {
#pragma unroll
                for (int h = 0; h < kHT; ++h)
                  r[b][h] = __float_as_uint(__uint_as_float(r[b][h]) * ((h & 1) ? alpha[h / 2].y : alpha[h / 2].x));
#pragma unroll
                for (int k = 0; k < kHT; k += 8) ptx::tmem_st8(ta + (uint32_t)(NH * b + k), r[b] + k);
              }
            }
            ptx::tmem_wait_st();
          }
        }
        // P[n % kPBufs] was last read by the PV of tile n - kPBufs
        if (n >= C::kPBufs && !failed) {
          const int64_t j = n - C::kPBufs;
          const bool wok = wait(bar(B_PD + (int)(j & 1)), (uint32_t)((j >> 1) & 1));
          if (!__all_sync(0xffffffffu, wok)) failed = true;
        }
        if (failed) continue;
        if (slot_ok) {
          // byte (row r, slot) of P: 32-slot planes of 32-byte rows, 32-byte swizzle
          uint8_t* pbuf = sgen + C::OFF_P + (int)(n % C::kPBufs) * C::kPB + qd * C::kPK;
          const float2 scaled = both(ratio * kPScale);
#pragma unroll
          for (int j = 0; j < kHT / 2; ++j) {
            const float2 e = make_float2(ptx::ex2(d[j].x), ptx::ex2(d[j].y));
            l_part[j] = add2(l_part[j], e);
            float2 v = mul2(e, scaled);
            const int r = kHT * hh + 2 * j;
#pragma unroll
            for (int term = 0; term < 3; ++term) {
              const uint32_t b = to_e4m3x2(v.x, v.y);
              if (term < 2) v = fma2(from_e4m3x2(b), both(-16.f), mul2(v, both(16.f)));
              pbuf[sw32_byte(term * NH + r, lane)] = (uint8_t)b;
              pbuf[sw32_byte(term * NH + r + 1, lane)] = (uint8_t)(b >> 8);
            }
          }
          if (p.weights != nullptr) {
            const int64_t at = (p.clustered ? un : (int64_t)blockIdx.x) * p.ntiles + split + (int64_t)live * S;
            float* s = p.scores + (at * NH + kHT * hh) * kTS + slot;
#pragma unroll
            for (int j = 0; j < kHT / 2; ++j) {
              s[2 * j * kTS] = x[j].x;
              s[(2 * j + 1) * kTS] = x[j].y;
            }
            if (threadIdx.x == 32 * kSm0) p.tiles[at] = tile;
          }
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (warp == kSm0) ptx::mbar_arrive(bar(B_KVE + st));
          ptx::mbar_arrive(bar(B_PF + pb));
        }
      }
      // ------------------------------------------------------------------ the unit's end
      // PD of tile n - 3 (two P buffers) or n - 2 was waited for above, on the same barrier or
      // before, so this wait is exact
      bool ok = !aborted;
      if (ok && live > 0) ok = wait(bar(B_PD + (int)((n - 1) & 1)), (uint32_t)(((n - 1) >> 1) & 1));
      aborted = ptx::bar_red_or(kSmBar, kSmThreads, !ok);
      // every warp has read the end's words
      if (!aborted && threadIdx.x == 32 * kSm0) ptx::mbar_arrive(bar(B_KVE + (int)((c - 1) % kStages)));
      ptx::tc_fence_after();
      float* red = reinterpret_cast<float*>(sgen + C::OFF_P);  // [half][quadrant][kHT]
#pragma unroll
      for (int h = 0; h < kHT; ++h) {
        float v = (h & 1) ? l_part[h / 2].y : l_part[h / 2].x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0 && slot_ok) red[(hh * kQuads + qd) * kHT + h] = v;
      }
      ptx::bar_sync(kSmBar, kSmThreads);
      if (p.clustered) break;
      // A unit of its own: O^T / L from tensor memory to the output.  The next unit's first PV
      // comes after these reads, as it needs this warp's P.
      // Lane h of every warp computes head h's weight 1 / L; quadrant 0's also its lse.
      float mine = 0.f;
      float* lse_s = reinterpret_cast<float*>(sgen + C::OFF_LSE);
      if (lane < kHT) {
        float L = 0.f, m = 0.f;
#pragma unroll
        for (int q = 0; q < kQuads; ++q) L += red[(hh * kQuads + q) * kHT + lane];
        mine = aborted ? NAN : L == 0.f ? 0.f : 1.f / L * (u * (1.f / kPScale));  // as the merge rounds it
        if (qd == 0) {
#pragma unroll
          for (int h = 0; h < kHT; ++h) m = lane == h ? -((h & 1) ? m_neg[h / 2].y : m_neg[h / 2].x) : m;
          const float lse = aborted ? NAN : L == 0.f ? -INFINITY : m + ptx::lg2(L);
          lse_s[kHT * hh + lane] = lse;
          p.lse[row * p.lse_sb + (int64_t)(h0 + kHT * hh + lane) * p.lse_sh] = lse;
        }
      }
      __syncwarp();
      float coef[kHT];
#pragma unroll
      for (int h = 0; h < kHT; ++h) coef[h] = __shfl_sync(0xffffffffu, mine, h);
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        uint32_t r[3][kHT];
#pragma unroll
        for (int t = 0; t < 3; ++t)
          tmem_ld<kHT>(tmem + lane_base + (uint32_t)(C::O_COL + NH * (3 * j + t) + kHT * hh), r[t]);
        ptx::tmem_wait_ld();
        __nv_bfloat16* dst = p.out + row * p.out_sb + (int64_t)(h0 + kHT * hh) * p.out_sh + 128 * j + 32 * qd + lane;
#pragma unroll
        for (int h = 0; h < kHT; ++h) {
          const float o = fmaf(fmaf(__uint_as_float(r[2][h]), 0.0625f, __uint_as_float(r[1][h])), 0.0625f,
                               __uint_as_float(r[0][h]));
          // 0: no weight, whatever O holds (nothing was written to it without a live tile)
          dst[(int64_t)h * p.out_sh] = __float2bfloat16_rn(coef[h] == 0.f ? 0.f : o * coef[h]);
        }
      }
      ptx::tc_fence_before();
      if (p.weights != nullptr) {
        ptx::bar_sync(kSmBar, kSmThreads);  // lse; every tile's scores are behind the barriers above
        if (aborted) {
          for (int k2 = sm_tid; k2 < p.topk; k2 += kSmThreads) p.weights[row * p.w_sb + k2] = NAN;
        } else {
          for (int64_t e = sm_tid; e < (int64_t)live * kTS; e += kSmThreads) {
            const int64_t at = (int64_t)blockIdx.x * p.ntiles + e / kTS;
            const int64_t k2 = (int64_t)p.tiles[at] * kTS + e % kTS;
            if (k2 < p.topk)
              p.weights[row * p.w_sb + k2] = head_sum<NH>(p.scores + at * NH * kTS + e % kTS, lse_s);
          }
        }
      }
    }
    if (p.clustered) {
      const float* red = reinterpret_cast<const float*>(sgen + C::OFF_P);
      if (qd == 0 && lane < kHT) {
        float L = 0.f, m = 0.f;
#pragma unroll
        for (int q = 0; q < kQuads; ++q) L += red[(hh * kQuads + q) * kHT + lane];
#pragma unroll
        for (int h = 0; h < kHT; ++h) m = lane == h ? -((h & 1) ? m_neg[h / 2].y : m_neg[h / 2].x) : m;
        ml[kHT * hh + lane] = m;
        ml[NH + kHT * hh + lane] = L;
        if (lane == 0) ml[2 * NH] = u;
      }
      // O to shared memory, [head][512] (nothing was ever written to it without a live tile)
      float* o_s = reinterpret_cast<float*>(sgen + C::OFF_O);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t r[3][kHT];
#pragma unroll
        for (int c = 0; c < 3; ++c)
          tmem_ld<kHT>(tmem + lane_base + (uint32_t)(C::O_COL + NH * (3 * j + c) + kHT * hh), r[c]);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int h = 0; h < kHT; ++h) {
          const float o = fmaf(fmaf(__uint_as_float(r[2][h]), 0.0625f, __uint_as_float(r[1][h])), 0.0625f,
                               __uint_as_float(r[0][h]));
          o_s[(kHT * hh + h) * kDCkv + 128 * j + 32 * qd + lane] = live > 0 ? o : 0.f;
        }
      }
    }
  }
  __syncwarp();

  // -------------------------------------------------------------------- merge of the splits
  // Behind this barrier every CTA of the cluster has its m, L, u and O in shared memory.
  if (p.clustered) ptx::cluster_sync();
  bool lost = false;  // a wait ran out somewhere in the cluster: the row is written as NaN
  if (p.clustered && warp >= kSm0) {
    const int h0 = group * NH;
    const int sm_tid = (int)threadIdx.x - 32 * kSm0;
    float* coef = reinterpret_cast<float*>(sgen + C::OFF_COEF);
    float* lse_s = coef + S * NH;
    const int rank0 = group * S;  // the rank of split 0 of this group
    if (sm_tid < S * G)
      lost = __float_as_uint(ld_cluster(
                 ptx::mapa(sbase + (uint32_t)C::OFF_MISC + 8u, (uint32_t)sm_tid))) != 0u;
    // split s sums and writes the heads [s NH / S, (s + 1) NH / S), four values a thread at a
    // time: NH / 2 reads whatever S, under way while the coefficients are computed
    const int ss = __ffs(S) - 1;  // S is a power of two
    const int per = NH >> ss;
    float4 part[NH / 2];
#pragma unroll
    for (int i = 0; i < NH / 2; ++i) {
      const int e = sm_tid + kSmThreads * (i >> ss);  // value 4 e of the heads of this split
      part[i] = ld_cluster4(ptx::mapa(sbase + (uint32_t)(C::OFF_O + 4 * (split * per * kDCkv + 4 * e)),
                                      (uint32_t)(rank0 + (i & (S - 1)))));
    }
    // thread (head, split): the head's lse, and what a value of the split's O counts for in its
    // output; the S threads of a head are neighbours in a warp
    static_assert(NH * kMaxCluster <= kSmThreads, "a thread per head and split");
    const int h = sm_tid >> ss, s = sm_tid & (S - 1);
    float ms = 0.f, ls = 0.f, us = 0.f;
    if (sm_tid < NH * S) {
      const uint32_t at = ptx::mapa(sbase + (uint32_t)C::OFF_SC, (uint32_t)(rank0 + s));
      ms = ld_cluster(at + 4u * (uint32_t)h);
      ls = ld_cluster(at + 4u * (uint32_t)(NH + h));
      us = ld_cluster(at + 8u * NH);
    }
    lost = ptx::bar_red_or(kSmBar, kSmThreads, lost);
    if (sm_tid < NH * S) {
      float M = ms;
      for (int k = 1; k < S; k <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
      const float w = ls == 0.f ? 0.f : ptx::ex2(ms - M);
      float L = ls == 0.f ? 0.f : ls * w;
      for (int k = 1; k < S; k <<= 1) L += __shfl_xor_sync(0xffffffffu, L, k);
      coef[s * NH + h] = w == 0.f ? 0.f : w / L * (us * (1.f / kPScale));
      const float lse = lost ? NAN : L == 0.f ? -INFINITY : M + ptx::lg2(L);
      if (s == 0) {
        lse_s[h] = lse;
        if (split == 0) p.lse[row * p.lse_sb + (int64_t)(h0 + h) * p.lse_sh] = lse;
      }
    }
    ptx::bar_sync(kSmBar, kSmThreads);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NH / 2; ++i) {
      const int e = sm_tid + kSmThreads * (i >> ss);
      const int hl = split * per + e / (kDCkv / 4), d = 4 * (e % (kDCkv / 4));
      const float c = coef[(i & (S - 1)) * NH + hl];
      if (c != 0.f) {  // 0: no weight, whatever the values
        o.x = fmaf(part[i].x, c, o.x);
        o.y = fmaf(part[i].y, c, o.y);
        o.z = fmaf(part[i].z, c, o.z);
        o.w = fmaf(part[i].w, c, o.w);
      }
      if ((i & (S - 1)) != S - 1) continue;
      if (lost) o = make_float4(NAN, NAN, NAN, NAN);
      __nv_bfloat16* dst = p.out + row * p.out_sb + (int64_t)(h0 + hl) * p.out_sh + d;
      const __nv_bfloat162 a = __floats2bfloat162_rn(o.x, o.y), b = __floats2bfloat162_rn(o.z, o.w);
      if (p.out8) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                                    *reinterpret_cast<const uint32_t*>(&b));
      } else {
        dst[0] = a.x;
        dst[1] = a.y;
        dst[2] = b.x;
        dst[3] = b.y;
      }
      o = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (p.weights != nullptr && lost) {
      for (int t = split + S * group; t < p.ntiles; t += S * G) {
        const int64_t k = (int64_t)t * kTS + sm_tid;
        if (sm_tid < kTS && k < p.topk) p.weights[row * p.w_sb + k] = NAN;
      }
    } else if (p.weights != nullptr) {
      // ---------------------------------------------------------------- weights
      // every tile's scores are behind the barriers above
      const int64_t first = (row * G + group) * p.ntiles + split;
      for (int64_t e = sm_tid; e < (int64_t)live * kTS; e += kSmThreads) {
        const int64_t at = first + e / kTS * S;
        const int slot = (int)(e % kTS);
        float* s = p.scores + at * NH * kTS + slot;
        const float w = head_sum<NH>(s, lse_s);
        if (G == 1) {
          const int64_t k = (int64_t)p.tiles[at] * kTS + slot;
          if (k < p.topk) p.weights[row * p.w_sb + k] = w;
        } else {
          s[0] = w;  // this group's sum, in the place of its first head's score
        }
      }
    }
  }
  if (p.clustered && G > 1 && p.weights != nullptr) {
    __syncwarp();
    ptx::cluster_sync();
    if (warp >= kSm0 && !lost) {
      // the groups ran the same tiles; each adds up the tiles it owns, group by group
      const int sm_tid = (int)threadIdx.x - 32 * kSm0;
      const int64_t first = row * G * p.ntiles + split;
      for (int64_t e = sm_tid; e < (int64_t)live * kTS; e += kSmThreads) {
        const int64_t at = first + e / kTS * S;
        const int tile = __ldcg(p.tiles + at + (int64_t)group * p.ntiles);
        const int slot = (int)(e % kTS);
        const int64_t k = (int64_t)tile * kTS + slot;
        if ((tile / S) % G != group || k >= p.topk) continue;
        float w = 0.f;
        for (int g = 0; g < G; ++g)
          w += __ldcg(p.scores + (at + (int64_t)g * p.ntiles) * NH * kTS + slot);
        p.weights[row * p.w_sb + k] = w;
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  // no CTA leaves while another may still read its shared memory
  if (S > 1) ptx::cluster_sync();
  if (warp == kScore) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, (uint32_t)C::TMEM_COLS);
  }
}

}  // namespace q8
}  // namespace dsa
