// bsa_bwd_sm100.cu -- gradient of block-sparse attention for sm_100a, 16-bit
// types, D = 64 (formulas and the split into work items: bsa_bwd.cuh).
//
// A work item owns 128 output rows of one head and walks the listed blocks of
// the other side in tiles of 128 rows (a 128-token block, or two listed
// 64-token blocks).  Both kinds of item run the same products on the tensor
// cores:
//               own operands    walked      S = own1 walk1^T   dP = own2 walk2^T
//   dk, dv      k, v            q, do       k q^T              v do^T
//   dq          q, do           k, v        q k^T              do v^T
// P = exp2(c S - lse) and dS = P (dP - delta) are formed in registers, one
// thread per own row and quarter of the walked columns, rounded to the 16-bit
// type and written back to TMEM, where they are the A operand of
//   dv += P walk2,   dk (or dq) += dS walk1
// (walk1 and walk2 read as K-by-64 operands from the same shared-memory tile
// that S and dP read).  So neither P nor dS touches shared memory.  lse and
// delta are per column for dk / dv (read from shared memory, a broadcast) and
// constants of the thread for dq.
//
// One persistent CTA per SM takes items (longest lists first) from a counter:
//   warp 0       producer: TMA loads of the own operands (two slots, so the
//                next item's are there when it starts) and of the walked tiles
//                (ring of kStages, with their lse and delta)
//   warp 1       TMEM allocation; one thread issues S and dP of tile after
//                tile, as soon as the ones before are read out of TMEM
//   warp 2       one thread issues the dv and dk (dq) products
//   warp 3       stores finished tiles by TMA from the item's own-operand slot
//   warps 4-19   compute: warpgroup w has columns [32 w, 32 w + 32) of a tile.
//                A tile costs a warp two hand-overs each way: S and dP are read
//                together (and may be overwritten at once), P and dS written
//                together.
// TMEM columns: S 128 | dP 128 | P 64 | dS 64 | dv 64 | dk or dq 64.
//
// f16: p below 2^-14 and ds of small gradients would leave the type's normal
// range, so P is formed times 2^4 and dS times a power of two that keeps it
// just inside the type for the largest |do| and the head's largest |v|,
// whatever their signs; the outputs are scaled back.  In dq items that |do| is
// the row's own largest (a row is one thread's, and its power goes into the
// exponent of P), in dk items the largest of the blocks listed for the key's
// half of the tile, so that a few rows with a large gradient take no bits from
// the others (with one power for the whole head, rows 2^12 below its largest
// were left with four bits).
//
// P and dS are rounded to the 16-bit type because the tensor cores want A and B
// of one type (walk1 and walk2 are the caller's); the sums over them, S, dP,
// lse and delta are fp32.  Against sums of unrounded values that makes the
// error of dk and dv 1.4 times the output's own rounding.  A row of dS sums to
// zero, so in dq a component that all keys share cancels, but its share of the
// rounding does not: with keys whose common part is eight times their spread, dq
// was off by 3.3 (bf16) and 3.4 to 3.7 (f16) times the output's rounding.  dq
// therefore adds the product of what the rounding took off too, from P's
// columns, which its items leave free: 1.0 times.  When it was added that cost
// 2.83 instead of 2.61 ms at the bf16 size below, and 735 instead of 661 us a
// call at 4 heads of 33976 tokens in f16 (strided).
//
// Bound (2 x 30 heads of 17776 tokens, a tenth of the 128-blocks, bf16): the
// tensor pipe, the exponentials and the issue slots share the SM, none of them
// full.  2.69 ms at 1965 MHz = 576 TFLOP/s of the five products that the
// gradient cannot do without (eight are run: S and dP in both kinds of items,
// dq in two parts), 3.1 to 3.2 ms once the 1000 W power cap holds the clock lower.
// f16, 4 heads of 33976 tokens, strided: 0.62 to 0.64 ms (by box), 536 to 554 TFLOP/s.
// Counters at 16 heads: tensor pipe 41 %, MUFU 41 %, issue 47 %, DRAM 11 %.
// Before dq's second product, with a part taken out (2.60 ms whole, timing
// only): no exponentials 2.24, no S and dP products 2.38, no dv and dk
// products 2.37, no products at all 1.96, no loads of the walked tiles 2.60,
// all items empty 0.26.  So the registers' work on a tile (~1400 cycles of a
// warp) is the longest chain and overlaps with the products only in part.
//
// Structures measured against those 2.60 ms and left: two compute warpgroups of
// 64 columns and one MMA thread 3.60 ms; 64-row units with MMA threads of their
// own 3.24; two pipelines of 64-row units 2.76; P of all columns before any dS
// 2.67; a finished item's results read out within the next item 2.89 (spills);
// exponentials in part on the FMA pipe 2.62 (1/8), 2.65 (1/4), 2.79 (1/2).  One
// kind of item that adds its share of dq in memory would save two of the
// products, but wants fp32 atomics, whose order changes the bits from run to run.
//
// Own tiles of two 64-token blocks: a half that does not list a walked unit has
// zeros for it, formed without the exponentials (16 heads of 8000 tokens, 15 %
// of the 64-blocks: 329 us, 363 with them).  0 times an infinity or NaN of the
// unit would reach that half all the same, so tiles whose S or dP show one are
// multiplied half by half, with the other half's lanes left out; done for every
// tile, that cost 8 % at the size above.
//
// Every wait is bounded, as in the forward kernel.
#include "bsa_bwd.cuh"

#include <cuda_fp16.h>

namespace saf {
namespace {

constexpr int kM = 128;  // own rows of an item, walked rows of a tile
constexpr int kUnit = 64;
constexpr int kD = 64;
constexpr int kStages = 4;
constexpr int kGroups = 4;  // compute warpgroups
constexpr int kCols = kM / kGroups;
constexpr int kComputeWarps = 4 * kGroups;
constexpr int kThreads = 128 + 32 * kComputeWarps;
// Launched at 96 registers a thread (640 x 96 = 61440): the control warpgroup
// drops to 64, the four compute warpgroups rise to 104.
constexpr uint32_t kRegsCtl = 64, kRegsCompute = 104;
constexpr int kLaunchRegs = 96;
static_assert(128 * kRegsCtl + 32 * kComputeWarps * kRegsCompute <= kThreads * kLaunchRegs, "register split");
constexpr uint32_t kColS = 0, kColDP = 128, kColP = 256, kColDS = 320, kColV = 384, kColK = 448, kTmemCols = 512;
constexpr float kF16PScale = 16.f;
constexpr int kOdd = 4;  // in a unit's entry, beside the halves: its rows hold infinities or NaN

struct Item {
  int32_t keys;  // 1: dk and dv of a key tile, 0: dq of a query tile, -1: no more items
  int32_t g, tile;
  int32_t n;     // walked tiles
  int32_t part;  // -1, or where the fp32 sums of this part of a line go
  int32_t ds_exp[2];  // f16: exponent of dS's power of two for each half of the own tile (dq: v's part)
  int32_t pad;
};

struct BwdParams {
  int H, Sq, Sk, BH, bm, bn;
  float scale, scale_log2;
  BwdWorkspace w;
  unsigned int* status;
  uint64_t budget_ns;
};

// Tensor maps, boxes of 64 rows.
struct Maps {
  CUtensorMap q, dout, k, v, dq, dk, dv;
};

// Shared memory: own operands [2 slots][2][128 x 64], the ring [kStages][2]
// [128 x 64], lse and delta of each stage, items, stage entries, barriers.
struct Layout {
  static constexpr int kTile = kM * kD * 2;
  static constexpr int kOffWalk = 4 * kTile;
  static constexpr int kOffStat = kOffWalk + kStages * 2 * kTile;
  static constexpr int kStat = 2 * kM * 4;
  static constexpr int kOffItem = kOffStat + kStages * kStat;
  static constexpr int kOffEnt = kOffItem + 2 * static_cast<int>(sizeof(Item));
  static constexpr int kOffBar = kOffEnt + kStages * 16;
  static constexpr int kBars = 4 + 2 * kStages + 10;
  static constexpr int kOffMisc = kOffBar + kBars * 8;
  static constexpr int kBytes = kOffMisc + 16;
  static constexpr int kDynSmem = kBytes + 1024;  // slack for 1024-byte alignment
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// 64 x 64 tile of shared memory -> rows [row, row + 64) of one head; rows past the end are not written.
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int row, int h, int b) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(0), "r"(row), "r"(h), "r"(b)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// What the roles share: addresses and the bounded wait.
struct Ctx {
  uint32_t bar0, own, walk, stat;
  Item* items;  // [2]
  int2* ents;   // [kStages][2 units]: first walked row, halves of the own tile that list it (0: no second unit)
  uint32_t* seen;  // [2 slots]: halves of the item's own tile whose sums were started
  const float* stats;
  volatile int* abort_flag;
  uint32_t tmem;
  const BwdParams& p;
  __device__ uint32_t own_full(int s) const { return bar0 + 8u * s; }
  __device__ uint32_t own_empty(int s) const { return bar0 + 8u * (2 + s); }
  __device__ uint32_t full(int s) const { return bar0 + 8u * (4 + s); }
  __device__ uint32_t empty(int s) const { return bar0 + 8u * (4 + kStages + s); }
  __device__ uint32_t at(int i) const { return bar0 + 8u * (4 + 2 * kStages + i); }
  __device__ uint32_t scores() const { return at(0); }     // S and dP are in TMEM
  __device__ uint32_t read() const { return at(1); }       // and read
  __device__ uint32_t written() const { return at(2); }    // P and dS are; the stage's values are read
  __device__ uint32_t added() const { return at(3); }      // and multiplied
  __device__ uint32_t acc_full() const { return at(4); }   // the item's sums are final
  __device__ uint32_t acc_empty() const { return at(5); }  // and read
  // The results of the item in slot s are in shared memory.  One barrier a
  // slot: an item without tiles waits for no product, so a compute warp may
  // arrive for it while another is still at the item before.  It cannot be a
  // whole round ahead: the slot's next item needs own_empty, which holds every
  // compute warp and the store warp.
  __device__ uint32_t staged(int s) const { return at(6 + s); }
  __device__ uint32_t drain(int w) const { return at(8 + w); }
  __device__ bool wait(uint32_t bar, uint32_t parity) const {
    return mbar_wait(bar, parity, abort_flag, p.status, p.budget_ns);
  }
  // the 32 lanes of a warp together
  __device__ bool wait_all(uint32_t bar, uint32_t parity) const {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, p.budget_ns));
  }
};

// A compute warp's wait: after a time-out it goes on (the abort flag is up, so
// no later wait holds it, and it leaves at the end of the item).
__device__ __forceinline__ void pass(const Ctx& c, uint32_t bar, uint32_t parity) {
  if (!mbar_try_wait(bar, parity)) (void)c.wait(bar, parity);
  __syncwarp();
}

__device__ __forceinline__ void warp_arrive(uint32_t bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// Shared-memory matrix descriptors as (low, high) words: the high word and the
// leading-dimension field are constants, so the next K slice is one addition
// (sdesc_sw128's fields: K-major rows 32 bytes on, MN-major 16 rows on).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ uint64_t desc64(uint32_t lo) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(kDescHi));
  return d;
}

// Register pairs by mov.b64, which costs nothing when they lie side by side.
__device__ __forceinline__ f2 pair(float lo, float hi) {
  f2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d.v) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ float first(f2 x) {
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x.v));
  return lo;
}
__device__ __forceinline__ float second(f2 x) {
  float lo, hi;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x.v));
  return hi;
}

template <bool kBF16>
__device__ __forceinline__ uint32_t pack2(f2 x) {
  return kBF16 ? pack_bf16x2(first(x), second(x)) : pack_f16x2(first(x), second(x));
}
__device__ __forceinline__ void zero16(uint32_t (&r)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) asm volatile("mov.b32 %0, 0;" : "=r"(r[e]));
}

// What rounding to the 16-bit type took off a pair.
template <bool kBF16>
__device__ __forceinline__ f2 rounded_off(f2 x, uint32_t r) {
  if constexpr (kBF16) return pair(first(x) - __uint_as_float(r << 16), second(x) - __uint_as_float(r & 0xffff0000u));
  const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&r));
  return pair(first(x) - y.x, second(x) - y.y);
}

// One tile: 32 columns of this thread's row; t is the tile's number in the
// CTA.  kKeys: lse and delta per column (shared
// memory; the MMA thread that arrives on `scores` has waited for the stage),
// and P goes to TMEM too.  dq: the low part of dS takes P's place.  A half
// of the own tile that does not list a unit has zeros there; infinities or NaN
// in the unit's rows (every row of S or dP shows them) are noted in its entry,
// since 0 times them would be NaN.
template <bool kKeys, bool kBF16>
__device__ __forceinline__ void compute_tile(const Ctx& c, const BwdParams& p, int w, int quarter, uint32_t t,
                                             float nl_row, float nd_row, float ds_scale) {
  const uint32_t s = t % kStages, par = t & 1;
  const uint32_t lane_addr = c.tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const uint32_t ts = lane_addr + w * kCols;
  const uint32_t tp = lane_addr + w * (kCols / 2);
  pass(c, c.scores(), par);
  tc_fence_after();
  uint32_t r[32], rd[32];
  tmem_ld32(ts + kColS, r);
  tmem_ld32(ts + kColDP, rd);
  const int2 ent = c.ents[2 * s + (w >> 1)];
  const float4* nl = reinterpret_cast<const float4*>(c.stats + s * 2 * kM + w * kCols);
  const float4* nd = nl + kM / 4;
  tmem_wait_ld(r);
  tmem_wait_ld(rd);
  tc_fence_before();
  mbar_arrive(c.read());
  const f2 sl = mk2(p.scale_log2, p.scale_log2);
  uint32_t pk[kCols / 2], dk[kCols / 2];
  if (!((ent.y >> (quarter >> 1)) & 1)) {  // not listed for this half of the own tile, or no second unit
    bool odd = false;
#pragma unroll
    for (int e = 0; e < kCols; ++e)
      odd |= !(fabsf(__uint_as_float(r[e])) < INFINITY) || !(fabsf(__uint_as_float(rd[e])) < INFINITY);
    if (odd && ent.y != 0) c.ents[2 * s + (w >> 1)].y = ent.y | kOdd;
    zero16(dk);
    zero16(pk);
  } else {
#pragma unroll
    for (int e4 = 0; e4 < kCols / 4; ++e4) {
      f2 ol[2] = {mk2(nl_row, nl_row), mk2(nl_row, nl_row)}, od[2] = {mk2(nd_row, nd_row), mk2(nd_row, nd_row)};
      if constexpr (kKeys) {
        const float4 l = nl[e4], d = nd[e4];
        ol[0] = pair(l.x, l.y), ol[1] = pair(l.z, l.w);
        od[0] = pair(d.x, d.y), od[1] = pair(d.z, d.w);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = 4 * e4 + 2 * i;
        const f2 y = fma2(pair(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), sl, ol[i]);
        const f2 pr = pair(ex2_approx(first(y)), ex2_approx(second(y)));
        if constexpr (kKeys) pk[e / 2] = pack2<kBF16>(pr);
        f2 z = mul2(add2(pair(__uint_as_float(rd[e]), __uint_as_float(rd[e + 1])), od[i]), pr);
        if constexpr (!kBF16 && kKeys) z = mul2(z, mk2(ds_scale, ds_scale));
        dk[e / 2] = pack2<kBF16>(z);
        if constexpr (!kKeys) pk[e / 2] = pack2<kBF16>(rounded_off<kBF16>(z, dk[e / 2]));
      }
    }
  }
  if constexpr (!kKeys) {
    // keys past the end: their scores are 0, not -inf
    const int valid = p.Sk - (ent.x + (w & 1) * kCols);
    if (valid < kCols) {
#pragma unroll
      for (int e = 0; e < kCols / 2; ++e) {
        const uint32_t live = 2 * e + 1 < valid ? 0xffffffffu : 2 * e < valid ? 0xffffu : 0u;
        dk[e] &= live;
        pk[e] &= live;
      }
    }
  }
  pass(c, c.added(), par ^ 1);  // the tile before is multiplied
  tc_fence_after();
  tmem_st16(tp + kColP, pk);
  tmem_st16(tp + kColDS, dk);
  tmem_wait_st();
  tc_fence_before();
  mbar_arrive(c.written());
}

// kParts: lines may be cut into parts (a template, so that the code of the
// parts costs the launches without them nothing).
template <bool kBF16, bool kParts>
__global__ void __launch_bounds__(kThreads, 1)
    bsa_bwd_sm100_kernel(const __grid_constant__ Maps maps, const __grid_constant__ BwdParams p) {
  using L = Layout;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  Ctx c{0, 0, 0, 0, nullptr, nullptr, nullptr, nullptr, nullptr, 0, p};
  c.bar0 = smem_u32(smem + L::kOffBar);
  c.own = smem_u32(smem);
  c.walk = smem_u32(smem + L::kOffWalk);
  c.stat = smem_u32(smem + L::kOffStat);
  c.stats = reinterpret_cast<const float*>(smem + L::kOffStat);
  c.items = reinterpret_cast<Item*>(smem + L::kOffItem);
  c.ents = reinterpret_cast<int2*>(smem + L::kOffEnt);
  c.abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  c.seen = reinterpret_cast<uint32_t*>(smem + L::kOffMisc + 8);
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(c.own_full(s), 1);
      mbar_init(c.own_empty(s), 3 + kComputeWarps);  // MMA threads, store warp, compute warps
      mbar_init(c.staged(s), kComputeWarps);
      mbar_init(c.drain(s), 1);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(c.full(s), 1);
      mbar_init(c.empty(s), 1);
    }
    mbar_init(c.scores(), 2);
    mbar_init(c.read(), 32 * kComputeWarps);
    mbar_init(c.written(), 32 * kComputeWarps);
    mbar_init(c.added(), 1);
    mbar_init(c.acc_full(), 2);
    mbar_init(c.acc_empty(), kComputeWarps);
    *c.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  c.tmem = *tmem_slot;
  // all of the above runs beside the end of the preparation (29.3 -> 28.6 us a
  // short call, 2.817 -> 2.812 ms the layer)
  asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp < 4) {
    setmaxnreg_dec<kRegsCtl>();
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      const int mine = lane < kClasses ? p.w.class_count[lane] : 0;  // items per length class
      int n_items = mine;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) n_items += __shfl_xor_sync(0xffffffffu, n_items, o);
      int it = 0, t = 0, nown = 0;
      bool ok = true;
      int lin = lane == 0 ? atomicAdd(p.w.next, 1) : 0;
      while (ok) {
        lin = __shfl_sync(0xffffffffu, lin, 0);
        // the class that holds position lin, and the place in it
        int left = lin, cls = 0;
        if (lin < n_items)
          for (; cls < kClasses - 1; ++cls) {
            const int cnt = __shfl_sync(0xffffffffu, mine, cls);
            if (left < cnt) break;
            left -= cnt;
          }
        Item im{};
        im.keys = -1;
        int n = 0, block = kM;
        const uint16_t* list = nullptr;
        if (lin < n_items) {
          const uint2 entry = p.w.items[static_cast<int64_t>(cls) * p.w.item_cap + left];
          const uint32_t id = entry.x;
          const PartOf part = unpack_part(entry.y);
          im.part = kParts && part.parts > 1 ? part.slot : -1;
          im.keys = static_cast<int32_t>(id >> 31);
          const int line = static_cast<int>(id & 0x7fffffffu);
          const int lines = im.keys ? p.w.lines_k : p.w.lines_q;
          im.g = line / lines;
          im.tile = line - im.g * lines;
          n = (im.keys ? p.w.count_k : p.w.count_q)[line];
          list = im.keys ? p.w.list_k + static_cast<int64_t>(line) * p.w.cap_k
                         : p.w.list_q + static_cast<int64_t>(line) * p.w.cap_q;
          block = im.keys ? p.bm : p.bn;
          im.n = block == kM ? n : (n + 1) / 2;
          if (kParts && part.parts > 1) {  // this part's tiles, and their entries of the list
            const int t0 = im.n * part.number / part.parts, t1 = im.n * (part.number + 1) / part.parts;
            const int per = kM / block;
            list += t0 * per;
            n = min(n - t0 * per, (t1 - t0) * per);
            im.n = t1 - t0;
          }
          if (!kBF16) im.ds_exp[0] = im.ds_exp[1] = f16_ds_exponent_v(__uint_as_float(p.w.vmax[im.g]));
          if (!kBF16 && im.keys) {  // the largest |do| of the listed query blocks
            const float* amax = p.w.amax + im.g * (p.w.Sp / kUnit);
            const int per = block / kUnit;
            float a0 = 0.f, a1 = 0.f;
#pragma unroll 4
            for (int i = lane; i < n; i += 32) {
              const uint32_t ent = list[i];
              const float* at = amax + (ent & 0x3fffu) * per;
              const float x = fmaxf(at[0], at[per - 1]);
              if (ent & 0x4000u) a0 = fmaxf(a0, x);
              if (ent & 0x8000u) a1 = fmaxf(a1, x);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
              a0 = fmaxf(a0, __shfl_xor_sync(0xffffffffu, a0, o));
              a1 = fmaxf(a1, __shfl_xor_sync(0xffffffffu, a1, o));
            }
            im.ds_exp[0] += f16_ds_exponent_do(a0);
            im.ds_exp[1] += f16_ds_exponent_do(a1);
          }
        }
        if (lane == 0 && lin < n_items) lin = atomicAdd(p.w.next, 1);  // the next one, in flight over this one
        const int slot = it & 1;
        ok = c.wait_all(c.own_empty(slot), ((it >> 1) & 1) ^ 1);
        if (!ok) break;
        ++it;
        const int b = im.g / p.H, h = im.g % p.H;
        if (lane == 0) {
          c.items[slot] = im;
          if (im.n > 0) {
            mbar_arrive_expect_tx(c.own_full(slot), 2 * L::kTile);
            const uint32_t dst = c.own + slot * 2 * L::kTile;
            for (int x = 0; x < 2; ++x) {
              const uint32_t at = dst + x * (L::kTile / 2);
              const int r = im.tile * kM + x * kUnit;
              tma_load_4d(at, im.keys ? &maps.k : &maps.q, c.own_full(slot), 0, r, h, b);
              tma_load_4d(at + L::kTile, im.keys ? &maps.v : &maps.dout, c.own_full(slot), 0, r, h, b);
            }
          } else {
            mbar_arrive(c.own_full(slot));
          }
        }
        nown = it;
        __syncwarp();
        if (im.keys < 0) break;
        if (lane == 0 && n > 0) {
          uint32_t next = list[0];
          for (int j = 0; j < n; ++t) {
            const int s = t % kStages;
            if (!c.wait(c.empty(s), ((t / kStages) & 1) ^ 1)) {
              ok = false;
              break;
            }
            const uint32_t ent0 = next;
            if (++j < n) next = list[j];
            const int row0 = static_cast<int>(ent0 & 0x3fffu) * block;
            int row1 = row0 + kUnit;
            uint32_t live1 = ent0 >> 14;
            if (block == kUnit) {  // the second unit is the next listed block, if there is one
              row1 = static_cast<int>(next & 0x3fffu) * kUnit;
              live1 = j < n ? next >> 14 : 0u;
              if (j < n && ++j < n) next = list[j];
            }
            const int units = live1 != 0u ? 2 : 1;
            c.ents[2 * s] = make_int2(row0, static_cast<int>(ent0 >> 14));
            c.ents[2 * s + 1] = make_int2(row1, static_cast<int>(live1));
            mbar_arrive_expect_tx(c.full(s), units * (L::kTile + (im.keys ? L::kStat / 2 : 0)));
            for (int x = 0; x < units; ++x) {
              const int row = x ? row1 : row0;
              const uint32_t dst = c.walk + s * 2 * L::kTile + x * (L::kTile / 2);
              tma_load_4d(dst, im.keys ? &maps.q : &maps.k, c.full(s), 0, row, h, b);
              tma_load_4d(dst + L::kTile, im.keys ? &maps.dout : &maps.v, c.full(s), 0, row, h, b);
              if (im.keys) {
                const int64_t at = im.g * p.w.Sp + row;
                const uint32_t st = c.stat + s * L::kStat + x * kUnit * 4;
                bulk_load(st, p.w.stat_lse + at, kUnit * 4, c.full(s));
                bulk_load(st + kM * 4, p.w.stat_delta + at, kUnit * 4, c.full(s));
              }
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        t = __shfl_sync(0xffffffffu, t, 0);
      }
      // every copy issued has landed before shared memory is given up
      if (lane == 0) {
        for (int s = 0; s < 2 && s < nown; ++s) {
          const int last = s + ((nown - 1 - s) / 2) * 2;
          mbar_drain(c.own_full(s), (last >> 1) & 1, p.status);
        }
        for (int s = 0; s < kStages && s < t; ++s) {
          const int last = s + ((t - 1 - s) / kStages) * kStages;
          mbar_drain(c.full(s), (last / kStages) & 1, p.status);
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ------------------------------------------------------ S and dP issuer
      if (lane == 0) {
        constexpr uint32_t kIdesc = idesc_f16(kM, kM, kBF16, false, false);
        const uint32_t own_lo = desc_lo(c.own), walk_lo = desc_lo(c.walk);
        // own tile (descriptor a) x walked tile (b)^T, both K-major, into column d
        auto scores = [&](uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
          for (int kk = 0; kk < kD / 16; ++kk)
            tc_mma_ss(c.tmem + d, desc64(a + kk * 2), desc64(b + kk * 2), kIdesc, kk > 0 ? 1u : 0u);
        };
        uint32_t it = 0, t = 0;
        bool ok = true;
        while (ok) {
          const uint32_t slot = it & 1;
          if (!c.wait(c.own_full(slot), (it >> 1) & 1)) break;
          ++it;
          const int keys = c.items[slot].keys, n = c.items[slot].n;
          if (keys < 0) break;
          const uint32_t a = own_lo + slot * (2 * L::kTile >> 4);
          for (int j = 0; j < n; ++j, ++t) {
            const uint32_t s = t % kStages;
            const uint32_t b = walk_lo + s * (2 * L::kTile >> 4);
            ok = c.wait(c.full(s), (t / kStages) & 1) && c.wait(c.read(), (t & 1) ^ 1);
            if (!ok) break;
            tc_fence_after();
            scores(kColS, a, b);
            scores(kColDP, a + (L::kTile >> 4), b + (L::kTile >> 4));
            tc_commit(c.scores());
            mbar_arrive(c.scores());  // hands on the order behind this thread's wait for the stage
          }
          if (n > 0)
            tc_commit(c.own_empty(slot));
          else
            mbar_arrive(c.own_empty(slot));
        }
        tc_commit(c.drain(0));
        mbar_drain(c.drain(0), 0, p.status);
      }
    } else if (warp == 2) {
      // ------------------------------------------------- dv, dk and dq issuer
      if (lane == 0) {
        constexpr uint32_t kIdesc = idesc_f16(kM, kD, kBF16, false, true);
        const uint32_t walk_lo = desc_lo(c.walk);
        // P or dS (TMEM column a) x walked tile (MN-major, b) added to column
        // d: 16 walked rows a step, of one or both units
        auto add = [&](uint32_t d, uint32_t a, uint32_t b, bool both, uint32_t accumulate) {
#pragma unroll
          for (int kk = 0; kk < kUnit / 16; ++kk)
            tc_mma_ts(c.tmem + d, c.tmem + a + kk * 8, desc64(b + kk * 128), kIdesc, kk > 0 ? 1u : accumulate);
          if (both) {
#pragma unroll
            for (int kk = kUnit / 16; kk < kM / 16; ++kk)
              tc_mma_ts(c.tmem + d, c.tmem + a + kk * 8, desc64(b + kk * 128), kIdesc, 1u);
          }
        };
        // the same, each unit for the halves that list it alone
        auto add_halves = [&](uint32_t d, uint32_t a, uint32_t b, uint32_t live0, uint32_t live1, uint32_t seen) {
          constexpr int kSlices = kUnit / 16;
          auto desc0 = [&](int kk) { return desc64(b + kk * 128); };
          auto desc1 = [&](int kk) { return desc64(b + (kSlices + kk) * 128); };
          tc_add_halves<kSlices>(c.tmem + d, c.tmem + a, desc0, kIdesc, live0, seen);
          if (live1 != 0u)
            tc_add_halves<kSlices>(c.tmem + d, c.tmem + a + kSlices * 8, desc1, kIdesc, live1, seen | live0);
        };
        uint32_t it = 0, t = 0, na = 0;  // na: items with tiles
        bool ok = true;
        while (ok) {
          const uint32_t slot = it & 1;
          if (!c.wait(c.own_full(slot), (it >> 1) & 1)) break;
          ++it;
          const int keys = c.items[slot].keys, n = c.items[slot].n;
          if (keys < 0) break;
          mbar_arrive(c.own_empty(slot));  // the entry is read
          if (n > 0) {
            ok = c.wait(c.acc_empty(), (na & 1) ^ 1);  // the sums of the item before are read
            if (!ok) break;
            ++na;
          }
          uint32_t seen = 0u;  // halves of the own tile whose sums are started
          for (int j = 0; j < n; ++j, ++t) {
            const uint32_t s = t % kStages;
            const uint32_t b = walk_lo + s * (2 * L::kTile >> 4);
            ok = c.wait(c.written(), t & 1);
            if (!ok) break;
            tc_fence_after();
            const uint32_t e0 = c.ents[2 * s].y, e1 = c.ents[2 * s + 1].y;
            const uint32_t b2 = keys ? b + (L::kTile >> 4) : b;
            const uint32_t d2 = keys ? kColV : kColK;  // dq: P's columns hold what rounding took off dS
            if (!((e0 | e1) & kOdd) && (seen == 3u || j == 0)) {
              add(d2, kColP, b2, e1 != 0u, j > 0);
              add(kColK, kColDS, b, e1 != 0u, !keys || j > 0);
              seen = 3u;
            } else {  // infinities or NaN that one half does not list
              const uint32_t live0 = e0 & 3u, live1 = e1 & 3u, now = seen | live0 | live1;
              add_halves(d2, kColP, b2, live0, live1, seen);
              add_halves(kColK, kColDS, b, live0, live1, keys ? seen : now);
              seen = now;
            }
            tc_commit(c.added());
            tc_commit(c.empty(s));
          }
          if (ok && n > 0) {
            c.seen[slot] = seen;
            tc_commit(c.acc_full());
            mbar_arrive(c.acc_full());  // hands on `seen`
          }
        }
        tc_commit(c.drain(1));
        mbar_drain(c.drain(1), 0, p.status);
      }
    } else {
      // --------------------------------------------------------- store warp
      int it = 0;
      while (true) {
        const int slot = it & 1;
        if (!c.wait_all(c.own_full(slot), (it >> 1) & 1)) break;
        const Item im = c.items[slot];
        if (im.keys < 0) break;
        if (!c.wait_all(c.staged(slot), (it >> 1) & 1)) break;
        if (lane == 0 && (!kParts || im.part < 0)) {
          const int h = im.g % p.H, b = im.g / p.H;
          const uint32_t src = c.own + slot * 2 * L::kTile;
          for (int x = 0; x < 2; ++x) {
            const uint32_t at = src + x * (L::kTile / 2);
            const int r = im.tile * kM + x * kUnit;
            if (r >= (im.keys ? p.Sk : p.Sq)) break;
            tma_store_4d(im.keys ? &maps.dv : &maps.dq, at, r, h, b);
            if (im.keys) tma_store_4d(&maps.dk, at + L::kTile, r, h, b);
          }
          bulk_commit();
          bulk_wait_read();
        }
        warp_arrive(c.own_empty(slot), lane);
        ++it;
      }
      if (lane == 0) bulk_wait();
    }
    __syncwarp();
    tc_fence_before();
    named_barrier_sync(1, kThreads);
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(c.tmem, kTmemCols);
    }
  } else {
    setmaxnreg_inc<kRegsCompute>();
    // ------------------------------------------------------------ compute
    const int w = (warp >> 2) - 1, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = c.tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    uint32_t it = 0, t = 0, na = 0;
    while (true) {
      const uint32_t slot = it & 1;
      if (!c.wait_all(c.own_full(slot), (it >> 1) & 1)) break;
      const int keys = c.items[slot].keys, n = c.items[slot].n;
      if (keys < 0) break;
      // f16: dS's power of two, for this half of the own tile (dk) or this thread's row (dq)
      int ds_exp = kBF16 ? 0 : c.items[slot].ds_exp[quarter >> 1];
      if (keys) {
        const float ds_scale = power_of_two(ds_exp);
        for (int j = 0; j < n; ++j, ++t) compute_tile<true, kBF16>(c, p, w, quarter, t, 0.f, 0.f, ds_scale);
      } else {
        const int64_t at = c.items[slot].g * p.w.Sp + c.items[slot].tile * kM + row;
        // dS's power of two goes into the exponent: dq does not need P itself
        if constexpr (!kBF16) ds_exp += static_cast<int>(p.w.stat_exp[at]);
        const float nl = p.w.stat_lse[at] + static_cast<float>(ds_exp);
        const float nd = p.w.stat_delta[at];
        for (int j = 0; j < n; ++j, ++t) compute_tile<false, kBF16>(c, p, w, quarter, t, nl, nd, 1.f);
      }
      if (__any_sync(0xffffffffu, *c.abort_flag)) break;
      // Results: warpgroups 0 and 1 take dv, 2 and 3 dk (32 channels each);
      // dq 16 channels each.  They go through this item's own-operand slot,
      // which no product reads once the sums are final.
      const bool dv = keys && w < 2;
      uint32_t r[32];
      if (n > 0) {
        if (!c.wait_all(c.acc_full(), na & 1)) break;
        ++na;
        tc_fence_after();
        tmem_ld32(lane_addr + (dv ? kColV + 32 * w : keys ? kColK + 32 * (w - 2) : kColK + (w >> 1) * 32), r);
        tmem_wait_ld(r);
        tc_fence_before();
        warp_arrive(c.acc_empty(), lane);
        if (!((c.seen[slot] >> (quarter >> 1)) & 1u)) {  // nothing was ever added for this half
#pragma unroll
          for (int e = 0; e < 32; ++e) asm volatile("mov.b32 %0, 0;" : "=r"(r[e]));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) r[e] = 0u;
      }
      const float unscale = kBF16 ? 1.f : 1.f / kF16PScale;
      const float scale = dv ? unscale : kBF16 ? p.scale : p.scale * unscale * power_of_two(-ds_exp);
      const int part = kParts ? c.items[slot].part : -1;
      if (kParts && part >= 0) {  // sums of a part of the line: fp32, scaled, to the workspace
        if (keys || (w & 1) == 0) {  // dq: one of the two warpgroups that hold the same 32 channels
          float* to = p.w.part + (static_cast<int64_t>(part) * 2 + dv) * (kM * kD) + row * kD + (keys ? (w & 1) * 32 : (w >> 1) * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            reinterpret_cast<float4*>(to)[i] =
                make_float4(__uint_as_float(r[4 * i]) * scale, __uint_as_float(r[4 * i + 1]) * scale,
                            __uint_as_float(r[4 * i + 2]) * scale, __uint_as_float(r[4 * i + 3]) * scale);
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(c.staged(slot));
          mbar_arrive(c.own_empty(slot));
        }
        ++it;
        continue;
      }
      const uint32_t dst = c.own + (2 * slot + (keys && !dv)) * L::kTile + row * 128;
      const int chunk0 = 4 * (keys ? w & 1 : w >> 1);  // 16-byte chunks of the row
#pragma unroll
      for (int i8 = 0; i8 < 4; ++i8) {
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = pack2<kBF16>(
              pair(__uint_as_float(r[8 * i8 + 2 * i]) * scale, __uint_as_float(r[8 * i8 + 2 * i + 1]) * scale));
        // dq: the two warpgroups that read the same 32 channels store 16 each
        if (keys || (i8 >> 1) == (w & 1)) st_shared_v4(dst + (((chunk0 + i8) ^ (row & 7)) << 4), x[0], x[1], x[2], x[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(c.staged(slot));
        mbar_arrive(c.own_empty(slot));
      }
      ++it;
    }
    tc_fence_before();
    named_barrier_sync(1, kThreads);
  }
}

// Adds the parts of a cut line in their order and stores its rows.  One CTA a
// cut line (the others leave), 8 threads a row of 64 channels; bound by the
// latency of reading the parts out of L2.
struct MergeParams {
  BwdWorkspace w;
  int H, Sq, Sk;
  void *dq, *dk, *dv;
  int64_t dq_sb, dq_sh, dq_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
};
template <bool kBF16>
__global__ void __launch_bounds__(256) bwd_merge_kernel(const MergeParams p) {
  if (static_cast<int>(blockIdx.x) >= *p.w.split_count) return;
  const uint2 entry = p.w.split[blockIdx.x];
  const bool keys = entry.x >> 31;
  const int line = static_cast<int>(entry.x & 0x7fffffffu), lines = keys ? p.w.lines_k : p.w.lines_q;
  const int g = line / lines, tile = line - g * lines, b = g / p.H, h = g % p.H;
  const PartOf part = unpack_part(entry.y);
  const int which = blockIdx.y;  // 0: dk or dq, 1: dv
  if (which == 1 && !keys) return;
  const float* src = p.w.part + (static_cast<int64_t>(part.slot) * 2 + which) * (kM * kD);
  uint8_t* dst = static_cast<uint8_t*>(keys ? (which ? p.dv : p.dk) : p.dq);
  const int64_t ss = keys ? (which ? p.dv_ss : p.dk_ss) : p.dq_ss;
  const int64_t at = keys ? (which ? b * p.dv_sb + h * p.dv_sh : b * p.dk_sb + h * p.dk_sh) : b * p.dq_sb + h * p.dq_sh;
  const int c0 = static_cast<int>(threadIdx.x & 7) * 8;
  for (int row = threadIdx.x >> 3; row < kM; row += 32) {
    const int out = tile * kM + row;
    if (out >= (keys ? p.Sk : p.Sq)) break;
    float sum[8] = {};
#pragma unroll 4
    for (int i = 0; i < part.parts; ++i) {
      const float4* x = reinterpret_cast<const float4*>(src + static_cast<int64_t>(i) * 2 * (kM * kD) + row * kD + c0);
      const float4 lo = x[0], hi = x[1];
      sum[0] += lo.x, sum[1] += lo.y, sum[2] += lo.z, sum[3] += lo.w;
      sum[4] += hi.x, sum[5] += hi.y, sum[6] += hi.z, sum[7] += hi.w;
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2<kBF16>(pair(sum[2 * i], sum[2 * i + 1]));
    *reinterpret_cast<uint4*>(dst + 2 * (at + out * ss + c0)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <bool kBF16, bool kParts>
int32_t launch(const Maps& maps, const BwdParams& p, int grid, cudaStream_t stream) {
  auto kern = bsa_bwd_sm100_kernel<kBF16, kParts>;
  // a build launched with fewer registers than the split hands out would wait forever
  static const int launch_regs = [] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, bsa_bwd_sm100_kernel<kBF16, kParts>) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (launch_regs < kLaunchRegs) return SAF_ERR_UNSUPPORTED;
  if (const int32_t rc = allow_smem<bsa_bwd_sm100_kernel<kBF16, kParts>>(Layout::kDynSmem); rc != SAF_OK) return rc;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Layout::kDynSmem;
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  SAF_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, maps, p));
  return SAF_OK;
}

}  // namespace

float bwd_f16_p_log2_scale() { return 4.f; }  // log2 of kF16PScale

// Launch after the preparation (validated by saf_bsa_bwd).
int32_t bsa_bwd_sm100(const saf_tensor4* dout, const saf_tensor4* q, const saf_tensor4* k, const saf_tensor4* v,
                      const saf_tensor4* dq, const saf_tensor4* dk, const saf_tensor4* dv, int bm, int bn,
                      float sm_scale, const BwdWorkspace& w, cudaStream_t stream) {
  if (!current_device_is_sm100()) return SAF_ERR_UNSUPPORTED;
  Maps maps;
  const struct {
    CUtensorMap* map;
    const saf_tensor4* t;
  } want[7] = {{&maps.q, q}, {&maps.dout, dout}, {&maps.k, k}, {&maps.v, v}, {&maps.dq, dq}, {&maps.dk, dk}, {&maps.dv, dv}};
  for (const auto& x : want) {
    const int32_t rc = make_qkv_map(x.map, x.t, kUnit);
    if (rc != SAF_OK) return rc;
  }
  BwdParams p{};
  p.H = static_cast<int>(q->H), p.Sq = static_cast<int>(q->S), p.Sk = static_cast<int>(k->S);
  p.BH = static_cast<int>(q->B * q->H);
  p.bm = bm, p.bn = bn;
  p.scale = sm_scale;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.w = w;
  p.status = device_status_ptr();
  p.budget_ns = wait_budget_ns();
  if (p.status == nullptr) return SAF_ERR_CUDA;
  const int sms = current_device_sms();
  if (sms <= 0) return SAF_ERR_CUDA;
  const int grid = w.item_cap < sms ? w.item_cap : sms;
  const bool bf16 = q->dtype == SAF_BF16;
  if (w.part_cap == 0)
    return bf16 ? launch<true, false>(maps, p, grid, stream) : launch<false, false>(maps, p, grid, stream);
  const int32_t rc = bf16 ? launch<true, true>(maps, p, grid, stream) : launch<false, true>(maps, p, grid, stream);
  if (rc != SAF_OK) return rc;
  MergeParams m{};
  m.w = w;
  m.H = p.H, m.Sq = p.Sq, m.Sk = p.Sk;
  m.dq = dq->data, m.dk = dk->data, m.dv = dv->data;
  m.dq_sb = dq->stride_b, m.dq_sh = dq->stride_h, m.dq_ss = dq->stride_s;
  m.dk_sb = dk->stride_b, m.dk_sh = dk->stride_h, m.dk_ss = dk->stride_s;
  m.dv_sb = dv->stride_b, m.dv_sh = dv->stride_h, m.dv_ss = dv->stride_s;
  // a cut line has two parts at least
  const int64_t lines = static_cast<int64_t>(p.BH) * (w.lines_q + w.lines_k);
  const dim3 mgrid(static_cast<unsigned>(lines < w.part_cap / 2 ? lines : w.part_cap / 2), 2);
  if (bf16)
    bwd_merge_kernel<true><<<mgrid, 256, 0, stream>>>(m);
  else
    bwd_merge_kernel<false><<<mgrid, 256, 0, stream>>>(m);
  SAF_CUDA_TRY(cudaGetLastError());
  return SAF_OK;
}

}  // namespace saf
