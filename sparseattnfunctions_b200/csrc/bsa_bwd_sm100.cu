// bsa_bwd_sm100.cu -- gradient of block-sparse attention for sm_100a, 16-bit
// types, D = 64 (formulas and the split into work items: bsa_bwd.cuh).
//
// A work item owns 128 output rows of one head and walks the listed blocks of
// the other side, N = 64 or 128 rows at a time.  Both kinds of item run the
// same products on the tensor cores, with R the rows of the own tile:
//               own operands    walked      S = own1 walk1^T   dP = own2 walk2^T
//   dk, dv      k, v            q, do       k q^T              v do^T
//   dq          q, do           k, v        q k^T              do v^T
// P = exp2(c S - lse) and dS = P (dP - delta) are formed in registers, one
// thread per own row and half of the walked columns, rounded to the 16-bit
// type and written back to TMEM, where they are the A operand of
//   dv += P walk2,   dk (or dq) += dS walk1
// (walk1 and walk2 read as K-by-64 operands from the same shared-memory tile
// that S and dP read).  So neither P nor dS touches shared memory, and lse and
// delta are per column for dk / dv (read from shared memory, a broadcast) and
// constants of the thread for dq.
//
// One persistent CTA per SM takes items (longest lists first) from a counter:
//   warp 0       producer: TMA loads of the own operands (two slots, so the
//                next item's are there when it starts) and of the walked tiles
//                (ring of kStages, with their lse and delta)
//   warp 1       TMEM allocation; one thread issues every MMA.  It runs one
//                block ahead with S and dP, across items, so that they are
//                done when the compute warps come to them
//   warps 2, 3   idle (they complete warpgroup 0 for the register split)
//   warps 4-11   compute: warpgroup w has columns [wN/2, (w+1)N/2) of a block
// TMEM columns: S 128 | dP 128 | P 64 | dS 64 | dv 64 | dk or dq 64.
//
// f16: p below 2^-14 and ds of small gradients would leave the type's normal
// range, so P is formed times 2^4 and dS times a power of two that takes the
// head's largest |do| to [2^-4, 2^-3); the outputs are scaled back.
//
// Every wait is bounded, as in the forward kernel.
#include "bsa_bwd.cuh"

namespace saf {
namespace {

constexpr int kM = 128;  // own rows of an item
constexpr int kD = 64;
constexpr int kStages = 4;
constexpr int kThreads = 384;
// Launched at 168 registers a thread (384 x 168 = 64512): the control
// warpgroup drops to 56, the two compute warpgroups rise to 224.
constexpr uint32_t kRegsCtl = 56, kRegsCompute = 224;
constexpr int kLaunchRegs = 168;
static_assert(128 * kRegsCtl + 256 * kRegsCompute <= kThreads * kLaunchRegs, "register split");
constexpr uint32_t kColS = 0, kColDP = 128, kColP = 256, kColDS = 320, kColV = 384, kColK = 448;
constexpr int kComputeWarps = 8;
constexpr float kF16PScale = 16.f;

struct Item {
  int32_t keys;   // 1: dk and dv of a key tile, 0: dq of a query tile, -1: no more items
  int32_t g, tile, n;
  float ds_scale;
  int32_t pad[3];
};

struct BwdParams {
  int H, Sq, Sk, BH;
  float scale, scale_log2;
  void *dq, *dk, *dv;
  int64_t dq_sb, dq_sh, dq_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
  BwdWorkspace w;
  unsigned int* status;
  uint64_t budget_ns;
};

// Shared memory: own operands [2 slots][2][128 x 64], then the ring
// [kStages][2][N x 64] (N the larger of the two walks), lse and delta of each
// stage, items, stage entries, barriers.
template <int NMax>
struct Layout {
  static constexpr int kOwn = kM * kD * 2;
  static constexpr int kWalk = NMax * kD * 2;
  static constexpr int kOffWalk = 4 * kOwn;
  static constexpr int kOffStat = kOffWalk + kStages * 2 * kWalk;
  static constexpr int kStat = 2 * NMax * 4;
  static constexpr int kOffItem = kOffStat + kStages * kStat;
  static constexpr int kOffEnt = kOffItem + 2 * static_cast<int>(sizeof(Item));
  static constexpr int kOffBar = kOffEnt + kStages * 8;
  static constexpr int kBars = 4 + 2 * kStages + 11;
  static constexpr int kOffMisc = kOffBar + kBars * 8;
  static constexpr int kBytes = kOffMisc + 16;
  static constexpr int kDynSmem = kBytes + 1024;  // slack for 1024-byte alignment
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// What the roles share: barrier addresses and the bounded wait.
struct Ctx {
  uint32_t bar0, own, walk, stat;
  const Item* items;
  const int32_t* ents;
  volatile int* abort_flag;
  unsigned int* status;
  uint64_t budget;
  uint32_t tmem;
  __device__ uint32_t own_full(int s) const { return bar0 + 8u * s; }
  __device__ uint32_t own_empty(int s) const { return bar0 + 8u * (2 + s); }
  __device__ uint32_t full(int s) const { return bar0 + 8u * (4 + s); }
  __device__ uint32_t empty(int s) const { return bar0 + 8u * (4 + kStages + s); }
  __device__ uint32_t at(int i) const { return bar0 + 8u * (4 + 2 * kStages + i); }
  __device__ uint32_t s_full() const { return at(0); }
  __device__ uint32_t s_empty() const { return at(1); }
  __device__ uint32_t dp_full() const { return at(2); }
  __device__ uint32_t dp_empty() const { return at(3); }
  __device__ uint32_t p_full() const { return at(4); }
  __device__ uint32_t p_empty() const { return at(5); }
  __device__ uint32_t ds_full() const { return at(6); }
  __device__ uint32_t ds_empty() const { return at(7); }
  __device__ uint32_t acc_full() const { return at(8); }
  __device__ uint32_t acc_empty() const { return at(9); }
  __device__ uint32_t drain() const { return at(10); }
  __device__ bool wait(uint32_t bar, uint32_t parity) const { return mbar_wait(bar, parity, abort_flag, status, budget); }
  // the 32 lanes of a warp together
  __device__ bool wait_all(uint32_t bar, uint32_t parity) const {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, budget));
  }
};

__device__ __forceinline__ void warp_arrive(uint32_t bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

template <bool kBF16>
__device__ __forceinline__ uint32_t pack2(f2 x) {
  return kBF16 ? pack_bf16x2(lo2(x), hi2(x)) : pack_f16x2(lo2(x), hi2(x));
}

// One block of a compute warpgroup: NC columns of this thread's row.
// kKeys: lse and delta per column (shared memory), and P goes to TMEM too.
// Returns false when a wait gave up.
template <int N, bool kKeys, bool kBF16>
__device__ __forceinline__ bool compute_block(const Ctx& c, const BwdParams& p, int wg, int lane, int quarter, int t,
                                              int tk, float nl_row, float nd_row, float ds_scale) {
  constexpr int NC = N / 2;
  const int s = t % kStages;
  const uint32_t par = (t / kStages) & 1;
  const uint32_t lane_addr = c.tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  if (!c.wait_all(c.full(s), par)) return false;
  const int ent = c.ents[2 * s];
  const bool live = ((static_cast<uint32_t>(ent) >> 14) >> (quarter >> 1)) & 1u;
  const float* nl = reinterpret_cast<const float*>(__cvta_shared_to_generic(c.stat + s * (2 * N * 4))) + wg * NC;
  const float* nd = nl + N;
  if (!c.wait_all(c.s_full(), t & 1)) return false;
  tc_fence_after();
  uint32_t r[NC / 32][32];
#pragma unroll
  for (int i = 0; i < NC / 32; ++i) tmem_ld32(lane_addr + kColS + wg * NC + 32 * i, r[i]);
#pragma unroll
  for (int i = 0; i < NC / 32; ++i) tmem_wait_ld(r[i]);
  tc_fence_before();
  warp_arrive(c.s_empty(), lane);

  const f2 sl = mk2(p.scale_log2, p.scale_log2);
  f2 pr[NC / 2];
#pragma unroll
  for (int e = 0; e < NC / 2; ++e) {
    const f2 x = mk2(__uint_as_float(r[e / 16][2 * e % 32]), __uint_as_float(r[e / 16][(2 * e + 1) % 32]));
    f2 off;
    if constexpr (kKeys) {
      const float2 l = *reinterpret_cast<const float2*>(nl + 2 * e);
      off = mk2(l.x, l.y);
    } else {
      off = mk2(nl_row, nl_row);
    }
    const f2 y = fma2(x, sl, off);
    pr[e] = mk2(ex2_approx(lo2(y)), ex2_approx(hi2(y)));
  }
  if constexpr (!kKeys) {
    // keys past the end: their scores are 0, not -inf
    const int valid = p.Sk - ((ent & 0x3fff) * N + wg * NC);
    if (valid < NC) {
#pragma unroll
      for (int e = 0; e < NC / 2; ++e)
        pr[e] = mk2(2 * e < valid ? lo2(pr[e]) : 0.f, 2 * e + 1 < valid ? hi2(pr[e]) : 0.f);
    }
  }
  uint32_t pk[NC / 2];
  if constexpr (kKeys) {
#pragma unroll
    for (int e = 0; e < NC / 2; ++e) pk[e] = live ? pack2<kBF16>(pr[e]) : 0u;
    // the dv product of the previous block has read P
    if (!c.wait_all(c.p_empty(), (tk & 1) ^ 1)) return false;
    tc_fence_after();
    if constexpr (NC == 64)
      tmem_st32(lane_addr + kColP + wg * (NC / 2), pk);
    else
      tmem_st16(lane_addr + kColP + wg * (NC / 2), pk);
    tmem_wait_st();
    tc_fence_before();
    warp_arrive(c.p_full(), lane);
  }
  if (!c.wait_all(c.dp_full(), t & 1)) return false;
  tc_fence_after();
#pragma unroll
  for (int i = 0; i < NC / 32; ++i) tmem_ld32(lane_addr + kColDP + wg * NC + 32 * i, r[i]);
#pragma unroll
  for (int i = 0; i < NC / 32; ++i) tmem_wait_ld(r[i]);
  tc_fence_before();
  warp_arrive(c.dp_empty(), lane);
#pragma unroll
  for (int e = 0; e < NC / 2; ++e) {
    const f2 x = mk2(__uint_as_float(r[e / 16][2 * e % 32]), __uint_as_float(r[e / 16][(2 * e + 1) % 32]));
    f2 off;
    if constexpr (kKeys) {
      const float2 d = *reinterpret_cast<const float2*>(nd + 2 * e);
      off = mk2(d.x, d.y);
    } else {
      off = mk2(nd_row, nd_row);
    }
    f2 y = mul2(add2(x, off), pr[e]);
    if constexpr (!kBF16) y = mul2(y, mk2(ds_scale, ds_scale));
    pk[e] = live ? pack2<kBF16>(y) : 0u;
  }
  warp_arrive(c.empty(s), lane);  // lse, delta and the entry are read
  if (!c.wait_all(c.ds_empty(), (t & 1) ^ 1)) return false;
  tc_fence_after();
  if constexpr (NC == 64)
    tmem_st32(lane_addr + kColDS + wg * (NC / 2), pk);
  else
    tmem_st16(lane_addr + kColDS + wg * (NC / 2), pk);
  tmem_wait_st();
  tc_fence_before();
  warp_arrive(c.ds_full(), lane);
  return true;
}

// 32 accumulator columns of this thread's row, scaled and stored.
template <bool kBF16>
__device__ __forceinline__ void store32(uint32_t (&r)[32], void* dst, float scale) {
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = pack2<kBF16>(mk2(__uint_as_float(r[8 * v + 2 * e]) * scale, __uint_as_float(r[8 * v + 2 * e + 1]) * scale));
    reinterpret_cast<uint4*>(dst)[v] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// NK: walked rows per step of dk / dv items (the query block), NQ: of dq items
// (the key block).  Maps: o* own tiles of 128 rows, w* walked tiles of NK / NQ.
struct Maps {
  CUtensorMap oq, odo, ok, ov, wq, wdo, wk, wv;
};

template <int NK, int NQ, bool kBF16>
__global__ void __launch_bounds__(kThreads, 1)
    bsa_bwd_sm100_kernel(const __grid_constant__ Maps maps, const __grid_constant__ BwdParams p) {
  constexpr int NMax = NK > NQ ? NK : NQ;
  using L = Layout<NMax>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Item* items = reinterpret_cast<Item*>(smem + L::kOffItem);
  int32_t* ents = reinterpret_cast<int32_t*>(smem + L::kOffEnt);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  Ctx c;
  c.bar0 = smem_u32(smem + L::kOffBar);
  c.own = smem_u32(smem);
  c.walk = smem_u32(smem + L::kOffWalk);
  c.stat = smem_u32(smem + L::kOffStat);
  c.items = items;
  c.ents = ents;
  c.abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  c.status = p.status;
  c.budget = p.budget_ns;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(c.own_full(s), 1);
      mbar_init(c.own_empty(s), 1 + kComputeWarps);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(c.full(s), 1);
      mbar_init(c.empty(s), 1 + kComputeWarps);
    }
    mbar_init(c.s_full(), 1);
    mbar_init(c.s_empty(), kComputeWarps);
    mbar_init(c.dp_full(), 1);
    mbar_init(c.dp_empty(), kComputeWarps);
    mbar_init(c.p_full(), kComputeWarps);
    mbar_init(c.p_empty(), 1);
    mbar_init(c.ds_full(), kComputeWarps);
    mbar_init(c.ds_empty(), 1);
    mbar_init(c.acc_full(), 1);
    mbar_init(c.acc_empty(), kComputeWarps);
    mbar_init(c.drain(), 1);
    *c.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  c.tmem = *tmem_slot;

  if (warp < 4) {
    setmaxnreg_dec<kRegsCtl>();
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      const int n_items = p.BH * (p.w.lines_q + p.w.lines_k);
      const int mine = lane < kClasses ? p.w.class_count[lane] : 0;  // items per length class
      int it = 0, t = 0, nown = 0, amax_g = -1;
      float ds_scale = 1.f;
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
        const uint16_t* list = nullptr;
        if (lin < n_items) {
          const uint32_t id = p.w.items[static_cast<int64_t>(cls) * n_items + left];
          im.keys = static_cast<int32_t>(id >> 31);
          const int line = static_cast<int>(id & 0x7fffffffu);
          const int lines = im.keys ? p.w.lines_k : p.w.lines_q;
          im.g = line / lines;
          im.tile = line - im.g * lines;
          im.n = (im.keys ? p.w.count_k : p.w.count_q)[line];
          list = im.keys ? p.w.list_k + static_cast<int64_t>(line) * p.w.cap_k
                         : p.w.list_q + static_cast<int64_t>(line) * p.w.cap_q;
          if (!kBF16 && im.g != amax_g) {
            amax_g = im.g;
            const int chunks = static_cast<int>(p.w.Sp / 128);
            float a = 0.f;
            for (int i = lane; i < chunks; i += 32) a = fmaxf(a, p.w.amax[static_cast<int64_t>(im.g) * chunks + i]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
            // exponent of the largest |do| -> [2^-4, 2^-3); all zero or not finite: unscaled
            ds_scale = a > 0.f && a <= 65504.f ? ldexpf(1.f, -4 - ilogbf(a)) : 1.f;
          }
          im.ds_scale = ds_scale;
        }
        if (lane == 0 && lin < n_items) lin = atomicAdd(p.w.next, 1);  // the next one, in flight over this one
        const int slot = it & 1;
        ok = c.wait_all(c.own_empty(slot), ((it >> 1) & 1) ^ 1);
        if (!ok) break;
        ++it;
        const int b = im.g / p.H, h = im.g % p.H;
        if (lane == 0) {
          items[slot] = im;
          if (im.keys >= 0 && im.n > 0) {
            mbar_arrive_expect_tx(c.own_full(slot), 2 * L::kOwn);
            const uint32_t dst = c.own + slot * 2 * L::kOwn;
            tma_load_4d(dst, im.keys ? &maps.ok : &maps.oq, c.own_full(slot), 0, im.tile * kM, h, b);
            tma_load_4d(dst + L::kOwn, im.keys ? &maps.ov : &maps.odo, c.own_full(slot), 0, im.tile * kM, h, b);
          } else {
            mbar_arrive(c.own_full(slot));
          }
        }
        nown = it;
        __syncwarp();
        if (im.keys < 0) break;
        if (lane == 0) {
          const int N = im.keys ? NK : NQ;
          uint32_t next = im.n > 0 ? list[0] : 0;
          for (int j = 0; j < im.n; ++j, ++t) {
            const int s = t % kStages;
            const uint32_t ent = next;
            if (j + 1 < im.n) next = list[j + 1];
            if (!c.wait(c.empty(s), ((t / kStages) & 1) ^ 1)) {
              ok = false;
              break;
            }
            const int row = static_cast<int>(ent & 0x3fffu) * N;
            ents[2 * s] = static_cast<int32_t>(ent);
            const uint32_t dst = c.walk + s * 2 * L::kWalk;
            mbar_arrive_expect_tx(c.full(s), 2 * N * kD * 2 + (im.keys ? 2 * N * 4 : 0));
            tma_load_4d(dst, im.keys ? &maps.wq : &maps.wk, c.full(s), 0, row, h, b);
            tma_load_4d(dst + L::kWalk, im.keys ? &maps.wdo : &maps.wv, c.full(s), 0, row, h, b);
            if (im.keys) {
              const int64_t at = im.g * p.w.Sp + row;
              bulk_load(c.stat + s * 2 * N * 4, p.w.stat_lse + at, N * 4, c.full(s));
              bulk_load(c.stat + s * 2 * N * 4 + N * 4, p.w.stat_delta + at, N * 4, c.full(s));
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
    } else if (warp == 1 && lane == 0) {
      // -------------------------------------------------------- MMA issuer
      constexpr uint32_t kIdescAcc = idesc_f16(kM, kD, kBF16, false, true);
      // S (own1 x walk1) or dP (own2 x walk2) of the item in `slot`, block in stage s
      auto issue_scores = [&](bool second, int keys, int slot, int s) {
        const uint32_t a = c.own + (2 * slot + second) * L::kOwn;
        const uint32_t w = c.walk + (2 * s + second) * L::kWalk;
        const uint32_t d = c.tmem + (second ? kColDP : kColS);
        const uint32_t idesc = keys ? idesc_f16(kM, NK, kBF16, false, false) : idesc_f16(kM, NQ, kBF16, false, false);
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk)
          tc_mma_ss(d, sdesc_sw128(a + kk * 32, 16, 1024), sdesc_sw128(w + kk * 32, 16, 1024), idesc, kk > 0 ? 1u : 0u);
        tc_commit(second ? c.dp_full() : c.s_full());
      };
      // acc += (P or dS in TMEM) x walk tile
      auto issue_acc = [&](uint32_t acc, uint32_t a, uint32_t w, int N, bool first) {
        for (int kk = 0; kk < N / 16; ++kk)
          tc_mma_ts(c.tmem + acc, c.tmem + a + kk * 8, sdesc_sw128(w + kk * 2048, L::kWalk, 1024), kIdescAcc,
                    (!first || kk > 0) ? 1u : 0u);
      };
      int it = 0;  // items taken
      int keys = 0, n = 0, slot = 0;
      auto fetch = [&](int& keys_, int& n_, int& slot_) -> bool {  // false: no more items
        slot_ = it & 1;
        if (!c.wait(c.own_full(slot_), (it >> 1) & 1)) return false;
        ++it;
        keys_ = c.items[slot_].keys;
        n_ = c.items[slot_].n;
        return keys_ >= 0;
      };
      int t = 0, tk = 0, na = 0;  // blocks, blocks of dk / dv items, items with blocks
      bool run = true;
      while (run) {
        if (!fetch(keys, n, slot)) break;
        if (n == 0) {  // nothing to multiply: the compute warps store zeros
          mbar_arrive(c.own_empty(slot));
          continue;
        }
        if (!c.wait(c.full(t % kStages), (t / kStages) & 1) || !c.wait(c.s_empty(), (t & 1) ^ 1) ||
            !c.wait(c.dp_empty(), (t & 1) ^ 1))
          break;
        tc_fence_after();
        issue_scores(false, keys, slot, t % kStages);
        issue_scores(true, keys, slot, t % kStages);
        if (n == 1) tc_commit(c.own_empty(slot));
        bool done = false;  // this chain of blocks is through
        int j = 0;
        while (!done) {
          // the block after this one, of this item or the next; the chain
          // ends before an item without blocks (waiting for the one behind it
          // would wait for this item's own slot)
          int nkeys = keys, nn = n, nslot = slot, nj = j + 1;
          bool more = true;
          if (nj >= n) {
            nj = 0;
            if (!fetch(nkeys, nn, nslot)) {
              more = run = false;
            } else if (nn == 0) {
              mbar_arrive(c.own_empty(nslot));
              more = false;
            }
          }
          run = run && !*c.abort_flag;
          const int s = t % kStages, s1 = (t + 1) % kStages;
          bool ok = true;
          if (more) {
            ok = c.wait(c.full(s1), ((t + 1) / kStages) & 1) && c.wait(c.s_empty(), t & 1);
            if (ok) {
              tc_fence_after();
              issue_scores(false, nkeys, nslot, s1);
            }
          }
          const bool first = j == 0;
          if (first) ok = ok && c.wait(c.acc_empty(), (na & 1) ^ 1);
          if (keys) {
            ok = ok && c.wait(c.p_full(), tk & 1);
            if (ok) {
              tc_fence_after();
              issue_acc(kColV, kColP, c.walk + (2 * s + 1) * L::kWalk, NK, first);
              tc_commit(c.p_empty());
              ++tk;
            }
          }
          if (more) {
            ok = ok && c.wait(c.dp_empty(), t & 1);
            if (ok) {
              tc_fence_after();
              issue_scores(true, nkeys, nslot, s1);
              if (nj == nn - 1) tc_commit(c.own_empty(nslot));
            }
          }
          ok = ok && c.wait(c.ds_full(), t & 1);
          if (!ok) {
            run = false;
            break;
          }
          tc_fence_after();
          issue_acc(kColK, kColDS, c.walk + 2 * s * L::kWalk, keys ? NK : NQ, first);
          tc_commit(c.ds_empty());
          tc_commit(c.empty(s));
          if (j == n - 1) {
            tc_commit(c.acc_full());
            ++na;
          }
          ++t;
          done = !more;
          keys = nkeys, n = nn, slot = nslot, j = nj;
        }
      }
      tc_commit(c.drain());
      mbar_drain(c.drain(), 0, p.status);
    }
    __syncwarp();
    tc_fence_before();
    named_barrier_sync(1, kThreads);
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(c.tmem, 512);
    }
  } else {
    setmaxnreg_inc<kRegsCompute>();
    // ------------------------------------------------------------ compute
    const int wg = (warp >> 2) - 1, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = c.tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    int it = 0, t = 0, tk = 0, na = 0;
    bool ok = true;
    while (ok) {
      const int slot = it & 1;
      if (!c.wait_all(c.own_full(slot), (it >> 1) & 1)) break;
      ++it;
      const Item im = c.items[slot];
      if (im.keys < 0) break;
      const int b = im.g / p.H, h = im.g % p.H;
      const int own = im.tile * kM + row;
      if (im.keys) {
        for (int j = 0; j < im.n && ok; ++j, ++t, ++tk)
          ok = compute_block<NK, true, kBF16>(c, p, wg, lane, quarter, t, tk, 0.f, 0.f, im.ds_scale);
      } else {
        const float nl = p.w.stat_lse[im.g * p.w.Sp + own], nd = p.w.stat_delta[im.g * p.w.Sp + own];
        for (int j = 0; j < im.n && ok; ++j, ++t)
          ok = compute_block<NQ, false, kBF16>(c, p, wg, lane, quarter, t, tk, nl, nd, im.ds_scale);
      }
      if (!ok) break;
      if (im.n > 0) {
        ok = c.wait_all(c.acc_full(), na & 1);
        if (!ok) break;
        ++na;
        tc_fence_after();
      }
      const float unscale = kBF16 ? 1.f : 1.f / kF16PScale;
      const float grad_scale = kBF16 ? p.scale : p.scale * unscale / im.ds_scale;
      // dk / dv: warpgroup 0 stores dv, 1 dk; dq: half of the channels each
      const bool dv = im.keys && wg == 0;
      const uint32_t col = dv ? kColV : im.keys ? kColK : kColK + wg * 32;
      uint8_t* dst = static_cast<uint8_t*>(im.keys ? (dv ? p.dv : p.dk) : p.dq) +
                     2 * (im.keys ? (dv ? b * p.dv_sb + h * p.dv_sh + own * p.dv_ss
                                        : b * p.dk_sb + h * p.dk_sh + own * p.dk_ss)
                                  : b * p.dq_sb + h * p.dq_sh + own * p.dq_ss + wg * 32);
      const float scale = dv ? unscale : grad_scale;
      const bool in = own < (im.keys ? p.Sk : p.Sq);
      uint32_t r0[32], r1[32];
      if (im.n > 0) {
        tmem_ld32(lane_addr + col, r0);
        if (im.keys) tmem_ld32(lane_addr + col + 32, r1);
        tmem_wait_ld(r0);
        tmem_wait_ld(r1);
        tc_fence_before();
        warp_arrive(c.acc_empty(), lane);
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) r0[e] = r1[e] = 0u;
      }
      warp_arrive(c.own_empty(slot), lane);
      if (in) {
        store32<kBF16>(r0, dst, scale);
        if (im.keys) store32<kBF16>(r1, dst + 64, scale);
      }
    }
    tc_fence_before();
    named_barrier_sync(1, kThreads);
  }
}

template <int NK, int NQ, bool kBF16>
int32_t launch(const Maps& maps, const BwdParams& p, int grid, cudaStream_t stream) {
  auto kern = bsa_bwd_sm100_kernel<NK, NQ, kBF16>;
  constexpr int smem = Layout<(NK > NQ ? NK : NQ)>::kDynSmem;
  // a build launched with fewer registers than the split hands out would wait forever
  static const int launch_regs = [] {
    cudaFuncAttributes fa{};
    return cudaFuncGetAttributes(&fa, bsa_bwd_sm100_kernel<NK, NQ, kBF16>) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (launch_regs < kLaunchRegs) return SAF_ERR_UNSUPPORTED;
  SAF_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kern<<<grid, kThreads, smem, stream>>>(maps, p);
  SAF_CUDA_TRY(cudaGetLastError());
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
  int32_t rc;
  if ((rc = make_qkv_map(&maps.oq, q, kM)) != SAF_OK || (rc = make_qkv_map(&maps.odo, dout, kM)) != SAF_OK ||
      (rc = make_qkv_map(&maps.ok, k, kM)) != SAF_OK || (rc = make_qkv_map(&maps.ov, v, kM)) != SAF_OK)
    return rc;
  maps.wq = maps.oq, maps.wdo = maps.odo, maps.wk = maps.ok, maps.wv = maps.ov;
  if (bm != kM &&
      ((rc = make_qkv_map(&maps.wq, q, bm)) != SAF_OK || (rc = make_qkv_map(&maps.wdo, dout, bm)) != SAF_OK))
    return rc;
  if (bn != kM && ((rc = make_qkv_map(&maps.wk, k, bn)) != SAF_OK || (rc = make_qkv_map(&maps.wv, v, bn)) != SAF_OK))
    return rc;
  BwdParams p{};
  p.H = static_cast<int>(q->H), p.Sq = static_cast<int>(q->S), p.Sk = static_cast<int>(k->S);
  p.BH = static_cast<int>(q->B * q->H);
  p.scale = sm_scale;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.dq = dq->data, p.dk = dk->data, p.dv = dv->data;
  p.dq_sb = dq->stride_b, p.dq_sh = dq->stride_h, p.dq_ss = dq->stride_s;
  p.dk_sb = dk->stride_b, p.dk_sh = dk->stride_h, p.dk_ss = dk->stride_s;
  p.dv_sb = dv->stride_b, p.dv_sh = dv->stride_h, p.dv_ss = dv->stride_s;
  p.w = w;
  p.status = device_status_ptr();
  p.budget_ns = wait_budget_ns();
  if (p.status == nullptr) return SAF_ERR_CUDA;
  int dev = 0, sms = 0;
  SAF_CUDA_TRY(cudaGetDevice(&dev));
  SAF_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const int64_t items = static_cast<int64_t>(p.BH) * (w.lines_q + w.lines_k);
  const int grid = static_cast<int>(items < sms ? items : sms);
#define SAF_BWD_CASE(NK_, NQ_)                                                  \
  if (bm == NK_ && bn == NQ_)                                                   \
    return q->dtype == SAF_BF16 ? launch<NK_, NQ_, true>(maps, p, grid, stream) \
                                : launch<NK_, NQ_, false>(maps, p, grid, stream);
  SAF_BWD_CASE(128, 128)
  SAF_BWD_CASE(64, 64)
  SAF_BWD_CASE(64, 128)
  SAF_BWD_CASE(128, 64)
#undef SAF_BWD_CASE
  return SAF_ERR_UNSUPPORTED;
}

}  // namespace saf
