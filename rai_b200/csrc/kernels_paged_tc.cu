// Attention of a chunk over a paged cache on the 5th-generation tensor cores:
// f16 / bf16, head sizes up to 128. The mathematics, the masks and the line of
// tiles cut over the CTAs are those of kernels_paged_attn.cu.
//
// A CTA walks a row tile of one KV head through the cache in tiles of 128
// tokens:
//   S = Q K^T   tcgen05.mma, Q and K in shared memory, S in TMEM (f32)
//   P = 2^(c S - c m), row sums   two warpgroups, one row per thread
//   O += P V    tcgen05.mma, P in TMEM over S, V in shared memory, O in TMEM
// with two S and O in TMEM, halves A and B, that take turns: while a
// warpgroup works on its S, the tensor core runs the other half's P V and next
// Q K^T. With many query rows (prompts) the halves are the upper and lower
// 128 of 256 flattened rows (group heads x chunk rows). With up to 128 (DUO:
// decoding, draft verification) both take the same rows, A the even and B the
// odd tiles of an item, and A joins the two at the item's end.
//
// Per tile of 256 rows and head size 128 that is 2,048 cycles of tensor core
// and, at 16 exponentials a cycle, 2,048 cycles of the special function units
// (1.1 us); a tile takes 2.1 to 2.4 us, the rest being the way S -> registers
// -> P that the halves do not wholly hide from each other. With few rows HBM
// bounds it: a tile's K and V are 64 KB, 1.45 us of an SM's share of the
// bandwidth, against 0.55 us of tensor core; warps whose rows do not exist
// skip the softmax.
//
// (Two row halves in turn, P in place of S and a maximum that seldom moves are
// a published arrangement of attention for these tensor cores; the line of
// tiles, the paged loads, the form for few rows and the handling of masked V
// are this file's own.)
//
// The running maximum is lazy: m only moves (and O is only rescaled, in TMEM)
// when a row's maximum passes it by more than 2^8; until then probabilities
// grow up to 2^8, which f32 sums and the 16-bit types hold.
//
// Warps: 0-3 and 4-7 softmax of halves A and B, 8 TMEM and MMA issue (one
// thread; the MMAs of one thread run in issue order, so the next Q K^T may be
// issued over a P that P V still reads), 9 K and V by TMA, a piece of a page
// per lane (DUO: and the queries, two buffers), 10-11 the masked V tiles, which
// are looked through before the MMA gets them, and the queries. Pages that
// TMA cannot fetch (sizes that are not 8 x 2^i or whole tiles) come by 16-byte
// copies of warps 10-11. Tiles lie in the 128-byte swizzle the MMA reads,
// K-major for Q K^T and N-major for P V. Every wait is bounded; on a timeout
// all roles stop, what is in flight is waited for and the TMEM columns are
// released.
#include <cuda_runtime.h>

#include <mutex>

#include "paged_attn.cuh"

namespace rai {

namespace {

using namespace paged_attn;

constexpr int kTcThreads = 12 * 32;
constexpr int kProducers = 64;

template <int DT_, int HD_, bool DUO_>
struct Tc {
  static constexpr int DT = DT_, HD = HD_, NT = 128;
  static constexpr bool DUO = DUO_;
  static constexpr int MT = DUO ? 128 : 256;
  static constexpr int kTileB = NT * HD * 2;  // a K or V tile
  static constexpr int kQB = 256 * HD * 2;    // DUO: two buffers
  static constexpr int kSlots = HD == 128 ? 5 : 10;
  static constexpr int kSmem = kQB + kSlots * kTileB + 1024;
  static constexpr int kPartFloats = MT * (HD + 2);
  // A probability is at most 2^8 of the kept maximum's: 2^15 with the factor.
  static constexpr float kPShift = DT == kF16 ? 7.f : 0.f;
  static constexpr uint32_t kFmt = DT == kBF16 ? 1u : 0u;
  // Instruction descriptor: D f32 (bits 4-5 = 1), A and B of one type (7-9,
  // 10-12), B's major-ness (16), N >> 3 (17-22), M >> 4 (24-28).
  static constexpr uint32_t kIdescQK = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr uint32_t kIdescPV =
      (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | (((uint32_t)HD >> 3) << 17) | ((128u >> 4) << 24);
};

constexpr float kLazy = 8.f;  // log2 units
// Few rows and heads wider than 64: from how many tokens a sequence, and a
// call's sequences and KV heads together, can have this kernel is the faster
// one. (Device time, calls in a captured graph, one row a sequence, tables as
// wide as the sequences; 8 KV heads of 128: 256 x 1,000 tokens 302 us here and
// 430 us on mma.sync, 64 x 2,000 151 / 213, 64 x 1,000 104 / 115, 16 x 2,000
// 50 / 61; 16 x 1,000 36 / 35, 1 x 16,000 39 / 38, 64 x 700 89 / 85, 1 x 4,000
// 34 / 20; 256 x 300 143 / 156 goes the slower way. Heads of 64, 64 x 2,000:
// 67 / 32.) The host knows the table's width, not the lengths: short sequences
// in a wide table come here too.
constexpr long long kTcFewRowsTokens = 768, kTcFewRowsTotal = 131072;

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// Operand descriptors: 128-byte swizzle, rows of 128 bytes, 8-row atoms 1024
// bytes apart (SBO); in the low word the address and the distance of the
// 64-element blocks of an N-major operand (LBO), the high word is constant.
// The issuing thread is on every tile's critical path, so a step of K costs it
// one addition to each low word.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return ((addr & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void tm_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// clean_chunk() of this thread's share of the V tile that begins at token t0.
template <typename C>
__device__ __forceinline__ bool look_through(uint32_t base, int t0, const Item& it, int tid) {
  constexpr int kChunks = C::HD / 8, kRowsPer = kProducers / kChunks;
  const int chunk = tid % kChunks, r0 = tid / kChunks;
  bool bad = false;
#pragma unroll 8
  for (int i = 0; i < C::NT / kRowsPer; ++i) {
    const int row = r0 + i * kRowsPer;
    bad |= clean_chunk<C::DT>(base + tile_at(C::NT, row, chunk), t0 + row, it);
  }
  return bad;
}

// Requests the item's query rows, by THREADS threads. Rows that do not exist
// keep what they held: no row of S depends on another's.
template <typename C, int THREADS>
__device__ __forceinline__ void load_queries(const Params& p, const Item& it, int kv_head, uint32_t sq, int tid) {
  constexpr int kChunks = C::HD / 8, kRowsPer = THREADS / kChunks;
  const int chunk = tid % kChunks, r0 = tid / kChunks;
  const bool in_head = chunk * 8 < p.a.c.hd;
  const uint16_t* q = static_cast<const uint16_t*>(p.a.q) + (long long)it.start * p.a.q_row + (long long)kv_head * p.a.group * p.a.q_head + chunk * 8;
#pragma unroll 1
  for (int i0 = 0; i0 * kRowsPer < it.nf; i0 += 8) {
    const uint16_t* src[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int f = it.f0 + r0 + (i0 + i) * kRowsPer, qi = (int)p.group_div.quot(f), j = f - qi * p.a.group;
      src[i] = in_head ? q + qi * p.a.q_row + j * p.a.q_head : q;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + (i0 + i) * kRowsPer;
      if (r < it.nf) cp_async16_or_zero(sq + tile_at(C::MT, r, chunk), src[i], in_head);
    }
  }
  cp_async_commit();
}

constexpr int kLanded = 8;  // V tiles between their landing and their hand-over
// V tile k goes through the hands of warps 10 and 11. (Besides the masked ones
// one in 1024, since their waits for the next are bounded.)
__device__ __forceinline__ bool by_hand(const Params& p, const Item& it, uint32_t k, int t0, int nt) {
  return (k & 1023u) == 1023u || tile_masked(it, t0, nt, p.a.window, p.group_div);
}

// What the issuing thread has to know of a tile: it is the last of its item;
// the last of its item here; the last of the CTA.
enum : uint32_t { kLastOfItem = 1, kLastHere = 2, kLastOfCta = 4 };
template <int MT, int NT>
__device__ __forceinline__ uint32_t flags_of(const Params& p, const Cursor<MT, NT>& cur, long long end) {
  uint32_t f = (cur.last_of_item() ? kLastOfItem : 0) | (cur.ends(end) ? kLastHere : 0);
  // The next tile of the line lies behind the next item's cost.
  if (cur.pos + 1 + (cur.last_of_item() ? p.item_cost : 0) >= end) f |= kLastOfCta;
  return f;
}

// The lowest n bits, n cut to 0 .. 32.
__device__ __forceinline__ uint32_t bits_to(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

template <typename C, bool CAP, bool TMA>
__global__ void __launch_bounds__(kTcThreads, 1)
    paged_attn_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ KvMaps maps, int box,
                         const __grid_constant__ CUtensorMap q_map, bool q_tma) {
  constexpr int DT = C::DT, HD = C::HD, MT = C::MT, NT = C::NT;
  constexpr bool DUO = C::DUO;
  constexpr int kQThreads = DUO ? 32 : kProducers;
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long sh[kPlanWords];
  __shared__ uint64_t kv_full[C::kSlots], kv_empty[C::kSlots], q_full[2], q_empty[2], s_full[2], p_full[2], o_done[2], drained;
  __shared__ uint64_t b_ready, b_read;  // DUO: half B's sums are there, were read
  __shared__ float2 b_sums[DUO ? 128 : 1];  // half B's (m, l)
  __shared__ uint64_t landed[kLanded], looked;
  __shared__ uint32_t flags[C::kSlots];  // of the tile whose K is in the slot
  __shared__ uint32_t tmem_slot;
  __shared__ int poison[4];  // ordinal + 1 of an item with masked V values that are not finite
  const uint32_t sq = (smem_u32(smem_raw) + 1023) & ~1023u, skv = sq + C::kQB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedChunk& ch = p.a.c;
  uint32_t* err = ch.err;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&kv_full[i], TMA ? 1 : kProducers);
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(&b_ready, 4);
    mbar_init(&b_read, 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], q_tma ? 1 : kQThreads);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(&drained, 1);
    mbar_init(&looked, 2);
    for (int i = 0; i < kLanded; ++i) mbar_init(&landed[i], 1);
    for (int i = 0; i < 4; ++i) poison[i] = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait_prior();
  pdl_launch_dependents();
  const Range rg = plan<MT, NT, kTcThreads>(p, blockIdx.x, sh);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  const long long begin = rg.begin, end = rg.end;

  // 3 x 168 registers at launch: 208 for each softmax warpgroup, 88 for the
  // others (208 + 208 + 88 = 504).
  if (begin >= end && threadIdx.x == 0) reinterpret_cast<Cut*>(p.a.part)[blockIdx.x] = Cut{};
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (begin < end && TMA && warp == 9) {
      // ---------------- K and V by TMA ----------------
      Cursor<MT, NT> cur;
      cur.seek(p, rg);
      TilePieces<NT, HD / 64, 2> pieces;
      pieces.fetch(ch, cur.it, (cur.it.first + cur.tile) * NT, box, lane);
      uint32_t issued = 0, by_hands = 0;
      uint32_t handed = 0;  // bit i: fetch issued - 1 - i is a V tile that goes by hand
      int items = 0;
      bool ok = true, fresh = true;
      for (uint32_t k = 0; cur.pos < end && ok; ++k) {
        const Item& it = cur.it;
        const int t0 = (it.first + cur.tile) * NT;
        const bool hand = by_hand(p, it, k, t0, NT);
        const bool queries = DUO && fresh;
        if (queries) {
          if (items >= 2) ok = __all_sync(~0u, wait_bar(&q_empty[items & 1], (items / 2 - 1) & 1, err));
          if (!ok) break;
          load_queries<C, 32>(p, it, cur.head, sq + (items & 1) * MT * HD * 2, lane);
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t n = 2 * k + kv, slot = n % C::kSlots, use = n / C::kSlots;
          if (ok && use > 0) ok = __all_sync(~0u, wait_bar(&kv_empty[slot], (use - 1) & 1, err));
          if (ok) {
            if (kv == 0 && lane == 0) flags[slot] = flags_of<MT, NT>(p, cur, end);
            pieces.load(ch, it, t0, box, lane, kv ? &maps.v : &maps.k, cur.head, skv + slot * C::kTileB,
                        kv && hand ? &landed[by_hands % kLanded] : &kv_full[slot]);
            ++issued;
            handed = handed << 1 | (kv && hand ? 1u : 0u);
            if (kv && hand) ++by_hands;
          }
        }
        if (queries) {
          cp_async_wait<0>();
          fence_async();
          mbar_arrive(&q_full[items & 1]);
          ++items;
        }
        fresh = cur.last_of_item();
        cur.next(p);
        if (cur.pos < end) pieces.fetch(ch, cur.it, (cur.it.first + cur.tile) * NT, box, lane);
      }
      // What was requested lands before the CTA ends.
      for (uint32_t i = 0; i < C::kSlots && i < issued; ++i, handed >>= 1) {
        const uint32_t n = issued - 1 - i;
        if (handed & 1u) {
          --by_hands;
          wait_bar(&landed[by_hands % kLanded], by_hands / kLanded & 1, nullptr);
        } else {
          wait_bar(&kv_full[n % C::kSlots], n / C::kSlots & 1, nullptr);
        }
      }
    } else if (begin < end && TMA && warp >= 10) {
      // ---------------- queries; masked V tiles ----------------
      const int tid = threadIdx.x - 10 * 32;
      Cursor<MT, NT> cur;
      cur.seek(p, rg);
      if (tid == 0) leave_cut<MT, NT>(p, rg, cur, blockIdx.x);
      int items = 0;
      bool fresh = true;
      uint32_t asked = 0, seen = 0;  // query tiles requested by TMA, V tiles that went by hand
      for (uint32_t k = 0; cur.pos < end; ++k) {
        const Item& it = cur.it;
        if (!DUO && fresh) {
          // (By TMA warp 10 alone asks. Warp 11 has no part in it, so nothing
          // would keep the next phase from completing before it looked.)
          if (k > 0 && (!q_tma || warp == 10) && !__all_sync(~0u, wait_bar(&q_empty[0], (items - 1) & 1, err))) break;
          if (q_tma) {
            // group heads x (256 / group) rows, as the flattened rows lie
            ++asked;
            if (tid == 0) {
              mbar_arrive_expect_tx(&q_full[0], MT * HD * 2);
              const int qi = it.start + (int)p.group_div.quot(it.f0);
#pragma unroll
              for (int x = 0; x < HD / 64; ++x) tma_load3(sq + x * MT * 128, &q_map, x * 64, cur.head * p.a.group, qi, &q_full[0]);
            }
          } else {
            load_queries<C, kProducers>(p, it, cur.head, sq, tid);
            cp_async_wait<0>();
            fence_async();
            mbar_arrive(&q_full[0]);
          }
          fresh = false;
        }
        const int t0 = (it.first + cur.tile) * NT;
        if (by_hand(p, it, k, t0, NT)) {
          if (!__all_sync(~0u, wait_bar(&landed[seen % kLanded], seen / kLanded & 1, err))) break;
          const uint32_t slot = (2 * k + 1) % C::kSlots;
          if (tile_masked(it, t0, NT, p.a.window, p.group_div) && look_through<C>(skv + slot * C::kTileB, t0, it, tid))
            *(volatile int*)&poison[items & 3] = items + 1;
          fence_async();
          __syncwarp();
          // Both wait for both shares, so that neither is ever two phases of
          // a barrier ahead of the other: a wait by parity takes two for none.
          // (Waits are bounded, so this is no bar.sync, which a warp that gave
          // up would leave the other in.)
          if (lane == 0) mbar_arrive(&looked);
          if (!__all_sync(~0u, wait_bar(&looked, seen & 1, err))) break;
          if (tid == 0) mbar_arrive(&kv_full[slot]);
          ++seen;
        }
        if (cur.last_of_item()) {
          fresh = true;
          ++items;
        }
        cur.next(p);
      }
      // What was requested lands before the CTA ends.
      if (asked && tid == 0) wait_bar(&q_full[0], (asked - 1) & 1, nullptr);
    } else if (begin < end && !TMA && warp >= 10) {
      // ---------------- K, V and queries by 16-byte copies ----------------
      const int tid = threadIdx.x - 10 * 32;
      constexpr int kChunks = HD / 8, kRowsPer = kProducers / kChunks;  // rows of 16-byte chunks at a time
      constexpr int kLag = 2;  // tiles in flight before the oldest is handed over
      const int chunk = tid % kChunks, r0 = tid / kChunks;
      const bool in_head = chunk * 8 < ch.hd;
      Cursor<MT, NT> cur;
      cur.seek(p, rg);
      if (tid == 0) leave_cut<MT, NT>(p, rg, cur, blockIdx.x);
      TilePages<NT> pages;
      pages.fetch(ch, cur.it, (cur.it.first + cur.tile) * NT, lane);
      int items = 0;
      uint32_t n = 0, handed = 0;  // K and V tiles fetched, handed over
      bool ok = true, fresh = true;
      uint32_t look = 0;  // bit i: fetch n - 1 - i is a V tile to look through
      Item seen = cur.it;  // the item of the fetches in flight
      int look_t0[2] = {0, 0};  // first tokens of the V tiles in flight
      auto hand = [&](int age) {  // the fetch `handed` has landed
        const uint32_t slot = handed % C::kSlots;
        if ((look >> age & 1u) && look_through<C>(skv + slot * C::kTileB, handed / 2 & 1 ? look_t0[1] : look_t0[0], seen, tid))
          *(volatile int*)&poison[items & 3] = items + 1;
        fence_async();
        mbar_arrive(&kv_full[slot]);
        ++handed;
      };
      bool first = true;
      while (cur.pos < end && ok) {
        if (fresh) {
          // A new item: what is in flight is handed over under the old one's
          // ordinal, then the query rows are fetched.
          cp_async_wait<0>();
          while (handed < n) hand((int)(n - 1 - handed));
          if (!first) {
            ++items;
            ok = wait_bar(&q_empty[0], (items - 1) & 1, err);
            if (!ok) break;
          }
          first = false;
          seen = cur.it;
          load_queries<C, kProducers>(p, cur.it, cur.head, sq, tid);
          cp_async_wait<0>();
          fence_async();
          mbar_arrive(&q_full[0]);
          fresh = false;
        }
        const Item& it = cur.it;
        const int t0 = (it.first + cur.tile) * NT;
        pages.check(ch, it, t0, lane);
#pragma unroll 1
        for (int kv = 0; kv < 2 && ok; ++kv) {
          const uint32_t slot = n % C::kSlots, use = n / C::kSlots;
          if (use > 0 && !wait_bar(&kv_empty[slot], (use - 1) & 1, err)) {
            ok = false;
            break;
          }
          const uint32_t base = skv + slot * C::kTileB;
          const uint16_t* src = static_cast<const uint16_t*>(kv ? ch.v : ch.k) + (long long)cur.head * (kv ? ch.v_head : ch.k_head) + chunk * 8;
          long long off[NT / 32];
          pages.offsets(ch, t0, lane, kv ? ch.v_page : ch.k_page, kv ? ch.v_slot : ch.k_slot, off);
          // Eight copies' addresses at a time: their shuffles overlap.
#pragma unroll
          for (int i0 = 0; i0 < NT / kRowsPer; i0 += 8) {
            long long o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int row = r0 + (i0 + i) * kRowsPer;
              const long long x = __shfl_sync(~0u, off[(i0 + i) * kRowsPer / 32], row & 31);
              o[i] = in_head ? x : -1;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
              cp_async16_or_zero(base + tile_at(NT, r0 + (i0 + i) * kRowsPer, chunk), o[i] >= 0 ? src + o[i] : src, o[i] >= 0);
          }
          cp_async_commit();
          if (kv == 0 && tid == 0) flags[slot] = flags_of<MT, NT>(p, cur, end);
          if (kv) (n / 2 & 1 ? look_t0[1] : look_t0[0]) = t0;
          look = look << 1 | (kv && tile_masked(it, t0, NT, p.a.window, p.group_div) ? 1u : 0u);
          ++n;
          if (n - handed > (uint32_t)kLag) {
            cp_async_wait<kLag>();
            hand(kLag);
          }
        }
        if (cur.last_of_item()) fresh = true;
        cur.next(p);
        if (cur.pos < end) pages.fetch(ch, cur.it, (cur.it.first + cur.tile) * NT, lane);
      }
      cp_async_wait<0>();
      if (ok)
        while (handed < n) hand((int)(n - 1 - handed));
    } else if (begin < end && warp == 8) {
      // ---------------- MMA issue ----------------
      if (lane == 0) {
        // K of tile k is fetch 2k, V is fetch 2k + 1, fetch n in slot n % kSlots.
        struct Slot {
          uint32_t i, phase;
          __device__ __forceinline__ void skip() {  // two fetches on
            i += 2;
            if (i >= (uint32_t)C::kSlots) i -= C::kSlots, phase ^= 1;
          }
        } ks = {0, 0}, vs = {1, 0};
        // (A range may hold nothing but the beginning of an item's cost.)
        Cursor<MT, NT> start;
        start.seek(p, rg);
        bool ok = start.pos < end;
        int items = 0;
        uint32_t k = 0;
        auto qk = [&](int half) {
          const uint32_t a0 = desc_lo(sq + (DUO ? (items & 1) * MT * HD * 2 : half * 128 * 128), 16);
          const uint32_t b0 = desc_lo(skv + ks.i * C::kTileB, 16);
#pragma unroll
          for (int x = 0; x < HD / 16; ++x) {
            const uint32_t in = (x & 3) * 2;
            mma_ss(tmem + half * 128, a0 + (x >> 2) * (MT * 8) + in, b0 + (x >> 2) * (NT * 8) + in, C::kIdescQK, x > 0);
          }
          commit(&s_full[half]);
        };
        auto pv = [&](int half, bool add) {
          const uint32_t b0 = desc_lo(skv + vs.i * C::kTileB, NT * 128);
#pragma unroll
          for (int x = 0; x < NT / 16; ++x)
            mma_ts(tmem + 256 + half * HD, tmem + half * 128 + x * 8, b0 + x * 128, C::kIdescPV, add || x > 0);
          commit(&o_done[half]);
        };
        if constexpr (!DUO) {
          bool first = true;  // tile k is its item's first here
          uint32_t now = 0, next = 0;
          ok = ok && wait_bar(&q_full[0], 0, err) && wait_bar(&kv_full[0], 0, err);
          if (ok) {
            fence_after();
            next = flags[0];
            qk(0);
            qk(1);
            commit(&kv_empty[0]);
            ks.skip();
            if (next & kLastHere) commit(&q_empty[0]);
          }
          for (; ok; ++k) {
            now = next;
            ok = wait_bar(&kv_full[vs.i], vs.phase, err) && wait_bar(&p_full[0], k & 1, err);
            if (!ok) break;
            fence_after();
            pv(0, !first);
            if (!(now & kLastOfCta)) {
              if (now & kLastOfItem) {
                ++items;
                ok = wait_bar(&q_full[0], items & 1, err);
              }
              ok = ok && wait_bar(&kv_full[ks.i], ks.phase, err);
              if (!ok) break;
              fence_after();
              next = flags[ks.i];
              qk(0);
            }
            ok = wait_bar(&p_full[1], k & 1, err);
            if (!ok) break;
            fence_after();
            pv(1, !first);
            commit(&kv_empty[vs.i]);
            vs.skip();
            if (now & kLastOfCta) break;
            qk(1);
            commit(&kv_empty[ks.i]);
            ks.skip();
            if (next & kLastHere) commit(&q_empty[0]);  // tile k + 1 is its item's last here: the queries may go
            first = now & kLastOfItem;
          }
        } else {
          // Q K^T runs ahead of P V by one S of each half, in the line's order.
          bool q_fresh = true, q_more = true;
          int q_half = 0, v_half = 0, v_in = 0;
          uint32_t phase = 0, busy = 0;  // bit per half
          uint32_t ahead = 0, n_ahead = 0;  // flags of the tiles between, 4 bits each
          while (ok) {
            while (ok && q_more && !(busy >> q_half & 1u)) {
              if (q_fresh) ok = wait_bar(&q_full[items & 1], items >> 1 & 1, err);
              ok = ok && wait_bar(&kv_full[ks.i], ks.phase, err);
              if (!ok) break;
              fence_after();
              const uint32_t f = flags[ks.i];
              if (q_half == 0) qk(0); else qk(1);
              commit(&kv_empty[ks.i]);
              ks.skip();
              busy |= 1u << q_half;
              ahead |= f << (4 * n_ahead++);
              q_more = !(f & kLastOfCta);
              q_fresh = f & kLastHere;
              if (q_fresh) {
                commit(&q_empty[items & 1]);
                ++items;
              }
              q_half = f & kLastOfItem ? 0 : q_half ^ 1;
            }
            if (!ok) break;
            ok = wait_bar(&kv_full[vs.i], vs.phase, err) && wait_bar(&p_full[v_half], phase >> v_half & 1u, err);
            if (!ok) break;
            phase ^= 1u << v_half;
            busy &= ~(1u << v_half);
            fence_after();
            if (v_half == 0) pv(0, v_in >= 2); else pv(1, v_in >= 2);
            commit(&kv_empty[vs.i]);
            vs.skip();
            const uint32_t f = ahead & 15u;
            ahead >>= 4, --n_ahead;
            if (f & kLastOfCta) break;
            v_in = f & kLastOfItem ? 0 : v_in + 1;
            v_half = f & kLastOfItem ? 0 : v_half ^ 1;
          }
        }
        commit(&drained);
        wait_bar(&drained, 0, nullptr);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    if (begin < end) {
      // ---------------- softmax, one row per thread ----------------
      const int half = warp >> 2, row = threadIdx.x & 127;
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
      const uint32_t ts = tmem + half * 128 + lanes, to = tmem + 256 + half * HD + lanes;
      Cursor<MT, NT> cur;
      cur.seek(p, rg);
      int items = 0, in = 0;  // in: tiles of the item so far
      bool ok = true;
      float m = -INFINITY, l = 0.f;  // m: of the raw scores
      uint32_t k = 0, k_first = 0;   // this half's tiles; the item's first
      for (; cur.pos < end; ++in) {
        const Item& it = cur.it;
        const int r = DUO ? row : half * 128 + row;
        const int f = it.f0 + r, qi = (int)p.group_div.quot(f);
        const bool real = r < it.nf;
        const bool idle = __all_sync(~0u, !real);
        const int pos = real ? it.len - it.n + qi : -1;
        if (!DUO || (in & 1) == half) {
          ok = __all_sync(~0u, wait_bar(&s_full[half], k & 1, err));
          if (!ok) break;
          if (!idle) {
            const int t0 = (it.first + cur.tile) * NT;
            fence_after();
            uint32_t v[128];
#pragma unroll
            for (int x = 0; x < 4; ++x) tm_ld32(ts + 32 * x, v + 32 * x);
            tm_wait_ld();
            if constexpr (CAP) {
#pragma unroll
              for (int x = 0; x < 128; x += 2) {
                const float2 y = capped<DT>({__uint_as_float(v[x]), __uint_as_float(v[x + 1])}, p.a.scale, p.a.softcap, p.inv_cap);
                v[x] = __float_as_uint(y.x);
                v[x + 1] = __float_as_uint(y.y);
              }
            }
            if (tile_masked(it, t0, NT, p.a.window, p.group_div)) {
              // Columns from .. till as bits: two instructions an element (a
              // comparison with both ends was a branch each, 4 us a tile).
              const int from = max(it.lo, p.a.window > 0 ? pos - p.a.window + 1 : 0) - t0, till = pos - t0;
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const uint32_t bits = bits_to(till + 1 - 32 * w) & ~bits_to(from - 32 * w);
#pragma unroll
                for (int x = 0; x < 32; ++x) v[32 * w + x] = bits >> x & 1u ? v[32 * w + x] : 0xff800000u;
              }
            }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int x = 0; x < 128; x += 2)
              tops[x / 2 & 3] = fmaxf(tops[x / 2 & 3], fmaxf(__uint_as_float(v[x]), __uint_as_float(v[x + 1])));
            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            const bool move = top > m && (m == -INFINITY || (top - m) * p.c > kLazy);
            if (__any_sync(~0u, move)) {
              const float next = move ? top : m;
              const float fix = move && m != -INFINITY ? exp2_fast((m - next) * p.c) : 1.f;
              l *= fix;
              m = next;
              if (k > k_first) {
                ok = __all_sync(~0u, wait_bar(&o_done[half], (k - 1) & 1, err));
                if (!ok) break;
                fence_after();
#pragma unroll 1
                for (int x = 0; x < HD; x += 32) {
                  uint32_t o[32];
                  tm_ld32(to + x, o);
                  tm_wait_ld();
#pragma unroll
                  for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * fix);
                  tm_st32(to + x, o);
                }
              }
            }
            const float mc = (m == -INFINITY ? 0.f : m * p.c) - C::kPShift;
            float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
            const float2 cc = {p.c, p.c}, nm = {-mc, -mc};
#pragma unroll
            for (int x = 0; x < 64; ++x) {
              const float2 y = fma2({__uint_as_float(v[2 * x]), __uint_as_float(v[2 * x + 1])}, cc, nm);
              const float2 e = {exp2_fast(y.x), exp2_fast(y.y)};
              sum[x & 1] = add2(sum[x & 1], e);
              v[x] = pack<DT>(e.x, e.y);
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tm_st32(ts, v);
            tm_st32(ts + 32, v + 32);
            tm_wait_st();
            fence_before();
          }
          // Half B's O of the last item has been read before it is written anew.
          if (DUO && half == 1 && in == 1 && items > 0) {
            ok = __all_sync(~0u, wait_bar(&b_read, (items - 1) & 1, err));
            if (!ok) break;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[half]);
          ++k;
        }

        if (cur.ends(end)) {
          // ---- end of the item, or of this CTA's part of it ----
          if (k > k_first) {
            ok = __all_sync(~0u, wait_bar(&o_done[half], (k - 1) & 1, err));
            if (!ok) break;
            fence_after();
          }
          if (DUO && half == 1) {
            // Half A joins: it reads these sums, and O from the TMEM lanes that
            // its warps share with this half's.
            if (items > 0) {
              ok = __all_sync(~0u, wait_bar(&b_read, (items - 1) & 1, err));
              if (!ok) break;
            }
            b_sums[row] = make_float2(m, l);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b_ready);
          } else {
            float fix_a = 1.f, fix_b = 0.f;
            if (DUO) {
              ok = __all_sync(~0u, wait_bar(&b_ready, items & 1, err));
              if (!ok) break;
              fence_after();
              const float2 o = b_sums[row];
              const float top = fmaxf(m, o.x), ref = top == -INFINITY ? 0.f : top;
              fix_a = exp2_fast((m - ref) * p.c);
              fix_b = exp2_fast((o.x - ref) * p.c);
              l = l * fix_a + o.y * fix_b;
              m = top;
            }
            const bool two = DUO && in >= 1;  // half B has had a tile
            if (!idle) {
              const long long item_at = cur.pos - cur.tile;  // of its first tile
              const bool whole = item_at >= begin && cur.last_of_item();
              const bool poisoned = *(volatile int*)&poison[items & 3] == items + 1;
              const int j = f - qi * p.a.group, head = cur.head * p.a.group + j;
              const float inv = !whole ? 1.f : l > 0.f || l != l ? 1.f / l : 0.f;
              float* part = part_of(p, C::kPartFloats, blockIdx.x, items ? 1 : 0);
              uint16_t* out = static_cast<uint16_t*>(p.a.out) + (long long)(it.start + qi) * p.a.o_row + (long long)head * p.a.o_head;
#pragma unroll 1
              for (int x = 0; x < HD; x += 32) {
                uint32_t o[32];
                __syncwarp();
                tm_ld32(to + x, o);
                tm_wait_ld();
                if (DUO) {
                  uint32_t ob[32];
                  if (two) tm_ld32(to + HD + x, ob);
                  tm_wait_ld();
#pragma unroll
                  for (int y = 0; y < 32; ++y) {
                    float w = __uint_as_float(o[y]) * fix_a;
                    if (two && fix_b != 0.f) w += __uint_as_float(ob[y]) * fix_b;
                    o[y] = __float_as_uint(w);
                  }
                }
                if (real && !whole) {
#pragma unroll
                  for (int y = 0; y < 32; y += 4)
                    *reinterpret_cast<uint4*>(part + r * HD + x + y) = make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
                } else if (real) {
#pragma unroll
                  for (int y = 0; y < 32; y += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int z = 0; z < 4; ++z)
                      w[z] = pack<DT>(__uint_as_float(o[y + 2 * z]) * inv, __uint_as_float(o[y + 2 * z + 1]) * inv);
                    if (x + y < ch.hd) *reinterpret_cast<uint4*>(out + x + y) = make_uint4(w[0], w[1], w[2], w[3]);
                  }
                }
              }
              if (poisoned && real) {
                // A row that sees a V value which is not finite gets it after all.
                const int ta = it.first * NT + (int)max(0ll, begin - item_at) * NT, tb = (it.first + cur.tile + 1) * NT;
                const int from = max(max(ta, it.lo), p.a.window > 0 ? pos - p.a.window + 1 : 0), till = min(min(tb, it.hi), pos + 1);
#pragma unroll 1
                for (int col = 0; col < ch.hd; ++col) {
                  const float v = lost_values<DT, NT>(p, it, cur.head, col, from, till);
                  if (v != 0.f) {
                    if (whole) put<DT>(out, col, v);
                    else part[r * HD + col] = v;
                  }
                }
              }
              if (real && !whole) {
                part[MT * HD + r] = m == -INFINITY ? -INFINITY : m * p.c;
                part[MT * HD + MT + r] = l;
              } else if (real && p.a.lse) {
                p.a.lse[(long long)(it.start + qi) * (ch.nkv * p.a.group) + head] =
                    l > 0.f || l != l ? (m * p.c - C::kPShift) * kLn2 + logf(l) : -INFINITY;
              }
            }
            fence_before();
            __syncwarp();
            if (DUO && lane == 0) mbar_arrive(&b_read);
          }
          ++items;
          in = -1;
          m = -INFINITY;
          l = 0.f;
          k_first = k;
        }
        cur.next(p);
      }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 8) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

template <typename C, bool CAP, bool TMA>
cudaError_t launch(const AttnArgs& a, const KvMaps& maps, int box, cudaStream_t s) {
  CUtensorMap q_map;
  const bool q_tma = TMA && !C::DUO && 256 % a.group == 0 && make_q_map(a, 256 / a.group, &q_map);
  static std::once_flag once[64];
  static cudaError_t ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&] {
    ready[dev] = cudaFuncSetAttribute(paged_attn_tc_kernel<C, CAP, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (ready[dev] != cudaSuccess) return ready[dev];
  Params p;
  p.a = a;
  const long long frows = (long long)a.c.max_rows * a.group;
  p.row_tiles = (int)((frows + C::MT - 1) / C::MT);
  p.row_tiles_div = FastDiv(p.row_tiles);
  p.group_div = FastDiv(a.group);
  p.grid = device_sm_count();
  p.whole = p.direct = false;
  p.min_tiles = 10;
  // An item costs about 7 us beside its tiles of 2.1 us (capped ones take 4.9
  // us): three prompts of 3,000 tokens take 280 / 278 / 280 / 290 us at 2 / 3 /
  // 4 / 6, the capped chunks 162 / 163 / 162 / 165.
  p.item_cost = 3;
  p.c = a.softcap > 0.f ? kLog2e : a.scale * kLog2e;
  p.inv_cap = a.softcap > 0.f ? 1.f / a.softcap : 0.f;
  // Not launched ahead of its predecessor's end: a batch of prompts took 344
  // us so and 357 us with it when that was tried, long verification the same.
  paged_attn_tc_kernel<C, CAP, TMA><<<p.grid, kTcThreads, C::kSmem, s>>>(p, maps, box, q_map, q_tma);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_combine_kernel<C>, dim3(p.grid - 1, combine_grid_y(C::MT)), dim3(kCombineThreads), 0, s, p);
}

template <int DT, int HD>
cudaError_t choose(const AttnArgs& a, cudaStream_t s) {
  KvMaps maps;
  const int box = tma_box((int)a.c.page.d, 128);
  const bool tma = box && make_maps(a.c, a.dtype, box, &maps);
  const bool duo = (long long)a.c.max_rows * a.group <= 128, cap = a.softcap > 0.f;
  if (!tma) return cap ? launch<Tc<DT, HD, false>, true, false>(a, maps, box, s) : launch<Tc<DT, HD, false>, false, false>(a, maps, box, s);
  if (duo) return cap ? launch<Tc<DT, HD, true>, true, true>(a, maps, box, s) : launch<Tc<DT, HD, true>, false, true>(a, maps, box, s);
  return cap ? launch<Tc<DT, HD, false>, true, true>(a, maps, box, s) : launch<Tc<DT, HD, false>, false, true>(a, maps, box, s);
}

}  // namespace

bool paged_attention_tc_takes(const AttnArgs& a) {
  if (a.dtype == kF32 || a.c.hd > 128) return false;
  if ((long long)a.c.max_rows * a.group > 64) return true;
  const long long tokens = (long long)a.c.max_pages * a.c.page.d;
  return a.c.hd > 64 && tma_box((int)a.c.page.d, 128) && tokens >= kTcFewRowsTokens &&
         tokens * a.c.n_seqs * a.c.nkv >= kTcFewRowsTotal;
}

size_t paged_attention_tc_workspace(const AttnArgs& a) {
  return cut_bytes(device_sm_count()) +
         2ull * device_sm_count() * (a.c.hd <= 64 ? Tc<kBF16, 64, false>::kPartFloats : Tc<kBF16, 128, false>::kPartFloats) * 4;
}

cudaError_t paged_attention_tc(const AttnArgs& a, cudaStream_t s) {
  if (a.dtype == kF16) return a.c.hd <= 64 ? choose<kF16, 64>(a, s) : choose<kF16, 128>(a, s);
  return a.c.hd <= 64 ? choose<kBF16, 64>(a, s) : choose<kBF16, 128>(a, s);
}

}  // namespace rai
