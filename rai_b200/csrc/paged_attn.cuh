// What the two kernels of paged attention share: the line of token tiles and
// its cuts, the fetching of pages, the join of cut items, and elements.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "paged.h"

namespace rai {
namespace paged_attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kPlanWords = 22;

// All (sequence, row tile, KV head) items lie one after the other on a line,
// each item_cost + tiles long: tile i of an item that begins at s is at
// s + item_cost + i. Cut in equal ranges, one per CTA, the line gives CTAs with
// many short items fewer tiles (an item costs its queries' load, the filling
// of the pipeline and its output beside its tiles).
struct Params {
  AttnArgs a;
  int row_tiles, min_tiles, item_cost, grid;
  bool whole;   // items are short: none is cut
  bool direct;  // one CTA per item, in order
  float c;  // log2(e) * scale, or log2(e) when the scores are capped
  float inv_cap;  // 1 / softcap
  FastDiv row_tiles_div, group_div;
};

struct Item {
  int seq, start, n, len;  // rows and length of the sequence
  int f0, nf;              // flattened rows of the row tile
  int lo, hi;              // tokens that some row of the tile sees
  int first, tiles;        // token tiles
};

template <int MT, int NT>
__device__ __forceinline__ Item item_of(const Params& p, int unit) {
  Item it;
  it.seq = p.row_tiles_div.quot(unit);
  const int rt = unit - it.seq * p.row_tiles;
  const SeqRows r = seq_rows(p.a.c, it.seq);
  it.start = r.start, it.n = r.n, it.len = r.len;
  it.f0 = rt * MT;
  it.nf = min(MT, r.n * p.a.group - it.f0);
  it.lo = it.hi = it.first = it.tiles = 0;
  if (it.nf <= 0) return it;
  const int p0 = r.len - r.n;
  it.hi = p0 + (int)p.group_div.quot(it.f0 + it.nf - 1) + 1;
  const int plo = p0 + (int)p.group_div.quot(it.f0);
  if (p.a.window > 0) it.lo = max(0, plo - p.a.window + 1);
  it.tiles = 1;
  if (it.hi <= 0) {
    it.lo = it.hi = 0;
  } else {
    it.first = it.lo / NT;
    it.tiles = (it.hi + NT - 1) / NT - it.first;
  }
  return it;
}

__device__ __forceinline__ int length_of(const Params& p, const Item& it) { return it.tiles ? it.tiles + p.item_cost : 0; }

// The CTA's range [begin, end) of the line and the unit (sequence, row tile)
// it starts in. Every thread sums a run of units; a block scan places the
// runs. With p.whole the cuts move down to the starts of the items they fall
// in.
struct Range {
  long long total, per, begin, end;
  int unit;          // unit of `begin`
  long long before;  // length of one KV head's line before it
};
template <int MT, int NT, int THREADS>
__device__ __forceinline__ Range plan(const Params& p, long long cta, long long (&sh)[kPlanWords]) {
  const int units = p.a.c.n_seqs * p.row_tiles;
  const int per = (units + THREADS - 1) / THREADS;
  const int u0 = min(units, (int)threadIdx.x * per), u1 = min(units, u0 + per);
  long long own = 0;
  for (int u = u0; u < u1; ++u) own += length_of(p, item_of<MT, NT>(p, u));
  long long incl = own;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh[warp] = incl;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) incl += sh[w];
    total += sh[w];
  }
  Range r;
  const int nkv = p.a.c.nkv;
  r.total = total * nkv;
  r.per = max((r.total + p.grid - 1) / p.grid, (long long)p.min_tiles);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const long long at = min((cta + side) * r.per, r.total);
    long long excl = incl - own;
    if (at == r.total) {
      if (threadIdx.x == 0) sh[16 + 3 * side] = at;
    } else if (own && at >= excl * nkv && at < incl * nkv) {
      int u = u0, t;
      for (;; ++u) {
        t = length_of(p, item_of<MT, NT>(p, u));
        if (at < (excl + t) * nkv) break;
        excl += t;
      }
      sh[16 + 3 * side] = p.whole ? at - (at - excl * nkv) % t : at;
      sh[17 + 3 * side] = u;
      sh[18 + 3 * side] = excl;
    }
  }
  __syncthreads();
  r.begin = sh[16];
  r.unit = (int)sh[17];
  r.before = sh[18];
  r.end = sh[19];
  return r;
}

// Walks the line's tiles; done when pos reaches the end of the range.
template <int MT, int NT>
struct Cursor {
  Item it;
  int unit, head, tile;
  long long pos;
  // To the first tile at or behind the range's beginning.
  __device__ __forceinline__ void seek(const Params& p, const Range& r) {
    unit = r.unit;
    it = item_of<MT, NT>(p, unit);
    const long long in = r.begin - r.before * p.a.c.nkv;
    const int len = length_of(p, it);
    head = (int)(in / len);
    const int off = (int)(in - (long long)head * len);
    tile = max(0, off - p.item_cost);
    pos = r.begin + max(0, p.item_cost - off);
  }
  __device__ __forceinline__ void next(const Params& p) {
    ++pos;
    if (++tile < it.tiles || p.direct) return;
    tile = 0;
    pos += p.item_cost;
    if (++head < p.a.c.nkv) return;
    head = 0;
    const int units = p.a.c.n_seqs * p.row_tiles;
    do {
      if (++unit >= units) return;
      it = item_of<MT, NT>(p, unit);
    } while (it.tiles == 0);
  }
  __device__ __forceinline__ bool last_of_item() const { return tile + 1 == it.tiles; }
  // The CTA's last tile of the item.
  __device__ __forceinline__ bool ends(long long end) const { return tile + 1 == it.tiles || pos + 1 >= end; }
};

// The pages of a tile's NT tokens, NT / 32 per lane. fetch() only issues the
// loads, a tile ahead of their use; check() reports numbers outside the pool
// and leaves -1 there and for tokens that no row of the item sees.
template <int NT>
struct TilePages {
  int page[NT / 32];
  __device__ __forceinline__ void fetch(const PagedChunk& c, const Item& it, int t0, int lane) {
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
      const int t = t0 + lane + 32 * i;
      page[i] = -1;
      if (t >= it.lo && t < it.hi) page[i] = c.table[(long long)it.seq * c.table_stride + c.page.quot(t)];
    }
  }
  __device__ __forceinline__ void check(const PagedChunk& c, const Item& it, int t0, int lane) {
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
      const int t = t0 + lane + 32 * i;
      if (t >= it.lo && t < it.hi && (unsigned)page[i] >= (unsigned)c.n_pages) {
        atomicOr(c.err, kErrBadInput);
        page[i] = -1;
      }
    }
  }
  // Offset in elements of each of the lane's tokens, -1 without a page.
  __device__ __forceinline__ void offsets(const PagedChunk& c, int t0, int lane, long long page_stride, long long slot_stride,
                                          long long (&off)[NT / 32]) const {
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
      const int t = t0 + lane + 32 * i, slot = t - (int)c.page.quot(t) * (int)c.page.d;
      off[i] = page[i] >= 0 ? page[i] * page_stride + slot * slot_stride : -1;
    }
  }
};

// Tiles of tokens in shared memory: 128-byte column blocks of [token][128
// bytes] under the 128-byte swizzle (16-byte chunk c of a row at c ^ (row &
// 7)), as TMA writes them and tcgen05 and (conflict free) ldmatrix read them.
__device__ __forceinline__ uint32_t tile_at(int rows, int row, int chunk) {
  return (uint32_t)((chunk >> 3) * rows * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

__device__ __forceinline__ bool try_bar(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait (about a second of SM clock), polling: a wait with a suspend
// hint wakes late.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, uint32_t* err) {
  const uint32_t a = smem_u32(bar);
  if (try_bar(a, parity)) return true;
  const long long t0 = clock64();
  while (!try_bar(a, parity))
    if (clock64() - t0 > 2000000000ll) {
      if (err) atomicOr(err, kErrWaitTimeout);
      return false;
    }
  return true;
}

__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Whether some row of the item may not see some token of the tile that
// begins at t0.
__device__ __forceinline__ bool tile_masked(const Item& it, int t0, int nt, int window, const FastDiv& group) {
  const int p0 = it.len - it.n, plo = p0 + (int)group.quot(it.f0), phi = it.hi - 1;
  return t0 + nt - 1 > plo || t0 < it.lo || (window > 0 && t0 <= phi - window);
}

// The elements of a 32-bit word that are not finite, replaced by zero.
template <int DT>
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
  if constexpr (DT == kF32) {
    return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
  } else {
    constexpr uint32_t e = DT == kBF16 ? 0x7f80u : 0x7c00u;
    if ((w & e) == e) w &= 0xffff0000u;
    if ((w >> 16 & e) == e) w &= 0x0000ffffu;
    return w;
  }
}

// Whether a word holds an element that is not finite: its magnitude's bits plus
// the exponent's unit reach the sign bit. (The bits of interest, not a flag.)
template <int DT>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if constexpr (DT == kF32) return ((w & 0x7fffffffu) + 0x00800000u) & 0x80000000u;
  else return ((w & 0x7fff7fffu) + (DT == kBF16 ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}
// Replaces the values of one 16-byte chunk of a V tile that are not finite by
// zero; whether there were any in a token that some row sees (t: the chunk's
// token). Slots outside that range may hold anything.
template <int DT>
__device__ __forceinline__ bool clean_chunk(uint32_t ad, int t, const Item& it) {
  uint4 w;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(ad));
  if (!(not_finite<DT>(w.x) | not_finite<DT>(w.y) | not_finite<DT>(w.z) | not_finite<DT>(w.w))) return false;
  const uint4 f = make_uint4(finite_or_zero<DT>(w.x), finite_or_zero<DT>(w.y), finite_or_zero<DT>(w.z), finite_or_zero<DT>(w.w));
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(ad), "r"(f.x), "r"(f.y), "r"(f.z), "r"(f.w) : "memory");
  return t >= it.lo && t < it.hi;
}

// Pages as TMA tensors (element, slot, head, page). A tile of NT tokens is
// fetched in pieces of `box` slots of one page by one 128-byte column block,
// one copy per lane of a warp: pages of 8 x 2^i slots, or of whole tiles.
struct KvMaps {
  CUtensorMap k, v;
};
// Slots of a piece, 0 where TMA cannot fetch such pages.
inline int tma_box(int page, int nt) {
  if (page % 8 == 0 && page <= nt && nt % page == 0) return page;
  return page % nt == 0 ? nt : 0;
}
// Whether the maps could be made (kernels_paged_attn.cu).
bool make_maps(const PagedChunk& c, int dtype, int box, KvMaps* maps);
// The queries of 16-bit types as a tensor (element, head, row), `rows` rows of
// one KV head's heads a box.
bool make_q_map(const AttnArgs& a, int rows, CUtensorMap* map);

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int page,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

template <int NT, int BLOCKS, int ELT>
struct TilePieces {
  int page;  // of the lane's piece of the next tile
  __device__ __forceinline__ bool mine(int box, int lane, int* block, int* piece) const {
    const int pieces = NT / box;
    *block = lane / pieces;
    *piece = lane - *block * pieces;
    return *block < BLOCKS;
  }
  // Only issues the load, a tile ahead of its use.
  __device__ __forceinline__ void fetch(const PagedChunk& c, const Item& it, int t0, int box, int lane) {
    int block, piece;
    page = -1;
    if (!mine(box, lane, &block, &piece)) return;
    const int t = t0 + piece * box;
    if (t < it.hi && t + box > it.lo) page = c.table[(long long)it.seq * c.table_stride + c.page.quot(t)];
  }
  // One tile of K or V into dst, completing on bar (one arrival). Pieces that
  // no row sees are left out: their slots hold what they held. A page outside
  // the pool is reported and its slots are zeros.
  __device__ __forceinline__ void load(const PagedChunk& c, const Item& it, int t0, int box, int lane, const CUtensorMap* map,
                                       int head, uint32_t dst, uint64_t* bar) const {
    load2(c, it, t0, box, lane, map, nullptr, head, dst, 0, bar);
  }
  // With map2: both, K into dst and V into dst2, on one barrier.
  __device__ __forceinline__ void load2(const PagedChunk& c, const Item& it, int t0, int box, int lane, const CUtensorMap* map,
                                        const CUtensorMap* map2, int head, uint32_t dst, uint32_t dst2, uint64_t* bar) const {
    int block, piece;
    const bool any = mine(box, lane, &block, &piece);
    const int t = t0 + piece * box;
    const bool want = any && t < it.hi && t + box > it.lo;
    const bool good = want && (unsigned)page < (unsigned)c.n_pages;
    const uint32_t at = block * (NT * 128) + piece * box * 128;
    if (__any_sync(~0u, want && !good)) {
      if (want && !good) {
        atomicOr(c.err, kErrBadInput);
        for (int i = 0; i < box * 8; ++i) {
          asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(dst + at + i * 16), "r"(0) : "memory");
          if (map2) asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(dst2 + at + i * 16), "r"(0) : "memory");
        }
      }
      fence_async();
      __syncwarp();  // lane 0's arrival below stands for every lane's zeros
    }
    const uint32_t n = __popc(__ballot_sync(~0u, good));
    if (lane == 0) mbar_arrive_expect_tx(bar, (map2 ? 2 : 1) * n * box * 128);
    __syncwarp();
    if (good) {
      const int slot = t - (int)c.page.quot(t) * (int)c.page.d;
      tma_load(dst + at, map, block * (128 / ELT), slot, head, page, bar);
      if (map2) tma_load(dst2 + at, map2, block * (128 / ELT), slot, head, page, bar);
    }
  }
};

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

template <int DT>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  if constexpr (DT == kBF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <int DT>
__device__ __forceinline__ float value(const void* base, long long i) {
  if constexpr (DT == kF32) return static_cast<const float*>(base)[i];
  else if constexpr (DT == kF16) return __half2float(static_cast<const __half*>(base)[i]);
  else return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// cap tanh(z / cap), z = scale s, of two scores, right relative to the score
// for any cap.
//
// 16-bit types: tanh x = 1 - 2 / (1 + e^2x) is right to 2^-21.6 of 1, which
// for small x is nothing of x; there z (1 - x^2 / 3 + 2 x^4 / 15), whose next
// term is 17/315 x^6 < 2^-22 below x = 1/8. At that border the first form is
// right to 2^-18.6 of the score. (y = 2 log2(e) x serves both.)
template <int DT>
__device__ __forceinline__ float2 capped(float2 s, float scale, float cap, float inv_cap) {
  const float2 z = mul2(s, {scale, scale});
  if constexpr (DT == kF32) {
    const float2 x = mul2(z, {inv_cap, inv_cap});
    // Below 2^-12 tanh x is x; z has not been through a quotient that may
    // lie below the normal numbers.
    return {fabsf(x.x) < 0x1p-12f ? z.x : cap * tanhf(x.x), fabsf(x.y) < 0x1p-12f ? z.y : cap * tanhf(x.y)};
  } else {
    const float k = 2.f * kLog2e * inv_cap;
    const float2 y = mul2(z, {k, k});
    const float2 e = add2({exp2_fast(y.x), exp2_fast(y.y)}, {1.f, 1.f});
    const float2 far = mul2(fma2({rcp_fast(e.x), rcp_fast(e.y)}, {-2.f, -2.f}, {1.f, 1.f}), {cap, cap});
    constexpr float k2 = 4.f * kLog2e * kLog2e, c1 = -1.f / (3.f * k2), c2 = 2.f / (15.f * k2 * k2);
    const float2 w = mul2(y, y);
    const float2 near = fma2(mul2(z, w), fma2(w, {c2, c2}, {c1, c1}), z);
    return {fabsf(y.x) < 0.36f ? near.x : far.x, fabsf(y.y) < 0.36f ? near.y : far.y};
  }
}
// The V values of column `col` that are not finite among the tokens [from,
// till) of the item's masked tiles, added up; 0: there are none. (The tiles'
// copies of them were zeroed, so that they do not reach rows that may not see
// them; the rows that do get them here.)
template <int DT, int NT>
__device__ __noinline__ float lost_values(const Params& p, const Item it, int kv_head, int col, int from, int till) {
  const PagedChunk& c = p.a.c;
  float sum = 0.f;
  // By tiles: what lies between the masked ones may be a long context, and the
  // other warps' waits are bounded.
  for (int t = from; t < till;) {
    const int next = min(till, (t / NT + 1) * NT);
    if (tile_masked(it, t / NT * NT, NT, p.a.window, p.group_div)) {
      for (; t < next; ++t) {
        const int pi = (int)c.page.quot(t), page = page_of(c, it.seq, pi);
        if (page < 0) continue;
        const float v = value<DT>(c.v, page * c.v_page + (long long)kv_head * c.v_head + (t - pi * (int)c.page.d) * c.v_slot + col);
        if (!(fabsf(v) <= 3.4028235e38f)) sum += v;
      }
    }
    t = next;
  }
  return sum;
}
template <int DT>
__device__ __forceinline__ void put(void* base, long long i, float v) {
  if constexpr (DT == kF32) static_cast<float*>(base)[i] = v;
  else if constexpr (DT == kF16) static_cast<__half*>(base)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
}

// What a CTA of the main kernel leaves for the join: whether the cut at its
// first tile is the first one through an item, and that item.
struct Cut {
  int first;       // 0: nothing to join here
  int last;        // the item's parts are in CTAs b - 1 .. last
  int slot0;       // the part's slot in CTA b - 1
  int start, f0, nf, head, pad;
};
constexpr size_t cut_bytes(int grid) { return (size_t)grid * sizeof(Cut); }

template <int MT, int NT>
__device__ __forceinline__ void leave_cut(const Params& p, const Range& rg, const Cursor<MT, NT>& cur, int cta) {
  Cut c = {};
  if (rg.begin < rg.total && !p.whole && cta > 0) {
    const long long tile0 = cur.pos - cur.tile, before = rg.begin - rg.per;  // where CTA b - 1 begins
    if (tile0 < rg.begin && tile0 >= before) {
      c.first = 1;
      c.last = (int)((tile0 + cur.it.tiles - 1) / rg.per);
      c.slot0 = tile0 - p.item_cost <= before ? 0 : 1;  // the first item of CTA b - 1?
      c.start = cur.it.start, c.f0 = cur.it.f0, c.nf = cur.it.nf, c.head = cur.head;
    }
  }
  reinterpret_cast<Cut*>(p.a.part)[cta] = c;
}
__device__ __forceinline__ float* part_of(const Params& p, int floats, int cta, int slot) {
  return p.a.part + cut_bytes(p.grid) / 4 + (2ll * cta + slot) * floats;
}

constexpr int kCombineThreads = 128;

// Joins the parts of the item whose first cut is at the beginning of CTA
// b = blockIdx.x + 1; each warp takes rows of the tile. Bound by latency: a
// lane finds the weight of one part, and the parts' loads are independent.
template <typename C>
__global__ void __launch_bounds__(kCombineThreads) paged_combine_kernel(const __grid_constant__ Params p) {
  constexpr int HD = C::HD, MT = C::MT, PL = HD / 32;  // columns per lane
  pdl_wait_prior();
  pdl_launch_dependents();
  const int b = blockIdx.x + 1;
  const Cut cut = reinterpret_cast<const Cut*>(p.a.part)[b];
  if (!cut.first) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, parts = cut.last - b + 2;
  auto part = [&](int i) { return part_of(p, C::kPartFloats, b - 1 + i, i == 0 ? cut.slot0 : 0); };
  for (int r = blockIdx.y * (kCombineThreads / 32) + warp; r < cut.nf; r += gridDim.y * (kCombineThreads / 32)) {
    float top = -INFINITY;
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, part(i)[MT * HD + r]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float mc = top == -INFINITY ? 0.f : top;
    float acc[PL] = {}, l = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 32) {
      float mine = 0.f, w = 0.f;
      if (i0 + lane < parts) {
        const float* x = part(i0 + lane) + MT * HD + r;
        w = exp2_fast(x[0] - mc);
        mine = x[MT] * w;
      }
      const int n = min(32, parts - i0);
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float wi = __shfl_sync(~0u, w, i);
        l += __shfl_sync(~0u, mine, i);
        const float* x = part(i0 + i) + r * HD;
#pragma unroll
        for (int e = 0; e < PL / 2; ++e) {
          const float2 v = *reinterpret_cast<const float2*>(x + e * 64 + lane * 2);
          if (wi != 0.f) {  // else the row sees nothing of the part
            acc[2 * e] += v.x * wi;
            acc[2 * e + 1] += v.y * wi;
          }
        }
      }
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const int f = cut.f0 + r, i = (int)p.group_div.quot(f), head = cut.head * p.a.group + f - i * p.a.group;
    const long long o = (long long)(cut.start + i) * p.a.o_row + (long long)head * p.a.o_head;
#pragma unroll
    for (int e = 0; e < PL / 2; ++e) {
      const int col = e * 64 + lane * 2;
      if (col >= p.a.c.hd) continue;
      if constexpr (C::DT == kF32)
        *reinterpret_cast<float2*>(static_cast<float*>(p.a.out) + o + col) = make_float2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
      else
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.a.out) + o + col) =
            pack<C::DT>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    }
    if (p.a.lse && lane == 0)
      p.a.lse[(long long)(cut.start + i) * (p.a.c.nkv * p.a.group) + head] =
          l > 0.f || l != l ? (mc - C::kPShift) * kLn2 + logf(l) : -INFINITY;
  }
}
constexpr int combine_grid_y(int mt) { return mt / 4 < 32 ? mt / 4 : 32; }

}  // namespace paged_attn
}  // namespace rai
