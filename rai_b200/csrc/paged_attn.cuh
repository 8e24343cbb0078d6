// What the two kernels of paged attention share: the line of token tiles and
// its cuts, the join of cut items, and elements.
#pragma once
#include <cuda_runtime.h>

#include "paged.h"

namespace rai {
namespace paged_attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kPlanWords = 22;

struct Params {
  AttnArgs a;
  int row_tiles, min_tiles, grid;
  bool whole;  // items are short: none is cut
  float c;  // log2(e) * scale, or log2(e) when the scores are capped
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

// The CTA's range [begin, end) of the line of tiles and the unit it starts
// in. Every thread sums a run of units; a block scan places the runs. With
// p.whole the cuts move down to the starts of the items they fall in.
struct Range {
  long long total, per, begin, end;
  int unit;          // unit of `begin`
  long long before;  // tiles of one KV head before it
};
template <int MT, int NT, int THREADS>
__device__ __forceinline__ Range plan(const Params& p, long long cta, long long (&sh)[kPlanWords]) {
  const int units = p.a.c.n_seqs * p.row_tiles;
  const int per = (units + THREADS - 1) / THREADS;
  const int u0 = min(units, (int)threadIdx.x * per), u1 = min(units, u0 + per);
  long long own = 0;
  for (int u = u0; u < u1; ++u) own += item_of<MT, NT>(p, u).tiles;
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
        t = item_of<MT, NT>(p, u).tiles;
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

// Walks the line of tiles.
template <int MT, int NT>
struct Cursor {
  Item it;
  int unit, head, tile;
  __device__ __forceinline__ void seek(const Params& p, const Range& r, long long at) {
    unit = r.unit;
    it = item_of<MT, NT>(p, unit);
    const long long in = at - r.before * p.a.c.nkv;
    head = (int)(in / it.tiles);
    tile = (int)(in - (long long)head * it.tiles);
  }
  __device__ __forceinline__ void next(const Params& p) {
    if (++tile < it.tiles) return;
    tile = 0;
    if (++head < p.a.c.nkv) return;
    head = 0;
    const int units = p.a.c.n_seqs * p.row_tiles;
    do {
      if (++unit >= units) return;
      it = item_of<MT, NT>(p, unit);
    } while (it.tiles == 0);
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
template <int DT>
__device__ __forceinline__ float capped(float s, float scale, float cap) {
  const float x = __fdividef(s * scale, cap);
  if constexpr (DT == kF32) {
    return cap * tanhf(x);
  } else {
    // tanh x = 1 - 2 / (1 + e^2x): a few 2^-23 of the cap, far below the
    // 2^-9 that a probability is rounded to.
    return cap * (1.f - __fdividef(2.f, 1.f + exp2_fast(2.f * kLog2e * x)));
  }
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

constexpr int kCombineThreads = 128;
constexpr int combine_grid_y(int mt) { return mt / 4 < 16 ? mt / 4 : 16; }

// Joins the parts of items that the cut between CTAs b - 1 and b goes
// through first (b = blockIdx.x + 1); the CTAs of one b share the tile's rows.
template <typename C>
__global__ void __launch_bounds__(kCombineThreads) paged_combine_kernel(const __grid_constant__ Params p) {
  constexpr int HD = C::HD, MT = C::MT, NT = C::NT;
  __shared__ long long sh[kPlanWords];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int b = blockIdx.x + 1;
  const Range rg = plan<MT, NT, kCombineThreads>(p, b, sh);
  const long long at = rg.begin;
  if (at >= rg.total) return;
  Cursor<MT, NT> cur;
  cur.seek(p, rg, at);
  const long long start = at - cur.tile, stop = start + cur.it.tiles;
  if (start == at || start < at - rg.per) return;  // not cut here, or cut before
  const int last = (int)((stop - 1) / rg.per);     // parts: CTAs b - 1 .. last
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto part = [&](int cta) {
    const bool head = cta >= b || start == (long long)cta * rg.per;  // the CTA's first item
    return p.a.part + (2ll * cta + (head ? 0 : 1)) * C::kPartFloats;
  };
  for (int r = blockIdx.y * 4 + warp; r < cur.it.nf; r += gridDim.y * 4) {
    float top = -INFINITY;
    for (int cta = b - 1 + lane; cta <= last; cta += 32) top = fmaxf(top, part(cta)[MT * HD + r]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float mc = top == -INFINITY ? 0.f : top;
    constexpr int PL = HD / 32;  // columns per lane
    float acc[PL] = {}, l = 0.f;
    for (int cta = b - 1; cta <= last; ++cta) {
      const float* x = part(cta);
      const float w = exp2_fast(x[MT * HD + r] - mc);
      l += x[MT * HD + MT + r] * w;
      if (w != 0.f)  // a part of which the row sees nothing
#pragma unroll
        for (int e = 0; e < PL / 2; ++e) {
          const float2 v = *reinterpret_cast<const float2*>(x + r * HD + e * 64 + lane * 2);
          acc[2 * e] += v.x * w;
          acc[2 * e + 1] += v.y * w;
        }
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const int f = cur.it.f0 + r, i = (int)p.group_div.quot(f), head = cur.head * p.a.group + f - i * p.a.group;
    const long long o = (long long)(cur.it.start + i) * p.a.o_row + (long long)head * p.a.o_head;
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
      p.a.lse[(long long)(cur.it.start + i) * (p.a.c.nkv * p.a.group) + head] =
          l > 0.f || l != l ? (mc - C::kPShift) * kLn2 + logf(l) : -INFINITY;
  }
}

}  // namespace paged_attn
}  // namespace rai
