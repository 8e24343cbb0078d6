// Filling and keeping a paged cache: rotary positions with the store of k and
// v, and the page operations (fork, resize with copy on write, compact, copy).
#include <cuda_runtime.h>

#include "paged.h"

namespace rai {

namespace {

// ---------------------------------------------------------------- elements

template <int DT>
struct Elt;
template <>
struct Elt<kF32> {
  using T = float;
  static __device__ __forceinline__ float get(T x) { return x; }
  static __device__ __forceinline__ T put(float x) { return x; }
};
template <>
struct Elt<kF16> {
  using T = __half;
  static __device__ __forceinline__ float get(T x) { return __half2float(x); }
  static __device__ __forceinline__ T put(float x) { return __float2half_rn(x); }
};
template <>
struct Elt<kBF16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float get(T x) { return __bfloat162float(x); }
  static __device__ __forceinline__ T put(float x) { return __float2bfloat16_rn(x); }
};

// N elements as 16-byte vectors (or one of 8 bytes), as they lie in memory
// until they are needed.
template <int DT, int N>
struct Raw {
  using T = typename Elt<DT>::T;
  static constexpr int kB = N * sizeof(T);
  static_assert(kB % 16 == 0 || kB == 8, "vector width");
  uint32_t w[kB / 4];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kB % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kB / 16; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (DT == kF32) return __uint_as_float(w[i]);
    else if constexpr (DT == kBF16) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __half2float(__ushort_as_half((uint16_t)(w[i / 2] >> (16 * (i & 1)))));
  }
};
template <int DT, int N>
__device__ __forceinline__ void store_n(typename Elt<DT>::T* p, const float (&x)[N]) {
  using T = typename Elt<DT>::T;
  constexpr int kB = N * sizeof(T);
  alignas(16) T v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = Elt<DT>::put(x[i]);
  if constexpr (kB % 16 == 0) {
#pragma unroll
    for (int i = 0; i < kB / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
  } else {
    static_assert(kB == 8, "vector width");
    reinterpret_cast<uint2*>(p)[0] = reinterpret_cast<const uint2*>(v)[0];
  }
}

// cos and sin of pos * inv_freq. The product and its reduction to a part of a
// turn are in 64 bits (a far position times a frequency has more than 24
// significant bits above the point); the part, within half a turn, has a
// 32-bit sine and cosine.
__device__ __forceinline__ void turn_of(int pos, float inv_freq, float mscale, float* c, float* s) {
  const double t = (double)pos * (double)inv_freq * 0.15915494309189533577;
  float sv, cv;
  sincospif((float)(2.0 * (t - rint(t))), &sv, &cv);
  *c = cv * mscale;
  *s = sv * mscale;
}

constexpr int kRopeThreads = 256;

struct RopeUnits {
  FastDiv rot, tail, whole;  // units of a head: rotated, behind the rotated part, all (v)
  int parts;                 // warps that share a row
};

// The last s with q_start[s] <= row, by a warp: 32 probes a round.
__device__ __forceinline__ int seq_of_row(const PagedChunk& c, int row, int lane) {
  int lo = 0, span = c.n_seqs;
  while (span > 1) {
    const int step = (span + 31) / 32, at = lane * step;
    const int n = __popc(__ballot_sync(~0u, at < span && c.q_start[lo + at] <= row));
    if (n == 0) return 0;
    lo += (n - 1) * step;
    span = min(step, span - (n - 1) * step);
  }
  return lo;
}

// A warp takes a row, or with few rows a part of one: the row's angles go to
// shared memory, then lanes take units of kV elements of every q, k and v
// head (half-split: the two vectors of kV pairs, so a rotation in place is
// safe), two units' loads before their stores. Bound: HBM, each element read
// and written once; rows in flight hide the look-up of sequence and page.
template <int IN, int OUT>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_append_kernel(const __grid_constant__ RopeArgs a,
                                                                   const __grid_constant__ RopeUnits un) {
  using TI = typename Elt<IN>::T;
  using TO = typename Elt<OUT>::T;
  constexpr int kV = IN == kF32 && OUT == kF32 ? 4 : 8;
  constexpr int kU = IN == kF32 ? 1 : 2;
  __shared__ float table[kRopeThreads / 32][2][128];
  const PagedChunk& ch = a.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float *cs = table[warp][0], *sn = table[warp][1];
  const int half = a.rot / 2, stride = 32 * un.parts;
  pdl_wait_prior();
  pdl_launch_dependents();
  for (long long id = (long long)blockIdx.x * (kRopeThreads / 32) + warp; id < (long long)ch.rows * un.parts;
       id += (long long)gridDim.x * (kRopeThreads / 32)) {
    const int row = (int)(id / un.parts), part = (int)(id - (long long)row * un.parts);
    const int seq = seq_of_row(ch, row, lane);
    const SeqRows r = seq_rows(ch, seq);
    if (row < r.start || row >= r.start + r.n) continue;  // behind the last sequence (or before the first)
    const int pos = r.len - r.n + (row - r.start);
    int page = -1, slot = 0;
    if (pos >= 0) {
      const int pi = (int)ch.page.quot(pos);
      page = page_of(ch, seq, pi);
      slot = pos - pi * (int)ch.page.d;
    }
    __syncwarp();  // the last row's angles have been read
    for (int i = lane; i < half; i += 32) turn_of(pos, a.inv_freq[i], a.mscale, &cs[i], &sn[i]);
    __syncwarp();
    const TI* qr = static_cast<const TI*>(a.q) + (long long)row * a.q_row;
    const TI* kr = static_cast<const TI*>(a.k) + (long long)row * a.k_row;
    const TI* vr = static_cast<const TI*>(a.v) + (long long)row * a.v_row;
    TO* qo = static_cast<TO*>(a.q_out) + (long long)row * a.o_row;
    TO* ko = static_cast<TO*>(ch.k) + page * ch.k_page + slot * ch.k_slot;
    TO* vo = static_cast<TO*>(ch.v) + page * ch.v_page + slot * ch.v_slot;
    const int turned = page >= 0 ? a.heads + ch.nkv : a.heads;  // heads of q, then of k
    auto from = [&](int h) { return h < a.heads ? qr + (long long)h * a.q_head : kr + (long long)(h - a.heads) * a.k_head; };
    auto into = [&](int h) { return h < a.heads ? qo + (long long)h * a.o_head : ko + (long long)(h - a.heads) * ch.k_head; };
    if (half % kV) {
      // Pairs do not fall on vectors: one pair, or one element behind the
      // rotated part, at a time.
      const int per = ch.hd - half;
      const int all = turned + (page >= 0 ? ch.nkv : 0);
      for (int x = lane + 32 * part; x < all * per; x += stride) {
        const int head = x / per, e = x - head * per;
        const bool turn = head < turned;
        const TI* src = turn ? from(head) : vr + (long long)(head - turned) * a.v_head;
        TO* dst = turn ? into(head) : vo + (long long)(head - turned) * ch.v_head;
        if (e >= half) {
          dst[half + e] = Elt<OUT>::put(Elt<IN>::get(src[half + e]));
          continue;
        }
        const int i = a.interleaved ? 2 * e : e, j = a.interleaved ? 2 * e + 1 : e + half;
        const float x0 = Elt<IN>::get(src[i]), x1 = Elt<IN>::get(src[j]);
        const float c = turn ? cs[e] : 1.f, s = turn ? sn[e] : 0.f;
        dst[i] = Elt<OUT>::put(turn ? x0 * c - x1 * s : x0);
        dst[j] = Elt<OUT>::put(turn ? x1 * c + x0 * s : x1);
      }
      continue;
    }
    // Rotated units.
    const int n_rot = turned * (int)un.rot.d;
    for (int x0 = lane + 32 * part; x0 < n_rot; x0 += stride * kU) {
      Raw<IN, kV> u[kU], w[kU];
#pragma unroll
      for (int k = 0; k < kU; ++k) {
        const int x = x0 + k * stride;
        if (x < n_rot) {
          const int h = (int)un.rot.quot(x);
          const TI* src = from(h) + (x - h * (int)un.rot.d) * kV;
          u[k].load(src);
          if (!a.interleaved) w[k].load(src + half);
        }
      }
#pragma unroll
      for (int k = 0; k < kU; ++k) {
        const int x = x0 + k * stride;
        if (x < n_rot) {
          const int h = (int)un.rot.quot(x), d = (x - h * (int)un.rot.d) * kV;
          TO* dst = into(h) + d;
          float y[kV];
          if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < kV; i += 2) {
              const float c = cs[d / 2 + i / 2], s = sn[d / 2 + i / 2], y0 = u[k].get(i), y1 = u[k].get(i + 1);
              y[i] = y0 * c - y1 * s;
              y[i + 1] = y1 * c + y0 * s;
            }
          } else {
            float z[kV];
#pragma unroll
            for (int i = 0; i < kV; ++i) {
              const float c = cs[d + i], s = sn[d + i], y0 = u[k].get(i), y1 = w[k].get(i);
              y[i] = y0 * c - y1 * s;
              z[i] = y1 * c + y0 * s;
            }
            store_n<OUT, kV>(dst + half, z);
          }
          store_n<OUT, kV>(dst, y);
        }
      }
    }
    // Copies: what lies behind the rotated part, then v.
    const int n_tail = a.rot < ch.hd ? turned * (int)un.tail.d : 0, n_all = n_tail + (page >= 0 ? ch.nkv * (int)un.whole.d : 0);
    for (int x0 = lane + 32 * part; x0 < n_all; x0 += stride * kU) {
      Raw<IN, kV> u[kU];
#pragma unroll
      for (int k = 0; k < kU; ++k) {
        const int x = x0 + k * stride;
        if (x < n_tail) {
          const int h = (int)un.tail.quot(x);
          u[k].load(from(h) + a.rot + (x - h * (int)un.tail.d) * kV);
        } else if (x < n_all) {
          const int h = (int)un.whole.quot(x - n_tail);
          u[k].load(vr + (long long)h * a.v_head + (x - n_tail - h * (int)un.whole.d) * kV);
        }
      }
#pragma unroll
      for (int k = 0; k < kU; ++k) {
        const int x = x0 + k * stride;
        if (x >= n_all) continue;
        float y[kV];
#pragma unroll
        for (int i = 0; i < kV; ++i) y[i] = u[k].get(i);
        if (x < n_tail) {
          const int h = (int)un.tail.quot(x);
          store_n<OUT, kV>(into(h) + a.rot + (x - h * (int)un.tail.d) * kV, y);
        } else {
          const int h = (int)un.whole.quot(x - n_tail);
          store_n<OUT, kV>(vo + (long long)h * ch.v_head + (x - n_tail - h * (int)un.whole.d) * kV, y);
        }
      }
    }
  }
}

// ---------------------------------------------------------------- pages

constexpr int kMetaThreads = 1024;

__device__ __forceinline__ int cells_of(int len, int page_size) { return (len + page_size - 1) / page_size; }

// A sequence's length within its table.
__device__ __forceinline__ int table_len(const TableArgs& t, const int* lens, int s) {
  const int v = lens[s], cap = (int)min((long long)t.max_pages * t.page_size, (long long)(INT_MAX - 1024));
  const int c = min(max(v, 0), cap);
  if (c != v) atomicOr(t.err, kErrBadInput);
  return c;
}
__device__ __forceinline__ bool good_page(const TableArgs& t, int page) {
  if ((unsigned)page < (unsigned)t.n_pages) return true;
  atomicOr(t.err, kErrBadInput);
  return false;
}

// CTA i: child i's table row, and parent i's change of references (its
// children less one for each page). Integer sums: the order does not matter.
__global__ void __launch_bounds__(256) kv_fork_kernel(TableArgs in, TableArgs out, const int* parents) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const int i = blockIdx.x;
  int mine = 0;
  for (int x = threadIdx.x; x < out.n_seqs; x += blockDim.x) mine += parents[x] == i;
  __shared__ int sum[8];
#pragma unroll
  for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
  if ((threadIdx.x & 31) == 0) sum[threadIdx.x >> 5] = mine;
  __syncthreads();
  int children = 0;
  for (int w = 0; w < 8; ++w) children += sum[w];
  if (i < in.n_seqs && children != 1) {
    const int cells = cells_of(table_len(in, in.lens, i), in.page_size);
    const int* row = in.table + (long long)i * in.stride;
    for (int x = threadIdx.x; x < cells; x += blockDim.x)
      if (good_page(in, row[x])) atomicAdd(in.refs + row[x], children - 1);
  }
  if (i < out.n_seqs) {
    int p = parents[i];
    if (p < -1 || p >= in.n_seqs) {
      atomicOr(in.err, kErrBadInput);
      p = -1;
    }
    const int len = p >= 0 ? table_len(in, in.lens, p) : 0, cells = cells_of(len, in.page_size);
    const int* row = in.table + (long long)p * in.stride;
    int* to = out.table + (long long)i * out.stride;
    for (int x = threadIdx.x; x < out.max_pages; x += blockDim.x) to[x] = x < cells ? row[x] : -1;
    if (threadIdx.x == 0) out.lens[i] = len;
  }
}

// Exclusive sum over kMetaThreads threads; in 64 bits, since many sequences can
// ask for more pages than 32 bits count.
__device__ __forceinline__ long long block_scan(long long v, long long* sh, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    long long w = sh[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(~0u, w, o);
      if (lane >= o) w += u;
    }
    sh[lane] = w;
  }
  __syncthreads();
  *total = sh[31];
  return incl - v + (warp ? sh[warp - 1] : 0);
}

// A warp's run of the pages: 32 * n consecutive ones.
struct Run {
  int first, groups;
};
__device__ __forceinline__ Run run_of(int n_pages) {
  const int groups = (n_pages + 31) / 32, warps = kMetaThreads / 32, per = (groups + warps - 1) / warps;
  const int g0 = min(groups, (int)(threadIdx.x >> 5) * per);
  return {g0 * 32, min(per, groups - g0)};
}
// f(page, whether the lane has one, its count) for each group of 32 pages of
// the run, eight groups' counts fetched at a time; with STOP until f is false.
template <bool STOP, typename F>
__device__ __forceinline__ void scan_run_of(const int* refs, int n_pages, const Run& run, F f) {
  const int lane = threadIdx.x & 31;
  for (int g0 = 0; g0 < run.groups; g0 += 8) {
    int v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = run.first + (g0 + i) * 32 + lane;
      v[i] = g0 + i < run.groups && p < n_pages ? __ldcg(refs + p) : 1;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (g0 + i >= run.groups) return;
      const int p = run.first + (g0 + i) * 32 + lane;
      if constexpr (STOP) {
        if (!f(p, p < n_pages, v[i])) return;
      } else {
        f(p, p < n_pages, v[i]);
      }
    }
  }
}
// Exclusive sum over the block's warps of a value that each warp agrees on.
__device__ __forceinline__ int warp_scan(int v, int* sh, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) sh[warp] = v;
  __syncthreads();
  const int mine = sh[lane];  // kMetaThreads / 32 = 32 warps
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += u;
  }
  *total = __shfl_sync(~0u, incl, 31);
  return __shfl_sync(~0u, incl - mine, warp);
}

// One CTA. Releases what shrinks, then gives the sequences that grow the
// lowest free pages in sequence order: first the copy of a shared last page
// that is partly filled (all holders but the last copy it), then new pages.
// Copies are listed as (src, dst) for kv_copy_kernel: ws = [count, src[n],
// dst[n]].
__global__ void __launch_bounds__(kMetaThreads) kv_resize_kernel(TableArgs t, const int* new_lens,
                                                                 int delta, int* status, int* ws) {
  __shared__ int tail[kMaxTableSeqs];   // page to copy on write, or -1
  __shared__ int place[kMaxTableSeqs];  // exclusive sum of the pages that sequences take
  __shared__ int sh[32];
  __shared__ long long wide[32];
  pdl_wait_prior();
  const int n = t.n_seqs, ps = t.page_size;
  const int cap = (int)min((long long)t.max_pages * ps, (long long)(INT_MAX - 1024));
  auto want = [&](int s, int len) {
    long long v = new_lens ? (long long)new_lens[s] : (long long)len + delta;
    if (v < 0 || v > cap) {
      if (new_lens || v > cap) atomicOr(t.err, kErrBadInput);
      v = v < 0 ? 0 : cap;
    }
    return (int)v;
  };
  // Shrinking sequences release the pages behind their new end.
  for (int s = threadIdx.x; s < n; s += kMetaThreads) {
    const int len = table_len(t, t.lens, s), to = want(s, len);
    tail[s] = -1;
    int* row = t.table + (long long)s * t.stride;
    if (to <= len) {
      for (int x = cells_of(to, ps); x < cells_of(len, ps); ++x) {
        if (good_page(t, row[x])) atomicSub(t.refs + row[x], 1);
        row[x] = -1;
      }
    } else if (len % ps) {
      const int page = row[len / ps];
      if (good_page(t, page)) tail[s] = page;
    }
  }
  __syncthreads();
  // Growing ones: of the holders of a shared last page the first
  // refs - 1 copy it.
  for (int s0 = 0; s0 < n; s0 += kMetaThreads) {
    const int s = s0 + threadIdx.x;
    int copies = 0;
    if (s < n && tail[s] >= 0) {
      const int refs = *(volatile int*)(t.refs + tail[s]);
      if (refs > 1) {
        int before = 0;
        for (int x = 0; x < s; ++x) before += tail[x] == tail[s];
        copies = before < refs - 1;
      }
    }
    if (s < n) place[s] = copies;
  }
  __syncthreads();
  long long sum = 0;
  const int per = (n + kMetaThreads - 1) / kMetaThreads;
  const int s0 = min(n, (int)threadIdx.x * per), s1 = min(n, s0 + per);
  for (int s = s0; s < s1; ++s) {
    const int len = table_len(t, t.lens, s), to = want(s, len);
    if (!place[s]) tail[s] = -1;
    if (to > len) place[s] += cells_of(to, ps) - cells_of(len, ps);
    else place[s] = 0;
    sum += place[s];
  }
  long long total;
  long long at = block_scan(sum, wide, &total);
  // (Where the sum passes 32 bits nothing is given, and place is not read.)
  for (int s = s0; s < s1; ++s) {
    const int c = place[s];
    place[s] = (int)at;
    at += c;
  }
  // Free pages, in order: each warp looks at a run of the counts, 32 at a
  // time.
  const Run run = run_of(t.n_pages);
  int mine = 0;
  scan_run_of<false>(t.refs, t.n_pages, run, [&](int p, bool in, int refs) { mine += __popc(__ballot_sync(~0u, in && refs == 0)); });
  int free_total;
  int rank = warp_scan(mine, sh, &free_total);
  const bool fits = total <= free_total;
  __shared__ int count;
  if (threadIdx.x == 0) {
    count = 0;
    *status = fits ? 0 : (int)min(total - free_total, (long long)INT_MAX);
  }
  __syncthreads();
  if (fits && total > 0) {
    scan_run_of<true>(t.refs, t.n_pages, run, [&](int p, bool in, int refs) {
      const bool free = in && refs == 0;
      const uint32_t mask = __ballot_sync(~0u, free);
      const int mine_at = rank + __popc(mask & ((1u << (threadIdx.x & 31)) - 1u));
      rank += __popc(mask);
      if (free && mine_at < total) {
        // The sequence that takes the page of this rank.
        int lo = 0, hi = n;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (place[mid] <= mine_at) lo = mid; else hi = mid;
        }
        const int s = lo, len = table_len(t, t.lens, s);
        int nth = mine_at - place[s], cell = cells_of(len, ps) + nth;
        if (tail[s] >= 0) {
          --cell;
          if (nth == 0) {
            const int c = atomicAdd(&count, 1);
            ws[1 + c] = tail[s];
            ws[1 + n + c] = p;
            atomicSub(t.refs + tail[s], 1);
          }
        }
        t.table[(long long)s * t.stride + cell] = p;
        t.refs[p] = 1;
      }
      return rank < total;
    });
  }
  __syncthreads();
  if (threadIdx.x == 0) ws[0] = count;
  for (int s = threadIdx.x; s < n; s += kMetaThreads) {
    const int len = table_len(t, t.lens, s), to = want(s, len);
    if (to <= len || fits) t.lens[s] = to;
  }
  __syncthreads();
  pdl_launch_dependents();
}

// One CTA. The i-th used page at or above the number of used pages moves to
// the i-th free page below it. ws = [count, src.., dst..] with room for
// n_pages / 2 pairs; `moved` is the page's new number.
__global__ void __launch_bounds__(kMetaThreads) kv_compact_kernel(TableArgs t, int* used_out, int* ws, int* moved) {
  __shared__ int sh[32];
  pdl_wait_prior();
  const Run run = run_of(t.n_pages);
  const uint32_t below = (1u << (threadIdx.x & 31)) - 1u;
  int mine = 0;
  scan_run_of<false>(t.refs, t.n_pages, run, [&](int p, bool in, int refs) { mine += __popc(__ballot_sync(~0u, in && refs > 0)); });
  int used;
  warp_scan(mine, sh, &used);
  int holes = 0, highs = 0;
  scan_run_of<false>(t.refs, t.n_pages, run, [&](int p, bool in, int refs) {
    holes += __popc(__ballot_sync(~0u, in && refs <= 0 && p < used));
    highs += __popc(__ballot_sync(~0u, in && refs > 0 && p >= used));
  });
  int n_holes, n_highs;
  int hole = warp_scan(holes, sh, &n_holes);
  int high = warp_scan(highs, sh, &n_highs);  // n_highs == n_holes
  int *src = ws + 1, *dst = ws + 1 + t.n_pages / 2;
  scan_run_of<false>(t.refs, t.n_pages, run, [&](int p, bool in, int refs) {
    const bool is_hole = in && refs <= 0 && p < used, is_high = in && refs > 0 && p >= used;
    const uint32_t mh = __ballot_sync(~0u, is_hole), mg = __ballot_sync(~0u, is_high);
    if (is_hole) dst[hole + __popc(mh & below)] = p;
    if (is_high) src[high + __popc(mg & below)] = p;
    hole += __popc(mh);
    high += __popc(mg);
    if (in) moved[p] = p;
  });
  __syncthreads();
  for (int i = threadIdx.x; i < n_highs; i += kMetaThreads) {
    const int a = src[i], b = dst[i];
    moved[a] = b;
    t.refs[b] = t.refs[a];
    t.refs[a] = 0;
  }
  if (threadIdx.x == 0) {
    ws[0] = n_highs;
    *used_out = used;
  }
  __syncthreads();
  pdl_launch_dependents();
}

__global__ void __launch_bounds__(256) kv_rename_kernel(TableArgs t, const int* moved) {
  pdl_wait_prior();
  pdl_launch_dependents();
  for (int s = blockIdx.x; s < t.n_seqs; s += gridDim.x) {
    int* row = t.table + (long long)s * t.stride;
    const int cells = cells_of(table_len(t, t.lens, s), t.page_size);
    for (int x = threadIdx.x; x < cells; x += blockDim.x)
      if (good_page(t, row[x])) row[x] = moved[row[x]];
  }
}

// Page data: CTAs walk (pair, plane, piece) with 16-byte vectors, several in
// flight per thread. Bound: HBM, 2 x bytes moved.
constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 8;
constexpr long long kPiece = kCopyThreads * kCopyVecs * 16ll;
__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(PagePool pool, const int* src,
                                                               const int* dst,
                                                               const int* n_dev, int n, uint32_t* err) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const int pairs = n_dev ? min(max(*n_dev, 0), n) : n;
  const long long pieces = (pool.bytes + kPiece - 1) / kPiece;
  const long long planes = 2ll * pool.layers, total = pairs * planes * pieces;
  for (long long x = blockIdx.x; x < total; x += gridDim.x) {
    const long long piece = x % pieces, y = x / pieces;
    const int plane = (int)(y % planes), pair = (int)(y / planes);
    const int a = src[pair], b = dst[pair];
    if ((unsigned)a >= (unsigned)pool.n_pages || (unsigned)b >= (unsigned)pool.n_pages) {
      if (threadIdx.x == 0) atomicOr(err, kErrBadInput);
      continue;
    }
    const bool is_v = plane >= pool.layers;
    const int layer = is_v ? plane - pool.layers : plane;
    char* base = is_v ? pool.v + layer * pool.v_layer : pool.k + layer * pool.k_layer;
    const long long ps = is_v ? pool.v_page : pool.k_page;
    const uint4* from = reinterpret_cast<const uint4*>(base + a * ps + piece * kPiece);
    uint4* to = reinterpret_cast<uint4*>(base + b * ps + piece * kPiece);
    const int vecs = (int)(min(kPiece, pool.bytes - piece * kPiece) / 16);
    uint4 v[kCopyVecs];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
      if (threadIdx.x + i * kCopyThreads < vecs) v[i] = __ldcs(from + threadIdx.x + i * kCopyThreads);
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
      if (threadIdx.x + i * kCopyThreads < vecs) __stcs(to + threadIdx.x + i * kCopyThreads, v[i]);
  }
}

}  // namespace

cudaError_t rope_append(const RopeArgs& a, cudaStream_t s) {
  const int kv = a.in_dtype == kF32 && a.cache_dtype == kF32 ? 4 : 8, half = a.rot / 2;
  RopeUnits un;
  un.parts = 1;
  if (half % kv == 0) {
    un.rot = FastDiv((a.interleaved ? a.rot : half) / kv);
    un.tail = FastDiv(a.rot < a.c.hd ? (a.c.hd - a.rot) / kv : 1);
    un.whole = FastDiv(a.c.hd / kv);
  }
  // Few rows: up to eight warps a row, until every SM has two CTAs' worth.
  while (un.parts < 8 && (long long)a.c.rows * un.parts * 2 <= 16ll * device_sm_count()) un.parts *= 2;
  const long long ctas = ((long long)a.c.rows * un.parts + kRopeThreads / 32 - 1) / (kRopeThreads / 32);
  const int grid = grid_cap(ctas < INT_MAX ? (int)ctas : INT_MAX, 8);
#define RAI_ROPE(I, O)                                                                                   \
  if (a.in_dtype == I && a.cache_dtype == O)                                                             \
    return launch_pdl(rope_append_kernel<I, O>, dim3(grid), dim3(kRopeThreads), 0, s, a, un);
  RAI_ROPE(kF32, kF32) RAI_ROPE(kF32, kF16) RAI_ROPE(kF32, kBF16)
  RAI_ROPE(kF16, kF32) RAI_ROPE(kF16, kF16) RAI_ROPE(kF16, kBF16)
  RAI_ROPE(kBF16, kF32) RAI_ROPE(kBF16, kF16) RAI_ROPE(kBF16, kBF16)
#undef RAI_ROPE
  return cudaErrorInvalidValue;
}

cudaError_t kv_fork(const TableArgs& in, const TableArgs& out, const int* parents, cudaStream_t s) {
  const int grid = in.n_seqs > out.n_seqs ? in.n_seqs : out.n_seqs;
  return launch_pdl(kv_fork_kernel, dim3(grid), dim3(256), 0, s, in, out, parents);
}

cudaError_t kv_copy(const PagePool& pool, const int* src, const int* dst, const int* n_dev, int n, uint32_t* err,
                    cudaStream_t s) {
  const long long pieces = (pool.bytes + kPiece - 1) / kPiece;
  const long long total = n * 2ll * pool.layers * pieces;
  const int cap = device_sm_count() * 4;
  return launch_pdl(kv_copy_kernel, dim3((unsigned)(total < cap ? total : cap)), dim3(kCopyThreads), 0, s, pool, src, dst,
                    n_dev, n, err);
}

size_t kv_resize_workspace(int n_seqs) { return (1 + 2 * (size_t)n_seqs) * 4; }
cudaError_t kv_resize(const TableArgs& t, const PagePool& pool, const int* new_lens, int delta, int* status, void* ws,
                      cudaStream_t s) {
  int* w = static_cast<int*>(ws);
  cudaError_t e = launch_pdl(kv_resize_kernel, dim3(1), dim3(kMetaThreads), 0, s, t, new_lens, delta, status, w);
  if (e != cudaSuccess || (!new_lens && delta <= 0)) return e;  // nothing can grow
  return kv_copy(pool, w + 1, w + 1 + t.n_seqs, w, t.n_seqs, t.err, s);
}

size_t kv_compact_workspace(int n_pages) { return (1 + 2 * (size_t)(n_pages / 2) + n_pages) * 4; }
cudaError_t kv_compact(const TableArgs& t, const PagePool& pool, int* used, void* ws, cudaStream_t s) {
  int *w = static_cast<int*>(ws), *moved = w + 1 + 2 * (t.n_pages / 2);
  cudaError_t e = launch_pdl(kv_compact_kernel, dim3(1), dim3(kMetaThreads), 0, s, t, used, w, moved);
  if (e != cudaSuccess) return e;
  if (t.n_seqs > 0) {
    e = launch_pdl(kv_rename_kernel, dim3(grid_cap(t.n_seqs, 4)), dim3(256), 0, s, t, (const int*)moved);
    if (e != cudaSuccess) return e;
  }
  const int most = t.n_pages / 2;
  if (most == 0) return e;
  return kv_copy(pool, w + 1, w + 1 + most, w, most, t.err, s);
}

}  // namespace rai
