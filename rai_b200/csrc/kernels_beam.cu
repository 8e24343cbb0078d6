// Beam search's choice: of the beams x vocabulary continuations of each
// request the `keep` with the largest score_b + log softmax(logits_b)[v],
// the first `beams` of them that do not end, and their token histories.
//
// One pass over the logits. Each row (request, beam) is cut into slices, one
// CTA each, that keep a running maximum and sum of exponentials per thread
// and a short buffer of the elements above the slice's keep-th best so far; a
// second kernel (one CTA per request) joins the slices' sums, scores their
// sorted lists and merges them. Bound: HBM for many rows, latency for few.
//
// Order: by score in 64 bits, equal scores by logit, then by beam and token
// (lowest first). Within a row the score grows with the logit, so a slice
// only needs the logit and the token. Exponentials are 32-bit, so a row's
// log-sum is right to lse_error() (some 1e-6) at first; where candidates of
// different beams are nearer than that, the second kernel sums the rows of
// these beams again in 64 bits (about 60 us for a row of 151,936, requests
// side by side, 8 loads a thread in flight; one by one 180 us. Few calls have
// such candidates, but ones whose beams are equal do).
#include <cuda_runtime.h>

#include "paged.h"

namespace rai {

namespace {

constexpr int kThreads = 256;
constexpr int kStepElements = kThreads * 16;
constexpr int kBufCap = 2048;  // candidates a slice holds between two sorts
constexpr float kLog2e = 1.4426950408889634f;

// A float's bits in the order of its value (-0 as +0).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float x, int token) {
  return ((uint64_t)ordered(x) << 32) | (0xffffffffu - (uint32_t)token);
}

// e^(x - m), where x = m also counts when both are infinite: a row with
// infinite logits shares its mass among them, a row of -inf among all.
__device__ __forceinline__ float exp_of(float d) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * kLog2e));
  return r;
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
__device__ __forceinline__ float2 exp2_of(float2 a) {
  float2 d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d.x) : "f"(a.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d.y) : "f"(a.y));
  return d;
}
__device__ __forceinline__ float weight(float x, float m) { return x == m ? 1.f : exp_of(x - m); }

template <int DT>
__device__ __forceinline__ float to_f32(uint32_t w, int half) {
  if constexpr (DT == kF16) return __half2float(__ushort_as_half((uint16_t)(w >> (16 * half))));
  else return __uint_as_float(half ? w & 0xffff0000u : w << 16);
}

struct Slice {
  float max;
  int pad;
  double sum;
};

__host__ __device__ inline size_t slice_bytes(int keep) { return sizeof(Slice) + (size_t)keep * 8; }

// Sorts n = 2^k keys, largest first.
__device__ __forceinline__ void bitonic(uint64_t* a, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step; step >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int lo = 2 * step * (i / step) + i % step, hi = lo + step;
        const bool down = (lo & size) == 0;
        const uint64_t x = a[lo], y = a[hi];
        if ((x < y) == down) a[lo] = y, a[hi] = x;
      }
    }
  __syncthreads();
}

// The `keep` largest of buf[0 .. n), sorted, in front; keys are unique. Up to
// a key per thread each counts the larger ones (n steps, two barriers; a sort
// of 256 has 36 barriers and takes three times as long), more are sorted.
__device__ __forceinline__ void prune(uint64_t* buf, int n, int keep) {
  if (n <= kThreads) {
    uint64_t k = 0;
    int rank = 0;
    if ((int)threadIdx.x < n) {
      k = buf[threadIdx.x];
#pragma unroll 8
      for (int i = 0; i < n; ++i) rank += buf[i] > k;
    }
    __syncthreads();
    if ((int)threadIdx.x < n && rank < keep) buf[rank] = k;
    __syncthreads();
    return;
  }
  int size = 512;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kThreads) buf[i] = 0;
  bitonic(buf, size);
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 4) beam_slice_kernel(BeamArgs a, int slices, int len) {
  constexpr int V = DT == kF32 ? 4 : 8;  // elements of 16 bytes
  constexpr int kE = DT == kF32 ? 4 : 2;
  constexpr int N = kStepElements / kThreads, kVecs = N / V;  // elements and 16-byte loads of a thread in a step
  __shared__ uint64_t buf[kBufCap];
  __shared__ uint64_t tops[kMaxKeep + 1];
  static_assert(kThreads / 4 == kMaxKeep, "groups");
  __shared__ int count;
  __shared__ float wm[kThreads / 32];
  __shared__ double wsum[kThreads / 32];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int row = blockIdx.y, slice = blockIdx.x;
  const int begin = slice * len, end = min(a.vocab, begin + len);
  const char* src = static_cast<const char*>(a.logits) + (long long)row * a.row * kE;
  // Vector slots from the 16-byte boundary at or before the slice's start.
  const int off = (int)((reinterpret_cast<uintptr_t>(src + (long long)begin * kE) & 15) / kE);
  const int base = begin - off;
  constexpr int kStep = kStepElements;
  if (threadIdx.x == 0) count = 0;
  float m = -INFINITY;
  double sum = 0.0;
  uint64_t bar = 0;  // keys at or above it are kept
  float bar_x = -INFINITY;
  auto first_of = [&](int at, int u) { return at + (u * kThreads + (int)threadIdx.x) * V; };
  auto inside = [&](int at) { return at >= begin && at + kStep <= end; };  // the step is whole
  auto fetch = [&](int at, uint4 (&w)[kVecs]) {  // whole vectors only
    const bool all = inside(at);
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int e0 = first_of(at, u);
      if (all || (e0 >= begin && e0 + V <= end)) w[u] = __ldcs(reinterpret_cast<const uint4*>(src + (long long)e0 * kE));
    }
  };
  // The step's elements; bit per element that is there.
  auto take = [&](int at, const uint4 (&w)[kVecs], float (&x)[N]) -> uint32_t {
    const bool all = inside(at);
    uint32_t there = 0;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int e0 = first_of(at, u);
      if (all || (e0 >= begin && e0 + V <= end)) {
        const uint32_t ws[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if constexpr (DT == kF32) x[u * V + i] = __uint_as_float(ws[i]);
          else x[u * V + i] = to_f32<DT>(ws[i / 2], i & 1);
        }
        there |= ((1u << V) - 1u) << (u * V);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[u * V + i] = -INFINITY;
          if (e0 + i >= begin && e0 + i < end) {
            if constexpr (DT == kF32) x[u * V + i] = reinterpret_cast<const float*>(src)[e0 + i];
            else x[u * V + i] = to_f32<DT>(reinterpret_cast<const uint16_t*>(src)[e0 + i], 0);
            there |= 1u << (u * V + i);
          }
        }
      }
    }
    return there;
  };
  // Elements of `among` at or above the bar go to the buffer; the ones that
  // find it full come back.
  auto push = [&](int at, const float (&x)[N], uint32_t among) -> uint32_t {
    uint32_t full = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (x[i] >= bar_x && (among >> i & 1u)) {
        const uint64_t k = key_of(x[i], first_of(at, i / V) + i % V);
        if (k >= bar) {
          const int slot = atomicAdd(&count, 1);
          if (slot < kBufCap) buf[slot] = k;
          else full |= 1u << i;
        }
      }
    return full;
  };
  // Cut the buffer's first n to the keep best, which raises the bar.
  auto cut = [&](int n) {
    prune(buf, n, a.keep);
    bar = n >= a.keep ? buf[a.keep - 1] : 0;
    bar_x = bar ? unordered((uint32_t)(bar >> 32)) : -INFINITY;
    if (threadIdx.x == 0) count = min(n, a.keep);
    __syncthreads();
  };
  uint4 w[kVecs];
  fetch(base, w);
  __syncthreads();
  // Rounds of kRound steps without a barrier: a buffer that overflows within
  // one (rising logits, many equal ones) is put back to where it was and the
  // round's elements are pushed again with a barrier each step.
  constexpr int kRound = 4;
  int held = 0;  // in the buffer at the round's start
  for (int r0 = base; r0 < end; r0 += kRound * kStep) {
    const int stop = min(end, r0 + kRound * kStep);
    for (int at = r0; at < stop; at += kStep) {
      float x[N];
      const uint32_t there = take(at, w, x);
      if (at + kStep < end) fetch(at + kStep, w);  // in flight through this step
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < N; ++i) top = fmaxf(top, x[i]);  // (elements that are not there are -inf)
      if (there) {
        if (top > m) {
          sum *= (double)weight(m, top);
          m = top;
        }
        // Pairs: (x - m) log2(e), exponentials, sums.
        float2 part[2] = {{0.f, 0.f}, {0.f, 0.f}};
        const float2 mm = {-m, -m};
#pragma unroll
        for (int i = 0; i < N; i += 2) part[i / 2 & 1] = add2(part[i / 2 & 1], exp2_of(mul2(add2({x[i], x[i + 1]}, mm), {kLog2e, kLog2e})));
        float all = (part[0].x + part[0].y) + (part[1].x + part[1].y);
        if (!(fabsf(m) <= 3.4028235e38f) || !(all == all)) {
          // An infinite maximum, or a NaN among them, which is not chosen.
          all = 0.f;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (!(x[i] == x[i])) x[i] = -INFINITY;
            if (there >> i & 1u) all += weight(x[i], m);
          }
        }
        sum += (double)all;
      }
      if (at == base) {
        // A first bar: the keep-th largest of the best of 64 groups of four
        // threads is no larger than the keep-th largest element.
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if ((there >> i & 1u) && x[i] == top) best = max(best, key_of(x[i], first_of(at, i / V) + i % V));
        best = max(best, __shfl_xor_sync(~0u, best, 1));
        best = max(best, __shfl_xor_sync(~0u, best, 2));
        if ((threadIdx.x & 3) == 0) tops[threadIdx.x >> 2] = best;
        __syncthreads();
        if (threadIdx.x < kMaxKeep) {
          const uint64_t k = tops[threadIdx.x];
          int rank = 0;
#pragma unroll 8
          for (int i = 0; i < kMaxKeep; ++i) rank += tops[i] > k || (tops[i] == k && i < (int)threadIdx.x);
          if (rank == a.keep - 1) tops[kMaxKeep] = k;
        }
        __syncthreads();
        bar = tops[kMaxKeep];
        bar_x = bar ? unordered((uint32_t)(bar >> 32)) : -INFINITY;
      }
      if (there && top >= bar_x) push(at, x, there);
    }
    __syncthreads();
    const int n = count;
    __syncthreads();  // everyone has read the count
    if (n > kBufCap) {
      if (threadIdx.x == 0) count = held;
      __syncthreads();
      for (int at = r0; at < stop; at += kStep) {
        uint4 v[kVecs];
        float x[N];
        fetch(at, v);
        uint32_t rest = take(at, v, x);
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (!(x[i] == x[i])) x[i] = -INFINITY;
        for (int again = 1; again;) {
          rest = push(at, x, rest);
          again = __syncthreads_or(rest != 0);
          const int now = min(count, kBufCap);
          __syncthreads();
          held = now;
          if (again || now > kBufCap / 2) {
            cut(now);
            held = min(now, a.keep);
          }
        }
      }
    } else if (n > a.keep + 80 || (r0 == base && n > a.keep)) {
      cut(n);
      held = min(n, a.keep);
    } else {
      held = n;
    }
  }
  const int n = held;
  prune(buf, n, a.keep);
  // Join the threads' sums.
  float top = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  if ((threadIdx.x & 31) == 0) wm[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) top = fmaxf(top, wm[i]);
  double s = sum == 0.0 ? 0.0 : sum * (double)weight(m, top);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if ((threadIdx.x & 31) == 0) wsum[threadIdx.x >> 5] = s;
  __syncthreads();
  char* out = static_cast<char*>(a.ws) + ((long long)row * slices + slice) * slice_bytes(a.keep);
  if (threadIdx.x == 0) {
    Slice r = {top, 0, 0.0};
    for (int i = 0; i < kThreads / 32; ++i) r.sum += wsum[i];
    *reinterpret_cast<Slice*>(out) = r;
  }
  for (int i = threadIdx.x; i < a.keep; i += kThreads)
    reinterpret_cast<uint64_t*>(out + sizeof(Slice))[i] = i < n ? buf[i] : 0;
}

constexpr int kMaxSlices = 16;

// A candidate's place in the order: its score's bits in order, then its
// logit's, then its flat number (beam * vocab + token) the other way round.
struct Cand {
  uint64_t score = 0;  // 0: none
  uint32_t logit = 0, flat = 0;
};
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
  return b ^ ((b >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double unordered(uint64_t o) {
  return __longlong_as_double((long long)(o ^ ((o >> 63) ? 1ull << 63 : ~0ull)));
}
// The first of the warp's candidates, in every lane.
__device__ __forceinline__ Cand first_of_warp(const Cand& c) {
  Cand b;
  const uint32_t hi = __reduce_max_sync(~0u, (uint32_t)(c.score >> 32));
  bool in = (uint32_t)(c.score >> 32) == hi;
  const uint32_t lo = __reduce_max_sync(~0u, in ? (uint32_t)c.score : 0u);
  in = in && (uint32_t)c.score == lo;
  b.score = (uint64_t)hi << 32 | lo;
  b.logit = __reduce_max_sync(~0u, in ? c.logit : 0u);
  in = in && c.logit == b.logit;
  b.flat = __reduce_min_sync(~0u, in ? c.flat : 0xffffffffu);
  return b;
}

// How far a row's log-sum may be off, by the steps of a thread of the pass. A
// weight is the product of at most steps + 2 exponentials (its own, one for
// each time its thread's maximum moved, one for the join), each off by 2^-22 of
// itself and by 2.25 x 2^-24 of its argument (difference, product, constant).
// The arguments of one weight add up to its distance from the maximum, whose
// mean over the mass is at most ln(vocab). Five more roundings add 16 weights.
__host__ __device__ inline double lse_error(int steps, int vocab) {
  return ((steps + 2) * 4.0 + 2.25 * log((double)vocab) + 5.0) * 0x1p-24;
}
template <int DT>
__device__ __forceinline__ float logit_at(const void* row, int i) {
  if constexpr (DT == kF32) return static_cast<const float*>(row)[i];
  else return to_f32<DT>(static_cast<const uint16_t*>(row)[i], 0);
}
// The sum of e^(x - top) over a row in 64 bits, by the CTA; the same for the
// same logits wherever they lie. `top` is finite.
template <int DT>
__device__ __noinline__ double exact_sum(const void* row, int vocab, float top, double* warps) {
  constexpr int kLoads = 8;  // in flight
  double sum = 0.0;
  for (int i0 = threadIdx.x; i0 < vocab; i0 += kLoads * blockDim.x) {
    float x[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const long long i = i0 + (long long)u * blockDim.x;
      x[u] = i < vocab ? logit_at<DT>(row, (int)i) : -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      if (x[u] == x[u]) sum += exp((double)x[u] - (double)top);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = sum;
  __syncthreads();
  double all = 0.0;
  for (int w = 0; w < (int)blockDim.x >> 5; ++w) all += warps[w];
  return all;
}

constexpr int kMergeThreads = 512;  // at least: the work but the lists' is shared among all

// One CTA per request, one thread per (beam, slice) list; each round takes
// the best of the lists' heads. Bound by the rounds' latency.
__global__ void __launch_bounds__(kMaxBeams * kMaxSlices) beam_merge_kernel(BeamArgs a, int slices, double error) {
  __shared__ double sums[kMaxBeams * kMaxSlices], lse[kMaxBeams];  // lse: log of the sum beside the maximum
  __shared__ float tops[kMaxBeams * kMaxSlices];
  __shared__ Cand warp_best[2][kMaxBeams * kMaxSlices / 32];
  __shared__ Cand chosen[kMaxKeep];
  __shared__ int next[kMaxBeams];
  __shared__ uint32_t again;  // beams whose sums are needed in 64 bits
  __shared__ double warp_sums[kMaxBeams * kMaxSlices / 32];
  __shared__ uint64_t heads[4096];  // the lists, where they fit
  pdl_wait_prior();
  pdl_launch_dependents();
  const int req = blockIdx.x, lists = a.beams * slices, warps = (lists + 31) / 32;  // that hold lists
  const size_t sb = slice_bytes(a.keep);
  const char* ws = static_cast<const char*>(a.ws) + (long long)req * lists * sb;
  const bool real = (int)threadIdx.x < lists;
  const int beam = threadIdx.x / slices;
  const char* mine_at = ws + (long long)threadIdx.x * sb;
  Slice s = {-INFINITY, 0, 0.0};
  float score = 0.f;
  if (real) {
    s = *reinterpret_cast<const Slice*>(mine_at);
    score = a.scores[req * a.beams + beam];
    if (!(score == score)) score = -INFINITY;
    tops[threadIdx.x] = s.max;
  }
  if (threadIdx.x == 0) again = 0;
  const bool fits = lists * a.keep <= 4096;
  if (fits)
    for (int i = threadIdx.x; i < lists * a.keep; i += blockDim.x)
      heads[i] = reinterpret_cast<const uint64_t*>(ws + (long long)(i / a.keep) * sb + sizeof(Slice))[i % a.keep];
  __syncthreads();
  float top = -INFINITY;
  if (real) {
    for (int i = 0; i < slices; ++i) top = fmaxf(top, tops[beam * slices + i]);
    sums[threadIdx.x] = s.sum * (s.max == top ? 1.0 : exp((double)s.max - (double)top));
  }
  __syncthreads();
  if (threadIdx.x < a.beams) {
    double sum = 0.0;
    for (int i = 0; i < slices; ++i) sum += sums[threadIdx.x * slices + i];
    lse[threadIdx.x] = log(sum);
  }
  __syncthreads();
  const uint64_t* list = fits ? heads + threadIdx.x * a.keep : reinterpret_cast<const uint64_t*>(mine_at + sizeof(Slice));
  int at = 0;
  auto head = [&]() {
    Cand c;
    c.flat = 0xffffffffu;
    if (!real || at >= a.keep) return c;
    const uint64_t k = list[at];
    if (!k) return c;
    c.logit = (uint32_t)(k >> 32);
    c.flat = (uint32_t)(beam * a.vocab) + (0xffffffffu - (uint32_t)k);
    const float x = unordered(c.logit);
    const double d = x == top ? 0.0 : (double)x - (double)top;
    const double total = (double)score + (d - lse[beam]);
    c.score = ordered(total == total ? total : -INFINITY);  // (a beam of +infinity, a token of weight 0)
    return c;
  };
  Cand mine;
  auto choose = [&]() {
    at = 0;
    mine = head();
    for (int r = 0; r < a.keep; ++r) {
      Cand best = first_of_warp(mine);
      if (warps > 1) {
        // Every warp reads all warps' best; two buffers, so one barrier a round.
        const int lane = threadIdx.x & 31;
        if (lane == 0) warp_best[r & 1][threadIdx.x >> 5] = best;
        asm volatile("bar.sync 1, %0;" ::"r"(warps * 32) : "memory");
        Cand c;
        c.flat = 0xffffffffu;
        if (lane < warps) c = warp_best[r & 1][lane];
        best = first_of_warp(c);
      }
      if (threadIdx.x == 0) chosen[r] = best;
      if (best.score && best.flat == mine.flat) {
        ++at;
        mine = head();
      }
    }
  };
  if ((int)threadIdx.x < warps * 32) choose();
  __syncthreads();
  // Candidates of different beams that the sums' error may have put in the
  // wrong order: neighbours among the chosen ones, and a list's first one left
  // against the last one chosen of another beam. (Equal scores of -inf are
  // equal whatever the sums; their difference is NaN.)
  auto near = [&](const Cand& x, const Cand& y) { return y.score && unordered(x.score) - unordered(y.score) <= 2.0 * error; };
  auto beam_of = [&](const Cand& c) { return (int)c.flat / a.vocab; };
  if ((int)threadIdx.x + 1 < a.keep) {
    const Cand x = chosen[threadIdx.x], y = chosen[threadIdx.x + 1];
    if (near(x, y) && beam_of(x) != beam_of(y)) atomicOr(&again, 1u << beam_of(x) | 1u << beam_of(y));
  }
  if (real && mine.score && near(chosen[a.keep - 1], mine)) {
    for (int r = a.keep - 1; r >= 0 && near(chosen[r], mine); --r)
      if (beam_of(chosen[r]) != beam) atomicOr(&again, 1u << beam_of(chosen[r]) | 1u << beam);
  }
  __syncthreads();
  if (again) {
    for (int b = 0; b < a.beams; ++b) {
      if (!(again >> b & 1u)) continue;
      float m = -INFINITY;
      for (int i = 0; i < slices; ++i) m = fmaxf(m, tops[b * slices + i]);
      if (!(fabsf(m) <= 3.4028235e38f)) continue;  // a number of equal ones: exact
      const char* row = static_cast<const char*>(a.logits) + (long long)(req * a.beams + b) * a.row * (a.dtype == kF32 ? 4 : 2);
      const double sum = a.dtype == kF32   ? exact_sum<kF32>(row, a.vocab, m, warp_sums)
                         : a.dtype == kF16 ? exact_sum<kF16>(row, a.vocab, m, warp_sums)
                                           : exact_sum<kBF16>(row, a.vocab, m, warp_sums);
      if (threadIdx.x == 0) lse[b] = log(sum);
    }
    __syncthreads();
    if ((int)threadIdx.x < warps * 32) choose();
  }
  __syncthreads();
  for (int r = threadIdx.x; r < a.keep; r += blockDim.x) {
    const Cand c = chosen[r];
    const long long o = (long long)req * a.keep + r;
    const int b = c.score ? (int)c.flat / a.vocab : -1;
    a.cand_score[o] = c.score ? (float)unordered(c.score) : -INFINITY;
    a.cand_beam[o] = b;
    a.cand_token[o] = c.score ? (int)c.flat - b * a.vocab : -1;
  }
  if (threadIdx.x < 32) {
    // Candidates that do not end, in order.
    int n = 0;
    for (int r0 = 0; r0 < a.keep; r0 += 32) {
      const int r = r0 + threadIdx.x;
      const bool goes = r < a.keep && chosen[r].score && (int)chosen[r].flat % a.vocab != a.eos;
      const uint32_t mask = __ballot_sync(~0u, goes);
      const int place = n + __popc(mask & ((1u << threadIdx.x) - 1u));
      if (goes && place < a.beams) next[place] = r;
      n += __popc(mask);
    }
    for (int i = n + threadIdx.x; i < a.beams; i += 32) next[i] = -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.beams; i += blockDim.x) {
    const long long o = (long long)req * a.beams + i;
    const bool some = next[i] >= 0;
    const Cand c = some ? chosen[next[i]] : Cand{};
    const int b = some ? (int)c.flat / a.vocab : 0;
    a.score[o] = some ? (float)unordered(c.score) : -INFINITY;
    a.parent[o] = some ? req * a.beams + b : -1;
    a.token[o] = some ? (int)c.flat - b * a.vocab : -1;
  }
  if (!a.history) return;
  for (int i = 0; i < a.beams; ++i) {
    const long long o = (long long)req * a.beams + i;
    if (next[i] < 0) {
      if (threadIdx.x == 0) a.out_len[o] = 0;
      continue;
    }
    const Cand c = chosen[next[i]];
    const int b = (int)c.flat / a.vocab;
    const long long p = (long long)req * a.beams + b;
    int n = a.hist_len[p];
    const bool ok = n >= 0 && n < a.hist_cap;
    if (!ok) n = min(max(n, 0), a.hist_cap);
    for (int x = threadIdx.x; x < n; x += blockDim.x) a.out_history[o * a.out_stride + x] = a.history[p * a.hist_stride + x];
    if (threadIdx.x == 0) {
      if (ok) a.out_history[o * a.out_stride + n] = (int)c.flat - b * a.vocab;
      else atomicOr(a.err, kErrBadInput);
      a.out_len[o] = ok ? n + 1 : n;
    }
  }
}

int slices_of(int batch, int beams, int vocab) {
  // As many CTAs as are resident at once (four on each SM), none with less
  // than 2048 elements.
  const long long rows = (long long)batch * beams;
  long long n = 4ll * device_sm_count() / rows;
  const long long most = (vocab + 2047) / 2048;
  n = n < most ? n : most;
  n = n < kMaxSlices ? n : kMaxSlices;
  return n < 1 ? 1 : (int)n;
}

}  // namespace

size_t beam_workspace(int batch, int beams, int vocab, int keep) {
  return (size_t)batch * beams * slices_of(batch, beams, vocab) * slice_bytes(keep);
}

cudaError_t beam_select(const BeamArgs& a, cudaStream_t s) {
  const int slices = slices_of(a.batch, a.beams, a.vocab);
  int len = (a.vocab + slices - 1) / slices;
  len = (len + 7) / 8 * 8;
  const dim3 grid(slices, a.batch * a.beams);
  cudaError_t e = a.dtype == kF32   ? launch_pdl(beam_slice_kernel<kF32>, grid, dim3(kThreads), 0, s, a, slices, len)
                  : a.dtype == kF16 ? launch_pdl(beam_slice_kernel<kF16>, grid, dim3(kThreads), 0, s, a, slices, len)
                                    : launch_pdl(beam_slice_kernel<kBF16>, grid, dim3(kThreads), 0, s, a, slices, len);
  if (e != cudaSuccess) return e;
  const int lists = a.beams * slices;
  const int threads = lists > kMergeThreads ? (lists + 31) / 32 * 32 : kMergeThreads;
  return launch_pdl(beam_merge_kernel, dim3(a.batch), dim3(threads), 0, s, a, slices, lse_error((len + kStepElements - 1) / kStepElements + 1, a.vocab));
}

}  // namespace rai
