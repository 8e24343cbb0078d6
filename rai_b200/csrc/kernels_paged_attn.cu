// Attention of a ragged chunk of new rows over a paged cache, for few query
// rows per KV head (decoding, draft verification) and for every type and head
// size the tcgen05 kernel does not take.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(s_ij - max_j s_ij),
//   s_ij = scale q_i . k_j   (or cap tanh(scale q_i . k_j / cap)),
// over the tokens j that row i sees: j <= pos_i, and j > pos_i - window.
//
// The query rows of one KV head (group heads x chunk rows, flattened) form
// row tiles of MT rows; K and V stream through shared memory in tiles of NT
// tokens, once per row tile, with the running maximum and sum of the softmax
// in registers (one pass over the cache). What bounds it is HBM: at 8 chunk
// rows x 4 heads a byte of K and V gets 32 multiply-adds, a few percent of
// the tensor rate, so mma.sync from registers carries it.
//
// Work split: all (sequence, row tile, KV head) items' token tiles form one
// line of W tiles, cut into equal ranges, one per resident CTA, so ragged
// lengths and few long sequences fill the machine alike. An item cut between
// CTAs leaves partial sums (m, l, unnormalized o in f32) in the workspace;
// paged_combine_kernel joins them in CTA order (the same bits every run).
//
// 16-bit types: products of 16-bit operands in f32 (m16n8k16); P is rounded
// to the operand type (relative 2^-9 bf16, 2^-12 f16, about the rounding of
// the 16-bit output itself), its sum is taken before the rounding. f16
// probabilities carry a factor 2^10 so that small ones stay normal.
// f32: each operand is split in two tf32 halves and the three products that
// matter are summed in f32 (2^-21 relative per product).
//
// Masked places never reach a result: scores are replaced, not biased; token
// slots outside a row tile's visible range are not loaded (zero filled); and
// a V value that is not finite in a tile where some row may not see it is
// replaced by zero and added back to the rows that do see it at the end.
#include <cuda_runtime.h>

#include <mutex>

#include "paged_attn.cuh"

namespace rai {

// kernels_paged_tc.cu
bool paged_attention_tc_takes(const AttnArgs& a);
size_t paged_attention_tc_workspace(const AttnArgs& a);
cudaError_t paged_attention_tc(const AttnArgs& a, cudaStream_t s);

namespace paged_attn {

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static Encode encoder() {
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<Encode>(f);
  }();
  return encode;
}

bool make_q_map(const AttnArgs& a, int rows, CUtensorMap* map) {
  const Encode encode = encoder();
  if (!encode || a.group > 256 || rows > 256) return false;
  const int heads = a.group * a.c.nkv;
  const cuuint64_t dims[3] = {(cuuint64_t)a.c.hd, (cuuint64_t)heads, (cuuint64_t)a.c.rows};
  // The stride of a dimension of one means nothing, but has to be valid.
  const cuuint64_t strides[2] = {(cuuint64_t)(heads == 1 ? 8 : a.q_head) * 2, (cuuint64_t)(a.c.rows == 1 ? 8 : a.q_row) * 2};
  if (!strides[0] || !strides[1] || strides[0] >= (1ull << 40) || strides[1] >= (1ull << 40)) return false;
  const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)rows}, ones[3] = {1, 1, 1};
  return encode(map, a.dtype == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                const_cast<void*>(a.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool make_maps(const PagedChunk& c, int dtype, int box, KvMaps* maps) {
  const Encode encode = encoder();
  if (!encode) return false;
  const int elt = dtype == kF32 ? 4 : 2;
  const CUtensorMapDataType type = dtype == kF32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const cuuint64_t dims[4] = {(cuuint64_t)c.hd, c.page.d, (cuuint64_t)c.nkv, (cuuint64_t)c.n_pages};
  const cuuint32_t boxes[4] = {128u / elt, (cuuint32_t)box, 1, 1}, ones[4] = {1, 1, 1, 1};
  for (int kv = 0; kv < 2; ++kv) {
    long long st[3] = {kv ? c.v_slot : c.k_slot, kv ? c.v_head : c.k_head, kv ? c.v_page : c.k_page};
    cuuint64_t strides[3];
    for (int i = 0; i < 3; ++i) {
      // The stride of a dimension of one means nothing, but has to be valid.
      if (dims[i + 1] == 1) st[i] = 16 / elt;
      strides[i] = (cuuint64_t)st[i] * elt;
      if (st[i] <= 0 || strides[i] >= (1ull << 40)) return false;
    }
    if (encode(kv ? &maps->v : &maps->k, type, 4, kv ? c.v : c.k, dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  }
  return true;
}

}  // namespace paged_attn

namespace {

using namespace paged_attn;

constexpr int kThreads = 128;

template <int DT_, int HD_, int MT_>
struct Cfg {
  static constexpr int DT = DT_, HD = HD_, MT = MT_;
  static constexpr int kElt = DT == kF32 ? 4 : 2;
  static constexpr int kRowB = HD * kElt;
  static constexpr int NT = DT == kF32 ? (HD >= 128 ? 32 : 64) : HD == 64 ? 128 : 64;
  static constexpr int kTileB = NT * kRowB;
  // Heads of 64: two stages of 32 KB leave room for three CTAs an SM (64
  // streams of 300 to 2,300 tokens: 27.8 us; three stages and two CTAs 31.2,
  // four of half the size 33.1).
  static constexpr int kStages = HD == 256 || HD == 64 ? 2 : 3;
  static constexpr int WM = MT / 16, WN = 4 / WM, NTW = NT / WN;
  static constexpr bool kQReg = DT != kF32 && HD <= 128;  // query fragments stay in registers
  static constexpr int kQB = kQReg ? 0 : MT * kRowB;
  static constexpr int kMergeB = WN > 1 ? 2 * 16 * (HD + 4) * 4 + 4 * 16 * 8 : 0;
  static constexpr int kBlocks = kRowB / 128;  // 128-byte column blocks
  static constexpr int kSmem = kStages * 2 * kTileB + kQB + kMergeB + 1024;
  static constexpr int kPartFloats = MT * (HD + 2);
  static constexpr float kPShift = DT == kF16 ? 10.f : 0.f;
};

// K and V of the cursor's tile, from pages looked up a tile ahead. Each lane
// knows the offsets of NT / 32 tokens; a token's copies get its offset by a
// shuffle, eight copies' addresses at a time.
template <typename C>
__device__ __forceinline__ void load_tile(const Params& p, const Cursor<C::MT, C::NT>& cur, TilePages<C::NT>& pages,
                                          uint32_t sk, uint32_t sv) {
  constexpr int kChunks = C::kRowB / 16;  // per row
  constexpr int kRowsPer = kThreads / kChunks, kIter = C::NT / kRowsPer;
  const PagedChunk& c = p.a.c;
  const int lane = threadIdx.x & 31, chunk = threadIdx.x % kChunks, r0 = threadIdx.x / kChunks;
  const int t0 = (cur.it.first + cur.tile) * C::NT;
  const bool in_head = chunk * 16 < c.hd * C::kElt;
  pages.check(c, cur.it, t0, lane);
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const char* base = static_cast<const char*>(kv ? c.v : c.k) + (long long)cur.head * (kv ? c.v_head : c.k_head) * C::kElt + chunk * 16;
    long long off[C::NT / 32];
    pages.offsets(c, t0, lane, kv ? c.v_page : c.k_page, kv ? c.v_slot : c.k_slot, off);
    constexpr int kB = kIter < 8 ? kIter : 8;
#pragma unroll
    for (int i0 = 0; i0 < kIter; i0 += kB) {
      long long o[kB];
#pragma unroll
      for (int i = 0; i < kB; ++i) {
        const int row = r0 + (i0 + i) * kRowsPer;
        // The lane's rows of one pass lie in one half of the tile or in
        // both (fewer chunks a row than lanes).
        long long x = __shfl_sync(~0u, off[0], row & 31);
#pragma unroll
        for (int y = 1; y < C::NT / 32; ++y) {
          const long long z = __shfl_sync(~0u, off[y], row & 31);
          if (row / 32 == y) x = z;
        }
        o[i] = in_head ? x : -1;
      }
#pragma unroll
      for (int i = 0; i < kB; ++i)
        cp_async16_or_zero((kv ? sv : sk) + tile_at(C::NT, r0 + (i0 + i) * kRowsPer, chunk), o[i] >= 0 ? base + o[i] * C::kElt : base, o[i] >= 0);
    }
  }
}

template <int DT>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == kBF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo with both in tf32: hi the upper 19 bits, lo the rest (exact),
// rounded by the half step added below the bits that the tensor core reads.
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) + 0x1000u;
}
// The same for the operand that meets K and V (q, probabilities): a lower half
// of zero would make NaN of an infinite one, so it gets 2^-40 of the upper
// half, which is nothing beside the product that is left out. (An infinite x
// has -0 for its lower half: the NaN of inf - inf and the half step.)
__device__ __forceinline__ void split_first(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  const float h = __uint_as_float(hi);
  lo = __float_as_uint(fmaf(h, 0x1p-40f, x - h)) + 0x1000u;
}
// d += a b of f32 operands: the small products first.
__device__ __forceinline__ void mma8x3(float (&d)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split(b0, h0, l0);
  split(b1, h1, l1);
  mma8(d, al, h0, h1);
  mma8(d, ah, l0, l1);
  mma8(d, ah, h0, h1);
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ float lds_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
template <typename C, bool TMA>
__global__ void __launch_bounds__(kThreads)
    paged_attn_kernel(const __grid_constant__ Params p, const __grid_constant__ KvMaps maps, int box) {
  constexpr int DT = C::DT, HD = C::HD, MT = C::MT, NT = C::NT, WN = C::WN, NTW = C::NTW, S = C::kStages;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ long long sh[kPlanWords];
  __shared__ uint64_t full[S], empty[S];  // TMA: a stage has landed, every warp is done with it
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t sq = base + S * 2 * C::kTileB;
  float* merge = reinterpret_cast<float*>(smem_raw + (sq + C::kQB - smem_u32(smem_raw)));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wm = warp % C::WM, wn = warp / C::WM;
  const int g = lane >> 2, t4 = lane & 3;
  const PagedChunk& ch = p.a.c;

  if (TMA && threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kThreads / 32);
    }
    fence_barrier_init();
  }
  pdl_wait_prior();
  pdl_launch_dependents();
  Range rg;
  Cursor<MT, NT> ld;
  if (p.direct) {
    ld.unit = blockIdx.x / ch.nkv, ld.head = blockIdx.x - ld.unit * ch.nkv;
    ld.it = item_of<MT, NT>(p, ld.unit);
    ld.tile = 0, ld.pos = 0;
    rg.begin = 0, rg.end = ld.it.tiles;
    if (TMA) __syncthreads();
  } else {
    rg = plan<MT, NT, kThreads>(p, blockIdx.x, sh);  // (with barriers of the CTA)
  }
  const long long begin = rg.begin, end = rg.end;
  if (begin >= end) {
    if (threadIdx.x == 0 && !p.whole) reinterpret_cast<Cut*>(p.a.part)[blockIdx.x] = Cut{};
    return;
  }

  if (!p.direct) ld.seek(p, rg);
  Cursor<MT, NT> cur = ld;
  if (threadIdx.x == 0 && !p.whole) leave_cut<MT, NT>(p, rg, cur, blockIdx.x);
  uint32_t loaded = 0, done = 0;  // tiles
  TilePages<NT> pages;
  TilePieces<NT, C::kBlocks, C::kElt> pieces;
  // The next tile of K and V (TMA: by warp 0 alone).
  auto fetch = [&] {
    if (ld.pos >= end) return;
    if constexpr (TMA) pieces.fetch(ch, ld.it, (ld.it.first + ld.tile) * NT, box, lane);
    else pages.fetch(ch, ld.it, (ld.it.first + ld.tile) * NT, lane);
  };
  auto load = [&] {
    const uint32_t i = loaded % S, st = base + i * 2 * C::kTileB;
    if constexpr (TMA) {
      const int t0 = (ld.it.first + ld.tile) * NT;
      pieces.load2(ch, ld.it, t0, box, lane, &maps.k, &maps.v, ld.head, st, st + C::kTileB, &full[i]);
    } else {
      load_tile<C>(p, ld, pages, st, st + C::kTileB);
    }
    ++loaded;
    ld.next(p);
    fetch();
  };
  bool ok = true;
  if (!TMA || warp == 0) {
    fetch();
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
      if (ld.pos < end) load();
      if (!TMA) cp_async_commit();
    }
  }

  uint32_t qf[C::kQReg ? HD / 16 : 1][4];
  float acc[HD / 8][4];
  float m[2], l[2];
  int pos[2];  // position of the thread's two rows, below 0: none
  bool poison = false, fresh = true;
  int first_slot = 0;  // of the workspace: 0 for the CTA's first item, 1 for its last
  for (; cur.pos < end; ++done) {
    const Item& it = cur.it;
    if (fresh) {
      // The item's rows: query fragments, positions, empty sums.
      const int p0 = it.len - it.n;
      const void* q = p.a.q;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = wm * 16 + g + 8 * h;
        const int f = it.f0 + r, i = (int)p.group_div.quot(f), j = f - i * p.a.group;
        const bool real = r < it.nf;
        pos[h] = real ? p0 + i : -1;
        if constexpr (C::kQReg) {
          const long long o = (long long)(it.start + i) * p.a.q_row + (long long)(cur.head * p.a.group + j) * p.a.q_head;
          const uint16_t* row = static_cast<const uint16_t*>(q) + o;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int col = kk * 16 + e * 8 + 2 * t4;
              qf[kk][2 * e + h] = real && col < ch.hd ? *reinterpret_cast<const uint32_t*>(row + col) : 0u;
            }
        }
        m[h] = -INFINITY;
        l[h] = 0.f;
      }
      if constexpr (!C::kQReg) {
        __syncthreads();  // the last item's reads of the query tile are over
        constexpr int kChunks = C::kRowB / 16;
        for (int x = threadIdx.x; x < MT * kChunks; x += kThreads) {
          const int r = x / kChunks, chunk = x % kChunks;
          const int f = it.f0 + r, i = (int)p.group_div.quot(f), j = f - i * p.a.group;
          const bool real = r < it.nf && chunk * 16 < ch.hd * C::kElt;
          const long long o = (long long)(it.start + i) * p.a.q_row + (long long)(cur.head * p.a.group + j) * p.a.q_head;
          uint4 w = make_uint4(0, 0, 0, 0);
          if (real) w = *reinterpret_cast<const uint4*>(static_cast<const char*>(q) + o * C::kElt + chunk * 16);
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(sq + tile_at(MT, r, chunk)), "r"(w.x), "r"(w.y),
                       "r"(w.z), "r"(w.w)
                       : "memory");
        }
        __syncthreads();
      }
#pragma unroll
      for (int x = 0; x < HD / 8; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = 0.f;
      poison = false;
      fresh = false;
    }
    if constexpr (TMA) {
      if (warp == 0 && ld.pos < end) {
        // The stage of the last tile is free once every warp is done with it.
        if (done > 0) ok = __all_sync(~0u, wait_bar(&empty[(done - 1) % S], (done - 1) / S & 1, ch.err));
        if (ok) load();
      }
      ok = __all_sync(~0u, ok && wait_bar(&full[done % S], done / S & 1, ch.err));
      if (!ok) break;
    } else {
      cp_async_wait<S - 2>();
      __syncthreads();
      // The stage that the last step read is free: fetch ahead.
      if (ld.pos < end) load();
      cp_async_commit();
    }
    const uint32_t sk = base + (done % S) * 2 * C::kTileB, sv = sk + C::kTileB;
    const int t0 = (it.first + cur.tile) * NT;
    const int p0 = it.len - it.n;
    const int plo = p0 + (int)p.group_div.quot(it.f0), phi = it.hi - 1;
    const bool masked = t0 + NT - 1 > plo || t0 < it.lo || (p.a.window > 0 && t0 <= phi - p.a.window);

    if (masked) {
      // V values that are not finite, where a row may not see them.
      bool bad = false;
#pragma unroll 4
      for (int x = threadIdx.x; x < C::kTileB / 16; x += kThreads) bad |= clean_chunk<DT>(sv + x * 16, t0 + x / 8 % NT, it);
      if (__syncthreads_or(bad)) poison = true;
      if (TMA) fence_async();  // the stage is TMA's again after this
    }

    // ---- S = Q K^T over this warp's tokens ----
    float s[NTW / 8][4];
#pragma unroll
    for (int x = 0; x < NTW / 8; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) s[x][y] = 0.f;
    const int w0 = wn * NTW;  // first token of the warp in the tile
    if constexpr (DT != kF32) {
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        uint32_t a[4];
        if constexpr (C::kQReg) {
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = qf[kk][e];
        } else {
          ldsm4(a, sq + tile_at(MT, wm * 16 + (lane & 15), kk * 2 + (lane >> 4)));
        }
#pragma unroll
        for (int x = 0; x < NTW / 16; ++x) {
          uint32_t b[4];
          ldsm4(b, sk + tile_at(NT, w0 + x * 16 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
          mma16<DT>(s[2 * x], a, b[0], b[1]);
          mma16<DT>(s[2 * x + 1], a, b[2], b[3]);
        }
      }
    } else {
      // The tensor core truncates as it adds, so each step's products get an
      // accumulator of their own and join the sum rounded to nearest.
#pragma unroll 4
      for (int kk = 0; kk < HD / 8; ++kk) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          split_first(lds_f32(sq + tile_at(MT, wm * 16 + g + 8 * (e & 1), kk * 2 + (e >> 1)) + 4 * t4), ah[e], al[e]);
#pragma unroll
        for (int x = 0; x < NTW / 8; ++x) {
          const int tk = w0 + x * 8 + g;
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma8x3(d, ah, al, lds_f32(sk + tile_at(NT, tk, kk * 2) + 4 * t4), lds_f32(sk + tile_at(NT, tk, kk * 2 + 1) + 4 * t4));
#pragma unroll
          for (int y = 0; y < 4; ++y) s[x][y] += d[y];
        }
      }
    }
    if (p.a.softcap > 0.f) {
#pragma unroll
      for (int x = 0; x < NTW / 8; ++x)
#pragma unroll
        for (int y = 0; y < 4; y += 2) {
          const float2 z = capped<DT>({s[x][y], s[x][y + 1]}, p.a.scale, p.a.softcap, p.inv_cap);
          s[x][y] = z.x;
          s[x][y + 1] = z.y;
        }
    }
    if (masked) {
#pragma unroll
      for (int x = 0; x < NTW / 8; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int t = t0 + w0 + x * 8 + 2 * t4 + (y & 1), pr = pos[y >> 1];
          const bool seen = t <= pr && t >= it.lo && (p.a.window <= 0 || t > pr - p.a.window);
          if (!seen) s[x][y] = -INFINITY;
        }
    }
    // ---- running softmax ----
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = m[h];
#pragma unroll
      for (int x = 0; x < NTW / 8; ++x) top = fmaxf(top, fmaxf(s[x][2 * h], s[x][2 * h + 1]));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      // Both products rounded before their difference: fused, a maximum that
      // stays would rescale by its own rounding at every tile (at 20,000 tokens
      // f32 outputs were off by 1.8e-5 so).
      const float mc = top == -INFINITY ? 0.f : __fmul_rn(top, p.c);
      const float fix = exp2_fast(__fmul_rn(m[h], p.c) - mc);  // m = -inf: 0
      m[h] = top;
      float sum = 0.f;
#pragma unroll
      for (int x = 0; x < NTW / 8; ++x)
#pragma unroll
        for (int y = 2 * h; y < 2 * h + 2; ++y) {
          s[x][y] = exp2_fast(fmaf(s[x][y], p.c, C::kPShift - mc));
          sum += s[x][y];
        }
      l[h] = l[h] * fix + sum;
#pragma unroll
      for (int x = 0; x < HD / 8; ++x) {
        acc[x][2 * h] *= fix;
        acc[x][2 * h + 1] *= fix;
      }
    }
    // ---- O += P V ----
    if constexpr (DT != kF32) {
#pragma unroll
      for (int kk = 0; kk < NTW / 16; ++kk) {
        const uint32_t a[4] = {pack<DT>(s[2 * kk][0], s[2 * kk][1]), pack<DT>(s[2 * kk][2], s[2 * kk][3]),
                               pack<DT>(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack<DT>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
        for (int x = 0; x < HD / 16; ++x) {
          uint32_t b[4];
          ldsm4t(b, sv + tile_at(NT, w0 + kk * 16 + (lane & 15), x * 2 + (lane >> 4)));
          mma16<DT>(acc[2 * x], a, b[0], b[1]);
          mma16<DT>(acc[2 * x + 1], a, b[2], b[3]);
        }
      }
    } else {
      // Column k of A is token 2k (k < 4) or 2 (k - 4) + 1, as the scores lie.
      uint32_t ah[NTW / 8][4], al[NTW / 8][4];
#pragma unroll
      for (int kk = 0; kk < NTW / 8; ++kk) {
        split_first(s[kk][0], ah[kk][0], al[kk][0]);
        split_first(s[kk][2], ah[kk][1], al[kk][1]);
        split_first(s[kk][1], ah[kk][2], al[kk][2]);
        split_first(s[kk][3], ah[kk][3], al[kk][3]);
      }
#pragma unroll
      for (int x = 0; x < HD / 8; ++x) {
        const int chunk = x * 2 + (g >> 2), off = 4 * (g & 3);
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NTW / 8; ++kk) {
          const int tk = w0 + kk * 8 + 2 * t4;
          mma8x3(d, ah[kk], al[kk], lds_f32(sv + tile_at(NT, tk, chunk) + off), lds_f32(sv + tile_at(NT, tk + 1, chunk) + off));
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] += d[y];
      }
    }

    if constexpr (TMA) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[done % S]);
    }

    // ---- end of the item, or of this CTA's part of it ----
    if (cur.ends(end)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(~0u, l[h], 1);
        l[h] += __shfl_xor_sync(~0u, l[h], 2);
      }
      if constexpr (WN > 1) {
        // Join the warps that took different tokens of the same rows.
        float* ml = merge + 2 * 16 * (HD + 4);  // [warp][16] (m, l)
        __syncthreads();
        if (t4 == 0)
#pragma unroll
          for (int h = 0; h < 2; ++h) *reinterpret_cast<float2*>(ml + (warp * 16 + g + 8 * h) * 2) = make_float2(m[h], l[h]);
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float2 w[WN];
          float top = -INFINITY;
#pragma unroll
          for (int x = 0; x < WN; ++x) {
            w[x] = *reinterpret_cast<const float2*>(ml + ((wm + x * C::WM) * 16 + g + 8 * h) * 2);
            top = fmaxf(top, w[x].x);
          }
          const float mc = top == -INFINITY ? 0.f : __fmul_rn(top, p.c);
          float sum = 0.f;
#pragma unroll
          for (int x = 0; x < WN; ++x) sum += w[x].y * exp2_fast(__fmul_rn(w[x].x, p.c) - mc);
          const float fix = exp2_fast(__fmul_rn(m[h], p.c) - mc);
          m[h] = top;
          l[h] = sum;
#pragma unroll
          for (int x = 0; x < HD / 8; ++x) {
            acc[x][2 * h] *= fix;
            acc[x][2 * h + 1] *= fix;
          }
        }
#pragma unroll
        for (int half = WN / 2; half >= 1; half >>= 1) {
          float* buf = merge + ((wn % half) * C::WM + wm) * 16 * (HD + 4);
          if (wn >= half && wn < 2 * half)
#pragma unroll
            for (int x = 0; x < HD / 8; ++x)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                *reinterpret_cast<float2*>(buf + (g + 8 * h) * (HD + 4) + x * 8 + 2 * t4) =
                    make_float2(acc[x][2 * h], acc[x][2 * h + 1]);
          __syncthreads();
          if (wn < half)
#pragma unroll
            for (int x = 0; x < HD / 8; ++x)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float2 o = *reinterpret_cast<const float2*>(buf + (g + 8 * h) * (HD + 4) + x * 8 + 2 * t4);
                acc[x][2 * h] += o.x;
                acc[x][2 * h + 1] += o.y;
              }
          __syncthreads();
        }
      }
      if (wn == 0) {
        const long long item_at = cur.pos - cur.tile;  // of its first tile
        const bool whole = item_at >= begin && cur.last_of_item();
        if (whole) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = wm * 16 + g + 8 * h;
            if (r >= it.nf) continue;
            const int f = it.f0 + r, i = (int)p.group_div.quot(f), j = f - i * p.a.group, head = cur.head * p.a.group + j;
            const float inv = l[h] > 0.f || l[h] != l[h] ? 1.f / l[h] : 0.f;
            const long long o = (long long)(it.start + i) * p.a.o_row + (long long)head * p.a.o_head;
#pragma unroll
            for (int x = 0; x < HD / 8; ++x) {
              const int col = x * 8 + 2 * t4;
              if (col >= ch.hd) continue;
              const float a0 = acc[x][2 * h] * inv, a1 = acc[x][2 * h + 1] * inv;
              if constexpr (DT == kF32)
                *reinterpret_cast<float2*>(static_cast<float*>(p.a.out) + o + col) = make_float2(a0, a1);
              else
                *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.a.out) + o + col) = pack<DT>(a0, a1);
            }
            if (p.a.lse && t4 == 0)
              p.a.lse[(long long)(it.start + i) * (ch.nkv * p.a.group) + head] =
                  l[h] > 0.f || l[h] != l[h] ? (m[h] * p.c - C::kPShift) * kLn2 + logf(l[h]) : -INFINITY;
          }
        } else {
          float* part = part_of(p, C::kPartFloats, blockIdx.x, first_slot);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = wm * 16 + g + 8 * h;
#pragma unroll
            for (int x = 0; x < HD / 8; ++x)
              *reinterpret_cast<float2*>(part + r * HD + x * 8 + 2 * t4) = make_float2(acc[x][2 * h], acc[x][2 * h + 1]);
            if (t4 == 0) {
              part[MT * HD + r] = m[h] == -INFINITY ? -INFINITY : m[h] * p.c;
              part[MT * HD + MT + r] = l[h];
            }
          }
        }
        if (poison) {
          // Rows that see a V value which is not finite get it after all.
          const int ta = it.first * NT + (int)max(0ll, begin - item_at) * NT, tb = (it.first + cur.tile + 1) * NT;
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            const int r = wm * 16 + g + 8 * h, f = it.f0 + r, i = (int)p.group_div.quot(f), at = h ? pos[1] : pos[0];
            if (r >= it.nf) continue;
            const int from = max(max(ta, it.lo), p.a.window > 0 ? at - p.a.window + 1 : 0), till = min(min(tb, it.hi), at + 1);
            const long long o = (long long)(it.start + i) * p.a.o_row + (long long)(cur.head * p.a.group + f - i * p.a.group) * p.a.o_head;
#pragma unroll 1
            for (int x = 0; x < HD / 4; ++x) {
              const int col = (x >> 1) * 8 + 2 * t4 + (x & 1);
              if (col >= ch.hd) continue;
              const float v = lost_values<DT, NT>(p, it, cur.head, col, from, till);
              if (v != 0.f) {
                if (whole) put<DT>(p.a.out, o + col, v);
                else part_of(p, C::kPartFloats, blockIdx.x, first_slot)[r * HD + col] = v;
              }
            }
          }
        }
      }
      first_slot = 1;
      fresh = true;
    }
    cur.next(p);
  }
  if constexpr (TMA) {
    // After a timeout: what was requested lands before the CTA ends.
    if (warp == 0 && !ok)
      for (uint32_t i = done; i < loaded; ++i) wait_bar(&full[i % S], i / S & 1, nullptr);
  } else {
    cp_async_wait<0>();
  }
}

template <typename C>
int resident_ctas() {
  // Per SM, from shared memory (228 KB with 1 KB kept for each CTA) and
  // registers: three CTAs of 128 threads have 168 each, which row tiles over
  // 16 pass.
  const int n = (228 * 1024) / (C::kSmem + 1024 + 512), most = C::MT == 16 ? 3 : 2;
  return n < 1 ? 1 : n > most ? most : n;
}

template <typename F>
auto with_cfg(int dtype, int hd, int rows, F f) {
#define RAI_MT(DT, HD)                            \
  (rows <= 16   ? f(Cfg<DT, HD, 16>{})            \
   : rows <= 32 ? f(Cfg<DT, HD, 32>{})            \
                : f(Cfg<DT, HD, 64>{}))
#define RAI_HD(DT) (hd <= 64 ? RAI_MT(DT, 64) : hd <= 128 ? RAI_MT(DT, 128) : RAI_MT(DT, 256))
  return dtype == kF32 ? RAI_HD(kF32) : dtype == kF16 ? RAI_HD(kF16) : RAI_HD(kBF16);
#undef RAI_HD
#undef RAI_MT
}

// Least tiles of a CTA's range: a cut costs a partial result (a few KB) and
// its share of the joining kernel.
constexpr int kMinTiles = 4;
constexpr int kItemCost = 1;  // tiles
// Caches of at most this many tiles a sequence are not cut.
constexpr int kWholeTiles = 8;
template <typename C>
bool whole_items(const AttnArgs& a) {
  return ((long long)a.c.max_pages * a.c.page.d + C::NT - 1) / C::NT <= kWholeTiles;
}

template <typename C, bool TMA>
cudaError_t launch_main(const Params& p, const KvMaps& maps, int box, cudaStream_t s) {
  static std::once_flag once[64];
  static cudaError_t ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&] {
    ready[dev] = cudaFuncSetAttribute(paged_attn_kernel<C, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (ready[dev] != cudaSuccess) return ready[dev];
  return launch_pdl(paged_attn_kernel<C, TMA>, dim3(p.grid), dim3(kThreads), C::kSmem, s, p, maps, box);
}

template <typename C>
cudaError_t launch(const AttnArgs& a, cudaStream_t s) {
  Params p;
  p.a = a;
  const long long frows = (long long)a.c.max_rows * a.group;
  p.row_tiles = (int)((frows + C::MT - 1) / C::MT);
  p.row_tiles_div = FastDiv(p.row_tiles);
  p.group_div = FastDiv(a.group);
  p.whole = whole_items<C>(a);
  p.min_tiles = p.whole ? 1 : kMinTiles;
  p.item_cost = kItemCost;
  p.grid = device_sm_count() * resident_ctas<C>();
  const long long items = (long long)a.c.n_seqs * p.row_tiles * a.c.nkv;
  p.direct = p.whole && items <= 2ll * p.grid;  // no need to share them out
  if (p.direct) p.grid = (int)items;
  p.c = a.softcap > 0.f ? kLog2e : a.scale * kLog2e;
  p.inv_cap = a.softcap > 0.f ? 1.f / a.softcap : 0.f;
  KvMaps maps;
  const int box = tma_box((int)a.c.page.d, C::NT);
  const bool tma = box && make_maps(a.c, a.dtype, box, &maps);
  cudaError_t e = tma ? launch_main<C, true>(p, maps, box, s) : launch_main<C, false>(p, maps, box, s);
  if (e != cudaSuccess || p.whole) return e;
  return launch_pdl(paged_combine_kernel<C>, dim3(p.grid - 1, combine_grid_y(C::MT)), dim3(kCombineThreads), 0, s, p);
}

}  // namespace

size_t paged_attention_workspace(const AttnArgs& a) {
  if (paged_attention_tc_takes(a)) return paged_attention_tc_workspace(a);
  const long long frows = (long long)a.c.max_rows * a.group;
  return with_cfg(a.dtype, a.c.hd, (int)(frows < 64 ? frows : 64), [&](auto c) -> size_t {
    using C = decltype(c);
    if (whole_items<C>(a)) return 0;  // nothing is cut
    const int grid = device_sm_count() * resident_ctas<C>();
    return cut_bytes(grid) + 2ull * grid * C::kPartFloats * 4;
  });
}

cudaError_t paged_attention(const AttnArgs& a, cudaStream_t s) {
  if (paged_attention_tc_takes(a)) return paged_attention_tc(a, s);
  const long long frows = (long long)a.c.max_rows * a.group;
  return with_cfg(a.dtype, a.c.hd, (int)(frows < 64 ? frows : 64), [&](auto c) { return launch<decltype(c)>(a, s); });
}

}  // namespace rai
