// Attention of one new token per sequence over a paged key-value cache: o = sum_j p_j v_j / sum_j p_j, p_j = exp(c q.k_j), for every
// query head, with the heads of a group as rows of one operand.
//
// What bounds it is HBM: every stored key and value is read once, 2 D bytes times the element's size, against 4 D operations per row.
// 64 sequences of up to 8000 tokens, 64 heads over 8 of 128 in bf16 (1018 MB): 161 us, 6.3 TB/s, 0.97 of the copy rate; one sequence of
// 131072 in f16 89 us (0.92); 128 of up to 4096 in e4m3 (560 MB) 102 us (0.84); 4 of up to 500 8.8 us, which are latencies: lengths (0.9 us),
// ranges (0.3), page numbers (1.1), the first keys (0.6), tiles, meeting (1) and joining (1).
// In 8 bits the 630 (e4m3) or 820 (int8) instructions of a tile of 32 keys come next to HBM: with pages out of L2 the same keys take 80 or 91 us.
//
// Work is cut into tiles of 16 to 64 keys of one item (a sequence, a key/value head, a row of up to 16 heads of its group); 4 KB of keys and
// 4 KB of values each.  The tiles of all items form one line that the warps of the grid share out in equal contiguous ranges, whatever the
// lengths are: every CTA finds the tiles before every sequence by a scan over the lengths, which only the device knows.  An item counts a
// tile more than it has, for its queries and results (64 x 500 keys in bf16 19.5 us without, 18.0 with).  Where the
// longest item has at most kWholeItems tiles (or there is no scratch for parts), ranges of CTAs end where items end, so that no CTA has to
// wait for another's part (figures at kWholeItems).  A warp leaves an item that it has as a whole with the output, otherwise with its part in
// shared memory (maxima, sums, unnormalised output); when the CTA's warps are done, each takes rows of parts to join, and items that several
// CTAs have are joined by the one that arrives last, in ascending order of the parts.  The ranges hang on the lengths alone, so that
// results are the same from run to run.
//
// A warp streams its range for itself: it asks for keys and values in turn, an entry of 4 KB of its ring in shared memory each, three
// entries ahead of the one that it reads (144 KB on the way per SM), by asynchronous copies of 16 bytes per lane.  Rows are exchanged in chunks
// as they are copied, so that no read meets a bank conflict.  Ways that were slower: keys and values straight into registers, 12 warps
// (the first of these 169 us, 8-bit caches 151 for 100); bulk and tensor copies by a lane of every warp (177, 154) or by a warp for all
// (181, 206): a copy costs its warp about 100 clocks, and pages of 16 tokens make many small ones; 8 or 10 warps with longer rings, 16 with
// shorter ones (8-bit caches 115, 112, 120).
//
// S^T = K Q^T and O^T += V^T P^T are m16n8k16 tensor-core instructions with the keys (the dimensions) as the 16 rows and up to eight heads as
// the columns: a tcgen05 tile of 128 rows would be 94 % padding, and the tensor work is an eighth of what this path delivers.
// A lane reads 16-byte chunks of a key and takes its dimensions in the order in which they come, queries accordingly.  Probabilities go from the
// accumulators' layout into the operand's by a transposition in registers, 16-bit values by transposing loads, 8-bit codes by byte
// permutes; codes become f16 as they are read (exact), their scales multiply scores and probabilities.  Probabilities enter as two 16-bit
// numbers, which leave 2^-16 of them at most: one f16 beside 8-bit codes (2^-11) took up to 7 % less time where a tile's instructions count.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <optional>
#include <type_traits>

#include "ctx.h"
#include "ptx.cuh"

using namespace ctb;
using namespace ctb_internal;

namespace {

enum Store { F16 = 0, BF16 = 1, E4M3 = 2, I8 = 3 };

constexpr int kMaxBatch = 1024;  // sequences of a launch (their lengths lie in shared memory)
constexpr unsigned kItemCost = 1;     // tiles that an item counts more than it has
// Tiles of the longest item up to which CTAs have whole items.  Items of 40, 78 and 100 tiles, whole and in parts, in us: 128 items (bf16) 12.7 and
// 16.6, 18.6 and 22.9, 22.2 and 26.7; 512 items 32.3 and 36.4, 56.1 and 59.8, 69.6 and 72.8; 64 items (e4m3) 14.5 and 16.0, 20.7 and 20.7,
// 24.0 and 22.5; one item 8.8 and 9.3, 11.7 and 9.7, 13.6 and 10.1.
constexpr unsigned kWholeItems = 80;
// Exponents' reference (in powers of two): it moves once a score stands kLazy above the largest that it knows.  What goes to f16 is lifted
// by kLift, so that the largest is at most 2^(kLazy + kLift + 1) and what f16 pairs cannot tell from 0 is 2^-(25 + kLift) of it.
constexpr int kLazy = 6, kLift = 8;

struct Params {
  const void *Q, *K, *V;
  const float *Ks, *Vs;
  void* Out;
  float* lse;
  const int32_t *table, *lengths;
  int64_t q_seq, q_head, k_page, v_page, ks_page, vs_page, table_ld;
  int batch, heads, kv_heads, group, row_tiles, width, page_log2, pages;
  int q_bf16;
  float scale_log2;
  unsigned whole_items;  // tiles of the longest item up to which CTAs have whole items: kWholeItems, or any number without scratch
  float* part;        // [CTA][first, last item of its range][rows x D, maxima, sums]
  unsigned* tickets;  // per CTA: parts left of the item that begins in its range and ends in another's
};

template <int STORE, int D_, int NT_>
struct Shape {
  static constexpr int D = D_, NT = NT_;
  static constexpr bool kBytes = STORE >= E4M3;
  static constexpr int kRow = D * (kBytes ? 1 : 2);  // bytes of a key's row
  static constexpr int KC = kRow / 64;               // 16-byte chunks that a lane has of a key's row
  static constexpr int KT = 256 / kRow;              // groups of 16 keys in a tile: K and V of a tile are 4 KB each
  static constexpr int VW = kRow / 32;               // 32-bit words that a lane has of a value's row
  static constexpr int MT = D / 16;                  // instructions along the dimensions of O
  static constexpr int QW = D / 8;                   // words that a lane has of a query row
  static constexpr int R = 8 * NT;
  static constexpr int kWarps = NT == 1 ? 12 : 8, kThreads = kWarps * 32;
  static constexpr int kEntry = 4096;                // bytes of keys or values of a tile
  static constexpr int kRing = NT == 1 ? 3 : 4;      // entries that a warp has or has asked for
  static constexpr int kPitch = D + 4;               // floats between rows of partial results in shared memory
  static constexpr int kSlotFloats = R * kPitch + 2 * R;
  static constexpr int kPartFloats = R * D + 2 * R;
  static constexpr int kScales = kBytes ? 16 * KT : 0;  // of an entry
  static constexpr size_t kSmem =
      128 + (size_t)kWarps * (kRing * (kEntry + kScales * 4) + kSlotFloats * 4) + 2 * kMaxBatch * 4;
};

template <int OFFSET>
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at), "n"(OFFSET));
  return v;
}
template <int OFFSET>
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4+%5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at), "n"(OFFSET)
               : "memory");
}
template <int OFFSET>
__device__ __forceinline__ uint2 lds8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2+%3];" : "=r"(v.x), "=r"(v.y) : "r"(at), "n"(OFFSET));
  return v;
}
template <int SRC, int DST>
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {  // all but the last N groups of every lane have landed
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  __syncwarp();
}
template <class F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F>
__device__ __forceinline__ void unrolled(F f) {  // f(std::integral_constant<int, i>()) for i = 0 .. N - 1
  each(f, std::make_integer_sequence<int, N>());
}
template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // of an 8 x 8 matrix of 16-bit elements
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// The four codes of w as f16 (both types are exact in it): lo has the first two, hi the others.
template <int STORE>
__device__ __forceinline__ void codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (STORE == E4M3) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {  // 0x6400 + u is the f16 1024 + u; u = code + 128
    w ^= 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}
__device__ __forceinline__ float max_over_keys(float v) {  // over the lanes that hold the same rows
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float sum_over_keys(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
__device__ __forceinline__ float from_minus_inf(float m) { return m == -INFINITY ? 0.f : m; }

// `n` tiles shared out among `workers`: the first ones have one more.
struct Shares {
  unsigned least, more;
  __device__ __forceinline__ Shares(unsigned n, unsigned workers) : least(n / workers), more(n - least * workers) {}
  __device__ __forceinline__ unsigned first(unsigned w) const { return w * least + min(w, more); }
  __device__ __forceinline__ unsigned owner(unsigned x) const {  // of tile x
    const unsigned large = more * (least + 1);
    return x < large ? x / (least + 1) : more + (x - large) / least;
  }
};

// Of the dimensions 8 i + g of a lane, those (bit i) of which some value of a sequence's keys first .. end - 1 is infinite, with one sign (bit
// 16 + i: minus) and no NaN beside it.  The four lanes of a dimension look at a key each.  A key that is not finite itself has a
// probability of 0 or NaN in every row: its infinite values are as good as NaN.  Not inlined: seldom called, and in the way otherwise.
template <bool BF, int D>
__device__ __noinline__ uint32_t infinite_values(const uint16_t* K, const uint16_t* V, int64_t k_page, int64_t v_page, const int32_t* pages,
                                                 int page_log2, int first, int end) {
  constexpr uint32_t kInf = BF ? 0x7f80 : 0x7c00;
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint32_t plus = 0, minus = 0, nan = 0;
  for (int key = first + c; key < end; key += 4) {
    const int64_t page = __ldg(pages + (key >> page_log2)) - 1, at = (key & ((1 << page_log2) - 1)) * D;
    const uint16_t *v = V + page * v_page + at, *k = K + page * k_page + at;
    uint32_t up = 0, down = 0;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const uint32_t x = __ldg(v + 8 * i + g);
      up |= (uint32_t)(x == kInf) << i;
      down |= (uint32_t)(x == (kInf | 0x8000)) << i;
      nan |= (uint32_t)((x & 0x7fff) > kInf) << i;
    }
    if (up | down) {
      bool finite = true;
      for (int i = 0; i < D; ++i) finite &= (__ldg(k + i) & 0x7fff) < kInf;
      if (!finite) nan |= up | down;
    }
    plus |= up;
    minus |= down;
  }
  __syncwarp();
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    plus |= __shfl_xor_sync(0xffffffffu, plus, x);
    minus |= __shfl_xor_sync(0xffffffffu, minus, x);
    nan |= __shfl_xor_sync(0xffffffffu, nan, x);
  }
  return ((plus ^ minus) & ~nan) | minus << 16;
}

// A tile: the sequence, the row of heads, and the keys.
struct Cursor {
  unsigned x;                 // its place on the line
  int b, head, rt, key, len;  // head: of the keys and values
};

template <int STORE, int D, int NT>
__global__ void __launch_bounds__(Shape<STORE, D, NT>::kThreads, 1)
    fmha_paged_kernel(const Params p, int* status) {
  using S = Shape<STORE, D, NT>;
  constexpr int KC = S::KC, KT = S::KT, VW = S::VW, MT = S::MT, QW = S::QW, R = S::R, kWarps = S::kWarps, kThreads = S::kThreads;
  constexpr int kTileKeys = 16 * KT, kRow = S::kRow, kRing = S::kRing;
  constexpr bool BF = STORE == BF16;
  constexpr float kAbove = STORE == F16 ? kLift : 0;  // what the known largest score stands above m
  constexpr float kNone = -3.4028235e38f;  // the reference of a row whose keys so far score -inf: whatever comes stands far above it
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  // [warp][entries], [warp][entries' scales], [warp][R rows, maxima, sums], lengths, tiles before
  float* all_scales = reinterpret_cast<float*>(smem + kWarps * kRing * S::kEntry);
  float* firsts = all_scales + kWarps * kRing * S::kScales;
  int* lens = reinterpret_cast<int*>(firsts + kWarps * S::kSlotFloats);
  unsigned* prefix = reinterpret_cast<unsigned*>(lens + kMaxBatch);
  __shared__ unsigned warp_sum[kWarps], warp_most[kWarps], ends[2];
  __shared__ uint4 segs[2 * kWarps];  // parts of items: first output row of the item (-1: no part), its live rows, its first tile, its last one's end
  __shared__ int last_s[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  // Results of a warp's part of an item: of the first item of its range beside the ring, of the last one in the ring, which is empty by then.
  auto slot_at = [&](int slot) {
    return slot & 1 ? reinterpret_cast<float*>(smem + (slot >> 1) * (kRing * S::kEntry)) : firsts + (slot >> 1) * S::kSlotFloats;
  };
  grid_dependency_sync();

  // ---- tiles before every sequence
  const int most = p.width << p.page_log2;
  const unsigned per_tile = (unsigned)p.kv_heads * p.row_tiles;
  unsigned longest, total = 0;
  {
    const int per = (p.batch + kThreads - 1) / kThreads, b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
    auto tiles = [&](int n) { return n ? (unsigned)(n + kTileKeys - 1) / kTileKeys + kItemCost : 0; };
    unsigned sum = 0, top = 0;
    for (int b = b0; b < b1; ++b) {
      const int n = min(max(__ldg(p.lengths + b), 0), most);
      lens[b] = n;
      sum += tiles(n) * per_tile;
      top = max(top, tiles(n));
    }
    unsigned up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += v;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 31) {
      warp_sum[warp] = up;
      warp_most[warp] = top;
    }
    if (tid < 2 * kWarps) segs[tid].x = ~0u;
    __syncthreads();
    unsigned before = up - sum;
    longest = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      total += warp_sum[w];
      before += w < warp ? warp_sum[w] : 0;
      longest = max(longest, warp_most[w]);
    }
    auto place = [&](auto&& at_sequence) {  // at_sequence(an item's tiles, the first one of all items, their end)
      for (int b = b0; b < b1; ++b) {
        const unsigned n = tiles(lens[b]), behind = before + n * per_tile;
        prefix[b] = before;
        at_sequence(n, before, behind);
        before = behind;
      }
    };
    if (longest <= p.whole_items) {
      // Whole items: a CTA's range ends where an item does that is next to the end of an equal range.  Whoever has that sequence says where.
      const Shares equal(total, gridDim.x);
      const unsigned at[2] = {equal.first(blockIdx.x), equal.first(blockIdx.x + 1)};
      if (tid < 2 && at[tid] >= total) ends[tid] = total;
      place([&](unsigned n, unsigned first, unsigned behind) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (first <= at[i] && at[i] < behind) ends[i] = first + (at[i] - first + n / 2) / n * n;
      });
    } else {
      place([](unsigned, unsigned, unsigned) {});
    }
    __syncthreads();
  }
  // sequences without keys
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (lens[b] > 0) continue;
    const bool wrong = __ldg(p.lengths + b) != 0;
    if (wrong && tid == 0) atomicMax(status, (int)DEV_BAD_INDEX);
    uint32_t* out = static_cast<uint32_t*>(p.Out) + (int64_t)b * p.heads * (D / 2);
    for (int i = tid; i < p.heads * (D / 2); i += kThreads) out[i] = wrong ? 0x7fff7fffu : 0u;
    if (p.lse)
      for (int i = tid; i < p.heads; i += kThreads) p.lse[(int64_t)b * p.heads + i] = wrong ? NAN : -INFINITY;
  }
  if (total == 0) return;
  // The sequence that has tile x: the last one that begins at or before it.  All lanes of a warp ask together.
  auto sequence_of = [&](unsigned x) {
    const int stride = (p.batch + 31) / 32;
    auto count = [&](int at, int end) { return __popc(__ballot_sync(0xffffffffu, at < end && prefix[at] <= x)); };
    const int start = (count(lane * stride, p.batch) - 1) * stride;
    return start + count(start + lane, min(start + stride, p.batch)) - 1;
  };
  // Ranges of the line of tiles: equal ones for all warps of the grid, or, where items are short, for the warps of a CTA, whose range
  // ends where an item ends.
  auto warp_shares = [&] { return Shares(total, min(gridDim.x * kWarps, total)); };
  unsigned lo, hi;
  if (longest <= p.whole_items) {
    const unsigned n = ends[1] - ends[0];
    lo = ends[0] + warp * n / kWarps;
    hi = ends[0] + (warp + 1) * n / kWarps;
  } else {
    const Shares shares = warp_shares();
    auto range_of = [&](unsigned w) { return min(shares.first(w), total); };
    if (tid < 2) ends[tid] = range_of((blockIdx.x + tid) * kWarps);
    lo = range_of(blockIdx.x * kWarps + warp);
    hi = range_of(blockIdx.x * kWarps + warp + 1);
  }

  auto write_lse = [&](int at, float m, float l) {
    if (p.lse) p.lse[at] = (m + log2f(l)) * 0.6931471805599453f;
  };
  auto pack = [&](float x, float y) { return p.q_bf16 ? pack2<true>(x, y) : pack2<false>(x, y); };
  auto next_item = [&](Cursor& t) {
    t.x += kItemCost;
    t.key = 0;
    if (++t.rt < p.row_tiles) return;
    t.rt = 0;
    if (++t.head < p.kv_heads) return;
    t.head = 0;
    do ++t.b;
    while (t.b < p.batch && (t.len = lens[t.b]) <= 0);
  };
  auto next = [&](Cursor& t) {
    ++t.x;
    t.key += kTileKeys;
    if (t.key >= t.len) next_item(t);
  };
  auto cursor_at = [&](unsigned x) {  // the first tile at x or behind it
    Cursor t;
    t.b = sequence_of(x);
    t.len = lens[t.b];
    const unsigned tiles = (unsigned)(t.len + kTileKeys - 1) / kTileKeys, n = tiles + kItemCost, at = x - prefix[t.b], item = at / n, tile = min(at - item * n, tiles);
    t.head = item / p.row_tiles;
    t.rt = item - t.head * p.row_tiles;
    t.key = (int)tile * kTileKeys;
    t.x = prefix[t.b] + item * n + tile;
    if (tile == tiles) next_item(t);
    return t;
  };
  if (lo < hi) {
    Cursor now = cursor_at(lo);  // the tile at hand
    // Tiles are asked for ahead of it: keys and values in turn, an entry of the warp's ring each.  A tile's groups of 16 keys are shared
    // out over the lanes; the number of a lane's page is read two tiles before that: (number, row in the page, -1 behind the last key).
    constexpr int kLanes = 32 / KT;  // of a group
    const int mine = lane / kLanes * 16;
    Cursor ahead = now;
    unsigned looked = 0, asked = 0, done = 0;  // tiles
    int id[3] = {}, row[3] = {};
    uint32_t bad_pages = 0;  // a bit per tile that has been asked for
    bool seen_bad = false;
    auto look_ahead = [&](int& to_id, int& to_row) {
      if (ahead.x >= hi) return;
      ++looked;
      const int key = ahead.key + mine;
      to_id = to_row = -1;
      if (key < ahead.len) {
        to_id = __ldg(p.table + ahead.b * p.table_ld + (key >> p.page_log2));
        to_row = (ahead.head << p.page_log2) + (key & ((1 << p.page_log2) - 1));
      }
      if (ahead.key == 0) {  // an item's queries are wanted at once when it is its turn
        const int r = lane / (D / 64);
        if (r < min(R, p.group - ahead.rt * R))
          asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const uint16_t*>(p.Q) + (int64_t)ahead.b * p.q_seq +
                                                          ((int64_t)ahead.head * p.group + ahead.rt * R + r) * p.q_head + lane % (D / 64) * 64));
      }
      next(ahead);
    };
#pragma unroll
    for (int i = 0; i < 3; ++i) look_ahead(id[i], row[i]);

    const uint32_t ring = smem_u32(smem) + warp * (kRing * S::kEntry);
    float* scales = all_scales + warp * (kRing * S::kScales);
    int put = 0, slot = 0;
    // Where a lane's 16 bytes go: rows in 128-byte lines whose chunks are exchanged by the line's number (in 64-byte rows by that of every
    // second one); the second halves of 256-byte rows in lines behind those of the first.
    const int l = lane % kLanes;
    const uint32_t to = kRow == 256   ? ((lane >> 3) & 1) * 2048 + (lane >> 4) * 128 + ((lane & 7) ^ (lane >> 4)) * 16
                        : kRow == 128 ? (lane >> 4) * 2048 + (l >> 3) * 128 + ((l & 7) ^ (l >> 3)) * 16
                                      : (lane >> 3) * 1024 + l * 16;
    auto ask = [&](auto values) {
      constexpr bool V = decltype(values)::value;
      if (asked < looked) {
        const bool good = (unsigned)(id[0] - 1) < (unsigned)p.pages;
        const int64_t page = good ? id[0] - 1 : 0;  // the first one where there is none
        if (KT == 1 || row[0] >= 0) {
          const uint32_t dst = ring + put * S::kEntry + to;
          const char* src = static_cast<const char*>(V ? p.V : p.K) + (page * (V ? p.v_page : p.k_page) + (int64_t)row[0] * D) * (S::kBytes ? 1 : 2) + l * 16;
          unrolled<8>([&](auto i_tag) {
            constexpr int i = decltype(i_tag)::value;
            copy16<i * 512 / KT, i * (kRow == 64 ? 128 : 256)>(dst ^ ((kRow == 64 ? 16 : 32) * (i & 3)), src);
          });
          if constexpr (S::kBytes) {
            const float* from = (V ? p.Vs + page * p.vs_page : p.Ks + page * p.ks_page) + row[0] + l;
            const uint32_t s_dst = smem_u32(scales + put * S::kScales + mine + l);
#pragma unroll
            for (int i = 0; i < 16; i += kLanes) copy4(s_dst + 4 * i, from + i);
          }
        }
        if constexpr (!V) {
          const bool wrong = __any_sync(0xffffffffu, row[0] >= 0 && !good);
          bad_pages = (bad_pages & ~(1u << (asked & 31))) | ((uint32_t)wrong << (asked & 31));
        } else {
          ++asked;
          id[0] = id[1];
          id[1] = id[2];
          row[0] = row[1];
          row[1] = row[2];
          look_ahead(id[2], row[2]);
        }
      }
      copies_commit();
      if (++put == kRing) put = 0;
    };
    constexpr std::false_type keys;
    constexpr std::true_type values;
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      if (i & 1) ask(values);
      else ask(keys);
    }
    auto leave_entry = [&](auto next_is) {
      __syncwarp();  // every lane has read it
      ask(next_is);
      if (++slot == kRing) slot = 0;
    };
    using AfterKeys = std::integral_constant<bool, (kRing & 1) != 0>;
    using AfterValues = std::integral_constant<bool, (kRing & 1) == 0>;
    // Dimensions of a lane in instruction j's output: with 16 bits 16 j + g and 16 j + g + 8, with 8 bits the pair at
    auto pair_of = [&](int j) { return g * (D / 8) + 2 * j; };
    // This lane's places in an entry.  Its chunks of a key are 2c and 2c + 1 of a line (c where a row is half a line): with the swizzle,
    // the eight lanes that a 16-byte load serves at a time (two keys) are in different banks.  16-bit values are read as matrices of
    // eight keys' chunks and transposed on the way, 8-bit ones as chunk g (half a chunk where a row is half a line) of four keys.
    const uint32_t k_at = kRow == 64 ? g * 64 + ((c ^ (g >> 1)) & 3) * 16 : g * 128 + ((2 * c) ^ g) * 16;
    const uint32_t v_at = !S::kBytes ? ((lane >> 4) * 8 + (lane & 7)) * 128 + (((lane >> 3) & 1) ^ (lane & 7)) * 16
                          : kRow == 64 ? c * 128 + ((g >> 1) ^ c) * 16 + (g & 1) * 8
                                       : c * 256 + (g ^ (2 * c)) * 16;

    while (now.x < hi) {
      // ---- an item or the part of it that is this warp's
      const int b = now.b, head = now.head, rt = now.rt, len = now.len;
      const unsigned item_lo = now.x - (unsigned)now.key / kTileKeys, item_hi = item_lo + (unsigned)(len + kTileKeys - 1) / kTileKeys;
      const int rows = p.group - rt * R;  // live rows, at least one
      bool bad = __ldg(p.lengths + b) > most;
      uint32_t q[NT][QW];
      float mult[NT][2];  // score in powers of two of the rows 2c, 2c + 1
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int row = n * 8 + g;
        const bool live = row < rows;
        const uint16_t* src = static_cast<const uint16_t*>(p.Q) + (int64_t)b * p.q_seq + ((int64_t)head * p.group + rt * R + (live ? row : 0)) * p.q_head;
        constexpr int kDims = S::kBytes ? 16 : 8;  // of a chunk
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
          for (int h = 0; h < kDims / 8; ++h) {
            const uint4 w = live ? __ldg(reinterpret_cast<const uint4*>(src + (kRow == 64 ? c : (i >> 1) * 8 + 2 * c + (i & 1)) * kDims + 8 * h)) : make_uint4(0, 0, 0, 0);
            const int at = (i * kDims / 8 + h) * 4;
            q[n][at] = w.x;
            q[n][at + 1] = w.y;
            q[n][at + 2] = w.z;
            q[n][at + 3] = w.w;
          }
        float factor = 1.f;
        if constexpr (S::kBytes) {
          // bf16 queries as f16 times a power of two that brings the row's largest element to 2^8: elements of at least 2^-25 of
          // that stay exact, smaller ones are off by 2^-33 of it at most
          if (p.q_bf16) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < QW; ++i) top = max(top, max(q[n][i] & 0x7fffu, (q[n][i] >> 16) & 0x7fffu));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = (int)(top >> 7);  // the exponent's field
            factor = e == 255 || top == 0 ? 1.f : __uint_as_float((uint32_t)min(254 - e + 8, 254) << 23);
#pragma unroll
            for (int i = 0; i < QW; ++i) {
              const float2 f = unpack2<true>(q[n][i]);
              q[n][i] = pack2<false>(f.x * factor, f.y * factor);
            }
          }
        }
        const float mine = p.scale_log2 / factor;
        mult[n][0] = __shfl_sync(0xffffffffu, mine, 8 * c);
        mult[n][1] = __shfl_sync(0xffffffffu, mine, 8 * c + 4);
      }
      float o[MT][NT][4], m[NT][2], ref[NT][2], l[NT][2], unit[NT][2], peak[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          m[n][r] = -INFINITY;
          ref[n][r] = kNone;
          l[n][r] = peak[n][r] = 0.f;
          unit[n][r] = S::kBytes ? 8.507059e37f : 1.f;  // 2^126
        }
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][n][e] = 0.f;
      auto tile = [&](auto tail_tag) {  // TAIL: some of its keys are behind the last one
        constexpr bool tail = decltype(tail_tag)::value;
        copies_wait<kRing - 1>();
        bad |= (bad_pages >> (done++ & 31)) & 1;
        float sc[KT][NT][4];
        [[maybe_unused]] float ks[KT][2];
        const uint32_t k_even = ring + slot * S::kEntry + k_at, k_odd = k_even ^ 16;
        if constexpr (S::kBytes) {
#pragma unroll
          for (int s = 0; s < KT; ++s) {
            ks[s][0] = scales[slot * S::kScales + 16 * s + g];
            ks[s][1] = scales[slot * S::kScales + 16 * s + g + 8];
          }
        }
        unrolled<KT>([&](auto tag) {
          constexpr int s = decltype(tag)::value;
          uint4 k[2][KC];
          unrolled<2 * KC>([&](auto hi_tag) {
            constexpr int h = decltype(hi_tag)::value / KC, i = decltype(hi_tag)::value % KC;
            constexpr int kAt = s * 16 * kRow + (i >> 1) * 2048 + h * 8 * (kRow == 64 ? 64 : 128);
            k[h][i] = lds16<kAt>(i & 1 ? k_odd : k_even);
          });
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[s][n][e] = 0.f;
#pragma unroll
          for (int i = 0; i < KC; ++i) {
            const uint32_t w0[4] = {k[0][i].x, k[0][i].y, k[0][i].z, k[0][i].w};
            const uint32_t w1[4] = {k[1][i].x, k[1][i].y, k[1][i].z, k[1][i].w};
            if constexpr (S::kBytes) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint32_t a0, a1, a2, a3;
                codes4<STORE>(w0[j], a0, a2);
                codes4<STORE>(w1[j], a1, a3);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma<false>(sc[s][n], a0, a1, a2, a3, q[n][8 * i + 2 * j], q[n][8 * i + 2 * j + 1]);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                  mma<BF>(sc[s][n], w0[2 * j], w1[2 * j], w0[2 * j + 1], w1[2 * j + 1], q[n][4 * i + 2 * j], q[n][4 * i + 2 * j + 1]);
            }
          }
        });
        leave_entry(AfterKeys());
        // ---- Scores in powers of two: e = 0, 1: key g, rows 2c, 2c + 1; e = 2, 3: key g + 8.  d is their distance from the reference.
        auto hidden = [&](int s, int e) { return tail && now.key + 16 * s + g + 8 * (e >> 1) >= len; };
        auto times = [&](int s, int n, int e) {
          if constexpr (S::kBytes) return mult[n][e & 1] * ks[s][e >> 1];
          else return mult[n][e & 1];
        };
        float d[KT][NT][4], top_d = -INFINITY;
#pragma unroll
        for (int s = 0; s < KT; ++s)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              d[s][n][e] = hidden(s, e) ? -INFINITY : fmaf(sc[s][n][e], times(s, n, e), -ref[n][e & 1]);
              top_d = fmaxf(top_d, d[s][n][e]);
            }
        const bool grown = __any_sync(0xffffffffu, top_d > kAbove + kLazy);
        if (grown) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float top = -INFINITY;
#pragma unroll
              for (int s = 0; s < KT; ++s)
#pragma unroll
                for (int e = r; e < 4; e += 2)
                  if (!hidden(s, e)) top = fmaxf(top, sc[s][n][e] * times(s, n, e));
              const float m_new = fmaxf(m[n][r], max_over_keys(top) - kAbove);
              ref[n][r] = m_new == -INFINITY ? kNone : m_new;
              const float alpha = ex2_approx_ftz(m[n][r] - ref[n][r]);
              m[n][r] = m_new;
              l[n][r] *= alpha;
              peak[n][r] *= alpha;
#pragma unroll
              for (int j = 0; j < MT; ++j) {
                o[j][n][r] *= alpha;
                o[j][n][r + 2] *= alpha;
              }
#pragma unroll
              for (int s = 0; s < KT; ++s)
#pragma unroll
                for (int e = r; e < 4; e += 2)
                  if (!hidden(s, e)) d[s][n][e] = fmaf(sc[s][n][e], times(s, n, e), -ref[n][r]);
            }
        }
        copies_wait<kRing - 1>();
#pragma unroll
        for (int s = 0; s < KT; ++s)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              d[s][n][e] = ex2_approx_ftz(d[s][n][e]);
              l[n][e & 1] += d[s][n][e];
            }
        if constexpr (S::kBytes) {
          // A probability times its value's scale goes to f16 in units of (about) the largest so far: scales differ from key to key by
          // any factor.  While all were 0 (rows of zeros have scales of 0) the unit is 2^126, the largest there is, with which the first
          // beyond 2^-111 is too large.
          float vs[KT][2];
#pragma unroll
          for (int s = 0; s < KT; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float v = scales[slot * S::kScales + 16 * s + g + 8 * h];
              vs[s][h] = hidden(s, 2 * h) ? 0.f : v;
            }
          float top_w = 0.f;
#pragma unroll
          for (int s = 0; s < KT; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                sc[s][n][e] = d[s][n][e] * vs[s][e >> 1] * unit[n][e & 1];  // not d (vs unit), which is 0 inf for a large scale behind tiny ones
                top_w = fmaxf(top_w, fabsf(sc[s][n][e]));
              }
          if (grown || __any_sync(0xffffffffu, top_w > (float)(2 << (kLift + kLazy)))) {
#pragma unroll
            for (int s = 0; s < KT; ++s) asm volatile("" : "+f"(vs[s][0]), "+f"(vs[s][1]));  // products again, below: kept, they cost registers in every tile
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                float top = peak[n][r];
#pragma unroll
                for (int s = 0; s < KT; ++s)
#pragma unroll
                  for (int e = r; e < 4; e += 2) top = fmaxf(top, fabsf(d[s][n][e] * vs[s][e >> 1]));
                top = max_over_keys(top);
                peak[n][r] = top;
                const int e = (int)(__float_as_uint(top) >> 23);
                const float u = e < 255 ? __uint_as_float((uint32_t)min(max(254 + kLift - e, 1), 253) << 23) : unit[n][r];
                const float f = u / unit[n][r];
                unit[n][r] = u;
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                  o[j][n][r] *= f;
                  o[j][n][r + 2] *= f;
                }
#pragma unroll
                for (int s = 0; s < KT; ++s)
#pragma unroll
                  for (int e2 = r; e2 < 4; e2 += 2) sc[s][n][e2] = d[s][n][e2] * vs[s][e2 >> 1] * u;
              }
          }
        }
        // ---- O += V P
        const uint32_t v_even = ring + slot * S::kEntry + v_at;
        [[maybe_unused]] const uint32_t v_odd = v_even ^ 16;
        unrolled<KT>([&](auto tag) {
          constexpr int s = decltype(tag)::value;
          uint32_t hi_[NT][2];
          uint32_t lo_[NT][2];  // what is left of a probability: one 16-bit number each would show in results whose terms cancel
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float a = S::kBytes ? sc[s][n][2 * h] : d[s][n][2 * h], z = S::kBytes ? sc[s][n][2 * h + 1] : d[s][n][2 * h + 1];
              const uint32_t w = pack2<BF>(a, z);
              hi_[n][h] = transposed(w);
              const float2 f = unpack2<BF>(w);
              lo_[n][h] = transposed(pack2<BF>(a - f.x, z - f.y));
            }
          // rows behind the last key may hold anything: 0 x NaN is NaN
          const int left = len - now.key - 16 * s;
          if constexpr (S::kBytes) {
            uint32_t v[4][VW];
            unrolled<4>([&](auto h_tag) {
              constexpr int h = decltype(h_tag)::value;
              constexpr int kLine = kRow == 64 ? 64 : 128, kAt = s * 16 * kRow + (8 * (h >> 1) + (h & 1)) * kLine;
              if constexpr (kRow == 64) {
                const uint2 w = lds8<kAt>(v_even);
                v[h][0] = w.x;
                v[h][1] = w.y;
              } else {
                const uint4 w = lds16<kAt>(h & 1 ? v_odd : v_even);
                v[h][0] = w.x;
                v[h][1] = w.y;
                v[h][2] = w.z;
                v[h][3] = w.w;
              }
              if (tail && 2 * c + (h & 1) + 8 * (h >> 1) >= left) {
#pragma unroll
                for (int i = 0; i < VW; ++i) v[h][i] = 0;
              }
            });
#pragma unroll
            for (int i = 0; i < VW; ++i) {  // four dimensions
              uint32_t a[2][4];
              codes4<STORE>(__byte_perm(v[0][i], v[1][i], 0x5140), a[0][0], a[0][1]);
              codes4<STORE>(__byte_perm(v[2][i], v[3][i], 0x5140), a[0][2], a[0][3]);
              codes4<STORE>(__byte_perm(v[0][i], v[1][i], 0x7362), a[1][0], a[1][1]);
              codes4<STORE>(__byte_perm(v[2][i], v[3][i], 0x7362), a[1][2], a[1][3]);
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma<false>(o[2 * i + h][n], a[h][0], a[h][1], a[h][2], a[h][3], hi_[n][0], hi_[n][1]);
                  mma<false>(o[2 * i + h][n], a[h][0], a[h][1], a[h][2], a[h][3], lo_[n][0], lo_[n][1]);
                }
            }
          } else {
            const uint32_t mask0 = (2 * c < left ? 0xffffu : 0u) | (2 * c + 1 < left ? 0xffff0000u : 0u);
            const uint32_t mask1 = (2 * c + 8 < left ? 0xffffu : 0u) | (2 * c + 9 < left ? 0xffff0000u : 0u);
            unrolled<MT>([&](auto j_tag) {
              constexpr int j = decltype(j_tag)::value;
              uint32_t a[4];
              ldmatrix4_trans<s * 16 * kRow + (j >> 2) * 2048>(a, v_even ^ (32 * (j & 3)));
              if (tail) {
                a[0] &= mask0;
                a[1] &= mask0;
                a[2] &= mask1;
                a[3] &= mask1;
              }
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma<BF>(o[j][n], a[0], a[1], a[2], a[3], hi_[n][0], hi_[n][1]);
                mma<BF>(o[j][n], a[0], a[1], a[2], a[3], lo_[n][0], lo_[n][1]);
              }
            });
          }
        });
        leave_entry(AfterValues());
      };
      const unsigned end = min(hi, item_hi);
      [[maybe_unused]] const int first_key = now.key;
      for (; now.x < end; ++now.x, now.key += kTileKeys) {
        if (now.key + kTileKeys <= len) tile(std::false_type());
        else tile(std::true_type());
      }
      if constexpr (!S::kBytes) {
        // An infinite value: its product with the low half of a probability, zero or negative, is a NaN beside the one with the high
        // half.  (8-bit rows with an infinity have a scale that is one, and codes of 0.)
        bool odd = false;
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= o[j][n][e] != o[j][n][e];
        if (__any_sync(0xffffffffu, odd) && !bad) {
          const int64_t at = ((int64_t)head << p.page_log2) * D;
          const uint32_t found = infinite_values<BF, D>(static_cast<const uint16_t*>(p.K) + at, static_cast<const uint16_t*>(p.V) + at, p.k_page, p.v_page,
                                                        p.table + b * p.table_ld, p.page_log2, first_key, min(now.key, len));
#pragma unroll
          for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t here = found >> (2 * j + (e >> 1));
                if (o[j][n][e] != o[j][n][e] && (here & 1)) o[j][n][e] = here & 0x10000 ? -INFINITY : INFINITY;
              }
        }
      }
      if (now.x == item_hi) next_item(now);
      // ---- leaving the item
      seen_bad |= bad;
      const bool whole = item_lo >= lo && item_hi <= hi;
      const int part_slot = warp * 2 + (item_lo <= lo ? 0 : 1);
      float* mine = slot_at(part_slot);
      const int out_row = b * p.heads + head * p.group + rt * R;
      float f[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float sum = bad ? NAN : sum_over_keys(l[n][r]);
          const int row = n * 8 + 2 * c + r;
          f[n][r] = (whole ? 1.f / sum : 1.f) / unit[n][r];
          if (g == 0) {
            if (whole) {
              if (row < rows) write_lse(out_row + row, m[n][r], sum);
            } else {
              mine[R * S::kPitch + row] = m[n][r];
              mine[R * S::kPitch + R + row] = sum;
            }
          }
        }
      if (whole) {  // outputs in pairs of dimensions of a row: those of 16-bit values by a transposition
        uint16_t* out = static_cast<uint16_t*>(p.Out) + (int64_t)out_row * D;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if constexpr (S::kBytes) {
                const int row = n * 8 + 2 * c + h;
                const uint32_t w = pack(o[j][n][h] * f[n][h], o[j][n][h + 2] * f[n][h]);
                if (row < rows) *reinterpret_cast<uint32_t*>(out + row * D + pair_of(j)) = w;
              } else {
                const int row = n * 8 + g;
                const uint32_t w = transposed(pack(o[j][n][2 * h] * f[n][0], o[j][n][2 * h + 1] * f[n][1]));
                if (row < rows) *reinterpret_cast<uint32_t*>(out + row * D + 16 * j + 8 * h + 2 * c) = w;
              }
            }
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int dim = S::kBytes ? pair_of(j) + (e >> 1) : 16 * j + g + 8 * (e >> 1);
              mine[(n * 8 + 2 * c + (e & 1)) * S::kPitch + dim] = o[j][n][e] * f[n][e & 1];
            }
        if (lane == 0) segs[part_slot] = make_uint4(out_row, min(rows, R), item_lo, item_hi);
      }
    }
    if (seen_bad && lane == 0) atomicMax(status, (int)DEV_BAD_INDEX);
  }
  __syncthreads();

  // ---- Items that several warps had.  A lane looks at a slot; neighbouring parts of one item are joined.
  constexpr int kEach = D / 32;  // dimensions of a lane
  static_assert(2 * kWarps <= 32, "a lane per slot");
  // One row of the parts in the slots of `members`, in ascending order: to the output, or to a part of the item in memory.
  auto join_row = [&](uint32_t members, int out_row, int row, float* part) {
    const bool member = (members >> lane) & 1;
    const float* stats = slot_at(member ? lane : 0) + R * S::kPitch + row;
    const float m = member ? stats[0] : -INFINITY;
    float M = m, L = member ? stats[R] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float f = ex2_approx_ftz(m - from_minus_inf(M));
    L *= f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    float acc[kEach] = {};
#pragma unroll 4
    for (uint32_t left = members; left; left &= left - 1) {
      const int s = __ffs(left) - 1;
      const float fs = __shfl_sync(0xffffffffu, f, s);
      const float* from = slot_at(s) + row * S::kPitch + lane * kEach;
      if constexpr (kEach == 4) {
        const float4 u = *reinterpret_cast<const float4*>(from);
        acc[0] += u.x * fs; acc[1] += u.y * fs; acc[2] += u.z * fs; acc[3] += u.w * fs;
      } else {
        const float2 u = *reinterpret_cast<const float2*>(from);
        acc[0] += u.x * fs; acc[1] += u.y * fs;
      }
    }
    if (part) {
#pragma unroll
      for (int i = 0; i < kEach; i += 2) *reinterpret_cast<float2*>(part + row * D + lane * kEach + i) = make_float2(acc[i], acc[i + 1]);
      if (lane == 0) {
        part[R * D + row] = M;
        part[R * D + R + row] = L;
      }
    } else {
      const float inv = 1.f / L;
      uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.Out) + (int64_t)(out_row + row) * D + lane * kEach);
      if constexpr (kEach == 4) *reinterpret_cast<uint2*>(out) = make_uint2(pack(acc[0] * inv, acc[1] * inv), pack(acc[2] * inv, acc[3] * inv));
      else *out = pack(acc[0] * inv, acc[1] * inv);
      if (lane == 0) write_lse(out_row + row, M, L);
    }
  };
  const unsigned cta_lo = ends[0], cta_hi = ends[1];
  const uint4 seg = lane < 2 * kWarps ? segs[lane] : make_uint4(~0u, 0, 0, 0);
  const uint32_t marked = __ballot_sync(0xffffffffu, seg.x != ~0u), below = marked & ((1u << lane) - 1);
  const uint32_t item_below = __shfl_sync(0xffffffffu, seg.x, below ? 31 - __clz(below) : 0);
  uint32_t leaders = __ballot_sync(0xffffffffu, seg.x != ~0u && (!below || item_below != seg.x));
  uint4 shared_first = make_uint4(~0u, 0, 0, 0), shared_last = shared_first;  // that other CTAs have a part of: the first and the last of the range
  for (int task = 0; leaders; leaders &= leaders - 1) {
    const int s = __ffs(leaders) - 1;
    const uint32_t later = leaders & (leaders - 1), members = marked & ~((1u << s) - 1) & (later ? (later & -later) - 1 : ~0u);
    const uint4 item = make_uint4(__shfl_sync(0xffffffffu, seg.x, s), __shfl_sync(0xffffffffu, seg.y, s), __shfl_sync(0xffffffffu, seg.z, s),
                                  __shfl_sync(0xffffffffu, seg.w, s));
    const bool inside = item.z >= cta_lo && item.w <= cta_hi;
    const int which = item.z < cta_lo ? 0 : 1;
    if (!inside && which == 0) shared_first = item;
    if (!inside && which == 1) shared_last = item;
    float* part = inside ? nullptr : p.part + ((int64_t)blockIdx.x * 2 + which) * S::kPartFloats;
    for (int row = (warp + kWarps - task % kWarps) % kWarps; row < (int)item.y; row += kWarps) join_row(members, item.x, row, part);
    task += item.y;
  }
  if (shared_first.x == ~0u && shared_last.x == ~0u) return;
  // ---- Items that several CTAs had: the one that is done last adds the parts.
  const Shares shares = warp_shares();
  auto cta_of = [&](unsigned x) { return (int)(shares.owner(x) / kWarps); };
  __syncthreads();
  if (tid < 2) {
    last_s[tid] = 0;
    const uint4 item = tid ? shared_last : shared_first;
    if (item.x != ~0u) {
      const int c0 = cta_of(item.z), parts = cta_of(item.w - 1) - c0;
      unsigned before;  // back to zero by the last; what the CTA has written (it met above) comes before, what it reads below behind
      asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;" : "=r"(before) : "l"(p.tickets + c0), "r"(parts) : "memory");
      last_s[tid] = before == (unsigned)parts;
    }
  }
  __syncthreads();
  const bool last[2] = {last_s[0] != 0, last_s[1] != 0};
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (!last[which]) continue;
    const uint4 item = which ? shared_last : shared_first;
    // warp w takes the parts c0 + w, c0 + w + kWarps, ...: vector i of a lane is number i * 32 + lane of the part's rows
    const int c0 = cta_of(item.z), c1 = cta_of(item.w - 1), rows = item.y;
    constexpr int kVecs = R * D / 4 / 32;
    const int row = lane & (R - 1);
    float M = -INFINITY, L = 0.f;
    float4 acc[kVecs];
#pragma unroll
    for (int e = 0; e < kVecs; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = c0 + warp; i <= c1; i += kWarps) {
      const float* from = p.part + ((int64_t)i * 2 + (i == c0 ? 1 : 0)) * S::kPartFloats;
      float4 u[kVecs];
#pragma unroll
      for (int e = 0; e < kVecs; ++e)  // rows behind the group's last are not written
        if ((e * 32 + lane) / (D / 4) < rows) u[e] = __ldcg(reinterpret_cast<const float4*>(from) + e * 32 + lane);
        else u[e] = make_float4(0.f, 0.f, 0.f, 0.f);
      const float m = row < rows ? __ldcg(from + R * D + row) : -INFINITY, l = row < rows ? __ldcg(from + R * D + R + row) : 0.f;
      const float top = fmaxf(M, m), ref = from_minus_inf(top), old = ex2_approx_ftz(M - ref), f = ex2_approx_ftz(m - ref);
      M = top;
      L = L * old + l * f;
#pragma unroll
      for (int e = 0; e < kVecs; ++e) {
        const int r = (e * 32 + lane) / (D / 4);
        const float fr = __shfl_sync(0xffffffffu, f, r), of = __shfl_sync(0xffffffffu, old, r);
        acc[e].x = acc[e].x * of + u[e].x * fr;
        acc[e].y = acc[e].y * of + u[e].y * fr;
        acc[e].z = acc[e].z * of + u[e].z * fr;
        acc[e].w = acc[e].w * of + u[e].w * fr;
      }
    }
    __syncthreads();  // the slots are free
    float* to = slot_at(2 * warp);
#pragma unroll
    for (int e = 0; e < kVecs; ++e) {
      const int at = e * 32 + lane, r = at / (D / 4);
      *reinterpret_cast<float4*>(to + r * S::kPitch + (at - r * (D / 4)) * 4) = acc[e];
    }
    if (lane < R) {
      to[R * S::kPitch + lane] = M;
      to[R * S::kPitch + R + lane] = L;
    }
    __syncthreads();
    const uint32_t used = 0x55555555u & ((1ull << 2 * min(kWarps, c1 - c0 + 1)) - 1);
    for (int r = warp; r < rows; r += kWarps) join_row(used, item.x, r, nullptr);
  }
}

template <int STORE, int D, int NT>
int launch(ctb_ctx* ctx, cudaStream_t st, Params p, int64_t batch) {
  using S = Shape<STORE, D, NT>;
  static_assert(S::kSmem <= 227 * 1024, "shared memory of a CTA");
  p.row_tiles = (p.group + S::R - 1) / S::R;
  // of a sequence, at most; one where the page table is empty
  const int64_t most = (((int64_t)p.width << p.page_log2) + 16 * S::KT - 1) / (16 * S::KT) + kItemCost;  // of an item
  const int64_t tiles = std::max<int64_t>(1, most * p.kv_heads * p.row_tiles);
  if (tiles > INT32_MAX) return fail(CTB_UNSUPPORTED, "ctb_fmha_paged: a sequence has too many keys");
  const int64_t chunk = std::min<int64_t>(kMaxBatch, INT32_MAX / tiles);
  auto kern = fmha_paged_kernel<STORE, D, NT>;
  cudaError_t e = allow_smem(kern, S::kSmem);
  if (e != cudaSuccess) return cuda_fail(e, "ctb_fmha_paged: shared memory opt-in");
  std::optional<StreamScratch> scratch;  // until the kernel is launched
  p.whole_items = UINT32_MAX;            // no scratch, or more SMs than it has room for
  if (most <= kWholeItems) {
    p.whole_items = kWholeItems;  // none is used
  } else if ((size_t)ctx->sm_count * 2 * S::kPartFloats * sizeof(float) <= kSlotBytes && ctx->sm_count <= kTickets) {
    scratch.emplace(ctx, st);
    if (scratch->data) {
      p.part = scratch->data;
      p.tickets = scratch->tickets;
      p.whole_items = kWholeItems;
    }
  }
  for (int64_t b = 0; b < batch; b += chunk) {
    Params q = p;
    q.batch = (int)std::min(chunk, batch - b);
    q.Q = static_cast<const uint16_t*>(p.Q) + b * p.q_seq;
    q.Out = static_cast<uint16_t*>(p.Out) + b * p.heads * D;
    q.lse = p.lse ? p.lse + b * p.heads : nullptr;
    q.table = p.table + b * p.table_ld;
    q.lengths = p.lengths + b;
    launch_kernel(kern, (unsigned)ctx->sm_count, S::kThreads, S::kSmem, st, 0, q, ctx->dev_status);
    CTB_CHECK_LAUNCH("ctb_fmha_paged launch");
  }
  return CTB_OK;
}

template <int STORE>
int pick(ctb_ctx* ctx, cudaStream_t st, const Params& p, int64_t batch, int64_t D) {
  const bool small = p.group <= 8;
  if (D == 64) return small ? launch<STORE, 64, 1>(ctx, st, p, batch) : launch<STORE, 64, 2>(ctx, st, p, batch);
  return small ? launch<STORE, 128, 1>(ctx, st, p, batch) : launch<STORE, 128, 2>(ctx, st, p, batch);
}

}  // namespace

extern "C" int ctb_fmha_paged(ctb_ctx* ctx, void* stream, void* Out, float* lse, const void* Q, const ctb_kv_cache* cache,
                              const int32_t* page_table, const int32_t* lengths, int64_t batch, int64_t heads, int64_t q_seq_stride,
                              int64_t q_head_stride, int64_t table_width, int64_t table_stride, float qk_scale, int dtype) {
  CTB_CHECK_CTX(ctx);
  CurrentDevice on(ctx);
  int r = check_kv_cache("ctb_fmha_paged", cache);
  if (r) return r;
  if (batch < 0 || heads <= 0 || table_width < 0) return fail(CTB_BAD_ARG, "ctb_fmha_paged: non-positive dimension");
  if (heads % cache->kv_heads)
    return fail(CTB_BAD_ARG, "ctb_fmha_paged: heads (%lld) is not a multiple of kv_heads (%lld)", (long long)heads, (long long)cache->kv_heads);
  if (dtype != CTB_F16 && dtype != CTB_BF16) return fail(CTB_UNSUPPORTED, "ctb_fmha_paged: queries are f16 or bf16");
  if (cache->dtype != dtype && cache->dtype != CTB_E4M3 && cache->dtype != CTB_I8)
    return fail(CTB_BAD_ARG, "ctb_fmha_paged: a cache of 16-bit elements has the type of the queries");
  const float scale_log2 = qk_scale * 1.4426950408889634f;
  if (!isfinite(scale_log2)) return fail(CTB_BAD_ARG, "ctb_fmha_paged: qk_scale is not finite (in powers of two)");
  const int64_t D = cache->head_dim, page = cache->page_size;
  if (heads > 65536 || table_width > (1 << 28) / page)
    return fail(CTB_UNSUPPORTED, "ctb_fmha_paged: shape too large");
  if (batch == 0) return CTB_OK;
  CTB_CHECK_DEV(Q); CTB_CHECK_DEV(Out); CTB_CHECK_DEV(lengths);
  if (lse) CTB_CHECK_DEV(lse);
  if (table_width) CTB_CHECK_DEV(page_table);
  if (table_stride < table_width && batch > 1) return fail(CTB_BAD_ARG, "ctb_fmha_paged: rows of the page table overlap");
  if (batch == 1) q_seq_stride = 0;  // none along what has one element
  if (heads == 1) q_head_stride = 0;
  if ((uintptr_t)Q % 16 || (uintptr_t)Out % 16 || q_seq_stride % 8 || q_head_stride % 8)
    return fail(CTB_BAD_ALIGN, "ctb_fmha_paged: Q and Out must be 16-byte aligned and the strides of Q multiples of 8 elements");
  Params p = {};
  p.Q = Q; p.Out = Out; p.lse = lse;
  p.K = cache->k; p.V = cache->v; p.Ks = cache->k_scale; p.Vs = cache->v_scale;
  p.table = page_table; p.lengths = lengths;
  p.q_seq = q_seq_stride; p.q_head = q_head_stride; p.table_ld = table_stride;
  p.k_page = cache->k_page_stride; p.v_page = cache->v_page_stride;
  p.ks_page = cache->k_scale_page_stride; p.vs_page = cache->v_scale_page_stride;
  p.heads = (int)heads; p.kv_heads = (int)cache->kv_heads; p.group = (int)(heads / cache->kv_heads);
  p.width = (int)table_width; p.pages = (int)cache->pages;
  while ((1ll << p.page_log2) < page) ++p.page_log2;
  p.q_bf16 = dtype == CTB_BF16;
  p.scale_log2 = scale_log2;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case CTB_F16: return pick<F16>(ctx, st, p, batch, D);
    case CTB_BF16: return pick<BF16>(ctx, st, p, batch, D);
    case CTB_E4M3: return pick<E4M3>(ctx, st, p, batch, D);
    default: return pick<I8>(ctx, st, p, batch, D);
  }
}
