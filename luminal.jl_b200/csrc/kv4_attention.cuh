// Attention over the 4-bit paged cache: the kernel and its parameters.  kv4_attention.cu picks and launches; kv4_attention_{bf16,f32}.cu hold the instantiations.
//
// Mathematics.  With k = m + n s per key and group of 32 features, and v likewise, for one query row
//   score_k = sum_g ( s_kg (q . n_k)_g + m_kg sum_g q )          out_d = sum_k (p_k s_kg) n_kd + sum_k p_k m_kg,  p = softmax(scale score)
// so the 4-bit numbers n go to the tensor core as they are, and scales meet 16 keys x 8 rows of scores and weights instead of 16 x 32 values.  A number n in the low bits
// of a half IS the half n 2^-24 (a subnormal), and four bits higher 16 n 2^-24: one AND per two values makes MMA operands, and the powers of two go into q (keys) and into the
// result (values).  Sums of such products keep about 17 bits (the tensor core aligns them by their exponent fields), enough under bf16 results; for float32 n is made a normal half
// (1024 + n, less 1024), q and the weights are two halves each, and every pair of products starts at zero and is added in float32, because the tensor core's own sums
// are cut off, not rounded: 3.4e-5 of the result as subnormals in one sum.  Both products are mma.sync m16n8k16 with keys or features as the 16 rows and up to 8 query rows of one kv head as columns, because a decoding
// step has 1 to 8 of them: on tcgen05 M would be padded to 128, and the 4-bit operand would have to be widened through shared memory instead of in registers.
//
// Work.  Units of 128 keys of all (sequence, row tile, kv head) triples in a row are cut into equal shares whatever the sequences' lengths, so a long sequence among short ones
// is shared by many CTAs.  Little work is cut into pieces of triples instead, one per CTA, if none becomes much longer than a share: a second triple costs a CTA about 7 us.  Each of a CTA's four warps takes 32 keys of a unit through a ring of bulk copies of its own, which is filled with the next triple's keys while the present
// one's sums are joined.  Where a triple is cut, its shares leave partial sums and the last one to finish joins them (many: in groups first).
//
// What bounds it, in bf16 with 8 kv heads of 128 and 4 query heads each.  32 sequences of 8184 keys: 75 to 77 us with other inputs every call, 4.4 TB/s, 0.67 of the copy rate (70.6 over and over on the
// same ones, of which L2 keeps a part); about 300 warp instructions per 16 keys and head, issued at 57 % by 3.3 warps a scheduler that wait for their own arithmetic.  One sequence: 9.6 us for 300 keys,
// 16 for 8192, 44 for 131072; about 8 of them are the chain of lengths, table, queries, first copy and join.  float32 has three products for one: 32 sequences of 4096 keys 74 us against 42.  Values
// whose products with the weights leave the halves (scales above 2^8 or so, or below 2^-14) are gone through twice: 32 x 8184 153 us recorded against 70.6, float32 32 x 4096 147 against 74.
#pragma once
#include <math_constants.h>

#include <type_traits>

#include "kv4.cuh"
#include "kv4_shares.cuh"
#include "pdl.cuh"
#include "tc.cuh"

namespace lmb {
namespace kv4 {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kUnit = 128, kMaxSeqs = 8192;
// Units by which the longest piece may be longer than a share for the work to be cut into pieces.  As shares and as pieces, us: 64 sequences of 300 keys 22.6 and 13.7, 32 of 1000 24.3 and
// 18.8 (3 units longer), 20 of 4000 31.1 and 30.4 (4 longer), 16 of 8192 38.7 and 41.2, 32 of 8184 70.6 and 73.0 (5 longer).
constexpr unsigned kLonger = 4;

struct Params {
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  int rows, n_seq, max_pages, n_pages, shift, heads, G, window;
  float scale;                               // of the scores, times log2(e)
  const int *cu_rows, *lens, *table;
  const uint8_t* pages;
  int *dev_err, *dev_arg;
  unsigned* counters;                        // [kCounters], zero between calls
  float2* part_ml;                           // [share][2][columns]: maximum (log2) and sum
  float* part_o;                             // [share][2][columns][D]
};

// shared memory that grows with the sequences
__host__ __device__ constexpr int seq_bytes(int n_seq) { return (2 * n_seq + 1) * 4; }

// One variant: widths of NG groups, NT tiles of 8 query rows.
struct Variant {
  void (*kernel)(Params) = nullptr;
  int smem = 0, ctas_per_sm = 0;
};
const Variant* variant_bf16(int NG, int NT);
const Variant* variant_f32(int NG, int NT);
int32_t configure_bf16();
int32_t configure_f32();
constexpr int kMostTiles = 2;

template <typename T, int NG, int NT> struct Shape {
  static constexpr bool kSplit = sizeof(T) == 4;          // float32: operands as two halves, 22 bits
  static constexpr int D = 32 * NG, COLS = 8 * NT;
  static constexpr int kStageBytes = 2 * 640 * NG;
  static constexpr int kStages = NG == 1 ? 8 : NG == 2 ? 4 : NG == 3 ? 3 : 2;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kPitch = D + 4;                    // of the joined sums: 2 kPitch = 8 banks
  static constexpr int kMerge = 2 * COLS * kPitch * 4;
  static_assert(kMerge >= kMostShares / kJoin * COLS * 4, "join_parts keeps a weight per part and row there");
  static constexpr int kQ = 2 * NG * NT * 32 * (kSplit ? 16 : 8);
  static constexpr int kQSum = NT * 32 * 8;
  static constexpr int kFixed = kRing + kMerge + kQ + kQSum + COLS * 16 + 2 * kWarps * COLS * 4 + kWarps * kStages * 8 + 64 + 3 * 96 + kWarps * 16;
};

__device__ __forceinline__ void mma_half(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c = a b
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// c (+)= a b with b = hi + lo
template <bool kFirst>
__device__ __forceinline__ void mma_split(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t h0, uint32_t h1, uint32_t l0, uint32_t l1) {
  float x[4];
  mma_first(x, a0, a1, a2, a3, l0, l1);
  mma_half(x, a0, a1, a2, a3, h0, h1);
#pragma unroll
  for (int k = 0; k < 4; ++k) c[k] = kFirst ? x[k] : c[k] + x[k];
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
// all ones in the halves that are infinite or no number
__device__ __forceinline__ uint32_t odd_halves(uint32_t u) { return __vcmpgtu2(u & 0x7fff7fffu, 0x7bff7bffu); }
// two of a word's numbers as MMA operand: n 2^-24 (16 n 2^-24 for the high ones), or, normal, n (16 n)
template <bool kNormal> __device__ __forceinline__ uint32_t numbers(uint32_t x, uint32_t mask) {
  x &= mask;
  if (!kNormal) return x;
  const __half2 h = __hsub2(as_half2(x | 0x64006400u), __float2half2_rn(1024.f));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// What a warp works on, and where it stands in its CTA's share: in shared memory, because the pass over the keys has no registers to spare.  The warps of a CTA all write the
// same segment, into one of three places in turn.
struct Segment {
  int64_t item0;                             // the triple's first piece in the common order
  const int* row_table;
  const uint8_t* head_pages;                 // of its kv head in page 0
  int tile, head, valid, pad;                // valid: query rows of the tile
  int rows0, position0;                      // of the sequence's first new token
  int n_pieces, from_piece, to_piece;        // of the triple: pieces [from_piece, to_piece)
  int n_stages;                              // units of those
  int first_block, highest, lowest;          // keys that some row sees
  int all_from, all_to;                      // keys that all rows see
};
struct Walk {
  int64_t u;                                 // first piece that is left of the share
  int b, pad;                                // its sequence
};

__device__ __forceinline__ int row_tiles(int T, int G, int cols) { return (T * G + cols - 1) / cols; }

template <typename T, int NG, int NT>
__global__ void __launch_bounds__(kThreads, NG >= 5 ? 2 : NT == 1 ? 4 : 3) attention_kernel(const Params p) {
  using S = Shape<T, NG, NT>;
  constexpr int D = S::D, COLS = S::COLS, kStages = S::kStages;
  constexpr bool kSplit = S::kSplit;
  constexpr int BK = 2;                      // blocks of 16 keys whose scores are in registers at once
  constexpr float kPScale = 7.f, kPMost = 15.f;            // weights are 2^7 p at the maximum, up to 2^15 while it lags
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* at = smem;
  uint8_t* my_ring = at + (threadIdx.x >> 5) * kStages * S::kStageBytes; at += S::kRing;
  float* merge = reinterpret_cast<float*>(at); at += S::kMerge;
  uint32_t* qfrag = reinterpret_cast<uint32_t*>(at); at += S::kQ;
  uint2* qsum = reinterpret_cast<uint2*>(at); at += S::kQSum;
  uint64_t* my_full = reinterpret_cast<uint64_t*>(at) + (threadIdx.x >> 5) * kStages; at += kWarps * kStages * 8;
  float* col_scale = reinterpret_cast<float*>(at); at += COLS * 4;
  int* col_end = reinterpret_cast<int*>(at); at += COLS * 4;
  int* col_from = reinterpret_cast<int*>(at); at += COLS * 4;
  unsigned* col_top = reinterpret_cast<unsigned*>(at); at += COLS * 4;
  float* warp_m = reinterpret_cast<float*>(at); at += kWarps * COLS * 4;
  float* warp_l = reinterpret_cast<float*>(at); at += kWarps * COLS * 4;
  int* shared_word = reinterpret_cast<int*>(at); at += 64;  // 0..3 sums of warps, 4 the last one's flag
  Segment* segments = reinterpret_cast<Segment*>(at); at += 3 * 96;
  Walk* walk = reinterpret_cast<Walk*>(at) + (threadIdx.x >> 5); at += kWarps * 16;
  unsigned* before = reinterpret_cast<unsigned*>(at);      // [n_seq + 1] pieces of the sequences before
  int* seq_len = reinterpret_cast<int*>(before + p.n_seq + 1);           // [n_seq] their tokens

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  if (lane < kStages) tc::mbar_init(my_full + lane, 1);
  tc::mbar_init_fence();
  if (tid < COLS) col_top[tid] = 0;
  for (int i = tid; i < NT * 32; i += kThreads) qsum[i] = make_uint2(0, 0);               // groups that are not there stay 0
  pdl_launch_dependents();
  pdl_wait();

  // pieces of every sequence
  unsigned piece = 1;
  auto units_of = [&](int T_, int len, int& first) __attribute__((always_inline)) {
    const int lowest = len - T_;                           // position of the first row
    first = p.window > 0 && lowest - p.window + 1 > 0 ? (lowest - p.window + 1) / kUnit : 0;
    return max(1, (len + kUnit - 1) / kUnit - first);      // a sequence without keys still has rows to write
  };
  {
    const int capacity = p.max_pages << p.shift;
    const int per = (p.n_seq + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, p.n_seq), b1 = min(b0 + per, p.n_seq);
    unsigned sum = 0, items = 0;
    bool bad = false, broken = false;
    for (int b = b0; b < b1; ++b) {
      const int r0 = p.cu_rows[b], r1 = p.cu_rows[b + 1], l = p.lens[b];
      const int len = min(max(l, 0), capacity);
      int T_ = r1 - r0, first;
      if (l != len) { bad = true; T_ = 0; }                // longer than its table, or negative: left out
      if (r0 < 0 || r1 < r0 || r1 > p.rows) { broken = true; T_ = 0; }
      const unsigned triples = T_ > 0 ? (unsigned)row_tiles(T_, p.G, COLS) * p.heads : 0u, n = triples * units_of(T_, len, first);
      seq_len[b] = len;
      before[b + 1] = n;
      sum += n;
      items += triples;
    }
    if ((bad || broken) && blockIdx.x == 0) atomicExch(p.dev_arg, kErrPage);
    // units per piece: 1, or so many that every CTA has one piece
    {
      unsigned all = sum, of = items;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, off);
        of += __shfl_xor_sync(0xffffffffu, of, off);
      }
      if (lane == 0) { shared_word[warp] = (int)all; shared_word[8 + warp] = (int)of; }
      // Offsets that descend could make sequences overlap, and more work than the host has counted.
      if (__syncthreads_or(broken)) return;
      all = of = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) { all += (unsigned)shared_word[w]; of += (unsigned)shared_word[8 + w]; }
      const unsigned room = gridDim.x - min(of, gridDim.x);
      if (room > 0 && all > room) {          // (else every unit has a CTA)
        const unsigned each = (all + room - 1) / room;       // sum of ceil(n / each) <= all / each + of <= the CTAs
        unsigned longest = 0, pieces = 0;
        for (int b = b0; b < b1; ++b) {
          if (before[b + 1] == 0) continue;
          int first;
          const int T_ = p.cu_rows[b + 1] - p.cu_rows[b];
          const unsigned n = units_of(T_, seq_len[b], first), k = (n + each - 1) / each;
          longest = max(longest, (n + k - 1) / k);
          pieces += (unsigned)row_tiles(T_, p.G, COLS) * p.heads * k;
        }
        if (!__syncthreads_or(longest > all / gridDim.x + kLonger)) {
          piece = each;
          sum = pieces;
          for (int b = b0; b < b1; ++b) {
            if (before[b + 1] == 0) continue;
            int first;
            const int T_ = p.cu_rows[b + 1] - p.cu_rows[b];
            before[b + 1] = (unsigned)row_tiles(T_, p.G, COLS) * p.heads * ((units_of(T_, seq_len[b], first) + each - 1) / each);
          }
        }
      }
    }
    unsigned incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += u;
    }
    if (lane == 31) shared_word[4 + warp] = (int)incl;
    __syncthreads();
    unsigned run = incl - sum;
    for (int w = 0; w < warp; ++w) run += (unsigned)shared_word[4 + w];
    for (int b = b0; b < b1; ++b) { run += before[b + 1]; before[b + 1] = run; }
    if (tid == 0) before[0] = 0;
    __syncthreads();
  }
  // every CTA that takes part has a share, every share a piece
  const int64_t U = before[p.n_seq];
  const int grid = (int)min((int64_t)gridDim.x, U);
  if ((int)blockIdx.x >= grid) return;

  const int per_page = 1 << (p.shift - 4);

  // the next segment of the CTA's share into *sg; false behind the last
  const int64_t u_end = share_begin((int)blockIdx.x + 1, U, grid);
  auto advance = [&](Segment* sg) __attribute__((always_inline)) -> bool {
    const int64_t u = walk->u;
    if (u >= u_end) return false;
    int b = walk->b;
    while ((int64_t)before[b + 1] <= u) ++b;
    int first_unit;
    const int rows0 = p.cu_rows[b], T_ = p.cu_rows[b + 1] - rows0, len = seq_len[b];
    const int n_units = units_of(T_, len, first_unit);
    const int n_pieces = (n_units + (int)piece - 1) / (int)piece;        // of as equal lengths as units allow
    const int triple = (int)((unsigned)(u - before[b]) / (unsigned)n_pieces), tile = triple / p.heads, head = triple - tile * p.heads;
    const int64_t item0 = (int64_t)before[b] + (int64_t)triple * n_pieces;
    const int valid = min(COLS, T_ * p.G - tile * COLS);                 // query rows of this tile; their positions ascend
    const int first_pos = len - T_ + tile * COLS / p.G, last_pos = len - T_ + (tile * COLS + valid - 1) / p.G;
    const int from_piece = (int)(u - item0), to_piece = (int)min((int64_t)n_pieces, u_end - item0);
    const int from_unit = (int)((int64_t)n_units * from_piece / n_pieces), to_unit = (int)((int64_t)n_units * to_piece / n_pieces);
    __syncwarp();
    if (lane == 0) {
      sg->item0 = item0;
      sg->row_table = p.table + (int64_t)b * p.max_pages;
      sg->head_pages = p.pages + (int64_t)head * per_page * (640 * NG);
      sg->tile = tile; sg->head = head; sg->valid = valid;
      sg->rows0 = rows0; sg->position0 = len - T_;
      sg->n_pieces = n_pieces; sg->from_piece = from_piece; sg->to_piece = to_piece;
      sg->n_stages = to_unit - from_unit;
      sg->first_block = (first_unit + from_unit) * (kUnit / 16);
      sg->highest = max(0, last_pos + 1);
      sg->lowest = p.window > 0 ? max(0, first_pos - p.window + 1) : 0;
      sg->all_from = p.window > 0 ? max(0, last_pos - p.window + 1) : 0;
      sg->all_to = max(0, first_pos + 1);
      walk->u = item0 + to_piece; walk->b = b;
    }
    __syncwarp();
    return true;
  };

  // ---- ring: stage j holds this warp's two blocks of unit from_unit + j --------------------------------------------------
  int slot = 0, ids = -1, ids_next = -1;
  uint32_t phases = 0, loaded = 0;           // per stage of the ring: parity of its next wait; two bits for the blocks that are there
  bool dead = false;
  auto place_of = [&](const Segment* sg, int batch) __attribute__((always_inline)) {       // lane: block lane % 2 of stage 16 batch + lane / 2; -1: not to be read
    const int j = batch * 16 + (lane >> 1), key = (sg->first_block + 2 * warp + j * (kUnit / 16) + (lane & 1)) * 16;
    return j < sg->n_stages && key < sg->highest && key + 16 > sg->lowest ? key >> p.shift : -1;
  };
  auto page_at = [&](const Segment* sg, int batch) __attribute__((always_inline)) {
    const int place = place_of(sg, batch);
    return place >= 0 ? sg->row_table[place] : -1;
  };
  auto checked = [&](const Segment* sg, int batch, int page) __attribute__((always_inline)) {
    if ((unsigned)page < (unsigned)p.n_pages) return page;
    if (place_of(sg, batch) >= 0) atomicExch(p.dev_arg, kErrPage);
    return -1;
  };
  auto issue = [&](const Segment* sg, int j, int s) __attribute__((always_inline)) {
    if (j > 0 && (j & 15) == 0) {
      ids = checked(sg, j >> 4, ids_next);
      ids_next = page_at(sg, (j >> 4) + 1);
    }
    const int p0 = __shfl_sync(0xffffffffu, ids, (j & 15) * 2), p1 = __shfl_sync(0xffffffffu, ids, (j & 15) * 2 + 1);
    const uint32_t bits = (p0 >= 0 ? 1u : 0u) | (p1 >= 0 ? 2u : 0u);
    loaded = (loaded & ~(3u << (2 * s))) | bits << (2 * s);
    if (bits && lane == 0) {
      const int inside = (sg->first_block + 2 * warp + j * (kUnit / 16)) & (per_page - 1);
      const int64_t page_pitch = (int64_t)(p.heads * per_page) * (640 * NG);
      uint8_t* dst = my_ring + s * S::kStageBytes;
      const uint8_t* src = sg->head_pages + p0 * page_pitch + inside * (640 * NG);
      if (bits == 3 && per_page > 1) {                     // neighbours in one page
        tc::mbar_expect_tx(my_full + s, 2 * 640 * NG);
        tc::bulk_g2s(dst, src, 2 * 640 * NG, my_full + s);
      } else {
        tc::mbar_expect_tx(my_full + s, (bits == 3 ? 2 : 1) * 640 * NG);
        if (bits & 1) tc::bulk_g2s(dst, src, 640 * NG, my_full + s);
        if (bits & 2) tc::bulk_g2s(dst + 640 * NG, sg->head_pages + p1 * page_pitch + ((inside + 1) & (per_page - 1)) * (640 * NG), 640 * NG, my_full + s);
      }
    }
  };
  auto start = [&](const Segment* sg, int page0, int page1) __attribute__((always_inline)) {
    ids = checked(sg, 0, page0);
    ids_next = page1;
    slot = 0;
    const int n = min(kStages, sg->n_stages);
#pragma unroll 1
    for (int s = 0; s < n; ++s) issue(sg, s, s);
  };

  // ---- queries: four threads have a group of a row ---------------------------------------------------------------------------
  constexpr int kTasks = COLS * NG * 4, kRounds = (kTasks + kThreads - 1) / kThreads;
  auto load_queries = [&](const Segment* sg, uint4 (&v)[kRounds][kSplit ? 2 : 1]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int task = tid + i * kThreads, c = task / (NG * 4), f = (task - c * (NG * 4)) * 8;
      v[i][0] = make_uint4(0, 0, 0, 0);
      if (kSplit) v[i][kSplit ? 1 : 0] = make_uint4(0, 0, 0, 0);
      if (task < kTasks && c < sg->valid) {
        const int rho = sg->tile * COLS + c, row = rho / p.G, hq = rho - row * p.G;
        const T* qr = reinterpret_cast<const T*>(p.q) + (int64_t)(sg->rows0 + row) * p.q_stride + (int64_t)(sg->head * p.G + hq) * D + f;
        v[i][0] = *reinterpret_cast<const uint4*>(qr);
        if (kSplit) v[i][kSplit ? 1 : 0] = *reinterpret_cast<const uint4*>(qr + 4);
      }
    }
  };
  auto feature = [&](const uint4 (&v)[kSplit ? 2 : 1], int k) __attribute__((always_inline)) {
    if (kSplit) {
      const uint4& w = v[kSplit ? k >> 2 : 0];
      return __uint_as_float((k & 3) == 0 ? w.x : (k & 3) == 1 ? w.y : (k & 3) == 2 ? w.z : w.w);
    }
    const uint32_t w = (k >> 1) == 0 ? v[0].x : (k >> 1) == 1 ? v[0].y : (k >> 1) == 2 ? v[0].z : v[0].w;
    return __uint_as_float(k & 1 ? w & 0xffff0000u : w << 16);
  };

  auto put = [&](const Segment* my, int c, int d, float4 v, float L) __attribute__((always_inline)) {
    const float inv = L > 0.f || L != L ? 1.f / L : 0.f;             // a row that sees no key is 0
    const int rho = my->tile * COLS + c, row = rho / p.G, hq = rho - row * p.G;
    T* out = reinterpret_cast<T*>(p.out) + (int64_t)(my->rows0 + row) * p.out_stride + (int64_t)(my->head * p.G + hq) * D + d;
    if (kSplit) {
      *reinterpret_cast<float4*>(out) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    } else {
      __nv_bfloat162 x = __floats2bfloat162_rn(v.x * inv, v.y * inv), y = __floats2bfloat162_rn(v.z * inv, v.w * inv);
      *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<uint32_t*>(&x), *reinterpret_cast<uint32_t*>(&y));
    }
  };

  // The last of the shares that cut a triple joins what all of them left; of more than kJoin + kJoin / 2 the last of every kJoin neighbours first joins theirs.
  auto counted = [&](unsigned* counter, int of) __attribute__((always_inline)) {           // thread 0, behind a barrier behind all threads' writes
    unsigned old;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;\n" : "=r"(old) : "l"(counter) : "memory");
    const bool last = old == (unsigned)of - 1u;
    if (last) *counter = 0u;
    shared_word[4] = last;
  };
  auto count_part = [&](const Segment* my) __attribute__((always_inline)) {
    const Part q = part_of(my->item0, my->n_pieces, (int)blockIdx.x, U, grid);
    if (tid == 0) counted(p.counters + part_counter(q), q.count);
    return q;
  };
  // behind the barrier behind count_part
  auto join_parts = [&](const Segment* my, Part q) __attribute__((always_inline)) {
    if (!shared_word[4]) return;
    const int my_valid = my->valid;
    float* weight = merge;                   // [count][my_valid]
    int first = q.first, count = q.count, step = 1;
#pragma unroll 1
    for (bool done = q.groups == 1;; done = true) {
      // parts k of `count`, `step` shares apart: to the output, or to the first one's place
      auto place = [&](int k) __attribute__((always_inline)) { return (int64_t)((first + k * step) * 2 + (first + k * step == q.sa)) * COLS; };
      for (int c = warp; c < my_valid; c += kWarps) {
        float top = -CUDART_INF_F, L = 0.f;
        for (int k = lane; k < count; k += 32) top = fmaxf(top, __ldcg(&p.part_ml[place(k) + c].x));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        for (int k = lane; k < count; k += 32) {
          const float2 ml = __ldcg(p.part_ml + place(k) + c);
          const float f = ml.x == -CUDART_INF_F ? (ml.y != ml.y ? 1.f : 0.f) : exp2_fast(ml.x - top);
          weight[k * my_valid + c] = f;
          L = fmaf(ml.y, f, L);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
        if (lane == 0) { warp_m[c] = top; warp_l[c] = L; }
      }
      __syncthreads();
      for (int i = tid; i < my_valid * (D / 4); i += kThreads) {
        const int c = i / (D / 4), d = (i - c * (D / 4)) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int k0 = 0; k0 < count; k0 += 8) {            // eight loads on their way at a time
          float4 x[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + (place(min(k0 + k, count - 1)) + c) * D + d));
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float f = k0 + k < count ? weight[(k0 + k) * my_valid + c] : 0.f;
            if (f != 0.f) { sum.x = fmaf(x[k].x, f, sum.x); sum.y = fmaf(x[k].y, f, sum.y); sum.z = fmaf(x[k].z, f, sum.z); sum.w = fmaf(x[k].w, f, sum.w); }
          }
        }
        if (done) {
          put(my, c, d, sum, warp_l[c]);
        } else {
          __stcg(reinterpret_cast<float4*>(p.part_o + (place(0) + c) * D + d), sum);
          if (d == 0) __stcg(p.part_ml + place(0) + c, make_float2(warp_m[c], warp_l[c]));
        }
      }
      __syncthreads();
      if (done) break;
      if (tid == 0) counted(p.counters + triple_counter(q), q.groups);
      __syncthreads();
      if (!shared_word[4]) break;
      first = q.sa;
      count = q.groups;
      step = kJoin;
    }
  };

  {
    const int64_t u = share_begin((int)blockIdx.x, U, grid);
    int lo = 0, hi = p.n_seq - 1;            // the last sequence with before[b] <= u
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)before[mid] <= u) lo = mid; else hi = mid - 1;
    }
    if (lane == 0) { walk->u = u; walk->b = lo; }
  }
  __syncwarp();
  int at_segment = 0;
  bool more = true, pending = false;         // a part of the segment before this one waits to be counted
  advance(segments);
  uint4 v[kRounds][kSplit ? 2 : 1];
  load_queries(segments, v);
  start(segments, page_at(segments, 0), page_at(segments, 1));
  for (;;) {
    const Segment* sg = segments + at_segment;
    // ---- queries: MMA operands, sums per group, each row scaled to [2^9, 2^10) ----------------------------------------------
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int task = tid + i * kThreads, c = task / (NG * 4);
      unsigned top = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(fabsf(feature(v[i], k))));
      if (task < kTasks && c < sg->valid) atomicMax(col_top + c, top);
    }
    __syncthreads();                         // also: the parts of the segment before are written
    Part before_this;
    if (pending) before_this = count_part(segments + (at_segment + 2) % 3);
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int task = tid + i * kThreads, c = task / (NG * 4), rest = task - c * (NG * 4), gr = rest >> 2, part = rest & 3;
      if (task < kTasks) {
        const unsigned top = col_top[c];
        const int e = top > 0 ? max((int)(top >> 23) - 127, -117) : 9;                     // 2^(9 - e) stays a float
        const float up = __uint_as_float((uint32_t)(min(127 + 9 - e, 253)) << 23), down = __uint_as_float((uint32_t)max(127 - 9 + e, 1) << 23);
        float sum = 0.f;
        const int tl = 2 * gr + (part >> 1), hid = part & 1;                               // features 16 tl + 8 hid ..: register hid of the B operand
        uint32_t* dst = qfrag + ((tl * NT + (c >> 3)) * 32 + (c & 7) * 4) * (kSplit ? 4 : 2) + hid;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x = feature(v[i], 2 * k) * up, y = feature(v[i], 2 * k + 1) * up, f = hid ? 0.0625f : 1.f;
          sum += x + y;
          const uint32_t h = pack(x * f, y * f);
          dst[k * (kSplit ? 4 : 2)] = h;
          if (kSplit) {
            const float2 back = __half22float2(as_half2(h));
            dst[k * 4 + 2] = pack(x * f - back.x, y * f - back.y);
          }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (part == 0) {
          const __half sh = __float2half_rn(sum);
          __half* qs = reinterpret_cast<__half*>(qsum + (c >> 3) * 32 + (c & 7) * 4 + (gr >> 1));
          qs[gr & 1] = sh;
          qs[2 + (gr & 1)] = __float2half_rn(sum - __half2float(sh));
          if (gr == 0) {
            const int position = sg->position0 + (sg->tile * COLS + c) / p.G;
            col_scale[c] = p.scale * (kSplit ? 1.f : 16777216.f) * down;
            col_end[c] = c < sg->valid ? max(0, position + 1) : sg->highest;               // columns that are no rows have scores of 0
            col_from[c] = c >= sg->valid ? sg->lowest : p.window > 0 ? max(0, position - p.window + 1) : 0;
          }
        }
      }
    }
    __syncthreads();
    if (pending) join_parts(segments + (at_segment + 2) % 3, before_this);
    // the segment after this one and its first pages, to be at hand when this one's keys are through
    const int next = at_segment == 2 ? 0 : at_segment + 1;
    more = advance(segments + next);
    const int page0 = more ? page_at(segments + next, 0) : -1, page1 = more ? page_at(segments + next, 1) : -1;
    float cs[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) { cs[nt][0] = col_scale[nt * 8 + 2 * t]; cs[nt][1] = col_scale[nt * 8 + 2 * t + 1]; }

    // ---- one pass over the keys ----------------------------------------------------------------------------------------
    // Weights times scales are halves, which end at 2^16 and at 2^-24.  The quick way takes them as they are; where its sums are no numbers, or so small that the roundings of
    // subnormals may show, the segment is gone through again with care: the maximum never lags, and the products of each block, row and group are brought to the top of the halves by a power of
    // two of their own, so no group, row or key takes bits from another.
    float m[NT][2], l[NT][2], o[2 * NG][NT][4], om[NT][4];
    uint32_t seen = 0;                       // columns that have a maximum; m of the others is 0
    const int n_stages = sg->n_stages, first_key = (sg->first_block + 2 * warp) * 16, all_from = sg->all_from, all_to = sg->all_to;
    auto pass = [&](auto with_care, auto from, auto to) __attribute__((always_inline)) {            // column tiles from .. to - 1
      constexpr bool careful = decltype(with_care)::value;
      constexpr int first = decltype(from)::value, last = decltype(to)::value;
      constexpr uint32_t every = (1u << (2 * last)) - (1u << (2 * first));
      seen &= ~every;
      bool ready = false;                    // all columns have one
#pragma unroll
      for (int nt = first; nt < last; ++nt) {
        m[nt][0] = m[nt][1] = 0.f;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) om[nt][k] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[i][nt][k] = 0.f;
      }
#pragma unroll 1
      for (int j = 0; j < n_stages; ++j) {
        const uint32_t bits = loaded >> (2 * slot) & 3u;
        if (bits) {
          tc::mbar_wait(my_full + slot, phases >> slot & 1u, dead, p.dev_err);
          phases ^= 1u << slot;
          const int key0 = first_key + j * kUnit;
          const bool cut = bits != 3u || key0 < all_from || key0 + 32 > all_to;              // some row does not see all of it
          const uint8_t* stage = my_ring + slot * S::kStageBytes;
          float s[BK][NT][4];
          // minima: one MMA whose k slots are the groups, sums of q as hi (k < 8) and lo
#pragma unroll
          for (int kb = 0; kb < BK; ++kb) {
            const uint32_t* minima = reinterpret_cast<const uint32_t*>(stage + kb * 640 * NG + 544 * NG);
            uint32_t x = 0, y = 0;
            if (2 * t < NG) x = minima[2 * t * 8 + g];
            if (2 * t + 1 < NG) y = minima[(2 * t + 1) * 8 + g];
            const uint32_t a0 = __byte_perm(x, y, 0x5410), a1 = __byte_perm(x, y, 0x7632);
#pragma unroll
            for (int nt = first; nt < last; ++nt) {
              const uint2 qs = qsum[nt * 32 + lane];
              mma_first(s[kb][nt], a0, a1, a0, a1, qs.x, qs.y);
              if (!kSplit)
#pragma unroll
                for (int k = 0; k < 4; ++k) s[kb][nt][k] *= 5.9604644775390625e-8f;        // 2^-24, as the numbers
            }
          }
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            float acc[BK][NT][4];
            uint2 w[BK];
#pragma unroll
            for (int kb = 0; kb < BK; ++kb) w[kb] = *reinterpret_cast<const uint2*>(stage + kb * 640 * NG + gr * 256 + lane * 8);
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
              uint32_t a[BK][4];
#pragma unroll
              for (int kb = 0; kb < BK; ++kb) {
                const uint32_t x = tile ? w[kb].y : w[kb].x;
                a[kb][0] = numbers<kSplit>(x, 0x000f000fu);
                a[kb][2] = numbers<kSplit>(x, 0x00f000f0u);
                a[kb][1] = numbers<kSplit>(x >> 8, 0x000f000fu);
                a[kb][3] = numbers<kSplit>(x >> 8, 0x00f000f0u);
              }
#pragma unroll
              for (int nt = first; nt < last; ++nt) {
                if (kSplit) {
                  const uint4 q = *reinterpret_cast<const uint4*>(qfrag + (((2 * gr + tile) * NT + nt) * 32 + lane) * 4);
#pragma unroll
                  for (int kb = 0; kb < BK; ++kb) {
                    if (tile) mma_split<false>(acc[kb][nt], a[kb][0], a[kb][1], a[kb][2], a[kb][3], q.x, q.y, q.z, q.w);
                    else mma_split<true>(acc[kb][nt], a[kb][0], a[kb][1], a[kb][2], a[kb][3], q.x, q.y, q.z, q.w);
                  }
                } else {
                  const uint2 q = *reinterpret_cast<const uint2*>(qfrag + (((2 * gr + tile) * NT + nt) * 32 + lane) * 2);
#pragma unroll
                  for (int kb = 0; kb < BK; ++kb) {
                    if (tile) mma_half(acc[kb][nt], a[kb][0], a[kb][1], a[kb][2], a[kb][3], q.x, q.y);
                    else mma_first(acc[kb][nt], a[kb][0], a[kb][1], a[kb][2], a[kb][3], q.x, q.y);
                  }
                }
              }
            }
#pragma unroll
            for (int kb = 0; kb < BK; ++kb) {
              const float2 sc = __half22float2(as_half2(reinterpret_cast<const uint32_t*>(stage + kb * 640 * NG + 512 * NG)[gr * 8 + g]));
#pragma unroll
              for (int nt = first; nt < last; ++nt) {
                s[kb][nt][0] = fmaf(sc.x, acc[kb][nt][0], s[kb][nt][0]);
                s[kb][nt][1] = fmaf(sc.x, acc[kb][nt][1], s[kb][nt][1]);
                s[kb][nt][2] = fmaf(sc.y, acc[kb][nt][2], s[kb][nt][2]);
                s[kb][nt][3] = fmaf(sc.y, acc[kb][nt][3], s[kb][nt][3]);
              }
            }
          }
          // scores in units of log2, less the maximum as far as it is known, plus 7: weights are 2^7 p.  The maximum is raised only when it lags by more than 2^8, so most
          // blocks need no exchange between lanes.
          bool raise = false;
#pragma unroll
          for (int nt = first; nt < last; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float top = -CUDART_INF_F;
              const float less = kPScale - m[nt][k];
#pragma unroll
              for (int kb = 0; kb < BK; ++kb) {
                s[kb][nt][k] = fmaf(s[kb][nt][k], cs[nt][k], less);
                s[kb][nt][k + 2] = fmaf(s[kb][nt][k + 2], cs[nt][k], less);
                top = fmaxf(top, fmaxf(s[kb][nt][k], s[kb][nt][k + 2]));
              }
              raise |= top > kPScale + 8.f;
            }
          bool odd_values = false;           // a scale or minimum of a value is no number
          if (cut || careful || !ready || __any_sync(0xffffffffu, raise)) {
            if (cut) {
#pragma unroll
              for (int kb = 0; kb < BK; ++kb) {
                const bool there = bits >> kb & 1;
#pragma unroll
                for (int nt = first; nt < last; ++nt)
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const int key = key0 + kb * 16 + g + (k >= 2 ? 8 : 0), c = nt * 8 + 2 * t + (k & 1);
                    if (key >= col_end[c] || key < col_from[c] || !there) s[kb][nt][k] = -CUDART_INF_F;
                  }
                // What is no number among the values' scales and minima counts for the rows that see its key alone, and nothing counts of a block that is not there.  The stage is this
                // warp's own, so it is put in order in place, a word per lane: such scales become -0 and their minima 0; below, the rows that give a -0 a weight get their NaN.
                uint32_t* scales = reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(stage) + kb * 640 * NG + 576 * NG);
                for (int i = lane; i < 8 * NG; i += 32) {
                  const uint32_t sc = scales[i], mi = scales[8 * NG + i], odd = there ? odd_halves(sc) | odd_halves(mi) : 0xffffffffu;
                  if (odd) {
                    scales[i] = there ? (sc & ~odd) | (odd & 0x80008000u) : 0u;
                    scales[8 * NG + i] = mi & ~odd;
                    odd_values |= there;
                  }
                }
              }
              odd_values = __any_sync(0xffffffffu, odd_values);
              tc::fence_async_smem();        // before the next copy into this stage
            }
            __syncwarp();
#pragma unroll
            for (int nt = first; nt < last; ++nt)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                float x = fmaxf(fmaxf(s[0][nt][k], s[0][nt][k + 2]), fmaxf(s[1][nt][k], s[1][nt][k + 2]));
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                const float rise = x - (careful ? kPMost : kPScale);
                const bool fresh = !(seen >> (2 * nt + k) & 1);
                if (fresh ? x > -CUDART_INF_F : rise > 0.f) {
                  seen |= 1u << (2 * nt + k);
                  m[nt][k] += rise;
                  if (!fresh) {
                    const float fade = exp2_fast(-rise);
                    l[nt][k] *= fade;
                    om[nt][k] *= fade;
                    om[nt][k + 2] *= fade;
#pragma unroll
                    for (int i = 0; i < 2 * NG; ++i) { o[i][nt][k] *= fade; o[i][nt][k + 2] *= fade; }
                  }
#pragma unroll
                  for (int kb = 0; kb < BK; ++kb) { s[kb][nt][k] -= rise; s[kb][nt][k + 2] -= rise; }
                }
              }
            ready = __all_sync(0xffffffffu, (seen & every) == every);
          }
          // weights as halves (float32: two of them), from accumulators to B operands; then values, whose minima are an operand with groups as rows.  bf16 rounds twice, p and p s, each by 2^-12
          // of a term at most: beside results of unrounded weights, both rounded to bf16, 1.1e-3 of their size, where that rounding alone is 1.7e-3; a second half each would double the products
#pragma unroll
          for (int kb = 0; kb < BK; ++kb) {
            uint32_t pb[NT][kSplit ? 4 : 2];
            uint2 mn = make_uint2(0, 0);
            if (g < NG) mn = *reinterpret_cast<const uint2*>(stage + kb * 640 * NG + 608 * NG + g * 32 + t * 8);
#pragma unroll
            for (int nt = first; nt < last; ++nt) {
              float e[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) e[k] = exp2_fast(s[kb][nt][k]);
              l[nt][0] += e[0] + e[2];
              l[nt][1] += e[1] + e[3];
              const uint32_t h0 = pack(e[0], e[1]), h1 = pack(e[2], e[3]);
              pb[nt][0] = transposed(h0);
              pb[nt][1] = transposed(h1);
              if (kSplit) {
                const float2 f0 = __half22float2(as_half2(h0)), f1 = __half22float2(as_half2(h1));
                pb[nt][kSplit ? 2 : 0] = transposed(pack(e[0] - f0.x, e[1] - f0.y));
                pb[nt][kSplit ? 3 : 0] = transposed(pack(e[2] - f1.x, e[3] - f1.y));
              }
              if (kSplit) mma_split<false>(om[nt], mn.x, 0u, mn.y, 0u, pb[nt][0], pb[nt][1], pb[nt][kSplit ? 2 : 0], pb[nt][kSplit ? 3 : 0]);
              else mma_half(om[nt], mn.x, 0u, mn.y, 0u, pb[nt][0], pb[nt][1]);
            }
            if (odd_values) {
#pragma unroll
              for (int gr = 0; gr < NG; ++gr) {
                const uint2 sc = *reinterpret_cast<const uint2*>(stage + kb * 640 * NG + 576 * NG + gr * 32 + t * 8);
                const uint32_t ox = __vcmpeq2(sc.x, 0x80008000u), oy = __vcmpeq2(sc.y, 0x80008000u);
#pragma unroll
                for (int nt = first; nt < last; ++nt) {            // lane (g, t): row g's weights of keys 2t, 2t + 1, 2t + 8, 2t + 9
                  const unsigned hit = __ballot_sync(0xffffffffu, (pb[nt][0] & ox) | (pb[nt][1] & oy));
#pragma unroll
                  for (int k = 0; k < 2; ++k)
                    if (hit >> (4 * (2 * t + k)) & 15) o[2 * gr][nt][k] = o[2 * gr][nt][k + 2] = o[2 * gr + 1][nt][k] = o[2 * gr + 1][nt][k + 2] = CUDART_NAN_F;
                }
              }
            }
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              const uint2 w = *reinterpret_cast<const uint2*>(stage + kb * 640 * NG + 256 * NG + gr * 256 + lane * 8);
              const uint2 vs = *reinterpret_cast<const uint2*>(stage + kb * 640 * NG + 576 * NG + gr * 32 + t * 8);        // in the order of the weights' operand
              uint32_t wb[NT][kSplit ? 4 : 2];
              if (careful) {
#pragma unroll
                for (int nt = first; nt < last; ++nt) {            // lane (g, t): row g's weights of keys 2t, 2t + 1, 2t + 8, 2t + 9
                  float x[4], top = 0.f;
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    float2 e = __half22float2(as_half2(pb[nt][i])), f = __half22float2(as_half2(i ? vs.y : vs.x));
                    if (kSplit) {
                      const float2 lo = __half22float2(as_half2(pb[nt][kSplit ? 2 + i : 0]));
                      e.x += lo.x;
                      e.y += lo.y;
                    }
                    x[2 * i] = e.x * f.x;
                    x[2 * i + 1] = e.y * f.y;
                    top = fmaxf(top, fmaxf(fabsf(x[2 * i]), fabsf(x[2 * i + 1])));
                  }
                  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                  const int e = max((int)(__float_as_uint(top) >> 23), 60);                // less than 2^-66 is nothing
                  const float up = __uint_as_float((uint32_t)(268 - e) << 23), down = __uint_as_float((uint32_t)(e - 14) << 23);       // to [2^14, 2^15), and back
                  uint32_t hi[2], lo[2] = {0, 0};
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    hi[i] = pack(x[2 * i] * up, x[2 * i + 1] * up);
                    const float2 f = __half22float2(as_half2(hi[i]));
                    if (kSplit) lo[i] = pack(fmaf(x[2 * i], up, -f.x), fmaf(x[2 * i + 1], up, -f.y));
                  }
                  const float d0 = __shfl_sync(0xffffffffu, down, 8 * t), d1 = __shfl_sync(0xffffffffu, down, 8 * t + 4);              // of rows 2t, 2t + 1
#pragma unroll
                  for (int tile = 0; tile < 2; ++tile) {
                    const uint32_t y = tile ? w.y : w.x;
                    const uint32_t a0 = numbers<kSplit>(y, 0x000f000fu), a1 = numbers<kSplit>(y, 0x00f000f0u), a2 = numbers<kSplit>(y >> 8, 0x000f000fu),
                                   a3 = numbers<kSplit>(y >> 8, 0x00f000f0u);
                    float acc[4];
                    if (kSplit) mma_split<true>(acc, a0, a1, a2, a3, hi[0], hi[1], lo[0], lo[1]);
                    else mma_first(acc, a0, a1, a2, a3, hi[0], hi[1]);
                    float (&to)[4] = o[2 * gr + tile][nt];
                    to[0] = fmaf(acc[0], d0, to[0]);
                    to[1] = fmaf(acc[1], d1, to[1]);
                    to[2] = fmaf(acc[2], d0, to[2]);
                    to[3] = fmaf(acc[3], d1, to[3]);
                  }
                }
                continue;
              }
#pragma unroll
              for (int nt = first; nt < last; ++nt) {
                if (kSplit) {
                  const float2 sx = __half22float2(as_half2(vs.x)), sy = __half22float2(as_half2(vs.y));
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    const float2 hi = __half22float2(as_half2(pb[nt][i])), lo = __half22float2(as_half2(pb[nt][kSplit ? 2 + i : 0]));
                    const float x = (hi.x + lo.x) * (i ? sy.x : sx.x), y = (hi.y + lo.y) * (i ? sy.y : sx.y);
                    wb[nt][i] = pack(x, y);
                    const float2 f = __half22float2(as_half2(wb[nt][i]));
                    wb[nt][kSplit ? 2 + i : 0] = pack(x - f.x, y - f.y);
                  }
                } else {
                  wb[nt][0] = as_u32(__hmul2(as_half2(pb[nt][0]), as_half2(vs.x)));
                  wb[nt][1] = as_u32(__hmul2(as_half2(pb[nt][1]), as_half2(vs.y)));
                }
              }
#pragma unroll
              for (int tile = 0; tile < 2; ++tile) {
                const uint32_t x = tile ? w.y : w.x;
                const uint32_t a0 = numbers<kSplit>(x, 0x000f000fu), a1 = numbers<kSplit>(x, 0x00f000f0u), a2 = numbers<kSplit>(x >> 8, 0x000f000fu),
                               a3 = numbers<kSplit>(x >> 8, 0x00f000f0u);
#pragma unroll
                for (int nt = first; nt < last; ++nt) {
                  if (kSplit) mma_split<false>(o[2 * gr + tile][nt], a0, a1, a2, a3, wb[nt][0], wb[nt][1], wb[nt][kSplit ? 2 : 0], wb[nt][kSplit ? 3 : 0]);
                  else mma_half(o[2 * gr + tile][nt], a0, a1, a2, a3, wb[nt][0], wb[nt][1]);
                }
              }
            }
          }
        }
        __syncwarp();
        if (j + kStages < n_stages) issue(sg, j + kStages, slot);
        slot = slot + 1 == kStages ? 0 : slot + 1;
      }
    };
    pass(std::false_type(), std::integral_constant<int, 0>(), std::integral_constant<int, NT>());
    bool again;
    {
      // As bits sums ascend, 0 up to infinity and NaN.  A product is off by 2^-26 (2^-25 at most) where it is subnormal, so a sum over k keys of n about 7 by sqrt(k) 2^-23: less than 2^-18
      // (bf16: 2^-13) of a group's largest where that is not below `least`, in units of the high numbers, which count 16 times.  (0 is no rounding's work: the key of the largest
      // weight has at least 2^7 2^-24.)  First each lane's largest sum of four features, then the group's.
      const uint32_t least = __float_as_uint(sqrtf(32.f * n_stages) * (kSplit ? 0.5f : 0x1p-30f)) - 1u;
      auto largest = [&](int gr, int nt, int k) __attribute__((always_inline)) {
        return max(max(__float_as_uint(o[2 * gr][nt][k]), __float_as_uint(o[2 * gr + 1][nt][k])), max(__float_as_uint(o[2 * gr][nt][k + 2]), __float_as_uint(o[2 * gr + 1][nt][k + 2])));
      };
      uint32_t top = 0, lowest = 0xffffffffu;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            const uint32_t x = largest(gr, nt, k);
            top = max(top, x);
            lowest = min(lowest, x - 1u);    // 0 is no small one
          }
      again = top >= 0x7f800000u;
      if (__builtin_expect(__any_sync(0xffffffffu, lowest < least), 0)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              uint32_t x = largest(gr, nt, k);
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) x = max(x, __shfl_xor_sync(0xffffffffu, x, off));
              again |= x - 1u < least;
            }
      }
    }
    if (__builtin_expect(__any_sync(0xffffffffu, again), 0)) {
      start(sg, page_at(sg, 0), page_at(sg, 1));
      pass(std::true_type(), std::integral_constant<int, 0>(), std::integral_constant<int, 1>());
      if constexpr (NT == 2) {               // a tile at a time, so that this takes no more registers than the quick way
        start(sg, page_at(sg, 0), page_at(sg, 1));
        pass(std::true_type(), std::integral_constant<int, NT - 1>(), std::integral_constant<int, NT>());
      }
    }

    // ---- the next segment's keys are asked for while this one's sums become one -------------------------------------------------
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (!(seen >> (2 * nt + k) & 1)) m[nt][k] = -CUDART_INF_F;
    if (more) {
      start(segments + next, page0, page1);
      load_queries(segments + next, v);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[nt][k] += __shfl_xor_sync(0xffffffffu, l[nt][k], off);
        if (g == 0) {
          warp_m[warp * COLS + nt * 8 + 2 * t + k] = m[nt][k];
          warp_l[warp * COLS + nt * 8 + 2 * t + k] = l[nt][k];
        }
      }
    __syncthreads();
    if (tid < COLS) col_top[tid] = 0;
    float fade[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float top = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_m[w * COLS + nt * 8 + 2 * t + k]);
        fade[nt][k] = m[nt][k] == -CUDART_INF_F ? (l[nt][k] != l[nt][k] ? 1.f : 0.f) : exp2_fast(m[nt][k] - top);
      }
    constexpr float kUp = kSplit ? 0x1p-4f : 0x1p20f;      // of 16 n; n takes another 16
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {   // warps 0 and 1 write, 2 and 3 add
      if (warp >> 1 == turn) {
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float b0 = __shfl_sync(0xffffffffu, om[nt][0], (i >> 1) * 4 + t), b1 = __shfl_sync(0xffffffffu, om[nt][1], (i >> 1) * 4 + t);
            float* dst = merge + ((warp & 1) * COLS + nt * 8 + 2 * t) * S::kPitch + 16 * i + g;
            const float x0 = fmaf(o[i][nt][0], kUp * 16.f, b0) * fade[nt][0], x1 = fmaf(o[i][nt][1], kUp * 16.f, b1) * fade[nt][1];
            const float x2 = fmaf(o[i][nt][2], kUp, b0) * fade[nt][0], x3 = fmaf(o[i][nt][3], kUp, b1) * fade[nt][1];
            if (turn == 0) {
              dst[0] = x0; dst[S::kPitch] = x1; dst[8] = x2; dst[S::kPitch + 8] = x3;
            } else {
              dst[0] += x0; dst[S::kPitch] += x1; dst[8] += x2; dst[S::kPitch + 8] += x3;
            }
          }
      }
      __syncthreads();
    }
    const bool alone = sg->from_piece == 0 && sg->to_piece == sg->n_pieces;
    const int part = (int)blockIdx.x * 2 + (sg->from_piece == 0 ? 1 : 0);
    for (int i = tid; i < sg->valid * (D / 4); i += kThreads) {
      const int c = i / (D / 4), d = (i - c * (D / 4)) * 4;
      float top = -CUDART_INF_F, L = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_m[w * COLS + c]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = warp_m[w * COLS + c], lw = warp_l[w * COLS + c];
        L += mw == -CUDART_INF_F ? (lw != lw ? lw : 0.f) : lw * exp2_fast(mw - top);
      }
      const float4 x = *reinterpret_cast<const float4*>(merge + c * S::kPitch + d), y = *reinterpret_cast<const float4*>(merge + (COLS + c) * S::kPitch + d);
      const float4 w = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
      if (alone) {
        put(sg, c, d, w, L);
      } else {
        __stcg(reinterpret_cast<float4*>(p.part_o + ((int64_t)part * COLS + c) * D + d), w);
        if (d == 0) __stcg(p.part_ml + part * COLS + c, make_float2(top, L));
      }
    }
    pending = !alone;
    if (!more) break;
    at_segment = next;
  }
  if (pending) {
    __syncthreads();
    const Part last = count_part(segments + at_segment);
    __syncthreads();
    join_parts(segments + at_segment, last);
  }
}

template <typename T, int NG, int NT> int32_t configure_one(Variant* v) {
  using S = Shape<T, NG, NT>;
  v->kernel = attention_kernel<T, NG, NT>;
  v->smem = S::kFixed;
  const int most = S::kFixed + seq_bytes(kMaxSeqs);
  LMB_CUDA(cudaFuncSetAttribute(v->kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  LMB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&v->ctas_per_sm, v->kernel, kThreads, (size_t)S::kFixed + seq_bytes(64)));
  return LMB200_OK;
}

}  // namespace kv4
}  // namespace lmb
