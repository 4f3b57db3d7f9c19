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
// Work.  Units of 128 keys of all (sequence, row tile, kv head) triples in a row are cut into equal shares, one per CTA, whatever the sequences' lengths, so a long
// sequence among short ones is shared by many CTAs.  Each of a CTA's four warps takes 32 keys of a unit through a ring of bulk copies of its own.  Where
// a triple is shared, its CTAs leave partial sums and the last one to finish joins them.
#pragma once
#include <math_constants.h>

#include <type_traits>

#include "kv4.cuh"
#include "pdl.cuh"
#include "tc.cuh"

namespace lmb {
namespace kv4 {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kUnit = 128, kMaxSeqs = 8192, kCounterBytes = 8192;

struct Params {
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  int rows, n_seq, max_pages, n_pages, shift, heads, G, window;
  float scale;                               // of the scores, times log2(e)
  const int *cu_rows, *lens, *table;
  const uint8_t* pages;
  int* dev_err;
  unsigned* counters;                        // [grid], zero between calls
  float2* part_ml;                           // [grid][2][columns]: maximum (log2) and sum
  float* part_o;                             // [grid][2][columns][D]
};

// One variant: widths of NG groups, NT tiles of 8 query rows.
struct Variant {
  void (*kernel)(Params) = nullptr;
  int smem = 0, ctas_per_sm = 0;
};
const Variant* variant_bf16(int NG, int NT);
const Variant* variant_f32(int NG, int NT);
int32_t configure_bf16();
int32_t configure_f32();
// most query rows that share a pass over the keys, in tiles of 8: what the registers hold of out (8 NG values of it per tile and thread)
__host__ __device__ constexpr int most_tiles(bool f32, int NG) { return f32 ? 2 : NG <= 4 ? 4 : 2; }

template <typename T, int NG, int NT> struct Shape {
  static constexpr bool kSplit = sizeof(T) == 4;          // float32: operands as two halves, 22 bits
  static constexpr int D = 32 * NG, COLS = 8 * NT;
  static constexpr int kStageBytes = 2 * 640 * NG;
  static constexpr int kStages = NG == 1 ? 8 : NG == 2 ? 6 : NG == 3 ? 4 : NG <= 5 ? 3 : 2;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kPitch = D + 4;                    // of the joined sums: 2 kPitch = 8 banks
  static constexpr int kMerge = kWarps * COLS * kPitch * 4;
  static constexpr int kBig = kRing > kMerge ? kRing : kMerge;
  static constexpr int kQ = 2 * NG * NT * 32 * (kSplit ? 16 : 8);
  static constexpr int kQSum = NT * 32 * 8;
  static constexpr int kFixed = kBig + kQ + kQSum + COLS * 12 + 2 * kWarps * COLS * 4 + kWarps * kStages * 8 + 64;
};

__device__ __forceinline__ void mma_half(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c += a b with b = hi + lo
__device__ __forceinline__ void mma_split(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t h0, uint32_t h1, uint32_t l0, uint32_t l1) {
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  mma_half(x, a0, a1, a2, a3, l0, l1);
  mma_half(x, a0, a1, a2, a3, h0, h1);
#pragma unroll
  for (int k = 0; k < 4; ++k) c[k] += x[k];
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
// two of a word's numbers as MMA operand: n 2^-24 (16 n 2^-24 for the high ones), or, normal, n (16 n)
template <bool kNormal> __device__ __forceinline__ uint32_t numbers(uint32_t x, uint32_t mask) {
  x &= mask;
  if (!kNormal) return x;
  const __half2 h = __hsub2(as_half2(x | 0x64006400u), __float2half2_rn(1024.f));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// Where a unit of work lies.
struct Segment {
  int b, tile, head;                         // triple
  int rows0, T, len;                         // the sequence's first row, its rows, its tokens
  int first_unit, n_units;                   // of the triple: keys kUnit first_unit ..
  int64_t item0;                             // the triple's first unit in the common order
};

__device__ __forceinline__ int row_tiles(int T, int G, int cols) { return (T * G + cols - 1) / cols; }

template <typename T, int NG, int NT>
__global__ void __launch_bounds__(kThreads, NT >= 3 || NG >= 5 ? 2 : 3) attention_kernel(const Params p) {
  using S = Shape<T, NG, NT>;
  constexpr int D = S::D, COLS = S::COLS, kStages = S::kStages;
  constexpr bool kSplit = S::kSplit;
  constexpr int BK = NT <= 2 ? 2 : 1;        // blocks of 16 keys whose scores are in registers at once
  constexpr float kPScale = 7.f;             // weights are 2^7 p at the maximum, up to 2^15 while it lags
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  float* merge = reinterpret_cast<float*>(smem);
  uint8_t* at = smem + S::kBig;
  uint32_t* qfrag = reinterpret_cast<uint32_t*>(at); at += S::kQ;
  uint2* qsum = reinterpret_cast<uint2*>(at); at += S::kQSum;
  uint64_t* full = reinterpret_cast<uint64_t*>(at); at += kWarps * kStages * 8;
  float* col_scale = reinterpret_cast<float*>(at); at += COLS * 4;
  int* col_end = reinterpret_cast<int*>(at); at += COLS * 4;
  int* col_from = reinterpret_cast<int*>(at); at += COLS * 4;
  float* warp_m = reinterpret_cast<float*>(at); at += kWarps * COLS * 4;
  float* warp_l = reinterpret_cast<float*>(at); at += kWarps * COLS * 4;
  int* shared_word = reinterpret_cast<int*>(at); at += 64;
  unsigned* before = reinterpret_cast<unsigned*>(at);      // [n_seq + 1] units of the sequences before

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  for (int i = tid; i < kWarps * kStages; i += kThreads) tc::mbar_init(full + i, 1);
  tc::mbar_init_fence();
  pdl_launch_dependents();
  pdl_wait();

  // units of every sequence
  const int capacity = p.max_pages << p.shift;
  auto look_at = [&](int b, int& r0, int& T_, int& len) {
    r0 = p.cu_rows[b];
    const int r1 = p.cu_rows[b + 1];
    len = p.lens[b];
    bool bad = len < 0 || len > capacity;
    len = min(max(len, 0), capacity);
    T_ = r1 - r0;
    if (r0 < 0 || r1 < r0 || r1 > p.rows) { bad = true; T_ = 0; }
    return bad;
  };
  auto units_of = [&](int T_, int len, int& first) {
    const int lowest = len - T_;                           // position of the first row
    first = p.window > 0 && lowest - p.window + 1 > 0 ? (lowest - p.window + 1) / kUnit : 0;
    return max(1, (len + kUnit - 1) / kUnit - first);      // a sequence without keys still has rows to write
  };
  {
    const int per = (p.n_seq + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, p.n_seq), b1 = min(b0 + per, p.n_seq);
    unsigned sum = 0;
    bool bad = false;
    for (int b = b0; b < b1; ++b) {
      int r0, T_, len, first;
      bad |= look_at(b, r0, T_, len);
      const unsigned n = T_ > 0 ? (unsigned)row_tiles(T_, p.G, COLS) * p.heads * units_of(T_, len, first) : 0u;
      before[b + 1] = n;
      sum += n;
    }
    if (bad && blockIdx.x == 0) atomicExch(p.dev_err, kErrPage);
    unsigned incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += u;
    }
    if (lane == 31) shared_word[warp] = (int)incl;
    __syncthreads();
    unsigned run = incl - sum;
    for (int w = 0; w < warp; ++w) run += (unsigned)shared_word[w];
    for (int b = b0; b < b1; ++b) { run += before[b + 1]; before[b + 1] = run; }
    if (tid == 0) before[0] = 0;
    __syncthreads();
  }
  const int64_t U = before[p.n_seq], grid = min((int64_t)gridDim.x, U);                  // every CTA that takes part has a unit
  if ((int64_t)blockIdx.x >= grid) return;
  int64_t u = U * blockIdx.x / grid;
  const int64_t u_end = U * (blockIdx.x + 1) / grid;
  int b;
  {
    int lo = 0, hi = p.n_seq - 1;                          // the last sequence with before[b] <= u
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)before[mid] <= u) lo = mid; else hi = mid - 1;
    }
    b = lo;
  }

  int slot = 0;                              // ring state, of this warp
  uint32_t phases = 0;                       // bit s: parity of the next wait on stage s
  bool dead = false;
  uint8_t* my_ring = ring + warp * kStages * S::kStageBytes;
  uint64_t* my_full = full + warp * kStages;

  while (u < u_end) {
    while ((int64_t)before[b + 1] <= u) ++b;
    Segment sg;
    sg.b = b;
    look_at(b, sg.rows0, sg.T, sg.len);
    sg.n_units = units_of(sg.T, sg.len, sg.first_unit);
    const int in_seq = (int)(u - before[b]), triple = in_seq / sg.n_units;
    sg.tile = triple / p.heads;
    sg.head = triple - sg.tile * p.heads;
    sg.item0 = (int64_t)before[b] + (int64_t)triple * sg.n_units;
    const int from_unit = (int)(u - sg.item0), to_unit = (int)min((int64_t)sg.n_units, u_end - sg.item0);
    const int valid = min(COLS, sg.T * p.G - sg.tile * COLS);            // query rows of this tile
    u = sg.item0 + to_unit;

    // ---- queries: MMA operands, sums per group, each row scaled to [2^9, 2^10) --------------------------------------
    __syncthreads();                         // the previous segment's shared memory is free
    for (int c = warp; c < COLS; c += kWarps) {
      const int rho = sg.tile * COLS + c, row = rho / p.G, hq = rho - row * p.G;
      const T* qr = reinterpret_cast<const T*>(p.q) + (int64_t)(sg.rows0 + row) * p.q_stride + (int64_t)(sg.head * p.G + hq) * D;
      float v[NG], top = 0.f;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        v[i] = c < valid ? to_f32(qr[i * 32 + lane]) : 0.f;
        top = fmaxf(top, fabsf(v[i]));
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const int e = top > 0.f ? max((int)(__float_as_uint(top) >> 23) - 127, -117) : 9;   // 2^(9 - e) stays a float
      const float up = __uint_as_float((uint32_t)(min(127 + 9 - e, 253)) << 23), down = __uint_as_float((uint32_t)max(127 - 9 + e, 1) << 23);
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const float x = v[i] * up;
        float s = x;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        // feature lane of group i: tile lane / 16, k = lane % 16; B operand of lane (c % 8, k % 8 / 2), register k / 8
        const int tile = 2 * i + (lane >> 4), k = lane & 15;
        const float y = k >= 8 ? x * 0.0625f : x;
        const __half hi = __float2half_rn(y);
        const int word = ((tile * NT + (c >> 3)) * 32 + (c & 7) * 4 + ((k & 7) >> 1)) * (kSplit ? 4 : 2) + (k >> 3);
        __half* dst = reinterpret_cast<__half*>(qfrag + word) + (k & 1);
        dst[0] = hi;
        if (kSplit) dst[4] = __float2half_rn(y - __half2float(hi));
        if (lane == 0) {
          const __half sh = __float2half_rn(s);
          __half* qs = reinterpret_cast<__half*>(qsum + (c >> 3) * 32 + (c & 7) * 4 + (i >> 1));
          qs[i & 1] = sh;
          qs[2 + (i & 1)] = __float2half_rn(s - __half2float(sh));
        }
      }
      if (NG < 8 && lane < 8 && lane >= NG) {                            // groups that are not there
        __half* qs = reinterpret_cast<__half*>(qsum + (c >> 3) * 32 + (c & 7) * 4 + (lane >> 1));
        qs[lane & 1] = __ushort_as_half(0);
        qs[2 + (lane & 1)] = __ushort_as_half(0);
      }
      if (lane == 0) {
        const int position = sg.len - sg.T + row;
        col_scale[c] = p.scale * (kSplit ? 1.f : 16777216.f) * down;
        col_end[c] = c < valid ? max(0, position + 1) : 0;
        col_from[c] = p.window > 0 ? max(0, position - p.window + 1) : 0;
      }
    }
    __syncthreads();
    // keys that some row sees, keys that all rows see: the rows' positions ascend
    const int lowest = col_from[0], highest = col_end[valid - 1], all_from = col_from[valid - 1], all_to = col_end[0];
    float cs[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) { cs[nt][0] = col_scale[nt * 8 + 2 * t]; cs[nt][1] = col_scale[nt * 8 + 2 * t + 1]; }

    // ---- ring: stage j holds this warp's two blocks of unit from_unit + j --------------------------------------------
    const int n_stages = to_unit - from_unit;
    const int block0 = (sg.first_unit + from_unit) * (kUnit / 16) + 2 * warp;
    const int* row_table = p.table + (int64_t)sg.b * p.max_pages;
    auto fetch_pages = [&](int batch) {                    // lane: block lane % 2 of stage 16 batch + lane / 2; -1: not to be read
      const int j = batch * 16 + (lane >> 1), key = (block0 + j * (kUnit / 16) + (lane & 1)) * 16;
      if (j >= n_stages || key >= highest || key + 16 <= lowest) return -1;
      const int page = row_table[key >> p.shift];
      if ((unsigned)page < (unsigned)p.n_pages) return page;
      atomicExch(p.dev_err, kErrPage);
      return -1;
    };
    int ids = fetch_pages(0), ids_next = fetch_pages(1);
    uint32_t loaded = 0;                                   // two bits per stage of the ring
    auto issue = [&](int j, int s) {
      if (j > 0 && (j & 15) == 0) {
        ids = ids_next;
        ids_next = fetch_pages((j >> 4) + 1);
      }
      const int p0 = __shfl_sync(0xffffffffu, ids, (j & 15) * 2), p1 = __shfl_sync(0xffffffffu, ids, (j & 15) * 2 + 1);
      const uint32_t bits = (p0 >= 0 ? 1u : 0u) | (p1 >= 0 ? 2u : 0u);
      loaded = (loaded & ~(3u << (2 * s))) | bits << (2 * s);
      if (bits && lane == 0) {
        const int key = (block0 + j * (kUnit / 16)) * 16, inside = (key & ((1 << p.shift) - 1)) >> 4, per_page = 1 << (p.shift - 4);
        uint8_t* dst = my_ring + s * S::kStageBytes;
        tc::mbar_expect_tx(my_full + s, (bits == 3 ? 2 : 1) * 640 * NG);
        if (bits == 3 && per_page > 1) {                   // neighbours in one page
          tc::bulk_g2s(dst, p.pages + (((int64_t)p0 * p.heads + sg.head) * per_page + inside) * (640 * NG), 2 * 640 * NG, my_full + s);
        } else {
          if (bits & 1) tc::bulk_g2s(dst, p.pages + (((int64_t)p0 * p.heads + sg.head) * per_page + inside) * (640 * NG), 640 * NG, my_full + s);
          if (bits & 2)
            tc::bulk_g2s(dst + 640 * NG, p.pages + (((int64_t)p1 * p.heads + sg.head) * per_page + ((inside + 1) & (per_page - 1))) * (640 * NG), 640 * NG, my_full + s);
        }
      }
    };
    slot = 0;
#pragma unroll
    for (int s = 0; s < kStages; ++s)
      if (s < n_stages) issue(s, s);

    // ---- one pass over the keys ----------------------------------------------------------------------------------------
    float m[NT][2], l[NT][2], o[2 * NG][NT][4], om[NT][4];
    int r = 0;                               // values' scales are taken times 2^-r
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -CUDART_INF_F;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) om[nt][k] = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][nt][k] = 0.f;
    }
    for (int j = 0; j < n_stages; ++j) {
      const uint32_t bits = loaded >> (2 * slot) & 3u;
      if (bits) {
        tc::mbar_wait(my_full + slot, phases >> slot & 1u, dead, p.dev_err);
        phases ^= 1u << slot;
      }
      const int key0 = (block0 + j * (kUnit / 16)) * 16;
      const bool whole = bits == 3u && key0 >= all_from && key0 + 32 <= all_to;
      const uint8_t* stage = my_ring + slot * S::kStageBytes;
      auto work = [&](auto masked_) {
        constexpr bool kMasked = decltype(masked_)::value;
#pragma unroll
        for (int k0 = 0; k0 < 2; k0 += BK) {
          if (kMasked && BK == 1 && !(bits >> k0 & 1)) continue;
          float s[BK][NT][4];
          // minima: one MMA whose k slots are the groups, sums of q as hi (k < 8) and lo
#pragma unroll
          for (int kb = 0; kb < BK; ++kb) {
            const uint32_t* minima = reinterpret_cast<const uint32_t*>(stage + (k0 + kb) * 640 * NG + 544 * NG);
            uint32_t x = 0, y = 0;
            if (2 * t < NG) x = minima[2 * t * 8 + g];
            if (2 * t + 1 < NG) y = minima[(2 * t + 1) * 8 + g];
            const uint32_t a0 = __byte_perm(x, y, 0x5410), a1 = __byte_perm(x, y, 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint2 qs = qsum[nt * 32 + lane];
              s[kb][nt][0] = s[kb][nt][1] = s[kb][nt][2] = s[kb][nt][3] = 0.f;
              mma_half(s[kb][nt], a0, a1, a0, a1, qs.x, qs.y);
              if (!kSplit)
#pragma unroll
                for (int k = 0; k < 4; ++k) s[kb][nt][k] *= 5.9604644775390625e-8f;        // 2^-24, as the numbers
            }
          }
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            float acc[BK][NT][4];
#pragma unroll
            for (int kb = 0; kb < BK; ++kb)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) acc[kb][nt][0] = acc[kb][nt][1] = acc[kb][nt][2] = acc[kb][nt][3] = 0.f;
            uint2 w[BK];
#pragma unroll
            for (int kb = 0; kb < BK; ++kb) w[kb] = *reinterpret_cast<const uint2*>(stage + (k0 + kb) * 640 * NG + gr * 256 + lane * 8);
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
              for (int nt = 0; nt < NT; ++nt) {
                if (kSplit) {
                  const uint4 q = *reinterpret_cast<const uint4*>(qfrag + (((2 * gr + tile) * NT + nt) * 32 + lane) * 4);
#pragma unroll
                  for (int kb = 0; kb < BK; ++kb) mma_split(acc[kb][nt], a[kb][0], a[kb][1], a[kb][2], a[kb][3], q.x, q.y, q.z, q.w);
                } else {
                  const uint2 q = *reinterpret_cast<const uint2*>(qfrag + (((2 * gr + tile) * NT + nt) * 32 + lane) * 2);
#pragma unroll
                  for (int kb = 0; kb < BK; ++kb) mma_half(acc[kb][nt], a[kb][0], a[kb][1], a[kb][2], a[kb][3], q.x, q.y);
                }
              }
            }
#pragma unroll
            for (int kb = 0; kb < BK; ++kb) {
              const float2 sc = __half22float2(as_half2(reinterpret_cast<const uint32_t*>(stage + (k0 + kb) * 640 * NG + 512 * NG)[gr * 8 + g]));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                s[kb][nt][0] = fmaf(sc.x, acc[kb][nt][0], s[kb][nt][0]);
                s[kb][nt][1] = fmaf(sc.x, acc[kb][nt][1], s[kb][nt][1]);
                s[kb][nt][2] = fmaf(sc.y, acc[kb][nt][2], s[kb][nt][2]);
                s[kb][nt][3] = fmaf(sc.y, acc[kb][nt][3], s[kb][nt][3]);
              }
            }
          }
          // scores in units of log2; the maximum is raised only when it lags by more than 2^8, so most blocks need no exchange between lanes
          float top[NT][2];
          bool raise = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int kb = 0; kb < BK; ++kb)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                s[kb][nt][k] *= cs[nt][k & 1];
                if (kMasked) {
                  const int key = key0 + (k0 + kb) * 16 + g + (k >= 2 ? 8 : 0), c = nt * 8 + 2 * t + (k & 1);
                  if (key >= col_end[c] || key < col_from[c] || !(bits >> (k0 + kb) & 1)) s[kb][nt][k] = -CUDART_INF_F;
                }
              }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              top[nt][k] = fmaxf(s[0][nt][k], s[0][nt][k + 2]);
              if (BK == 2) top[nt][k] = fmaxf(top[nt][k], fmaxf(s[BK - 1][nt][k], s[BK - 1][nt][k + 2]));
              raise |= top[nt][k] > m[nt][k] + 8.f;
            }
          }
          // values' scales, in the order of the weights' operand
          uint2 vs[BK][NG];
          __half2 most = __float2half2_rn(0.f);
#pragma unroll
          for (int kb = 0; kb < BK; ++kb)
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              vs[kb][gr] = *reinterpret_cast<const uint2*>(stage + (k0 + kb) * 640 * NG + 576 * NG + gr * 32 + t * 8);
              if (kMasked && !(bits >> (k0 + kb) & 1)) vs[kb][gr] = make_uint2(0, 0);
              most = __hmax2(most, __hmax2(as_half2(vs[kb][gr].x), as_half2(vs[kb][gr].y)));
            }
          const float most_s = fmaxf(__low2float(most), __high2float(most));
          const float limit = __uint_as_float((uint32_t)(127 + r) << 23);                  // 2^r: weights up to 2^15 times scales up to 1 stay halves
          if (__any_sync(0xffffffffu, raise || most_s > limit)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                float x = top[nt][k];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                if (x > m[nt][k]) {
                  const float fade = exp2f(m[nt][k] - x);
                  m[nt][k] = x;
                  l[nt][k] *= fade;
                  om[nt][k] *= fade;
                  om[nt][k + 2] *= fade;
#pragma unroll
                  for (int i = 0; i < 2 * NG; ++i) { o[i][nt][k] *= fade; o[i][nt][k + 2] *= fade; }
                }
              }
            float x = most_s;
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
            if (x > limit && x <= 65504.f) {
              const int rn = (int)(__float_as_uint(x) >> 23) - 126;                        // x < 2^rn
              const float fade = __uint_as_float((uint32_t)(127 + r - rn) << 23);
              r = rn;
#pragma unroll
              for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int k = 0; k < 4; ++k) o[i][nt][k] *= fade;
            }
          }
          // weights: 2^7 exp2(score - m) as halves (float32: two of them), from accumulators to B operands
          uint32_t pb[BK][NT][kSplit ? 4 : 2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float m0 = (m[nt][0] == -CUDART_INF_F ? 0.f : m[nt][0]) - kPScale, m1 = (m[nt][1] == -CUDART_INF_F ? 0.f : m[nt][1]) - kPScale;
#pragma unroll
            for (int kb = 0; kb < BK; ++kb) {
              float e[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) e[k] = exp2f(s[kb][nt][k] - (k & 1 ? m1 : m0));
              l[nt][0] += e[0] + e[2];
              l[nt][1] += e[1] + e[3];
              const uint32_t h0 = pack(e[0], e[1]), h1 = pack(e[2], e[3]);
              pb[kb][nt][0] = transposed(h0);
              pb[kb][nt][1] = transposed(h1);
              if (kSplit) {
                const float2 f0 = __half22float2(as_half2(h0)), f1 = __half22float2(as_half2(h1));
                pb[kb][nt][kSplit ? 2 : 0] = transposed(pack(e[0] - f0.x, e[1] - f0.y));
                pb[kb][nt][kSplit ? 3 : 0] = transposed(pack(e[2] - f1.x, e[3] - f1.y));
              }
            }
          }
          // values: minima (rows = groups), then numbers times scales
#pragma unroll
          for (int kb = 0; kb < BK; ++kb) {
            uint2 mn = make_uint2(0, 0);
            if (g < NG) mn = *reinterpret_cast<const uint2*>(stage + (k0 + kb) * 640 * NG + 608 * NG + g * 32 + t * 8);
            if (kMasked) {
              // a key without a page has no minima; a minimum that is no number counts through its scale, and so only for the rows that see its key
              if (!(bits >> (k0 + kb) & 1)) mn = make_uint2(0, 0);
              const uint32_t ox = __vcmpgtu2(mn.x & 0x7fff7fffu, 0x7bff7bffu), oy = __vcmpgtu2(mn.y & 0x7fff7fffu, 0x7bff7bffu);
              mn.x &= ~ox;
              mn.y &= ~oy;
#pragma unroll
              for (int gr = 0; gr < NG; ++gr) {
                vs[kb][gr].x |= __shfl_sync(0xffffffffu, ox, gr * 4 + t) & 0x7fff7fffu;
                vs[kb][gr].y |= __shfl_sync(0xffffffffu, oy, gr * 4 + t) & 0x7fff7fffu;
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (kSplit) mma_split(om[nt], mn.x, 0u, mn.y, 0u, pb[kb][nt][0], pb[kb][nt][1], pb[kb][nt][kSplit ? 2 : 0], pb[kb][nt][kSplit ? 3 : 0]);
              else mma_half(om[nt], mn.x, 0u, mn.y, 0u, pb[kb][nt][0], pb[kb][nt][1]);
            }
            const float down_r = __uint_as_float((uint32_t)(127 - r) << 23);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
              const uint2 w = *reinterpret_cast<const uint2*>(stage + (k0 + kb) * 640 * NG + 256 * NG + gr * 256 + lane * 8);
              uint32_t wb[NT][kSplit ? 4 : 2];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if (kSplit) {
                  const float2 sx = __half22float2(as_half2(vs[kb][gr].x)), sy = __half22float2(as_half2(vs[kb][gr].y));
#pragma unroll
                  for (int i = 0; i < 2; ++i) {
                    const float2 hi = __half22float2(as_half2(pb[kb][nt][i])), lo = __half22float2(as_half2(pb[kb][nt][kSplit ? 2 + i : 0]));
                    const float2 sc = i ? sy : sx;
                    float x = (hi.x + lo.x) * (sc.x * down_r), y = (hi.y + lo.y) * (sc.y * down_r);
                    if (kMasked) {
                      if (hi.x == 0.f) x = 0.f;
                      if (hi.y == 0.f) y = 0.f;
                    }
                    wb[nt][i] = pack(x, y);
                    const float2 f = __half22float2(as_half2(wb[nt][i]));
                    wb[nt][kSplit ? 2 + i : 0] = pack(x - f.x, y - f.y);
                  }
                } else {
                  __half2 sx = as_half2(vs[kb][gr].x), sy = as_half2(vs[kb][gr].y);
                  if (r) {
                    const __half2 dr = __float2half2_rn(down_r);
                    sx = __hmul2(sx, dr);
                    sy = __hmul2(sy, dr);
                  }
                  wb[nt][0] = as_u32(__hmul2(as_half2(pb[kb][nt][0]), sx));
                  wb[nt][1] = as_u32(__hmul2(as_half2(pb[kb][nt][1]), sy));
                  if (kMasked) {
                    wb[nt][0] &= __vcmpne2(pb[kb][nt][0] & 0x7fff7fffu, 0u);
                    wb[nt][1] &= __vcmpne2(pb[kb][nt][1] & 0x7fff7fffu, 0u);
                  }
                }
              }
#pragma unroll
              for (int tile = 0; tile < 2; ++tile) {
                const uint32_t x = tile ? w.y : w.x;
                const uint32_t a0 = numbers<kSplit>(x, 0x000f000fu), a1 = numbers<kSplit>(x, 0x00f000f0u), a2 = numbers<kSplit>(x >> 8, 0x000f000fu),
                               a3 = numbers<kSplit>(x >> 8, 0x00f000f0u);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  if (kSplit) mma_split(o[2 * gr + tile][nt], a0, a1, a2, a3, wb[nt][0], wb[nt][1], wb[nt][kSplit ? 2 : 0], wb[nt][kSplit ? 3 : 0]);
                  else mma_half(o[2 * gr + tile][nt], a0, a1, a2, a3, wb[nt][0], wb[nt][1]);
                }
              }
            }
          }
        }
      };
      if (whole) work(std::false_type());
      else if (bits) work(std::true_type());
      __syncwarp();
      if (j + kStages < n_stages) issue(j + kStages, slot);
      slot = slot + 1 == kStages ? 0 : slot + 1;
    }

    // ---- the warps' sums become one ------------------------------------------------------------------------------------
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
    __syncthreads();                         // all warps are through with the ring
    float fade[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float top = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_m[w * COLS + nt * 8 + 2 * t + k]);
        fade[nt][k] = m[nt][k] == -CUDART_INF_F ? (l[nt][k] != l[nt][k] ? 1.f : 0.f) : exp2f(m[nt][k] - top);
      }
    const float up_r = __uint_as_float((uint32_t)(127 + (kSplit ? -4 : 20) + r) << 23);  // of 16 n; n takes another 16
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float b0 = __shfl_sync(0xffffffffu, om[nt][0], (i >> 1) * 4 + t), b1 = __shfl_sync(0xffffffffu, om[nt][1], (i >> 1) * 4 + t);
        float* dst = merge + (warp * COLS + nt * 8 + 2 * t) * S::kPitch + 16 * i + g;
        dst[0] = fmaf(o[i][nt][0], up_r * 16.f, b0) * fade[nt][0];
        dst[S::kPitch] = fmaf(o[i][nt][1], up_r * 16.f, b1) * fade[nt][1];
        dst[8] = fmaf(o[i][nt][2], up_r, b0) * fade[nt][0];
        dst[S::kPitch + 8] = fmaf(o[i][nt][3], up_r, b1) * fade[nt][1];
      }
    __syncthreads();
    const bool alone = from_unit == 0 && to_unit == sg.n_units;
    const int part = (int)blockIdx.x * 2 + (from_unit == 0 ? 1 : 0);
    auto put = [&](int c, int d, float4 v, float L) {
      const float inv = L > 0.f || L != L ? 1.f / L : 0.f;             // a row that sees no key is 0
      const int rho = sg.tile * COLS + c, row = rho / p.G, hq = rho - row * p.G;
      T* out = reinterpret_cast<T*>(p.out) + (int64_t)(sg.rows0 + row) * p.out_stride + (int64_t)(sg.head * p.G + hq) * D + d;
      if (kSplit) {
        *reinterpret_cast<float4*>(out) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      } else {
        __nv_bfloat162 x = __floats2bfloat162_rn(v.x * inv, v.y * inv), y = __floats2bfloat162_rn(v.z * inv, v.w * inv);
        *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<uint32_t*>(&x), *reinterpret_cast<uint32_t*>(&y));
      }
    };
    for (int i = tid; i < valid * (D / 4); i += kThreads) {
      const int c = i / (D / 4), d = (i - c * (D / 4)) * 4;
      float top = -CUDART_INF_F, L = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_m[w * COLS + c]);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = warp_m[w * COLS + c], lw = warp_l[w * COLS + c];
        L += mw == -CUDART_INF_F ? (lw != lw ? lw : 0.f) : lw * exp2f(mw - top);
        const float4 x = *reinterpret_cast<const float4*>(merge + (w * COLS + c) * S::kPitch + d);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
      }
      if (alone) {
        put(c, d, v, L);
      } else {
        __stcg(reinterpret_cast<float4*>(p.part_o + ((int64_t)part * COLS + c) * D + d), v);
        if (d == 0) __stcg(p.part_ml + part * COLS + c, make_float2(top, L));
      }
    }
    if (!alone) {
      // the last of the CTAs that share the triple joins what all of them left
      const int64_t last_unit = sg.item0 + sg.n_units - 1;
      const int ca = (int)(((sg.item0 + 1) * grid - 1) / U), cb = (int)(((last_unit + 1) * grid - 1) / U), n = cb - ca + 1;
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const bool last = atomicAdd(p.counters + ca, 1u) == (unsigned)n - 1u;
        if (last) p.counters[ca] = 0u;
        shared_word[0] = last;
      }
      __syncthreads();
      if (shared_word[0]) {
        __threadfence();
        for (int i = tid; i < valid * (D / 4); i += kThreads) {
          const int c = i / (D / 4), d = (i - c * (D / 4)) * 4;
          float top = -CUDART_INF_F;
#pragma unroll 8
          for (int k = 0; k < n; ++k) top = fmaxf(top, __ldcg(&p.part_ml[((ca + k) * 2 + (k == 0)) * COLS + c].x));
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          float L = 0.f;
#pragma unroll 8
          for (int k = 0; k < n; ++k) {
            const int64_t from = (int64_t)((ca + k) * 2 + (k == 0)) * COLS + c;
            const float2 ml = __ldcg(p.part_ml + from);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part_o + from * D + d));
            const float f = ml.x == -CUDART_INF_F ? (ml.y != ml.y ? 1.f : 0.f) : exp2f(ml.x - top);
            L = fmaf(ml.y, f, L);
            v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
          }
          put(c, d, v, L);
        }
      }
    }
    tc::fence_async_smem();                  // the next segment's copies overwrite what was joined here
  }
}

template <typename T, int NG, int NT> int32_t configure_one(Variant* v) {
  using S = Shape<T, NG, NT>;
  v->kernel = attention_kernel<T, NG, NT>;
  v->smem = S::kFixed;
  const int most = S::kFixed + (kMaxSeqs + 1) * 4;
  LMB_CUDA(cudaFuncSetAttribute(v->kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  LMB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&v->ctas_per_sm, v->kernel, kThreads, (size_t)S::kFixed + 260 * 4));
  return LMB200_OK;
}

}  // namespace kv4
}  // namespace lmb
