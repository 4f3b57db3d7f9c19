// Block tables on the GPU (lmb200_kv_reserve, lmb200_kv_shrink) and the 4-bit cache's store and load (lmb200_kv4_append, lmb200_kv4_read).
#include <cooperative_groups.h>
#include <limits.h>

#include <algorithm>

#include "kv4.cuh"
#include "pdl.cuh"

namespace lmb {
namespace {

constexpr int kTableThreads = 1024;
int g_most_ctas = 8;                         // of reserve_kernel's cluster
constexpr int kMaxSeqs = 8192;               // three words of shared memory each

struct TableParams {
  int n_seq, shift, max_pages, n_pages, rows;
  const int *lens, *change, *n_free;
  int *table, *free_list;                    // reserve writes the table, shrink the free list
  int *lens_out, *n_free_out, *cu_rows, *slots, *status;
  int* dev_arg;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_sync_all() {
  cluster_arrive();
  cluster_wait();
}
__device__ __forceinline__ int cluster_rank() { int r; asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r)); return r; }
__device__ __forceinline__ int cluster_size() { int r; asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(r)); return r; }

// Exclusive sums over the block of two counts per thread, and their totals.
__device__ __forceinline__ void scan2(long long a, long long b, long long& ea, long long& eb, long long& ta, long long& tb) {
  __shared__ long long sa[32], sb[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long ia = a, ib = b;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long ua = __shfl_up_sync(0xffffffffu, ia, off), ub = __shfl_up_sync(0xffffffffu, ib, off);
    if (lane >= off) { ia += ua; ib += ub; }
  }
  if (lane == 31) { sa[warp] = ia; sb[warp] = ib; }
  __syncthreads();
  if (warp == 0) {
    long long va = sa[lane], vb = sb[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long ua = __shfl_up_sync(0xffffffffu, va, off), ub = __shfl_up_sync(0xffffffffu, vb, off);
      if (lane >= off) { va += ua; vb += ub; }
    }
    sa[lane] = va;
    sb[lane] = vb;
  }
  __syncthreads();
  ea = ia - a + (warp ? sa[warp - 1] : 0);
  eb = ib - b + (warp ? sb[warp - 1] : 0);
  ta = sa[31];
  tb = sb[31];
}

// the last index in [lo, hi] with at[index] <= x (at ascending, at[lo] <= x)
__device__ __forceinline__ int last_at_most(const int* at, int lo, int hi, int x) {
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    const bool up = at[mid] <= x;
    lo = up ? mid : lo;
    hi = up ? hi : mid - 1;
  }
  return lo;
}

// One cluster.  Every CTA reads all lengths and forms the same sums (a thread takes neighbouring sequences); behind the cluster's barrier, when
// nobody reads them any more, the outputs, which may be the inputs' arrays, are written.  Rows and pages are dealt out to all warps in groups
// of 32 neighbours, whose sequence is found by bisection: what it takes is the chain of those searches and loads, so it wants many warps.  77000 rows of 2048 sequences on 1, 2, 4, 8, 16
// CTAs: 88, 48, 28, 17, 13 us; 26000 rows of 256: 19, 13, 9.6, 6.9, 6.8.
__global__ void __launch_bounds__(kTableThreads) reserve_kernel(const TableParams p) {
  extern __shared__ int sm[];
  int* len = sm;
  int* row0 = len + p.n_seq;                 // first row of a sequence
  int* page0 = row0 + p.n_seq;               // its first new page
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, per = (p.n_seq + kTableThreads - 1) / kTableThreads;
  const int first = min(tid * per, p.n_seq), last = min(first + per, p.n_seq);
  const int free_now = *p.n_free, size1 = (1 << p.shift) - 1;
  long long rows = 0, pages = 0;
  int bad = 0;
  for (int b = first; b < last; ++b) {
    const long long l = p.lens[b], a = p.change[b];
    if (l < 0 || a < 0) { bad |= 8; continue; }
    if (((l + a + size1) >> p.shift) > p.max_pages) bad |= 4;
    rows += a;
    pages += ((l + a + size1) >> p.shift) - ((l + size1) >> p.shift);
  }
  long long er, ep, tr, tp;
  scan2(rows, pages, er, ep, tr, tp);
  bad = __syncthreads_or(bad & 8 ? 1 : 0) * 8 | __syncthreads_or(bad & 4 ? 1 : 0) * 4;
  if (tr > p.rows) bad |= 2;
  if (free_now < 0 || free_now > p.n_pages) bad |= 8;
  else if (tp > free_now) bad |= 1;
  if (!bad)
    for (int b = first; b < last; ++b) {
      const long long l = p.lens[b], a = p.change[b];
      len[b] = (int)l;
      row0[b] = (int)er;
      page0[b] = (int)ep;
      er += a;
      ep += ((l + a + size1) >> p.shift) - ((l + size1) >> p.shift);
    }
  __syncthreads();
  const int n_rows = bad ? 0 : (int)tr, n_new = bad ? 0 : (int)tp;
  const int lane = tid & 31, warps = kTableThreads / 32 * cluster_size(), warp = cluster_rank() * (kTableThreads / 32) + (tid >> 5);
  // slots: the token's page is a new one, or the last that its sequence holds.  (`table` is read at places that this call does not write.)
  // Four groups of 32 at a time, so that their searches and loads overlap.
  constexpr int kTogether = 4;
  for (int r00 = warp * 32; r00 < p.rows; r00 += kTogether * warps * 32) {
    int lo[kTogether], hi[kTogether], seq[kTogether], page[kTogether], pos[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {    // the sequences of a group's first and last row, between which its rows' lie
      const int r0 = min(r00 + i * warps * 32, max(0, n_rows - 1));
      lo[i] = last_at_most(row0, 0, p.n_seq - 1, lane == 0 ? r0 : min(r0 + 31, max(0, n_rows - 1)));       // lane 0: first, the others: last
      hi[i] = __shfl_sync(0xffffffffu, lo[i], 1);
      lo[i] = __shfl_sync(0xffffffffu, lo[i], 0);
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int r = r00 + i * warps * 32 + lane;
      page[i] = -1;
      if (r < n_rows) {
        const int b = lo[i] == hi[i] ? lo[i] : last_at_most(row0, lo[i], hi[i], r);
        pos[i] = len[b] + (r - row0[b]);
        const int j = (pos[i] >> p.shift) - ((len[b] + size1) >> p.shift);
        page[i] = j >= 0 ? p.free_list[free_now - 1 - (page0[b] + j)] : p.table[(int64_t)b * p.max_pages + (pos[i] >> p.shift)];
      }
      seq[i] = r;
    }
    bool lost = false;                       // pages that are none of the cache's, of the table or the free list: their tokens have no slot
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const bool there = (unsigned)page[i] < (unsigned)p.n_pages;
      if (seq[i] < p.rows) p.slots[seq[i]] = there ? (page[i] << p.shift) + (pos[i] & size1) : -1;
      lost |= seq[i] < n_rows && !there;
    }
    if (lost) atomicExch(p.dev_arg, kv4::kErrPage);
  }
  for (int k0 = warp * 32; k0 < n_new; k0 += kTogether * warps * 32) {
    int id[kTogether];
    int64_t to[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int k = k0 + i * warps * 32 + lane;
      to[i] = -1;
      if (k < n_new) {
        const int b = last_at_most(page0, 0, p.n_seq - 1, k);
        to[i] = (int64_t)b * p.max_pages + ((len[b] + size1) >> p.shift) + (k - page0[b]);
        id[i] = p.free_list[free_now - 1 - k];
      }
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i)
      if (to[i] >= 0) p.table[to[i]] = id[i];
  }
  if (cluster_size() > 1) cluster_sync_all(); else __syncthreads();   // lens and n_free are read by no one any more
  if (cluster_rank() != 0) return;
  for (int b = tid; b < p.n_seq; b += kTableThreads) {
    const int up = b + 1 < p.n_seq ? row0[b + 1] : n_rows;
    if (!bad) p.lens_out[b] = len[b] + up - row0[b];
    else if (p.lens_out != p.lens) p.lens_out[b] = p.lens[b];
    p.cu_rows[b + 1] = bad ? 0 : up;
  }
  if (tid == 0) {
    p.cu_rows[0] = 0;
    *p.n_free_out = free_now - n_new;
    *p.status = bad;
  }
}

// The way back.  A sequence's pages go back behind those of the sequences after it, its last page first: the reverse of taking them.  All of them are looked at before any is
// written, so a table that names a page outside the cache leaves the list as it was.
__global__ void __launch_bounds__(kTableThreads) shrink_kernel(const TableParams p) {
  extern __shared__ int sm[];
  int* len = sm;
  int* left = len + p.n_seq;
  int* page0 = left + p.n_seq;               // pages that the sequences before it give back
  __shared__ int lost;                       // some CTA of the cluster found a page outside the cache
  if (threadIdx.x == 0) lost = 0;
  if (cluster_size() > 1) cluster_arrive();  // (waited for before anyone writes into another's `lost`)
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, per = (p.n_seq + kTableThreads - 1) / kTableThreads;
  const int first = min(tid * per, p.n_seq), last = min(first + per, p.n_seq);
  const int free_now = *p.n_free, size1 = (1 << p.shift) - 1;
  long long pages = 0;
  int bad = 0;
  for (int b = first; b < last; ++b) {
    const long long l = p.lens[b];
    const long long to = max(0ll, l - max(p.change[b], 0));
    if (l < 0 || ((l + size1) >> p.shift) > p.max_pages) { bad = 1; continue; }
    len[b] = (int)l;
    left[b] = (int)to;
    pages += ((l + size1) >> p.shift) - ((to + size1) >> p.shift);
  }
  long long ep, ez, tp, tz;
  scan2(pages, 0, ep, ez, tp, tz);
  bad = __syncthreads_or(bad);
  if (free_now < 0 || free_now + tp > p.n_pages) bad = 1;
  if (!bad)
    for (int b = first; b < last; ++b) {
      page0[b] = (int)ep;
      ep += ((len[b] + size1) >> p.shift) - ((left[b] + size1) >> p.shift);
    }
  __syncthreads();
  int n_back = bad ? 0 : (int)tp;
  const int stride = kTableThreads * cluster_size(), k0 = cluster_rank() * kTableThreads + tid;
  auto page_of = [&](int k) {
    const int b = last_at_most(page0, 0, p.n_seq - 1, k);
    return p.table[(int64_t)b * p.max_pages + ((left[b] + size1) >> p.shift) + (k - page0[b])];
  };
  int mine = 0;                              // page k0; mostly the only one
  bool outside = false;
  for (int k = k0; k < n_back; k += stride) {
    const int page = page_of(k);
    outside |= (unsigned)page >= (unsigned)p.n_pages;
    if (k == k0) mine = page;
  }
  outside = __syncthreads_or(outside);
  if (cluster_size() > 1) {
    cluster_wait();
    if (outside && tid < cluster_size()) *cooperative_groups::this_cluster().map_shared_rank(&lost, tid) = 1;
    cluster_sync_all();                      // lens and n_free are read by no one any more
    outside = lost;
  }
  if (outside) { bad = 1; n_back = 0; }
  for (int k = k0; k < n_back; k += stride) p.free_list[free_now + (n_back - 1 - k)] = k == k0 ? mine : page_of(k);      // k counts upwards over sequences and places; the list's top is the first
  if (cluster_rank() != 0) return;
  for (int b = tid; b < p.n_seq; b += kTableThreads) {
    if (!bad) p.lens_out[b] = left[b];
    else if (p.lens_out != p.lens) p.lens_out[b] = p.lens[b];
  }
  if (tid == 0) {
    *p.n_free_out = free_now + n_back;
    if (bad) atomicExch(p.dev_arg, kv4::kErrFree);
  }
}

struct StoreParams {
  void *k, *v;                               // append reads them, read writes them
  int64_t k_stride, v_stride;                // elements between rows
  int rows, heads, D, shift, n_pages;
  const int* slots;
  uint8_t* pages;
  int* dev_arg;
};

// The 32 features of one group of one row as a lane holds them.
template <typename T> struct Group;
template <> struct Group<float> {
  float4 v[8];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __ldcs(reinterpret_cast<const float4*>(p) + i);
  }
  __device__ __forceinline__ float at(int i) const { const float4& x = v[i >> 2]; return (i & 3) == 0 ? x.x : (i & 3) == 1 ? x.y : (i & 3) == 2 ? x.z : x.w; }
  // smallest and largest; NaN if there is one
  __device__ __forceinline__ void range(float& lo, float& hi) const {
    lo = hi = at(0);
#pragma unroll
    for (int i = 1; i < 32; ++i) {
      asm("min.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(at(i)));
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(at(i)));
    }
  }
  static constexpr int kParts = 8;           // of 16 bytes
  static __device__ __forceinline__ uint4 part(const float (&x)[32], int i) {
    return make_uint4(__float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]), __float_as_uint(x[4 * i + 2]), __float_as_uint(x[4 * i + 3]));
  }
};
template <> struct Group<__nv_bfloat16> {
  uint32_t w[16];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 x = __ldcs(reinterpret_cast<const uint4*>(p) + i);
      w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
    }
  }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
  __device__ __forceinline__ void range(float& lo, float& hi) const {
    uint32_t a = w[0], b = w[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) {
      asm("min.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(w[i]));
      asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(b) : "r"(w[i]));
    }
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(lo) : "f"(__uint_as_float(a << 16)), "f"(__uint_as_float(a & 0xffff0000u)));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(hi) : "f"(__uint_as_float(b << 16)), "f"(__uint_as_float(b & 0xffff0000u)));
  }
  static constexpr int kParts = 4;
  static __device__ __forceinline__ uint4 part(const float (&x)[32], int i) {
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[8 * i + 2 * k], x[8 * i + 2 * k + 1]);
      u[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

__device__ __forceinline__ uint64_t as_pair(float2 v) { return (uint64_t)__float_as_uint(v.y) << 32 | __float_as_uint(v.x); }
__device__ __forceinline__ float2 of_pair(uint64_t u) { return make_float2(__uint_as_float((uint32_t)u), __uint_as_float((uint32_t)(u >> 32))); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(as_pair(a)), "l"(as_pair(b)));
  return of_pair(d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(as_pair(a)), "l"(as_pair(b)), "l"(as_pair(c)));
  return of_pair(d);
}

// n of one value: rint of the float32 quotient, 0..15
__device__ __forceinline__ uint32_t level(float x, float m, float s) {
  return s > 0.f ? (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(x - m, s)), 0.f), 15.f) : 0u;
}

// A group's scale, minimum and levels, as the pairs (feature i % 16 < 8, the one 8 further) that share a byte: byte 8 (i / 16) + i % 8 of `pairs`.  A level is the rint of a
// float32 quotient; it is formed with the reciprocal, off by less than 1e-5, and by the quotient where that is near a half: for one value of 1500 in bf16, whose quotients are
// halves that often, so half of the warps have one.
template <typename T>
__device__ __forceinline__ void quantise(const Group<T>& x, const T* from, __half& s, __half& m, uint32_t (&pairs)[4]) {
  float lo, hi;
  x.range(lo, hi);
  m = __float2half_rn(lo);
  s = __float2half_rn(__fdiv_rn(hi - lo, 15.f));
  const float mf = __half2float(m), sf = __half2float(s);
  if (!(fabsf(mf) <= 65504.f) || !(sf <= 65504.f)) {        // a group without a 4-bit form reads back as NaN
    m = s = __ushort_as_half(0x7fff);
    pairs[0] = pairs[1] = pairs[2] = pairs[3] = 0;
    return;
  }
  const float inv = sf > 0.f ? __fdividef(1.f, 15.f * sf) : 0.f;
  constexpr float kInt = 12582912.f;         // 1.5 2^23: a small number added to it leaves its rint in the low bits
  uint32_t near_half = 0;                    // bit i: feature i
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t n[8];
#pragma unroll
    for (int k = 0; k < 8; k += 2) {         // two features an instruction where there is one for two
      const int f = (i >> 1) * 16 + (i & 1) * 4 + (k & 3) + (k >> 2) * 8;
      const float2 y = add2(make_float2(x.at(f), x.at(f + 1)), make_float2(-mf, -mf));
      const float2 q = make_float2(__saturatef(y.x * inv), __saturatef(y.y * inv));        // of 15 levels
      const float2 r = fma2(q, make_float2(15.f, 15.f), make_float2(kInt, kInt));
      const float2 off = fma2(q, make_float2(15.f, 15.f), fma2(r, make_float2(-1.f, -1.f), make_float2(kInt, kInt)));
      if (fabsf(off.x) > 0.49999f) near_half |= 1u << f;
      if (fabsf(off.y) > 0.49999f) near_half |= 2u << f;
      n[k] = __float_as_uint(r.x);
      n[k + 1] = __float_as_uint(r.y);
    }
    uint32_t byte[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) byte[k] = n[k + 4] * 16u + n[k];
    pairs[i] = __byte_perm(__byte_perm(byte[0], byte[1], 0x0040), __byte_perm(byte[2], byte[3], 0x0040), 0x5410);
  }
  while (near_half) {
    const int f = __ffs(near_half) - 1, shift = 8 * (f & 3) + (f & 8 ? 4 : 0), word = (f >> 4) * 2 + (f >> 2 & 1);
    near_half &= near_half - 1;
    const uint32_t n = level(to_f32(from[f]), mf, sf) << shift, keep = ~(15u << shift);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i == word) pairs[i] = (pairs[i] & keep) | n;
  }
}

__device__ __forceinline__ uint8_t* block_of(const StoreParams& p, int slot, int head) {
  return p.pages + (((int64_t)(slot >> p.shift) * p.heads + head) * (1 << (p.shift - 4)) + ((slot & ((1 << p.shift) - 1)) >> 4)) * kv4::block_bytes(p.D);
}

// Bytes bound it in principle (2 rows in, 0.31 of that out in bf16); what it takes is instructions, of which the exact levels are most, so it wants
// warps (32768 rows of 8 x 128, both sides, bf16: 53 us, 3.3 TB/s, with five blocks of 256 an SM, 68 with three; float32 71 us, 4.4 TB/s).
// A warp has 16 rows and two groups of a head's keys or values, a lane a row's 32 features, so the range needs no exchange.  Where 16 neighbouring rows go to the 16 places of a block, their
// bytes become words by exchange between lanes and the warp writes whole sectors; other rows write their bytes one by one.  Rows come in windows of 16; a block that begins in a
// window and goes on into the next belongs to the first.
template <typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 5 : 4) append_kernel(const StoreParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int NG = kv4::groups(p.D), lane = threadIdx.x, key = lane & 15, head = blockIdx.x, side = threadIdx.y & 1, g = (threadIdx.y >> 1) * 2 + (lane >> 4);
  const int64_t row0 = (((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * blockDim.z + threadIdx.z) * 16;
  if (row0 >= p.rows) return;
  // rows row0 - 16 .. row0 + 31: bit i of `follows`: row i + 1 goes to the place behind row i's
  auto slot_at = [&](int64_t r) { return r >= 0 && r < p.rows ? p.slots[r] : -1; };
  const int a = slot_at(row0 - 16 + lane), b = slot_at(row0 + 16 + key);
  const int a_next = __shfl_down_sync(0xffffffffu, a, 1), first_b = __shfl_sync(0xffffffffu, b, 0);
  const int b_next = __shfl_down_sync(0xffffffffu, b, 1);
  const int places = p.n_pages << p.shift;
  const uint64_t follows = (uint64_t)__ballot_sync(0xffffffffu, a >= 0 && (lane == 31 ? first_b : a_next) == a + 1) |
                           (uint64_t)(__ballot_sync(0xffffffffu, lane < 15 && b >= 0 && b_next == b + 1) & 0x7fffu) << 32;
  const uint32_t begins = __ballot_sync(0xffffffffu, a >= 0 && (a & 15) == 0 && a < places);
  uint64_t run = follows;                    // bit i: rows i .. i + 15 follow one another
  run &= run >> 1;
  run &= run >> 2;
  run &= run >> 4;
  run &= run >> 7;
  const uint32_t whole = begins & (uint32_t)run;
  const int mine = whole >> 16 ? __ffs(whole >> 16) - 1 : 16;            // first row of this window whose block is whole
  const int others = whole & 0xffffu ? __ffs(whole & 0xffffu) - 1 : 0;   // rows below it belong to the last window's block
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const bool block = pass == 0;
    const int64_t row = row0 + (block ? mine + key : key);
    if (block && mine == 16) continue;
    const bool live = g < NG && (block || (key >= others && key < mine && slot_at(row) >= 0));
    if (!block && !__any_sync(0xffffffffu, live)) continue;
    const int slot = slot_at(row);
    __half s = __ushort_as_half(0), m = s;
    uint32_t pairs[4] = {0, 0, 0, 0};
    if (live) {
      const T* from = reinterpret_cast<const T*>(side ? p.v : p.k) + row * (side ? p.v_stride : p.k_stride) + head * p.D + g * 32;
      Group<T> x;
      x.load(from);
      quantise<T>(x, from, s, m, pairs);
    }
    if (block) {
      uint8_t* out = block_of(p, slot, head);
      uint32_t w[4];
      if (side == 0) {
        // lanes key and key + 8 (xor 8) have the bytes of the same words: words t, tile of row key % 8.  The lower lane makes those of t = 0, 1, the other one t = 2, 3
        const bool up = key >= 8;
        // bytes (tile, 2t + e): register 2 tile + t / 2
        const uint32_t give0 = up ? pairs[0] : pairs[1], give1 = up ? pairs[2] : pairs[3];
        const uint32_t got0 = __shfl_xor_sync(0xffffffffu, give0, 8), got1 = __shfl_xor_sync(0xffffffffu, give1, 8);
        const uint32_t keep0 = up ? pairs[1] : pairs[0], keep1 = up ? pairs[3] : pairs[2];
        const uint32_t l0 = up ? got0 : keep0, h0 = up ? keep0 : got0, l1 = up ? got1 : keep1, h1 = up ? keep1 : got1;
        w[0] = __byte_perm(l0, h0, 0x5140);              // t even, tile 0: e = 0 of both keys, e = 1 of both
        w[1] = __byte_perm(l1, h1, 0x5140);              // tile 1
        w[2] = __byte_perm(l0, h0, 0x7362);              // t odd
        w[3] = __byte_perm(l1, h1, 0x7362);
        if (g < NG) *reinterpret_cast<uint4*>(out + g * 256 + (key & 7) * 32 + (up ? 16 : 0)) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        // keys 2t, 2t + 1, 2t + 8, 2t + 9 (xor 1, 8) have the bytes of the same words; each lane makes those of two features d % 8 of both tiles.  First bytes of keys 8 apart,
        // then of neighbours
        const bool up = key >= 8, odd = key & 1;
        const uint32_t give0 = up ? pairs[0] : pairs[1], give1 = up ? pairs[2] : pairs[3];
        const uint32_t got0 = __shfl_xor_sync(0xffffffffu, give0, 8), got1 = __shfl_xor_sync(0xffffffffu, give1, 8);
        const uint32_t keep0 = up ? pairs[1] : pairs[0], keep1 = up ? pairs[3] : pairs[2];
        const uint32_t l0 = up ? got0 : keep0, h0 = up ? keep0 : got0, l1 = up ? got1 : keep1, h1 = up ? keep1 : got1;
        // features d % 8 = 4 up + 0..3: halfwords (key, key + 8) of features 0, 1 and 2, 3
        const uint32_t a0 = __byte_perm(l0, h0, 0x5140), a1 = __byte_perm(l0, h0, 0x7362), b0 = __byte_perm(l1, h1, 0x5140), b1 = __byte_perm(l1, h1, 0x7362);
        const uint32_t sa = odd ? a0 : a1, sb = odd ? b0 : b1;
        const uint32_t ga = __shfl_xor_sync(0xffffffffu, sa, 1), gb = __shfl_xor_sync(0xffffffffu, sb, 1);
        const uint32_t ka = odd ? a1 : a0, kb = odd ? b1 : b0;
        const uint32_t ea = odd ? ga : ka, oa = odd ? ka : ga, eb = odd ? gb : kb, ob = odd ? kb : gb;
        const int j = (up ? 4 : 0) + (odd ? 2 : 0), t = (key & 7) >> 1;
        w[0] = __byte_perm(ea, oa, 0x5410);              // feature j, tile 0: keys 2t, 2t + 8, 2t + 1, 2t + 9
        w[1] = __byte_perm(eb, ob, 0x5410);
        w[2] = __byte_perm(ea, oa, 0x7632);              // feature j + 1
        w[3] = __byte_perm(eb, ob, 0x7632);
        if (g < NG) {
          uint8_t* to = out + 8 * p.D + g * 256 + (j * 4 + t) * 8;
          *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
          *reinterpret_cast<uint2*>(to + 32) = make_uint2(w[2], w[3]);
        }
      }
      if (g < NG) {
        __half* meta = reinterpret_cast<__half*>(out + 16 * p.D) + side * p.D;
        const int at = side ? kv4::value_meta(key, g) : kv4::key_meta(key, g);
        meta[at] = s;
        meta[p.D / 2 + at] = m;
      }
    } else if (live) {
      if (slot >= places) {
        atomicExch(p.dev_arg, kv4::kErrPage);
      } else {
        const int k16 = slot & 15;
        uint8_t* out = block_of(p, slot, head);
        uint8_t* data = out + (side ? 8 * p.D : 0);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int d = g * 32 + (i >> 3) * 16 + (i & 7);
          data[side ? kv4::value_byte(k16, d) : kv4::key_byte(k16, d)] = (uint8_t)(pairs[i >> 2] >> 8 * (i & 3));
        }
        __half* meta = reinterpret_cast<__half*>(out + 16 * p.D) + side * p.D;
        const int at = side ? kv4::value_meta(k16, g) : kv4::key_meta(k16, g);
        meta[at] = s;
        meta[p.D / 2 + at] = m;
      }
    }
  }
}

// One thread per row, side, head and group: its bytes lie in one run of 32 bytes (keys) or in 8 bytes of each of 8 (values), which the neighbouring keys' threads read too.  The values go
// through shared memory, so that a warp writes runs of 128 bytes.  32768 rows of 8 x 128: bf16 41 us, 4.3 TB/s; float32 53 us, 5.9 TB/s.  Slots, bytes and values wait for one another; more rows
// per warp with the next slots asked for ahead were slower (49 us).
template <typename T>
__global__ void __launch_bounds__(256) read_kernel(const StoreParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int NG = kv4::groups(p.D), lane = threadIdx.x, head = blockIdx.x, side = threadIdx.y & 1, g0 = (threadIdx.y >> 1) * 2, g = g0 + (lane >> 4);
  const int64_t row0 = (((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * blockDim.z + threadIdx.z) * 16;
  constexpr int kParts = Group<T>::kParts, kPitch = kParts + 1;          // 16-byte pieces of a lane's group, and one to spread the banks
  __shared__ uint4 staged[8][32 * kPitch];
  uint4* mine = staged[threadIdx.z * blockDim.y + threadIdx.y];
  const int64_t row = row0 + (lane & 15);
  if (row0 >= p.rows) return;
  int slot = row < p.rows && g < NG ? p.slots[row] : -1;
  if (slot >= p.n_pages << p.shift) { atomicExch(p.dev_arg, kv4::kErrPage); slot = -1; }
  const unsigned live = __ballot_sync(0xffffffffu, slot >= 0);
  if (slot >= 0) {
    const int key = slot & 15;
    const uint8_t* block = block_of(p, slot, head);
    uint32_t pairs[4];                         // as quantise() forms them
    if (side == 0) {
      const uint4* src = reinterpret_cast<const uint4*>(block + g * 256 + (key & 7) * 32);
      const uint4 x = src[0], y = src[1];      // words (t, tile): bytes e = 0 of keys key % 8 and + 8, e = 1
      const uint32_t pick = key & 8 ? 0x7531 : 0x6420;
      pairs[0] = __byte_perm(x.x, x.z, pick);
      pairs[2] = __byte_perm(x.y, x.w, pick);
      pairs[1] = __byte_perm(y.x, y.z, pick);
      pairs[3] = __byte_perm(y.y, y.w, pick);
    } else {
      const uint8_t* src = block + 8 * p.D + g * 256 + ((key & 7) >> 1) * 8;
      const int byte = 2 * (key & 1) + (key >> 3);
      uint2 x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = *reinterpret_cast<const uint2*>(src + j * 32);
      const uint32_t two = byte | (4 + byte) << 4;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pairs[h] = __byte_perm(__byte_perm(x[4 * h].x, x[4 * h + 1].x, two), __byte_perm(x[4 * h + 2].x, x[4 * h + 3].x, two), 0x5410);
        pairs[2 + h] = __byte_perm(__byte_perm(x[4 * h].y, x[4 * h + 1].y, two), __byte_perm(x[4 * h + 2].y, x[4 * h + 3].y, two), 0x5410);
      }
    }
    const __half* meta = reinterpret_cast<const __half*>(block + 16 * p.D) + side * p.D;
    const int at = side ? kv4::value_meta(key, g) : kv4::key_meta(key, g);
    const float s = __half2float(meta[at]), m = __half2float(meta[p.D / 2 + at]);
    float out[32];
#pragma unroll
    for (int i = 0; i < 16; ++i) {             // a level n in place, at bit e of a word, becomes 2^23 + n 2^e, and n 2^e meets s 2^-e: exactly n s before the one rounding
      const int f = (i >> 3) * 16 + (i & 7), e = 8 * (i & 1);
      const uint32_t b = i & 2 ? pairs[i >> 2] >> 16 : pairs[i >> 2];
      const float2 n = add2(make_float2(__uint_as_float(b & 15u << e | 0x4b000000u), __uint_as_float(b & 240u << e | 0x4b000000u)), make_float2(-8388608.f, -8388608.f));
      const float2 x = fma2(n, e ? make_float2(s * 0x1p-8f, s * 0x1p-12f) : make_float2(s, s * 0x1p-4f), make_float2(m, m));
      out[f] = x.x;
      out[f + 8] = x.y;
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i) mine[lane * kPitch + i] = Group<T>::part(out, i);
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const int piece = i * 32 + lane, of = piece / kParts, part = piece - of * kParts;      // lane `of` has row row0 + of % 16, group g0 + of / 16
    if (live >> of & 1) {
      T* to = reinterpret_cast<T*>(side ? p.v : p.k) + (row0 + (of & 15)) * (side ? p.v_stride : p.k_stride) + head * p.D + (g0 + (of >> 4)) * 32;
      __stcs(reinterpret_cast<uint4*>(to) + part, mine[of * kPitch + part]);
    }
  }
}

template <typename T> struct Pair;           // two neighbouring features
template <> struct Pair<float> {
  static __device__ __forceinline__ float2 load(const float* p) { return *reinterpret_cast<const float2*>(p); }
  static __device__ __forceinline__ void store(float* p, float2 v) { *reinterpret_cast<float2*>(p) = v; }
};
template <> struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 load(const __nv_bfloat16* p) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p)); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float2 v) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y); }
};

// Few rows: eight lanes per row, side, head and group, a quarter of the work for each; lane (tile, t) has features 16 tile + 2t, 2t + 1, 2t + 8, 2t + 9, which are two bytes of either form.
template <typename T>
__global__ void __launch_bounds__(256) append_few_kernel(const StoreParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int l8 = threadIdx.x & 7, tile = l8 >> 2, t = l8 & 3, g = threadIdx.x >> 3, pair = blockIdx.x * blockDim.y + threadIdx.y;
  const int side = pair >= p.heads, head = pair - (side ? p.heads : 0);
  const int64_t row = (int64_t)blockIdx.y * blockDim.z + threadIdx.z;
  const bool there = row < p.rows && pair < 2 * p.heads;
  const int slot = there ? p.slots[row] : -1;
  float2 a = make_float2(0.f, 0.f), b = a;
  if (there) {
    const T* x = reinterpret_cast<const T*>(side ? p.v : p.k) + row * (side ? p.v_stride : p.k_stride) + head * p.D + g * 32 + tile * 16 + 2 * t;
    a = Pair<T>::load(x);
    b = Pair<T>::load(x + 8);
  }
  float lo = fminf(fminf(a.x, a.y), fminf(b.x, b.y)), hi = fmaxf(fmaxf(a.x, a.y), fmaxf(b.x, b.y));
  const unsigned eight = 0xffu << ((threadIdx.z * blockDim.y + threadIdx.y) * blockDim.x + threadIdx.x & 24);      // the lanes of this group
  bool odd = a.x != a.x || a.y != a.y || b.x != b.x || b.y != b.y;
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(eight, lo, off));
    hi = fmaxf(hi, __shfl_xor_sync(eight, hi, off));
    odd = __shfl_xor_sync(eight, (int)odd, off) | (int)odd;
  }
  if (!there || slot < 0) return;
  if (slot >= p.n_pages << p.shift) { atomicExch(p.dev_arg, kv4::kErrPage); return; }
  __half m = __float2half_rn(lo), s = __float2half_rn(__fdiv_rn(hi - lo, 15.f));
  if (odd || __hisinf(m) || __hisinf(s) || __hisnan(s)) m = s = __ushort_as_half(0x7fff);   // a group without a 4-bit form reads back as NaN
  const float mf = __half2float(m), sf = __half2float(s);
  const uint32_t e0 = level(a.x, mf, sf) | level(b.x, mf, sf) << 4, e1 = level(a.y, mf, sf) | level(b.y, mf, sf) << 4;
  const int key = slot & 15;
  uint8_t* block = block_of(p, slot, head);
  uint8_t* data = block + (side ? 8 * p.D : 0);
  const int d = g * 32 + tile * 16 + 2 * t;
  data[side ? kv4::value_byte(key, d) : kv4::key_byte(key, d)] = (uint8_t)e0;
  data[side ? kv4::value_byte(key, d + 1) : kv4::key_byte(key, d + 1)] = (uint8_t)e1;
  if (l8 == 0) {
    __half* meta = reinterpret_cast<__half*>(block + 16 * p.D) + side * p.D;
    const int at = side ? kv4::value_meta(key, g) : kv4::key_meta(key, g);
    meta[at] = s;
    meta[p.D / 2 + at] = m;
  }
}

// The same lanes the other way.
template <typename T>
__global__ void __launch_bounds__(256) read_few_kernel(const StoreParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int l8 = threadIdx.x & 7, tile = l8 >> 2, t = l8 & 3, g = threadIdx.x >> 3, pair = blockIdx.x * blockDim.y + threadIdx.y;
  const int side = pair >= p.heads, head = pair - (side ? p.heads : 0);
  const int64_t row = (int64_t)blockIdx.y * blockDim.z + threadIdx.z;
  if (row >= p.rows || pair >= 2 * p.heads) return;
  const int slot = p.slots[row];
  if (slot < 0) return;
  if (slot >= p.n_pages << p.shift) { atomicExch(p.dev_arg, kv4::kErrPage); return; }
  const int key = slot & 15;
  const uint8_t* block = block_of(p, slot, head);
  const uint8_t* data = block + (side ? 8 * p.D : 0);
  const int d = g * 32 + tile * 16 + 2 * t;
  const uint32_t e0 = data[side ? kv4::value_byte(key, d) : kv4::key_byte(key, d)], e1 = data[side ? kv4::value_byte(key, d + 1) : kv4::key_byte(key, d + 1)];
  const __half* meta = reinterpret_cast<const __half*>(block + 16 * p.D) + side * p.D;
  const int at = side ? kv4::value_meta(key, g) : kv4::key_meta(key, g);
  const float s = __half2float(meta[at]), m = __half2float(meta[p.D / 2 + at]);
  T* x = reinterpret_cast<T*>(side ? p.v : p.k) + row * (side ? p.v_stride : p.k_stride) + head * p.D + d;
  Pair<T>::store(x, make_float2(fmaf((float)(e0 & 15), s, m), fmaf((float)(e1 & 15), s, m)));
  Pair<T>::store(x + 8, make_float2(fmaf((float)(e0 >> 4), s, m), fmaf((float)(e1 >> 4), s, m)));
}

template <typename K>
cudaError_t launch_cluster(K kernel, int ctas, size_t smem, cudaStream_t st, const TableParams& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kTableThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

int32_t check_tables(const char* who, int n_seq, int page, int max_pages, int n_pages) {
  LMB_REQUIRE(n_seq >= 1 && n_seq <= kMaxSeqs, "%s: %d sequences (1 to %d)", who, n_seq, kMaxSeqs);
  LMB_REQUIRE(max_pages >= 1 && (int64_t)max_pages * page <= kv4::kMostTokens, "%s: block tables of %d pages (up to 2^30 tokens)", who, max_pages);
  return kv4::check_cache(who, 1, 32, n_pages, page);
}

int32_t store_params(const char* who, Ctx* ctx, int32_t dtype, const void* k, const void* v, int64_t k_stride, int64_t v_stride, int32_t rows, int32_t heads, int32_t D,
                     const int32_t* slots, const void* pages, int32_t n_pages, int32_t page, StoreParams* p) {
  LMB_REQUIRE(dtype == LMB200_F32 || dtype == LMB200_BF16, "%s: dtype %d", who, dtype);
  LMB_TRY(kv4::check_cache(who, heads, D, n_pages, page));
  LMB_REQUIRE(rows >= 0, "%s: %d rows", who, rows);
  LMB_REQUIRE(rows == 0 || (k && v && slots && pages), "%s: null pointer", who);
  const int64_t width = (int64_t)heads * D;
  LMB_REQUIRE(k_stride >= width && v_stride >= width, "%s: row strides %lld and %lld for rows of %lld elements", who, (long long)k_stride, (long long)v_stride, (long long)width);
  const int vec = dtype == LMB200_F32 ? 4 : 8;
  LMB_REQUIRE(k_stride % vec == 0 && v_stride % vec == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)pages % 16 == 0,
              "%s: rows and pages must start on 16-byte boundaries", who);
  p->k = const_cast<void*>(k); p->v = const_cast<void*>(v);
  p->k_stride = k_stride; p->v_stride = v_stride;
  p->rows = rows; p->heads = heads; p->D = D; p->shift = kv4::page_shift(page); p->n_pages = n_pages;
  p->slots = slots;
  p->pages = static_cast<uint8_t*>(const_cast<void*>(pages));
  p->dev_arg = ctx->dev_arg;
  return LMB200_OK;
}

// Both ways give the same bits.  The wide one has a quarter of the threads, each with four times the work: below kFewGroups groups its chain is longer than what it saves.
// 512 rows of 8 heads of 128 (32768 groups), bf16: append 5.1 as few, 4.7 wide, read 2.9 and 2.4; 256 rows: 3.5 and 4.7, 2.2 and 2.4.  What a thread has follows from its places in
// grid and block without a division.  The wide blocks have `warps` warps: append 52.5 us with 4 and 54.9 with 8 (32768 rows), read 46 and 43.
constexpr int64_t kFewGroups = 24576;
template <typename K>
int32_t launch_store(Ctx* ctx, K few, K many, int warps, const StoreParams& p) {
  const int NG = kv4::groups(p.D);
  dim3 grid, block;
  if ((int64_t)p.rows * 2 * p.heads * NG > kFewGroups) {
    // warps of a block: sides, pairs of groups, windows; blocks: heads, windows
    const int per_window = 2 * ((NG + 1) / 2);
    block = dim3(32, (unsigned)per_window, (unsigned)std::max(1, warps / per_window));
    const int64_t blocks = ceil_div(ceil_div((int64_t)p.rows, 16), (int64_t)block.z), y = std::min<int64_t>(blocks, 32768);
    grid = dim3((unsigned)p.heads, (unsigned)y, (unsigned)ceil_div(blocks, y));
    LMB_REQUIRE(ceil_div(blocks, y) <= 65535 && (int64_t)p.heads * blocks <= INT_MAX, "kv4: %d rows of %d heads are too many for one call", p.rows, p.heads);
  } else {
    // groups of eight lanes of a block: groups of 32 features, heads of both sides, rows
    const int pairs = std::min(2 * p.heads, 256 / (8 * NG));
    block = dim3(8u * NG, (unsigned)pairs, (unsigned)std::max(1, std::min(p.rows, 256 / (8 * NG * pairs))));
    grid = dim3((unsigned)ceil_div(2 * p.heads, pairs), (unsigned)ceil_div(p.rows, (int)block.z));
  }
  LMB_CUDA(cudaSetDevice(ctx->device));
  LMB_CUDA(launch_k_opt(false, (int64_t)p.rows * 2 * p.heads * NG > kFewGroups ? many : few, grid, block, 0, ctx->stream, p));
  ctx->launches++;
  return LMB200_OK;
}

}  // namespace

int32_t paged_configure() {
  const int smem = kMaxSeqs * 3 * 4;
  LMB_CUDA(cudaFuncSetAttribute(reserve_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  LMB_CUDA(cudaFuncSetAttribute(shrink_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  // 16 CTAs are one cluster where the GPU has room for it
  LMB_CUDA(cudaFuncSetAttribute(reserve_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(16);
  cfg.blockDim = dim3(kTableThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 16;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, reserve_kernel, &cfg) == cudaSuccess && clusters >= 1) g_most_ctas = 16;
  else cudaGetLastError();
  return LMB200_OK;
}

}  // namespace lmb

using namespace lmb;

extern "C" int32_t lmb200_kv4_page_bytes(int32_t page_size, int32_t n_kv_heads, int32_t head_dim, int64_t* bytes) {
  LMB_REQUIRE(bytes, "kv4_page_bytes: null argument");
  LMB_TRY(kv4::check_cache("kv4_page_bytes", n_kv_heads, head_dim, 1, page_size));
  *bytes = (int64_t)n_kv_heads * (page_size / 16) * kv4::block_bytes(head_dim);
  return LMB200_OK;
}

extern "C" int32_t lmb200_kv_reserve(lmb200_ctx h, int32_t n_seq, int32_t page_size, int32_t max_pages, int32_t n_pages, int32_t rows, const int32_t* lens,
                                     const int32_t* add, int32_t* table, const int32_t* free_list, const int32_t* n_free, int32_t* lens_out, int32_t* n_free_out,
                                     int32_t* cu_rows, int32_t* slots, int32_t* status) {
  Ctx* ctx = ctx_from(h);
  if (!ctx) return LMB200_EINVAL;
  LMB_TRY(check_tables("kv_reserve", n_seq, page_size, max_pages, n_pages));
  LMB_REQUIRE(rows >= 0 && rows <= kv4::kMostTokens, "kv_reserve: %d rows (up to 2^30)", rows);
  LMB_REQUIRE(lens && add && table && free_list && n_free && lens_out && n_free_out && cu_rows && status && (slots || rows == 0), "kv_reserve: null pointer");
  LMB_CUDA(cudaSetDevice(ctx->device));
  TableParams p = {n_seq, kv4::page_shift(page_size), max_pages, n_pages, rows, lens, add, n_free, table, const_cast<int32_t*>(free_list),
                   lens_out, n_free_out, cu_rows, slots, status, ctx->dev_arg};
  LMB_CUDA(launch_cluster(reserve_kernel, n_seq <= 512 && rows <= 2048 ? 1 : rows <= 32768 ? 8 : g_most_ctas, (size_t)n_seq * 12, ctx->stream, p));
  ctx->launches++;
  return LMB200_OK;
}

extern "C" int32_t lmb200_kv_shrink(lmb200_ctx h, int32_t n_seq, int32_t page_size, int32_t max_pages, int32_t n_pages, const int32_t* lens, const int32_t* drop,
                                    const int32_t* table, int32_t* free_list, const int32_t* n_free, int32_t* lens_out, int32_t* n_free_out) {
  Ctx* ctx = ctx_from(h);
  if (!ctx) return LMB200_EINVAL;
  LMB_TRY(check_tables("kv_shrink", n_seq, page_size, max_pages, n_pages));
  LMB_REQUIRE(lens && drop && table && free_list && n_free && lens_out && n_free_out, "kv_shrink: null pointer");
  LMB_CUDA(cudaSetDevice(ctx->device));
  TableParams p = {n_seq, kv4::page_shift(page_size), max_pages, n_pages, 0, lens, drop, n_free, const_cast<int32_t*>(table), free_list,
                   lens_out, n_free_out, nullptr, nullptr, nullptr, ctx->dev_arg};
  LMB_CUDA(launch_cluster(shrink_kernel, n_seq > 512 ? 8 : 1, (size_t)n_seq * 12, ctx->stream, p));
  ctx->launches++;
  return LMB200_OK;
}

extern "C" int32_t lmb200_kv4_append(lmb200_ctx h, int32_t dtype, const void* k, const void* v, int64_t k_stride, int64_t v_stride, int32_t rows, int32_t n_kv_heads,
                                     int32_t head_dim, const int32_t* slots, void* pages, int32_t n_pages, int32_t page_size) {
  Ctx* ctx = ctx_from(h);
  if (!ctx) return LMB200_EINVAL;
  StoreParams p;
  LMB_TRY(store_params("kv4_append", ctx, dtype, k, v, k_stride, v_stride, rows, n_kv_heads, head_dim, slots, pages, n_pages, page_size, &p));
  if (rows == 0) return LMB200_OK;
  return dtype == LMB200_F32 ? launch_store(ctx, append_few_kernel<float>, append_kernel<float>, 4, p) : launch_store(ctx, append_few_kernel<__nv_bfloat16>, append_kernel<__nv_bfloat16>, 4, p);
}

extern "C" int32_t lmb200_kv4_read(lmb200_ctx h, int32_t dtype, void* k_out, void* v_out, int64_t k_stride, int64_t v_stride, int32_t rows, int32_t n_kv_heads,
                                   int32_t head_dim, const int32_t* slots, const void* pages, int32_t n_pages, int32_t page_size) {
  Ctx* ctx = ctx_from(h);
  if (!ctx) return LMB200_EINVAL;
  StoreParams p;
  LMB_TRY(store_params("kv4_read", ctx, dtype, k_out, v_out, k_stride, v_stride, rows, n_kv_heads, head_dim, slots, pages, n_pages, page_size, &p));
  if (rows == 0) return LMB200_OK;
  const int64_t size = dtype == LMB200_F32 ? 4 : 2;
  LMB_REQUIRE(kv4::apart(k_out, k_stride * size, v_out, v_stride * size, rows, (int64_t)n_kv_heads * head_dim * size), "kv4_read: k_out and v_out share memory");
  return dtype == LMB200_F32 ? launch_store(ctx, read_few_kernel<float>, read_kernel<float>, 8, p) : launch_store(ctx, read_few_kernel<__nv_bfloat16>, read_kernel<__nv_bfloat16>, 8, p);
}
