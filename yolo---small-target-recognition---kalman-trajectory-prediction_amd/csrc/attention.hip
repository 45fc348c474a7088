// Softmax attention over tokens, forward and backward (include/yk.h, yk_attention).
//
//   S = scale q k^T (masked), P = softmax(S), o = P v, lse = ln sum exp S
//   backward: delta = rowsum(do o), P = exp(S - lse), dP = do v^T, dS = P (dP - delta) scale,
//             dq = dS k, dk = dS^T q, dv = P^T do
//
// The heads that share a key head are packed into one list of rows: row r of key head hk is query
// r / G of head hk G + r % G, so a key block is read once for all of them and their dk / dv meet in
// one accumulator.  Keys (queries) at and behind a batch element's length are never read.
//
// Layout of every kernel here: an MFMA's 16 x 16 result has one column per lane l % 16 and rows
// 4 (l / 16) + i.  The score tiles are computed with the side that is summed over next (keys
// forward and for dq, queries for dk / dv) as rows, so the four values a lane holds of two
// neighbouring tiles are 8 summands of ITS column: exactly a B operand of the next product, if that
// product's K order is taken as {4g .. 4g+3, 16+4g .. 16+4g+3} for lane group g.  The A operand is
// read from LDS in the same order (two transposing reads), and P never leaves its registers.  Row
// statistics of a column are one scalar per lane.
#include "token_common.h"

namespace yk {
namespace tok {

struct AttnArgs {
  const char *q, *k, *v, *o, *go;
  char *out, *dq, *dk, *dv;
  float* lse;         // [b][hq][nq]
  const int32_t *q_lengths, *lengths;
  int64_t qs[3], ks[3], vs[3], os[3], gos[3], dqs[3], dks[3], dvs[3];
  float* part;        // keys split: [16 rows][split][16][d_pad + 4] (sums, exponents' reference, denominator); backward: lse2, delta [b][hk][rows]
  float* kv_part;     // backward, rows split: [split][b * hk * nk][dk, dv: 2 d_pad]
  float* q_part;      // backward, keys split: [split][b * hk * rows][d_pad]
  float scale;
  int b, hk, group, d, nq, nk, causal, rows, splits, key_splits;  // rows = nq * group
};

struct Seq {          // one batch element's lengths
  int qlen, klen, off;  // causal: query i sees keys below i + off + 1
};
__device__ __forceinline__ int clamp_len(const int32_t* p, int b, int n) {
  if (!p) return n;
  const int v = p[b];
  return v < 0 ? 0 : v > n ? n : v;
}
__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int b) {
  Seq s;
  s.qlen = clamp_len(a.q_lengths, b, a.nq);
  s.klen = clamp_len(a.lengths, b, a.nk);
  s.off = s.klen - s.qlen;
  return s;
}
__device__ __forceinline__ int query_of(int r, int group) { return group == 1 ? r : r / group; }
// keys that row r may see: [0, key_limit)
__device__ __forceinline__ int key_limit(const AttnArgs& a, const Seq& s, int r) {
  const int i = query_of(r, a.group);
  if (r >= a.rows || i >= s.qlen) return 0;
  if (!a.causal) return s.klen;
  const int n = i + s.off + 1;
  return n < 0 ? 0 : n;  // i < qlen: at most klen
}
template <class T>
__device__ __forceinline__ T* row_ptr(T* base, const int64_t* st, int b, int hk, int group, int r) {
  const int i = query_of(r, group);
  return base + b * st[0] + (int64_t)i * st[1] + (int64_t)(hk * group + (r - i * group)) * st[2];
}

// 8 elements of a row from element d0 on, those at or past d (all without `ok`) zero
template <class Tr>
__device__ __forceinline__ typename Tr::V8 load8(const typename Tr::T* p, const typename Tr::T* safe, int d0, int d, bool ok) {
  const bool whole = d % (16 / Tr::kBytes) == 0;
  if constexpr (Tr::kBytes == 2) {
    return __builtin_bit_cast(typename Tr::V8, load16_if<Tr>(p + d0, safe, d - d0, ok, whole));
  } else {
    const f32x4 lo = __builtin_bit_cast(f32x4, load16_if<Tr>(p + d0, safe, d - d0, ok, whole));
    const f32x4 hi = __builtin_bit_cast(f32x4, load16_if<Tr>(p + d0 + 4, safe, d - d0 - 4, ok, whole));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}
// two C tiles of a column -> 8 summands.  16-bit P and dS are rounded to the operands' type: half a
// step each, relative, as any operand of a 16-bit MFMA, where float32 operands would cost the whole
// second product four times the time.  An output is then off by some 1.4 of its own rounding.  What
// keeps fp16's short exponent range out of it: kShiftP and GradScale below.
template <class Tr>
__device__ __forceinline__ typename Tr::V8 pack8(f32x4 lo, f32x4 hi) {
  if constexpr (Tr::kBytes == 4) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    typename Tr::T t[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = from_f32<Tr>(lo[i]);
      t[4 + i] = from_f32<Tr>(hi[i]);
    }
    typename Tr::V8 v;
    __builtin_memcpy(&v, t, 16);
    return v;
  }
}

// kBN x kDP block of rows in LDS (kDP = d padded to 32, zero filled) in 16-byte chunks.  Chunk c of a
// row lies at c ^ twist(row) within its group of kGroup chunks.  The 16-bit twist serves both reads without
// bank conflicts (SQ_LDS_BANK_CONFLICT 0): 16 rows of one chunk (16 lanes a cycle, which are rows 0-3 and 12-15 of one lane
// group with rows 4-11 of the next), and 8 rows of 32 bytes (the transposing read's 32 lanes).
template <class Tr, int kDP>
struct Block {
  using T = typename Tr::T;
  static constexpr int kBN = 128 / Tr::kBytes;  // 64 rows of 16-bit, 32 of float32
  static constexpr int kEpc = 16 / Tr::kBytes;
  static constexpr int kRow = kDP * Tr::kBytes;
  static constexpr int kRowChunks = kDP / kEpc;
  static constexpr int kN = kDP / 32;           // chunks per thread of 256
  static constexpr int kBytesAll = kBN * kRow;
  static constexpr int kGroup = kRow % 256 == 0 ? 16 : kRow % 128 == 0 ? 8 : 4;

  static __device__ __forceinline__ int place(int row, int c) {  // (its own inverse in c)
    const int twist = Tr::kBytes == 4 ? (kGroup == 16 ? row & 15 : (row >> 1) & 7)
                      : kGroup == 16  ? (row & 7) << 1
                      : kGroup == 8   ? row & 7
                                      : (row >> 1) & 2;
    return c ^ twist;
  }
  // A operand: row 16 t + l, elements 32 s + 8 g ..
  static __device__ __forceinline__ typename Tr::V8 row_frag(const char* lds, int t, int s, int lane) {
    const int l = lane & 15, g = lane >> 4;
    const char* row = lds + (t * 16 + l) * kRow;
    if constexpr (Tr::kBytes == 2) {
      return *(const typename Tr::V8*)(row + place(l, s * 4 + g) * 16);
    } else {
      const f32x4 lo = *(const f32x4*)(row + place(l, s * 8 + 2 * g) * 16);
      const f32x4 hi = *(const f32x4*)(row + place(l, s * 8 + 2 * g + 1) * 16);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // A operand, transposed: element 16 dt + l of rows 32 u + {4g .. 4g+3, 16+4g .. 16+4g+3}
  static __device__ __forceinline__ typename Tr::V8 col_frag(const char* lds, int dt, int u, int lane) {
    const int l = lane & 15, g = lane >> 4;
    if constexpr (Tr::kBytes == 2) {
      const int row = 4 * g + (l >> 2);
      const char* p = lds + (u * 32 + row) * kRow + place(row, dt * 2 + ((l & 3) >> 1)) * 16 + (l & 1) * 8;
      typedef __attribute__((address_space(3))) s16x4* lp;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 16 * kRow));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      typename Tr::V8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = u * 32 + (e & 4) * 4 + 4 * g + (e & 3);
        v[e] = *(const float*)(lds + row * kRow + place(row, dt * 4 + (l >> 2)) * 16 + (l & 3) * 4);
      }
      return v;
    }
  }
};

// A stream of blocks of rows from memory to LDS by 256 threads: the packed rows of a group of
// heads, or (group 1) the keys of a head.  kAsync: without registers, through a buffer descriptor
// that moves with the block, whose range check turns what is not there into zeros; needs whole,
// 16-byte aligned chunks and a group that divides the block (feed_async).
template <class Tr, int kDP, bool kAsync>
struct Feed {
  using Bl = Block<Tr, kDP>;
  using T = typename Tr::T;
  static constexpr unsigned kOut = 0x80000000u;
  const T* base;  // row `first`'s query, head 0 of the group (kAsync); row 0 (else)
  int64_t st1, st2;
  int group, d, first;
  unsigned off[kAsync ? Bl::kN : 1];
  u32x4 reg[kAsync ? 1 : Bl::kN];

  __device__ __forceinline__ void init(const char* p, const int64_t* st, int b, int head0, int grp, int dd, int first_row) {
    group = grp, d = dd, first = first_row;
    st1 = st[1], st2 = st[2];
    base = (const T*)p + b * st[0] + head0 * st[2];
    if constexpr (kAsync) {
      base += (int64_t)query_of(first, group) * st1;
#pragma unroll
      for (int i = 0; i < Bl::kN; ++i) {
        const int j = i * 256 + threadIdx.x, row = j / Bl::kRowChunks, c = Bl::place(row, j % Bl::kRowChunks) * Bl::kEpc;
        const int q = query_of(row, group);
        off[i] = c < d ? (unsigned)((q * (int)st1 + (row - q * group) * (int)st2 + c) * Tr::kBytes) : kOut;
      }
    }
  }
  // the block that begins at `first`, rows at and past `limit` zero
  __device__ __forceinline__ void issue(char* lds, int limit) {
    if constexpr (kAsync) {
      const size_t b = (size_t)base;
      const size_t ub = ((size_t)(unsigned)rfl((int)(b >> 32)) << 32) | (unsigned)rfl((int)b);
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)ub, (short)0, 0x7ffffff0, 0x00020000);
      auto one = [&](int i, unsigned o) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc, (__attribute__((address_space(3))) void*)(lds + (i * 256 + rfl(threadIdx.x & ~63)) * 16), 16, o, 0, 0, 0);
      };
      if (first + Bl::kBN <= limit) {
#pragma unroll
        for (int i = 0; i < Bl::kN; ++i) one(i, off[i]);
      } else {
#pragma unroll
        for (int i = 0; i < Bl::kN; ++i)
          one(i, first + (int)((i * 256 + threadIdx.x) / Bl::kRowChunks) < limit ? off[i] : kOut);
      }
    } else {
#pragma unroll
      for (int i = 0; i < Bl::kN; ++i) {
        const int j = i * 256 + threadIdx.x, row = first + j / Bl::kRowChunks, c = (j % Bl::kRowChunks) * Bl::kEpc;
        const int q = query_of(row, group);
        reg[i] = load16_if<Tr>(base + q * st1 + (row - q * group) * st2 + c, base, d - c, row < limit, d % Bl::kEpc == 0);
      }
    }
  }
  __device__ __forceinline__ void advance() {
    first += Bl::kBN;
    if constexpr (kAsync) base += (int64_t)(group == 1 ? Bl::kBN : Bl::kBN / group) * st1;
  }
  __device__ __forceinline__ void commit(char* lds) const {
    if constexpr (!kAsync) {
#pragma unroll
      for (int i = 0; i < Bl::kN; ++i) {
        const int j = i * 256 + threadIdx.x, row = j / Bl::kRowChunks, c = j % Bl::kRowChunks;
        *(u32x4*)(lds + row * Bl::kRow + Bl::place(row, c) * 16) = reg[i];
      }
    }
  }
};

// Until this wave's loads have landed and its LDS reads are done; then until all waves are there.
__device__ __forceinline__ void block_landed() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
}

// Runs `body(buffer)` over the blocks of two feeds, [first, end) in rows; `buf`: kBuffers of them, the
// next block on its way while one is worked on, one barrier per block.  extra(buffer, first) loads what else
// belongs to a block (kAsync: straight to LDS).
template <class Tr, int kDP, bool kAsync, class F, class X, class B>
__device__ __forceinline__ void for_blocks(F& f0, F& f1, int first, int end, int limit, char* buf, int stride, X&& extra, B&& body) {
  constexpr int kBN = Block<Tr, kDP>::kBN, kHalf = Block<Tr, kDP>::kBytesAll;
  if (first >= end) return;
  auto issue = [&](char* p, int r) {
    f0.issue(p, limit);
    f1.issue(p + kHalf, limit);
    extra(p + 2 * kHalf, r);
    f0.advance();
    f1.advance();
  };
  int cur = 0;
  issue(buf, first);
  if constexpr (!kAsync) {
    f0.commit(buf);
    f1.commit(buf + kHalf);
  }
  for (int r = first; r < end; r += kBN) {
    block_landed();
    char* next = buf + (cur ^ 1) * stride;
    if (r + kBN < end) issue(next, r + kBN);
    body(buf + cur * stride, r);
    if constexpr (!kAsync) {
      if (r + kBN < end) {
        f0.commit(next);
        f1.commit(next + kHalf);
      }
    }
    cur ^= 1;
  }
}

// 4 elements d0 .. of an output row
template <class Tr>
__device__ __forceinline__ void store_out(typename Tr::T* p, int d0, int d, f32x4 v) {
  if (d0 + 4 <= d) {
    store4<Tr>(p + d0, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d0 + i < d) p[d0 + i] = from_f32<Tr>(v[i]);
  }
}

// One column's running softmax over a block of kT score tiles: raw scores in st, p comes back in
// it, keys beyond `lim` left out.  m is the reference of the column's exponents, in score * scale *
// log2 e: a maximum seen so far, renewed only when a lane's p add up to more than 2^8 under it.
// Most blocks then need no maximum at all, neither a lane's nor the other lanes', and no rescaling;
// that p may exceed 1 costs no accuracy (fp16 holds 2^15).  l: this lane's share of the denominator,
// from p as it is before any rounding.  rescale(f): what else was accumulated so far times f.
constexpr float kRenew = 256.f;
template <int kT, class R>
__device__ __forceinline__ void softmax_step(f32x4* st, int key0, int lim, float sl2, float& m, float& l, R&& rescale) {
  const int left = lim - key0 - ((threadIdx.x & 63) >> 4) * 4;  // this lane's keys t * 16 + i below it are seen
  if (__any(lim < key0 + kT * 16)) {
#pragma unroll
    for (int t = 0; t < kT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) st[t][i] = t * 16 + i < left ? st[t][i] : -INFINITY;
  }
  f32x4 p[kT];
  auto exps = [&](float ref) {
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < kT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[t][i] = exp2_f(fmaf(st[t][i], sl2, -ref));
        sum += p[t][i];
      }
    return sum;
  };
  // (nothing seen yet: m is -infinity, and every p of a column that sees nothing here exp2(-inf) = 0)
  float sum = exps(m == -INFINITY ? 0.f : m);
  if (__any(sum > kRenew || (m == -INFINITY && lim > key0))) {
    float mx = st[0][0];
#pragma unroll
    for (int t = 0; t < kT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, st[t][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx * sl2), ref = mn == -INFINITY ? 0.f : mn;
    const float f = exp2_f(m - ref);
    l *= f;
    rescale(f);
    m = mn;
    sum = exps(ref);
  }
  l += sum;
#pragma unroll
  for (int t = 0; t < kT; ++t) st[t] = p[t];
}

// A column's sum over the lanes that share it.
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// Two waves per SIMD for the 16-bit types: with 256 registers a wave the compiler keeps the MFMA's
// results where the vector instructions read them, with more it moves them there and back (a third of
// the forward kernel's instructions).
template <class Tr>
constexpr int kWavesPerSimd = Tr::kBytes == 2 ? 2 : 1;

// Keys that a block of rows [r0, r0 + n) sees: its last row in use sees most.
__device__ __forceinline__ int key_end(const AttnArgs& a, const Seq& s, int r0, int n) {
  if (query_of(r0, a.group) >= s.qlen) return 0;
  if (!a.causal) return s.klen;
  int i = query_of((r0 + n < a.rows ? r0 + n : a.rows) - 1, a.group);
  i = i < s.qlen ? i : s.qlen - 1;
  return i + s.off + 1;
}

// Range blockIdx.y of the keys [0, k_stop), in whole blocks.
template <int kBN>
__device__ __forceinline__ void key_range(int& k_begin, int& k_stop) {
  const int end = k_stop > 0 ? k_stop : 0, per = ((end + kBN - 1) / kBN + (int)gridDim.y - 1) / (int)gridDim.y * kBN;
  k_begin = (int)blockIdx.y * per < end ? (int)blockIdx.y * per : end;
  k_stop = end - k_begin < per ? end : k_begin + per;
}

// Forward: 4 waves of 16 kNT rows; with few row blocks, blockIdx.y a range of the keys, whose sums
// attn_join_rows_kernel joins.  Bound by issue: per block and lane 32 kNT exponentials, their sums and
// conversions next to the MFMAs, neither of which hides the other wholly with two waves per SIMD.
// bf16, 4 x 5120 x 5120, 8 heads of 64: 242 us, 887 TFLOP/s (under the profiler 258-272); 8 x 1280 x 1280,
// 8 heads of 40 (computed as 64): 39 us.
template <class Tr, int kDP, int kNT, bool kAsync>
__global__ __launch_bounds__(256, kWavesPerSimd<Tr>) void attn_kernel(AttnArgs a, int row_blocks) {
  using T = typename Tr::T;
  using V8 = typename Tr::V8;
  using Bl = Block<Tr, kDP>;
  constexpr int kKT = Bl::kBN / 16, kS = kDP / 32, kDT = kDP / 16, kRows = 64 * kNT, kBuf = 2 * Bl::kBytesAll;
  __shared__ __attribute__((aligned(16))) char lds[2 * kBuf];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int item = xcd_item(blockIdx.x, gridDim.x);
  // long causal rows first
  const int bh = item / row_blocks, rb = a.causal ? row_blocks - 1 - (item - bh * row_blocks) : item - bh * row_blocks;
  const int b = bh / a.hk, hk = bh - b * a.hk;
  const Seq s = seq_of(a, b);
  const int r0 = rb * kRows;
  V8 qf[kNT][kS];
  int lim[kNT];
  float m[kNT], l[kNT];
  f32x4 acc[kNT][kDT];
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    const int r = r0 + (wave * kNT + j) * 16 + l16;
    lim[j] = key_limit(a, s, r);
    m[j] = -INFINITY;
    l[j] = 0.f;
#pragma unroll
    for (int c = 0; c < kS; ++c)
      qf[j][c] = load8<Tr>(row_ptr((const T*)a.q, a.qs, b, hk, a.group, r), (const T*)a.q, c * 32 + g * 8, a.d, lim[j] > 0);
#pragma unroll
    for (int t = 0; t < kDT; ++t) acc[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float sl2 = a.scale * kLog2e;
  Feed<Tr, kDP, kAsync> fk, fv;
  int k_begin = 0, k_stop = key_end(a, s, r0, kRows);
  if (gridDim.y > 1) key_range<Bl::kBN>(k_begin, k_stop);
  fk.init(a.k, a.ks, b, hk, 1, a.d, k_begin);
  fv.init(a.v, a.vs, b, hk, 1, a.d, k_begin);
  for_blocks<Tr, kDP, kAsync>(fk, fv, k_begin, k_stop, s.klen, lds, kBuf, [](char*, int) {}, [&](const char* lk, int k0) {
    const char* lv = lk + Bl::kBytesAll;
    f32x4 st[kNT][kKT];
#pragma unroll
    for (int t = 0; t < kKT; ++t) {
#pragma unroll
      for (int j = 0; j < kNT; ++j) st[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kS; ++c) {
        const V8 kf = Bl::row_frag(lk, t, c, lane);
#pragma unroll
        for (int j = 0; j < kNT; ++j) st[j][t] = mma<Tr>(kf, qf[j][c], st[j][t]);
      }
    }
    V8 pf[kNT][kKT / 2];
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      softmax_step<kKT>(st[j], k0, lim[j], sl2, m[j], l[j], [&](float f) {
#pragma unroll
        for (int t = 0; t < kDT; ++t) acc[j][t] *= f;
      });
#pragma unroll
      for (int u = 0; u < kKT / 2; ++u) pf[j][u] = pack8<Tr>(st[j][2 * u], st[j][2 * u + 1]);
    }
#pragma unroll
    for (int u = 0; u < kKT / 2; ++u)
#pragma unroll
      for (int t = 0; t < kDT; ++t) {
        const V8 vf = Bl::col_frag(lv, t, u, lane);
#pragma unroll
        for (int j = 0; j < kNT; ++j) acc[j][t] = mma<Tr>(vf, pf[j][u], acc[j][t]);
      }
  });
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    const int r = r0 + (wave * kNT + j) * 16 + l16;
    const float sum = column_sum(l[j]);
    if (r >= a.rows) continue;
    if (gridDim.y > 1) {
      const int64_t at = ((int64_t)bh * ((a.rows + 15) / 16) + r / 16) * gridDim.y + blockIdx.y;
      float* part = a.part + (at * 16 + r % 16) * (kDP + 4);
#pragma unroll
      for (int t = 0; t < kDT; ++t) *(f32x4*)(part + t * 16 + g * 4) = acc[j][t];
      if (g == 0) {
        part[kDP] = m[j];
        part[kDP + 1] = sum;
      }
      continue;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* o = row_ptr((T*)a.out, a.os, b, hk, a.group, r);
#pragma unroll
    for (int t = 0; t < kDT; ++t) store_out<Tr>(o, t * 16 + g * 4, a.d, acc[j][t] * inv);
    if (a.lse && g == 0) {
      const int i = query_of(r, a.group);
      a.lse[((int64_t)(b * a.hk + hk) * a.group + (r - i * a.group)) * a.nq + i] = sum == 0.f ? -INFINITY : fmaf(m[j], kLn2, logf(sum));
    }
  }
}

// Few rows, long keys: 16 rows per workgroup and blockIdx.y a range of keys, which the waves walk 32
// keys at a time on their own, each through two slabs of LDS of its own (no barrier; the next slab on
// its way while one is worked on).  The waves' sums meet in LDS; ranges go to scratch unless there is
// one.  Bound by the keys' and values' bytes: what counts is how many are on their way per CU
// (64 KiB with two workgroups of four waves at d = 64).  fp16, 8 streams against 20480 keys at most, 16
// heads of 64 on 4: 22 us, and 3.8 for the join.
template <class Tr, int kDP, int kWaves, bool kAsync>
__global__ __launch_bounds__(64 * kWaves) void attn_split_kernel(AttnArgs a, int row_blocks) {
  using T = typename Tr::T;
  using V8 = typename Tr::V8;
  using Bl = Block<Tr, kDP>;
  constexpr int kKeys = 32, kS = kDP / 32, kDT = kDP / 16, kHalf = kKeys * Bl::kRow, kN = kHalf / 1024;
  constexpr unsigned kOut = 0x80000000u;
  __shared__ __attribute__((aligned(16))) char lds[kWaves * 4 * kHalf];
  __shared__ float stat[kWaves][2][16];
  static_assert(kDT * 1024 <= 4 * kHalf, "a wave's sums fit its slabs");
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int bh = blockIdx.x / row_blocks, rb = blockIdx.x - bh * row_blocks;
  const int b = bh / a.hk, hk = bh - b * a.hk;
  const Seq s = seq_of(a, b);
  const int r = rb * 16 + l16;
  const int lim = key_limit(a, s, r);
  const T* kb = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vb = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
  // the range of this workgroup: whole slabs for each of its waves
  const int turns = (s.klen + kKeys * kWaves - 1) / (kKeys * kWaves), per = (turns + a.splits - 1) / a.splits;
  const int64_t k_begin = (int64_t)blockIdx.y * per * kKeys * kWaves;
  const int k_end = (int)(k_begin + per * kKeys * kWaves < s.klen ? k_begin + per * kKeys * kWaves : s.klen);
  V8 qf[kS];
#pragma unroll
  for (int c = 0; c < kS; ++c)
    qf[c] = load8<Tr>(row_ptr((const T*)a.q, a.qs, b, hk, a.group, r), (const T*)a.q, c * 32 + g * 8, a.d, lim > 0);
  float m = -INFINITY, l = 0.f;
  f32x4 acc[kDT];
#pragma unroll
  for (int t = 0; t < kDT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float sl2 = a.scale * kLog2e;
  char* mine = lds + wave * 4 * kHalf;

  unsigned ko[kAsync ? kN : 1], vo[kAsync ? kN : 1];
  if constexpr (kAsync) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int j = i * 64 + lane, row = j / Bl::kRowChunks, c = Bl::place(row, j % Bl::kRowChunks) * Bl::kEpc;
      ko[i] = c < a.d ? (unsigned)((row * (int)a.ks[1] + c) * Tr::kBytes) : kOut;
      vo[i] = c < a.d ? (unsigned)((row * (int)a.vs[1] + c) * Tr::kBytes) : kOut;
    }
  }
  auto issue = [&](char* to, int k0) {
    if constexpr (kAsync) {
      const bool tail = k0 + kKeys > k_end;
      auto one = [&](const T* p, const unsigned* off, char* at) {
        const size_t u = (size_t)p;
        const size_t us = ((size_t)(unsigned)rfl((int)(u >> 32)) << 32) | (unsigned)rfl((int)u);
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)us, (short)0, 0x7ffffff0, 0x00020000);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          unsigned o = off[i];
          if (tail && k0 + (i * 64 + lane) / Bl::kRowChunks >= k_end) o = kOut;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(at + i * 1024), 16, o, 0, 0, 0);
        }
      };
      one(kb + (int64_t)k0 * a.ks[1], ko, to);
      one(vb + (int64_t)k0 * a.vs[1], vo, to + kHalf);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int j = i * 64 + lane, row = j / Bl::kRowChunks, c = j % Bl::kRowChunks, e = c * Bl::kEpc;
        const bool whole = a.d % Bl::kEpc == 0, in = k0 + row < k_end;
        *(u32x4*)(to + row * Bl::kRow + Bl::place(row, c) * 16) =
            load16_if<Tr>(kb + (int64_t)(k0 + row) * a.ks[1] + e, kb, a.d - e, in, whole);
        *(u32x4*)(to + kHalf + row * Bl::kRow + Bl::place(row, c) * 16) =
            load16_if<Tr>(vb + (int64_t)(k0 + row) * a.vs[1] + e, vb, a.d - e, in, whole);
      }
    }
  };
  int cur = 0;
  const int first = (int)k_begin + wave * kKeys;
  if (k_begin < k_end && first < k_end) issue(mine, first);
  for (int k0 = first; k_begin < k_end && k0 < k_end; k0 += kKeys * kWaves) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other slab's last reads are done
    if (k0 + kKeys * kWaves < k_end) {
      issue(mine + (cur ^ 1) * 2 * kHalf, k0 + kKeys * kWaves);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kAsync ? 2 * kN : 0) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const char* lk = mine + cur * 2 * kHalf;
    const char* lv = lk + kHalf;
    f32x4 st[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kS; ++c) st[t] = mma<Tr>(Bl::row_frag(lk, t, c, lane), qf[c], st[t]);
    }
    const int lim2 = lim < k_end ? lim : k_end;
    softmax_step<2>(st, k0, lim2, sl2, m, l, [&](float f) {
#pragma unroll
      for (int t = 0; t < kDT; ++t) acc[t] *= f;
    });
    const V8 pf = pack8<Tr>(st[0], st[1]);
#pragma unroll
    for (int t = 0; t < kDT; ++t) acc[t] = mma<Tr>(Bl::col_frag(lv, t, 0, lane), pf, acc[t]);
    cur ^= 1;
  }
  l = column_sum(l);
  if (g == 0) {
    stat[wave][0][l16] = m;
    stat[wave][1][l16] = l;
  }
  __syncthreads();
  float mm = stat[0][0][l16];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) mm = fmaxf(mm, stat[w][0][l16]);
  const float ref = mm == -INFINITY ? 0.f : mm;
  const float f = exp2_f(m - ref);
  float ll = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) ll += stat[w][1][l16] * exp2_f(stat[w][0][l16] - ref);
  float* sum = (float*)mine;  // [kDT][64 lanes][4] of each wave
#pragma unroll
  for (int t = 0; t < kDT; ++t) *(f32x4*)(sum + (t * 64 + lane) * 4) = acc[t] * f;
  __syncthreads();
  if (r >= a.rows) return;
  const bool one = a.splits == 1;
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  float* part = one ? nullptr : a.part + (((int64_t)blockIdx.x * a.splits + blockIdx.y) * 16 + l16) * (kDP + 4);
  for (int t = wave; t < kDT; t += kWaves) {
    f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += *(const f32x4*)((float*)(lds + w * 4 * kHalf) + (t * 64 + lane) * 4);
    if (one) store_out<Tr>(row_ptr((T*)a.out, a.os, b, hk, a.group, r), t * 16 + g * 4, a.d, v * inv);
    else *(f32x4*)(part + t * 16 + g * 4) = v;
  }
  if (wave || g) return;
  if (!one) {
    part[kDP] = mm;
    part[kDP + 1] = ll;
  } else if (a.lse) {
    const int i = query_of(r, a.group);
    a.lse[((int64_t)(b * a.hk + hk) * a.group + (r - i * a.group)) * a.nq + i] = ll == 0.f ? -INFINITY : fmaf(mm, kLn2, logf(ll));
  }
}

// The ranges of one row joined, in a fixed order: 4 waves take every fourth range each (8 at a time, so
// that their loads overlap), two elements of the row per lane.
template <class Tr>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int row_blocks, int dp) {
  using T = typename Tr::T;
  __shared__ float sums[4][128], denom[4];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6), bh = blockIdx.x / a.rows, r = blockIdx.x - bh * a.rows;
  const int b = bh / a.hk, hk = bh - b * a.hk;
  const float* p = a.part + (((int64_t)(bh * row_blocks + r / 16) * a.splits) * 16 + r % 16) * (dp + 4);
  const int64_t step = (int64_t)16 * (dp + 4);
  float mm = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) mm = fmaxf(mm, p[s * step + dp]);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) mm = fmaxf(mm, __shfl_xor(mm, x, 64));
  const float ref = mm == -INFINITY ? 0.f : mm;
  const bool b0 = lane < a.d, b1 = lane + 64 < a.d;
  float ll = 0.f, v0 = 0.f, v1 = 0.f;
  for (int s0 = wave; s0 < a.splits; s0 += 32) {
    float e[8], n[8], x0[8], x1[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = s0 + 4 * i < a.splits ? s0 + 4 * i : s0;
      const float* q = p + s * step;
      e[i] = q[dp];
      n[i] = q[dp + 1];
      x0[i] = b0 ? q[lane] : 0.f;
      x1[i] = b1 ? q[lane + 64] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = s0 + 4 * i < a.splits ? exp2_f(e[i] - ref) : 0.f;
      ll += n[i] * f;
      v0 += x0[i] * f;
      v1 += x1[i] * f;
    }
  }
  sums[wave][lane] = v0;
  sums[wave][lane + 64] = v1;
  if (lane == 0) denom[wave] = ll;
  __syncthreads();
  ll = (denom[0] + denom[1]) + (denom[2] + denom[3]);
  const int e = threadIdx.x;
  if (e < a.d) {
    const float v = (sums[0][e] + sums[1][e]) + (sums[2][e] + sums[3][e]);
    row_ptr((T*)a.out, a.os, b, hk, a.group, r)[e] = from_f32<Tr>(ll == 0.f ? 0.f : v / ll);
  }
  if (a.lse && e == 0) {
    const int i = query_of(r, a.group);
    a.lse[((int64_t)(b * a.hk + hk) * a.group + (r - i * a.group)) * a.nq + i] = ll == 0.f ? -INFINITY : fmaf(mm, kLn2, logf(ll));
  }
}

// The same for many rows in few ranges: 4 elements of a row per thread.
template <class Tr>
__global__ __launch_bounds__(256) void attn_join_rows_kernel(AttnArgs a, int dp) {
  using T = typename Tr::T;
  const int per = dp / 4, c = threadIdx.x % per;
  const int64_t all = (int64_t)a.b * a.hk * a.rows, id = (int64_t)blockIdx.x * (256 / per) + threadIdx.x / per;
  if (threadIdx.x >= 256 / per * per || id >= all) return;
  const int bh = (int)(id / a.rows), r = (int)(id - (int64_t)bh * a.rows), b = bh / a.hk, hk = bh - b * a.hk;
  const int64_t step = (int64_t)16 * (dp + 4);
  const float* p = a.part + ((int64_t)bh * ((a.rows + 15) / 16) + r / 16) * a.splits * step + (r % 16) * (dp + 4);
  float mm = -INFINITY;
  for (int s = 0; s < a.splits; ++s) mm = fmaxf(mm, p[s * step + dp]);
  const float ref = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f;
  f32x4 v{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const float f = exp2_f(p[s * step + dp] - ref);
    ll += p[s * step + dp + 1] * f;
    v += *(const f32x4*)(p + s * step + c * 4) * f;
  }
  store_out<Tr>(row_ptr((T*)a.out, a.os, b, hk, a.group, r), c * 4, a.d, v * (ll == 0.f ? 0.f : 1.f / ll));
  if (a.lse && c == 0) {
    const int i = query_of(r, a.group);
    a.lse[((int64_t)bh * a.group + (r - i * a.group)) * a.nq + i] = ll == 0.f ? -INFINITY : fmaf(mm, kLn2, logf(ll));
  }
}

// fp16 holds no digits below 2^-24, and a normalised P is about 1 / nk: the backward kernels compute
// P 2^15 (at most 2^15 of 2^16), by their exponents' reference, and take the power out of dv.
template <class Tr>
constexpr float kShiftP = 0.f;
template <>
constexpr float kShiftP<H16> = 15.f;

// dS in fp16 likewise times a power of two, one per column (a lane's query or key, shared by the four
// lanes of it): c, which only falls, whenever a |dS| c passes 2^15, and then to 2^9 .. 2^10, so that what
// is rounded to fp16 is off by half a step of itself or 2^-34 of the column's largest so far.  It begins
// at 2^64: |dS| 2^15 <= 2^15 128 65504^2 < 2^55 of fp16 operands stays finite times that, and what never
// reaches 2^15 needs no less.  The other types' range is float32's, and nothing of this is compiled.
// 4 x 5120 x 5120, 8 heads of 64, backward: 869-880 us, 819 without it (bf16 787-796).
template <class Tr>
struct GradScale {
  static constexpr bool kOn = Tr::kBytes == 2 && kShiftP<Tr> != 0.f;
  static constexpr float kTop = 32768.f;
  float c = kOn ? 18446744073709551616.f : 1.f;
  // before two tiles of dS c (P's shift included) are rounded; rescale(f): what was summed so far times f
  template <class R>
  __device__ __forceinline__ void fit(f32x4 (&ds)[2], R&& rescale) {
    if constexpr (kOn) {
      float mx = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fabsf(ds[h][i]));
      if (__any(mx > kTop)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        // (an infinite dS stays one)
        const float f = mx > kTop && mx < INFINITY ? ldexpf(1.f, 10 - __builtin_amdgcn_frexp_expf(mx)) : 1.f;
        c *= f;
        rescale(f);
#pragma unroll
        for (int h = 0; h < 2; ++h) ds[h] *= f;
      }
    }
  }
  // 1 / (c 2^shift), exact: what takes both powers out of a sum
  __device__ __forceinline__ float undo() const { return kOn ? ldexpf(1.f / c, -(int)kShiftP<Tr>) : 1.f; }
};

// Row statistics of the backward pass in packed-row order: lse * log2 e less P's shift (+infinity where a
// row has no key, which makes its P zero) and delta = sum over d of do o.  16 lanes per row.
template <class Tr>
__global__ __launch_bounds__(256) void attn_delta_kernel(AttnArgs a) {
  using T = typename Tr::T;
  const int lane = threadIdx.x & 15;
  const int64_t all = (int64_t)a.b * a.hk * a.rows, id = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int64_t idc = id < all ? id : all - 1;
  const int bh = (int)(idc / a.rows), r = (int)(idc - (int64_t)bh * a.rows), b = bh / a.hk, hk = bh - b * a.hk;
  const int i = query_of(r, a.group);
  const bool live = i < clamp_len(a.q_lengths, b, a.nq);
  float s = 0.f;
  if (live && lane * 8 < a.d) {
    const typename Tr::V8 o = load8<Tr>(row_ptr((const T*)a.o, a.os, b, hk, a.group, r), (const T*)a.o, lane * 8, a.d, true);
    const typename Tr::V8 d = load8<Tr>(row_ptr((const T*)a.go, a.gos, b, hk, a.group, r), (const T*)a.go, lane * 8, a.d, true);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (Tr::kBytes == 4) s += o[e] * d[e];
      else s += to_f32<Tr>(__builtin_bit_cast(T, (short)o[e])) * to_f32<Tr>(__builtin_bit_cast(T, (short)d[e]));
    }
  }
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) s += __shfl_xor(s, x, 64);
  if (id >= all || lane) return;
  const float lse = live ? a.lse[((int64_t)bh * a.group + (r - i * a.group)) * a.nq + i] : -INFINITY;
  a.part[id] = lse == -INFINITY ? INFINITY : fmaf(lse, kLog2e, -kShiftP<Tr>);
  a.part[all + id] = s;
}

// dk and dv: 4 waves of 16 kNT keys, blocks of packed rows (q, do and their statistics) through LDS;
// with few keys, blockIdx.y a range of the rows, whose float32 sums attn_dkv_sum_kernel adds.  S and dP are
// computed here and once more for dq, instead of sums that several workgroups add to: 14 products' work
// for 10, but no atomics and equal bits.  bf16, 4 x 5120 x 5120, 8 heads of 64: 471-497 us under the
// profiler, 864-912 TFLOP/s; fp16, whose dS is scaled, 513-535.
template <class Tr, int kDP, int kNT, bool kAsync>
__global__ __launch_bounds__(256, kWavesPerSimd<Tr>) void attn_dkv_kernel(AttnArgs a, int key_blocks) {
  using T = typename Tr::T;
  using V8 = typename Tr::V8;
  using Bl = Block<Tr, kDP>;
  constexpr int kRT = Bl::kBN / 16, kS = kDP / 32, kDT = kDP / 16, kKeys = 64 * kNT, kBuf = 2 * Bl::kBytesAll + 8 * Bl::kBN;
  __shared__ __attribute__((aligned(16))) char lds[2 * kBuf];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const int bh = item / key_blocks, key0 = (item - bh * key_blocks) * kKeys;
  const int b = bh / a.hk, hk = bh - b * a.hk;
  const Seq s = seq_of(a, b);
  const int64_t all = (int64_t)a.b * a.hk * a.rows;
  V8 kf[kNT][kS], vf[kNT][kS];
  f32x4 dk[kNT][kDT], dv[kNT][kDT];
  GradScale<Tr> gsc[kNT];
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    const int key = key0 + (wave * kNT + j) * 16 + l16;
    const bool live = key < s.klen;
#pragma unroll
    for (int c = 0; c < kS; ++c) {
      kf[j][c] = load8<Tr>((const T*)a.k + b * a.ks[0] + (int64_t)key * a.ks[1] + hk * a.ks[2], (const T*)a.k, c * 32 + g * 8, a.d, live);
      vf[j][c] = load8<Tr>((const T*)a.v + b * a.vs[0] + (int64_t)key * a.vs[1] + hk * a.vs[2], (const T*)a.v, c * 32 + g * 8, a.d, live);
    }
#pragma unroll
    for (int t = 0; t < kDT; ++t) dk[j][t] = dv[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // rows in use that see a key of this block
  const int r_end = key0 < s.klen ? s.qlen * a.group : 0;
  int r_begin = 0;
  if (a.causal && key0 > s.off) r_begin = (int)((int64_t)(key0 - s.off) * a.group < r_end ? (int64_t)(key0 - s.off) * a.group : r_end);
  r_begin = r_begin / Bl::kBN * Bl::kBN;
  int r_stop = r_end;
  if (gridDim.y > 1 && r_begin < r_end) {
    const int per = ((r_end - r_begin + Bl::kBN - 1) / Bl::kBN + gridDim.y - 1) / gridDim.y * Bl::kBN;
    r_begin = blockIdx.y * per < r_end - r_begin ? r_begin + blockIdx.y * per : r_end;
    r_stop = r_end - r_begin < per ? r_end : r_begin + per;
  }
  const float sl2 = a.scale * kLog2e;
  Feed<Tr, kDP, kAsync> fq, fo;
  fq.init(a.q, a.qs, b, hk * a.group, a.group, a.d, r_begin);
  fo.init(a.go, a.gos, b, hk * a.group, a.group, a.d, r_begin);
  // lse and delta of a block: waves 0 and 1, a lane a row.  Rows at and past the end read as zero,
  // which with their q = do = 0 leaves nothing.
  auto stats = [&](char* to, int r0) {
    const int i = threadIdx.x & 63;
    if (wave >= 2 || i >= Bl::kBN) return;
    const float* p = a.part + (wave ? all : 0) + (int64_t)bh * a.rows + r0;
    char* at = to + wave * 4 * Bl::kBN;
    if constexpr (kAsync) {
      const size_t ub = (size_t)p;
      const size_t us = ((size_t)(unsigned)rfl((int)(ub >> 32)) << 32) | (unsigned)rfl((int)ub);
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)us, (short)0, 0x7ffffff0, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)at, 4,
                                               r0 + i < r_end ? i * 4u : 0x80000000u, 0, 0, 0);
    } else {
      *(float*)(at + i * 4) = r0 + i < r_end ? p[i] : 0.f;
    }
  };
  for_blocks<Tr, kDP, kAsync>(fq, fo, r_begin, r_stop, r_end, lds, kBuf, stats, [&](const char* lq, int r0) {
    const char* lo = lq + Bl::kBytesAll;
    const float* stat = (const float*)(lo + Bl::kBytesAll);
    // the block's first query sees least
    const bool mask = a.causal && key0 + kKeys - 1 > query_of(r0, a.group) + s.off;
#pragma unroll
    for (int u = 0; u < kRT / 2; ++u) {
      f32x4 p[kNT][2], ds[kNT][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = 2 * u + h;
#pragma unroll
        for (int j = 0; j < kNT; ++j) p[j][h] = ds[j][h] = f32x4{0.f, 0.f, 0.f, 0.f};
        // (fp16: dP's sum begins at -delta, which leaves the subtraction's place to c)
        if constexpr (GradScale<Tr>::kOn) {
#pragma unroll
          for (int j = 0; j < kNT; ++j) ds[j][h] = -*(const f32x4*)(stat + Bl::kBN + t * 16 + g * 4);
        }
#pragma unroll
        for (int c = 0; c < kS; ++c) {
          const V8 qf = Bl::row_frag(lq, t, c, lane), of = Bl::row_frag(lo, t, c, lane);
#pragma unroll
          for (int j = 0; j < kNT; ++j) {
            p[j][h] = mma<Tr>(qf, kf[j][c], p[j][h]);
            ds[j][h] = mma<Tr>(of, vf[j][c], ds[j][h]);
          }
        }
        const f32x4 ls = *(const f32x4*)(stat + t * 16 + g * 4), dl = *(const f32x4*)(stat + Bl::kBN + t * 16 + g * 4);
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) p[j][h][i] = exp2_f(fmaf(p[j][h][i], sl2, -ls[i]));
          if (mask) {
            const int sees = key0 + (wave * kNT + j) * 16 + l16 - s.off;  // the first query that sees this key
            if (a.group == 1) {
              const int skip = sees - r0 - g * 4;
#pragma unroll
              for (int i = 0; i < 4; ++i) p[j][h][i] = t * 16 + i < skip ? 0.f : p[j][h][i];
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (query_of(r0 + t * 16 + g * 4 + i, a.group) < sees) p[j][h][i] = 0.f;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) ds[j][h][i] = p[j][h][i] * (GradScale<Tr>::kOn ? ds[j][h][i] * gsc[j].c : ds[j][h][i] - dl[i]);
        }
      }
      V8 pf[kNT], df[kNT];
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        gsc[j].fit(ds[j], [&](float f) {
#pragma unroll
          for (int t = 0; t < kDT; ++t) dk[j][t] *= f;
        });
        pf[j] = pack8<Tr>(p[j][0], p[j][1]);
        df[j] = pack8<Tr>(ds[j][0], ds[j][1]);
      }
#pragma unroll
      for (int t = 0; t < kDT; ++t) {
        const V8 of = Bl::col_frag(lo, t, u, lane), qf = Bl::col_frag(lq, t, u, lane);
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          dv[j][t] = mma<Tr>(of, pf[j], dv[j][t]);
          dk[j][t] = mma<Tr>(qf, df[j], dk[j][t]);
        }
      }
    }
  });
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    const int key = key0 + (wave * kNT + j) * 16 + l16;
    if (key >= a.nk) continue;
    const bool live = key < s.klen;  // a column behind the length holds P of zeros, not a gradient
    if constexpr (GradScale<Tr>::kOn) {
      const float rk = gsc[j].undo(), rv = ldexpf(1.f, -(int)kShiftP<Tr>);
#pragma unroll
      for (int t = 0; t < kDT; ++t) dk[j][t] *= rk, dv[j][t] *= rv;
    }
    if (gridDim.y > 1) {
      float* to = a.kv_part + (((int64_t)blockIdx.y * a.b * a.hk + bh) * a.nk + key) * (2 * kDP) + g * 4;
#pragma unroll
      for (int t = 0; t < kDT; ++t) {
        *(f32x4*)(to + t * 16) = dk[j][t];
        *(f32x4*)(to + kDP + t * 16) = dv[j][t];
      }
      continue;
    }
    T* pk = (T*)a.dk + b * a.dks[0] + (int64_t)key * a.dks[1] + hk * a.dks[2];
    T* pv = (T*)a.dv + b * a.dvs[0] + (int64_t)key * a.dvs[1] + hk * a.dvs[2];
#pragma unroll
    for (int t = 0; t < kDT; ++t) {
      const f32x4 z{0.f, 0.f, 0.f, 0.f};
      store_out<Tr>(pk, t * 16 + g * 4, a.d, live ? dk[j][t] * a.scale : z);
      store_out<Tr>(pv, t * 16 + g * 4, a.d, live ? dv[j][t] : z);
    }
  }
}

// The row ranges' sums of dk and dv added in order: 4 elements of a key's row per thread.
template <class Tr>
__global__ __launch_bounds__(256) void attn_dkv_sum_kernel(AttnArgs a, int dp, int splits) {
  using T = typename Tr::T;
  const int per = dp / 2, c = threadIdx.x % per;  // (dp / 4 quads of dk, then of dv)
  const int64_t keys = (int64_t)a.b * a.hk * a.nk, id = (int64_t)blockIdx.x * (256 / per) + threadIdx.x / per;
  if (threadIdx.x >= 256 / per * per || id >= keys) return;
  const int bh = (int)(id / a.nk), key = (int)(id - (int64_t)bh * a.nk), b = bh / a.hk, hk = bh - b * a.hk;
  f32x4 v{0.f, 0.f, 0.f, 0.f};
  if (key < clamp_len(a.lengths, b, a.nk)) {
    const float* p = a.kv_part + id * (2 * dp) + c * 4;
    for (int s = 0; s < splits; ++s) v += *(const f32x4*)(p + s * keys * (2 * dp));
  }
  const bool k = c < per / 2;
  T* to = k ? (T*)a.dk + b * a.dks[0] + (int64_t)key * a.dks[1] + hk * a.dks[2]
            : (T*)a.dv + b * a.dvs[0] + (int64_t)key * a.dvs[1] + hk * a.dvs[2];
  store_out<Tr>(to, (k ? c : c - per / 2) * 4, a.d, k ? v * a.scale : v);
}

// The key ranges' sums of dq added in order: 4 elements of a packed row per thread.
template <class Tr>
__global__ __launch_bounds__(256) void attn_dq_sum_kernel(AttnArgs a, int dp, int splits) {
  using T = typename Tr::T;
  const int per = dp / 4, c = threadIdx.x % per;
  const int64_t all = (int64_t)a.b * a.hk * a.rows, id = (int64_t)blockIdx.x * (256 / per) + threadIdx.x / per;
  if (threadIdx.x >= 256 / per * per || id >= all) return;
  const int bh = (int)(id / a.rows), r = (int)(id - (int64_t)bh * a.rows), b = bh / a.hk, hk = bh - b * a.hk;
  f32x4 v{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) v += *(const f32x4*)(a.q_part + (s * all + id) * dp + c * 4);
  store_out<Tr>(row_ptr((T*)a.dq, a.dqs, b, hk, a.group, r), c * 4, a.d, v * a.scale);
}

// dq: 4 waves of 16 kNT rows, key blocks (k, v) through LDS; with few rows, blockIdx.y a range of the keys,
// whose float32 sums attn_dq_sum_kernel adds.  bf16, 4 x 5120 x 5120, 8 heads of 64: 325-345 us under the
// profiler, 934-991 TFLOP/s; fp16 337-350.
template <class Tr, int kDP, int kNT, bool kAsync>
__global__ __launch_bounds__(256, kWavesPerSimd<Tr>) void attn_dq_kernel(AttnArgs a, int row_blocks) {
  using T = typename Tr::T;
  using V8 = typename Tr::V8;
  using Bl = Block<Tr, kDP>;
  constexpr int kKT = Bl::kBN / 16, kS = kDP / 32, kDT = kDP / 16, kRows = 64 * kNT, kBuf = 2 * Bl::kBytesAll;
  __shared__ __attribute__((aligned(16))) char lds[2 * kBuf];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const int bh = item / row_blocks, rb = a.causal ? row_blocks - 1 - (item - bh * row_blocks) : item - bh * row_blocks;
  const int b = bh / a.hk, hk = bh - b * a.hk;
  const Seq s = seq_of(a, b);
  const int r0 = rb * kRows;
  const int64_t all = (int64_t)a.b * a.hk * a.rows;
  const float* lse2 = a.part + (int64_t)bh * a.rows;
  V8 qf[kNT][kS], of[kNT][kS];
  int lim[kNT];
  float ls[kNT], dl[kNT];
  f32x4 dq[kNT][kDT];
  GradScale<Tr> gsc[kNT];
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    const int r = r0 + (wave * kNT + j) * 16 + l16;
    lim[j] = key_limit(a, s, r);
    ls[j] = lim[j] > 0 ? lse2[r] : INFINITY;
    dl[j] = lim[j] > 0 ? lse2[all + r] : 0.f;
#pragma unroll
    for (int c = 0; c < kS; ++c) {
      qf[j][c] = load8<Tr>(row_ptr((const T*)a.q, a.qs, b, hk, a.group, r), (const T*)a.q, c * 32 + g * 8, a.d, lim[j] > 0);
      of[j][c] = load8<Tr>(row_ptr((const T*)a.go, a.gos, b, hk, a.group, r), (const T*)a.go, c * 32 + g * 8, a.d, lim[j] > 0);
    }
#pragma unroll
    for (int t = 0; t < kDT; ++t) dq[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float sl2 = a.scale * kLog2e;
  Feed<Tr, kDP, kAsync> fk, fv;
  int k_begin = 0, k_stop = key_end(a, s, r0, kRows);
  if (gridDim.y > 1) key_range<Bl::kBN>(k_begin, k_stop);
  fk.init(a.k, a.ks, b, hk, 1, a.d, k_begin);
  fv.init(a.v, a.vs, b, hk, 1, a.d, k_begin);
  for_blocks<Tr, kDP, kAsync>(fk, fv, k_begin, k_stop, s.klen, lds, kBuf, [](char*, int) {}, [&](const char* lk, int k0) {
    const char* lv = lk + Bl::kBytesAll;
#pragma unroll
    for (int u = 0; u < kKT / 2; ++u) {
      f32x4 p[kNT][2], ds[kNT][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = 2 * u + h;
#pragma unroll
        for (int j = 0; j < kNT; ++j) p[j][h] = ds[j][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kS; ++c) {
          const V8 kf = Bl::row_frag(lk, t, c, lane), vf = Bl::row_frag(lv, t, c, lane);
#pragma unroll
          for (int j = 0; j < kNT; ++j) {
            p[j][h] = mma<Tr>(kf, qf[j][c], p[j][h]);
            ds[j][h] = mma<Tr>(vf, of[j][c], ds[j][h]);
          }
        }
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) p[j][h][i] = exp2_f(fmaf(p[j][h][i], sl2, -ls[j]));
          if (__any(lim[j] < k0 + Bl::kBN)) {
            const int left = lim[j] - k0 - g * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) p[j][h][i] = t * 16 + i < left ? p[j][h][i] : 0.f;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            ds[j][h][i] = p[j][h][i] * (GradScale<Tr>::kOn ? fmaf(ds[j][h][i], gsc[j].c, -dl[j] * gsc[j].c) : ds[j][h][i] - dl[j]);
        }
      }
      V8 df[kNT];
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        gsc[j].fit(ds[j], [&](float f) {
#pragma unroll
          for (int t = 0; t < kDT; ++t) dq[j][t] *= f;
        });
        df[j] = pack8<Tr>(ds[j][0], ds[j][1]);
      }
#pragma unroll
      for (int t = 0; t < kDT; ++t) {
        const V8 kf = Bl::col_frag(lk, t, u, lane);
#pragma unroll
        for (int j = 0; j < kNT; ++j) dq[j][t] = mma<Tr>(kf, df[j], dq[j][t]);
      }
    }
  });
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    const int r = r0 + (wave * kNT + j) * 16 + l16;
    if (r >= a.rows) continue;
    const bool live = lim[j] > 0;
    if constexpr (GradScale<Tr>::kOn) {
      const float rq = gsc[j].undo();
#pragma unroll
      for (int t = 0; t < kDT; ++t) dq[j][t] *= rq;
    }
    if (gridDim.y > 1) {
      float* to = a.q_part + (((int64_t)blockIdx.y * a.b * a.hk + bh) * a.rows + r) * kDP + g * 4;
#pragma unroll
      for (int t = 0; t < kDT; ++t) *(f32x4*)(to + t * 16) = live ? dq[j][t] : f32x4{0.f, 0.f, 0.f, 0.f};
      continue;
    }
    T* p = row_ptr((T*)a.dq, a.dqs, b, hk, a.group, r);
#pragma unroll
    for (int t = 0; t < kDT; ++t)
      store_out<Tr>(p, t * 16 + g * 4, a.d, live ? dq[j][t] * a.scale : f32x4{0.f, 0.f, 0.f, 0.f});
  }
}

// ---- launch rules -----------------------------------------------------------------------------
constexpr int kCUs = 256;
inline int pad_d(int d) { return (d + 31) / 32 * 32; }
// Two 16-wide tiles per wave (a fragment read from LDS serves both) where they fit the registers:
// 16-bit heads, while the workgroups still fill the chip.  dk and dv (two sets of sums): at d = 96
// only, 775 against 1018 us for 4 x 4096 x 16 heads; up to 64 one tile is as fast, and faster where
// rows are causal or few (8 x 1280 x 8 heads of 40: 72 against 80), at 128 two do not fit
inline bool two_tiles(int64_t bh, int64_t n) { return bh * cdiv(n, 128) >= kCUs; }
// Rows of a key head that attn_split_kernel takes (128 rows against 16384 keys: 13.6 us, in row blocks 42; from there
// on the row blocks, which share their keys' reads, are as many).
constexpr int64_t kFewRows = 128;
// Key ranges of the forward pass.  Few rows: two workgroups per CU, and at least four slabs for each wave of
// one.  Else one where the workgroups fill the chip, or as many as fill it twice, of 16 blocks at least
// (bf16, 8192 x 8192, one head of 64: 77 us whole, 37 in four; 1280 x 1280, 8 heads: 16 whole, 19 in two of 10).
inline int split_count(int bytes, int64_t bh, int64_t rows, int64_t nk) {
  int64_t s;
  if (rows <= kFewRows) {
    s = cdiv(2 * kCUs, bh * cdiv(rows, 16));
    const int64_t most = cdiv(nk, 512);
    return (int)(s > most ? most > 1 ? most : 1 : s > 256 ? 256 : s);
  }
  const int64_t wgs = bh * cdiv(rows, 64), most = cdiv(nk, 128 / bytes) / 16;
  s = wgs < kCUs ? cdiv(2 * kCUs, wgs) : 1;
  return (int)(s > most ? most > 1 ? most : 1 : s > 64 ? 64 : s);
}

// What Feed's kAsync needs of one operand: chunks whole and on 16-byte boundaries, a block's offsets
// below 2^30.
inline bool feed_async(const char* p, const int64_t* st, int d, int group, int bytes) {
  const int64_t bn = 128 / bytes;
  for (int i = 0; i < 3; ++i)
    if (st[i] * bytes % 16) return false;
  return (uintptr_t)p % 16 == 0 && d * bytes % 16 == 0 && bn % group == 0 && st[1] >= 0 && st[2] >= 0 &&
         (bn / group * st[1] + group * st[2]) * bytes < (int64_t(1) << 30);
}

// Ranges of the backward kernels (rows for dk / dv, keys for dq: `n` of the side that stays, `over` of
// the one that is walked): one where the workgroups fill the chip, else as many as fill it twice, of
// two blocks at least (5 x 333 tokens, 3 heads on a key head, float32: dk / dv 61 us whole, 17 in eight;
// one query against 12731 keys, 48 heads of 80, forward and backward: 528 us with dq whole, 261 split).
inline int range_splits(int bytes, int64_t bh, int64_t n, int64_t over) {
  const int64_t wgs = bh * cdiv(n, 64), blocks = cdiv(over, 128 / bytes);
  int64_t s = wgs < kCUs ? cdiv(2 * kCUs, wgs) : 1;
  if (s > blocks / 2) s = blocks / 2;
  return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
}
inline int64_t stat_words(int64_t bh, int64_t rows) { return cdiv(2 * bh * rows, 4) * 4; }

// Whether a launch holds the workgroups of every kernel of a call.  Forward: of 16 rows, or of 64 (128
// where two_tiles takes them); joins are of calls with few workgroups only.  Backward: 16 rows' statistics, 64 (128)
// rows and 64 keys.
inline bool fits_launch(const AttnArgs& a, int bytes, bool bwd) {
  const int64_t bh = (int64_t)a.b * a.hk, most = most_groups(256);
  const bool two = bytes == 2 && two_tiles(bh, a.rows) && feed_async(a.k, a.ks, a.d, 1, bytes) && feed_async(a.v, a.vs, a.d, 1, bytes);
  if (!bwd) return bh * cdiv(a.rows, a.rows <= kFewRows ? 16 : two ? 128 : 64) <= most;
  return cdiv(bh * a.rows, 16) <= most && bh * cdiv(a.rows, two ? 128 : 64) <= most && bh * cdiv(a.nk, 64) <= most;
}

template <class Tr, int kDP>
void run_split(const AttnArgs& a, hipStream_t st) {
  const int64_t bh = (int64_t)a.b * a.hk;
  const int rb = (int)cdiv(a.rows, 16);
  constexpr int kWaves = kDP * Tr::kBytes > 256 ? 2 : 4;  // (as many as have their slabs in 160 KB)
  const dim3 grid((unsigned)(bh * rb), a.splits);
  if (feed_async(a.k, a.ks, a.d, 1, Tr::kBytes) && feed_async(a.v, a.vs, a.d, 1, Tr::kBytes))
    launch((attn_split_kernel<Tr, kDP, kWaves, true>), grid, dim3(64 * kWaves), 0, st, a, rb);
  else
    launch((attn_split_kernel<Tr, kDP, kWaves, false>), grid, dim3(64 * kWaves), 0, st, a, rb);
  if (a.splits > 1)
    launch(attn_join_kernel<Tr>, dim3((unsigned)(bh * a.rows)), dim3(256), 0, st, a, rb, kDP);
}

template <class Tr, int kDP, int kNT, bool kAsync = true>
void launch_fwd(const AttnArgs& a, hipStream_t st) {
  const int rb = (int)cdiv(a.rows, 64 * kNT);
  launch((attn_kernel<Tr, kDP, kNT, kAsync>), dim3((unsigned)((int64_t)a.b * a.hk * rb), a.splits), dim3(256), 0, st, a, rb);
  if (a.splits > 1)
    launch(attn_join_rows_kernel<Tr>, dim3((unsigned)cdiv((int64_t)a.b * a.hk * a.rows, 256 / (kDP / 4))), dim3(256), 0, st,
                       a, kDP);
}
template <class Tr, int kDP, int kNT, bool kAsync = true>
void launch_dkv(const AttnArgs& a, hipStream_t st) {
  const int kb = (int)cdiv(a.nk, 64 * kNT), s = a.splits;
  launch((attn_dkv_kernel<Tr, kDP, kNT, kAsync>), dim3((unsigned)((int64_t)a.b * a.hk * kb), s), dim3(256), 0, st, a, kb);
  if (s > 1)
    launch(attn_dkv_sum_kernel<Tr>, dim3((unsigned)cdiv((int64_t)a.b * a.hk * a.nk, 256 / (kDP / 2))), dim3(256), 0, st,
                       a, kDP, s);
}
template <class Tr, int kDP, int kNT, bool kAsync = true>
void launch_dq(const AttnArgs& a, hipStream_t st) {
  const int rb = (int)cdiv(a.rows, 64 * kNT), s = a.key_splits;
  launch((attn_dq_kernel<Tr, kDP, kNT, kAsync>), dim3((unsigned)((int64_t)a.b * a.hk * rb), s), dim3(256), 0, st, a, rb);
  if (s > 1)
    launch(attn_dq_sum_kernel<Tr>, dim3((unsigned)cdiv((int64_t)a.b * a.hk * a.rows, 256 / (kDP / 4))), dim3(256), 0, st,
                       a, kDP, s);
}

template <class Tr, int kDP>
void run_fwd(const AttnArgs& a, hipStream_t st) {
  constexpr int kTwo = Tr::kBytes == 2 ? 2 : 1;
  const int64_t bh = (int64_t)a.b * a.hk;
  if (!feed_async(a.k, a.ks, a.d, 1, Tr::kBytes) || !feed_async(a.v, a.vs, a.d, 1, Tr::kBytes)) launch_fwd<Tr, kDP, 1, false>(a, st);
  else if (two_tiles(bh, a.rows)) launch_fwd<Tr, kDP, kTwo>(a, st);
  else launch_fwd<Tr, kDP, 1>(a, st);
}

template <class Tr, int kDP>
void run_bwd(const AttnArgs& a, hipStream_t st) {
  const int64_t bh = (int64_t)a.b * a.hk;
  launch(attn_delta_kernel<Tr>, dim3((unsigned)cdiv(bh * a.rows, 16)), dim3(256), 0, st, a);
  const bool rows = feed_async(a.q, a.qs, a.d, a.group, Tr::kBytes) && feed_async(a.go, a.gos, a.d, a.group, Tr::kBytes);
  const bool keys = feed_async(a.k, a.ks, a.d, 1, Tr::kBytes) && feed_async(a.v, a.vs, a.d, 1, Tr::kBytes);
  constexpr int kTwo = Tr::kBytes == 2 ? 2 : 1, kTwoKeys = kDP == 96 ? kTwo : 1;
  if (!rows) launch_dkv<Tr, kDP, 1, false>(a, st);
  else if (two_tiles(bh, a.nk)) launch_dkv<Tr, kDP, kTwoKeys>(a, st);
  else launch_dkv<Tr, kDP, 1>(a, st);
  if (!keys) launch_dq<Tr, kDP, 1, false>(a, st);
  else if (two_tiles(bh, a.rows)) launch_dq<Tr, kDP, kTwo>(a, st);
  else launch_dq<Tr, kDP, 1>(a, st);
}

template <class Tr>
void run_attn(const AttnArgs& a, bool bwd, hipStream_t st) {
  if (!bwd && a.rows <= kFewRows) {
    switch (pad_d(a.d)) {
      case 32: run_split<Tr, 32>(a, st); break;
      case 64: run_split<Tr, 64>(a, st); break;
      case 96: run_split<Tr, 96>(a, st); break;
      default: run_split<Tr, 128>(a, st); break;
    }
    return;
  }
  switch (pad_d(a.d)) {
    case 32: bwd ? run_bwd<Tr, 32>(a, st) : run_fwd<Tr, 32>(a, st); break;
    case 64: bwd ? run_bwd<Tr, 64>(a, st) : run_fwd<Tr, 64>(a, st); break;
    case 96: bwd ? run_bwd<Tr, 96>(a, st) : run_fwd<Tr, 96>(a, st); break;
    default: bwd ? run_bwd<Tr, 128>(a, st) : run_fwd<Tr, 128>(a, st); break;
  }
}

template <class A>
int check_attn(const char* fn, const A* a) {
  YK_CHECK_ARG(tok_bytes(a->dtype), std::string(fn) + ": dtype must be YK_ACT_BF16, YK_ACT_F32 or YK_ACT_F16");
  YK_CHECK_ARG(a->b >= 0 && a->h_q >= 1 && a->h_kv >= 1 && a->h_q % a->h_kv == 0,
               std::string(fn) + ": heads must be >= 1 and h_q a multiple of h_kv");
  YK_CHECK_ARG(a->d >= 1 && a->d <= 128, std::string(fn) + ": head size must be in [1, 128]");
  YK_CHECK_ARG(a->nq >= 0 && a->nk >= 0 && a->nk < (1 << 30) && a->nq * (a->h_q / a->h_kv) < (1 << 30),
               std::string(fn) + ": sizes out of range (nk and nq * h_q / h_kv below 2^30)");
  YK_CHECK_ARG((int64_t)a->b * a->h_kv * cdiv(a->nq * (a->h_q / a->h_kv), 16) < (int64_t(1) << 31) &&
                   (int64_t)a->b * a->h_kv * cdiv(a->nk, 64) < (int64_t(1) << 31),
               std::string(fn) + ": more work items than a launch holds");
  YK_CHECK_ARG(a->scale > 0.f && a->scale < INFINITY, std::string(fn) + ": scale must be positive and finite");
  return YK_OK;
}
template <class A>
AttnArgs common_args(const A* a) {
  AttnArgs k{};
  k.q = (const char*)a->q, k.k = (const char*)a->k, k.v = (const char*)a->v;
  k.q_lengths = a->q_lengths, k.lengths = a->lengths;
  for (int i = 0; i < 3; ++i) k.qs[i] = a->q_stride[i], k.ks[i] = a->k_stride[i], k.vs[i] = a->v_stride[i], k.os[i] = a->o_stride[i];
  k.scale = a->scale;
  k.b = a->b, k.hk = a->h_kv, k.group = a->h_q / a->h_kv, k.d = a->d, k.nq = (int)a->nq, k.nk = (int)a->nk;
  k.causal = a->causal != 0;
  k.rows = k.nq * k.group;
  k.part = (float*)a->ws;
  return k;
}

}  // namespace tok
}  // namespace yk

using namespace yk::tok;

extern "C" {

int yk_attention_workspace(const yk_attention_args* a, int64_t* bytes) {
  YK_CHECK_ARG(a && bytes, "yk_attention_workspace: NULL argument");
  if (const int rc = check_attn("yk_attention_workspace", a)) return rc;
  const int64_t bh = (int64_t)a->b * a->h_kv, rows = a->nq * (a->h_q / a->h_kv);
  *bytes = 0;
  if (bh == 0 || rows == 0) return YK_OK;
  const int s = split_count(tok_bytes(a->dtype), bh, rows, a->nk);
  if (s > 1) *bytes = bh * cdiv(rows, 16) * s * 16 * (pad_d(a->d) + 4) * 4;
  return YK_OK;
}

int yk_attention(yk_ctx* ctx, const yk_attention_args* a, void* stream) {
  YK_CHECK_ARG(ctx && a, "yk_attention: NULL argument");
  if (const int rc = check_attn("yk_attention", a)) return rc;
  if (a->b == 0 || a->nq == 0) return YK_OK;
  YK_CHECK_ARG(a->q && a->o && (a->nk == 0 || (a->k && a->v)), "yk_attention: q, k, v and o must be set");
  int64_t need = 0;
  if (const int rc = yk_attention_workspace(a, &need)) return rc;
  YK_CHECK_ARG(need == 0 || !a->ws || (a->ws_bytes >= need && (uintptr_t)a->ws % 16 == 0),
               "yk_attention: ws must be yk_attention_workspace bytes, 16-byte aligned (or NULL: the keys are not split)");
  yk::DeviceGuard g(ctx->device);
  AttnArgs k = common_args(a);
  k.out = (char*)a->o;
  k.lse = a->lse;
  k.splits = split_count(tok_bytes(a->dtype), (int64_t)k.b * k.hk, k.rows, k.nk);
  if (k.splits > 1 && !a->ws) k.splits = 1;
  YK_CHECK_ARG(fits_launch(k, tok_bytes(a->dtype), false), "yk_attention: more work items than a launch holds");
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == YK_ACT_F32) run_attn<F32>(k, false, st);
  else if (a->dtype == YK_ACT_BF16) run_attn<B16>(k, false, st);
  else run_attn<H16>(k, false, st);
  return launched("yk_attention");
}

int yk_attention_backward_workspace(const yk_attention_grad_args* a, int64_t* bytes) {
  YK_CHECK_ARG(a && bytes, "yk_attention_backward_workspace: NULL argument");
  if (const int rc = check_attn("yk_attention_backward_workspace", a)) return rc;
  const int64_t bh = (int64_t)a->b * a->h_kv, rows = a->nq * (a->h_q / a->h_kv);
  *bytes = stat_words(bh, rows) * 4;
  if (bh == 0 || rows == 0 || a->nk == 0) return YK_OK;
  const int s = range_splits(tok_bytes(a->dtype), bh, a->nk, rows), ks = range_splits(tok_bytes(a->dtype), bh, rows, a->nk);
  if (s > 1) *bytes += (int64_t)s * bh * a->nk * 2 * pad_d(a->d) * 4;
  if (ks > 1) *bytes += (int64_t)ks * bh * rows * pad_d(a->d) * 4;
  return YK_OK;
}

int yk_attention_backward(yk_ctx* ctx, const yk_attention_grad_args* a, void* stream) {
  YK_CHECK_ARG(ctx && a, "yk_attention_backward: NULL argument");
  if (const int rc = check_attn("yk_attention_backward", a)) return rc;
  YK_CHECK_ARG(a->nq >= 1 && a->nk >= 1, "yk_attention_backward: nq and nk must be >= 1");
  if (a->b == 0) return YK_OK;
  YK_CHECK_ARG(a->go && a->q && a->k && a->v && a->o && a->lse && a->dq && a->dk && a->dv,
               "yk_attention_backward: every pointer but the lengths must be set");
  int64_t need = 0;
  if (const int rc = yk_attention_backward_workspace(a, &need)) return rc;
  YK_CHECK_ARG(a->ws && a->ws_bytes >= need && (uintptr_t)a->ws % 16 == 0,
               "yk_attention_backward: ws must be yk_attention_backward_workspace bytes, 16-byte aligned");
  yk::DeviceGuard g(ctx->device);
  AttnArgs k = common_args(a);
  k.o = (const char*)a->o, k.go = (const char*)a->go;
  k.dq = (char*)a->dq, k.dk = (char*)a->dk, k.dv = (char*)a->dv;
  k.lse = (float*)a->lse;
  YK_CHECK_ARG(fits_launch(k, tok_bytes(a->dtype), true), "yk_attention_backward: more work items than a launch holds");
  const int64_t bh = (int64_t)k.b * k.hk;
  k.splits = range_splits(tok_bytes(a->dtype), bh, k.nk, k.rows);
  k.key_splits = range_splits(tok_bytes(a->dtype), bh, k.rows, k.nk);
  k.kv_part = k.part + stat_words(bh, k.rows);
  k.q_part = k.kv_part + (k.splits > 1 ? (int64_t)k.splits * bh * k.nk * 2 * pad_d(k.d) : 0);
  for (int i = 0; i < 3; ++i) k.gos[i] = a->go_stride[i], k.dqs[i] = a->dq_stride[i], k.dks[i] = a->dk_stride[i], k.dvs[i] = a->dv_stride[i];
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == YK_ACT_F32) run_attn<F32>(k, true, st);
  else if (a->dtype == YK_ACT_BF16) run_attn<B16>(k, true, st);
  else run_attn<H16>(k, true, st);
  return launched("yk_attention_backward");
}

}  // extern "C"
