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
  float* part;        // split: [item][split][16][d_pad + 2]; backward: lse2, delta [b][hk][rows]
  float scale;
  int b, hk, group, d, nq, nk, causal, rows, splits;  // rows = nq * group
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
// two C tiles of a column -> 8 summands.  16-bit P and dS are rounded to the operands' type.
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

// kBN x kDP block of rows in LDS (kDP = d padded to 32, zero filled), rows 16 bytes apart beyond
// their data so that the 16 rows of a fragment start on different banks.
template <class Tr, int kDP>
struct Block {
  using T = typename Tr::T;
  static constexpr int kBN = 128 / Tr::kBytes;  // 64 rows of 16-bit, 32 of float32
  static constexpr int kEpc = 16 / Tr::kBytes;
  static constexpr int kPitch = kDP * Tr::kBytes + 16;
  static constexpr int kRowChunks = kDP / kEpc;
  static constexpr int kN = kDP / 32;           // chunks per thread of 256
  static constexpr int kBytesAll = kBN * kPitch;

  // A operand: row 16 t + l, elements 32 s + 8 g ..
  static __device__ __forceinline__ typename Tr::V8 row_frag(const char* lds, int t, int s, int lane) {
    const int l = lane & 15, g = lane >> 4;
    return *(const typename Tr::V8*)__builtin_assume_aligned(lds + (t * 16 + l) * kPitch + (s * 32 + g * 8) * Tr::kBytes, 16);
  }
  // A operand, transposed: element 16 dt + l of rows 32 u + {4g .. 4g+3, 16+4g .. 16+4g+3}
  static __device__ __forceinline__ typename Tr::V8 col_frag(const char* lds, int dt, int u, int lane) {
    const int l = lane & 15, g = lane >> 4;
    if constexpr (Tr::kBytes == 2) {
      const char* p = lds + (u * 32 + 4 * g + (l >> 2)) * kPitch + dt * 32 + (l & 3) * 8;
      typedef __attribute__((address_space(3))) s16x4* lp;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 16 * kPitch));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      typename Tr::V8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = *(const float*)(lds + (u * 32 + (e & 4) * 4 + 4 * g + (e & 3)) * kPitch + (dt * 16 + l) * 4);
      return v;
    }
  }
};

template <class Tr, int kDP>
struct Stage {  // a block on its way from memory to LDS, by 256 threads
  using Bl = Block<Tr, kDP>;
  using T = typename Tr::T;
  u32x4 reg[Bl::kN];
  // rows first .. of a key head's keys, below `limit`
  __device__ __forceinline__ void load_keys(const T* base, int64_t stride, int first, int limit, int d) {
#pragma unroll
    for (int i = 0; i < Bl::kN; ++i) {
      const int j = i * 256 + threadIdx.x, row = j / Bl::kRowChunks, c = (j % Bl::kRowChunks) * Bl::kEpc;
      reg[i] = load16_if<Tr>(base + (int64_t)(first + row) * stride + c, base, d - c, first + row < limit, d % Bl::kEpc == 0);
    }
  }
  // packed rows first .. of (b, hk), below `limit`
  __device__ __forceinline__ void load_rows(const T* base, const int64_t* st, int b, int hk, int group, int first,
                                            int limit, int d) {
#pragma unroll
    for (int i = 0; i < Bl::kN; ++i) {
      const int j = i * 256 + threadIdx.x, row = j / Bl::kRowChunks, c = (j % Bl::kRowChunks) * Bl::kEpc;
      reg[i] = load16_if<Tr>(row_ptr(base, st, b, hk, group, first + row) + c, base, d - c, first + row < limit, d % Bl::kEpc == 0);
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < Bl::kN; ++i) {
      const int j = i * 256 + threadIdx.x, row = j / Bl::kRowChunks, c = j % Bl::kRowChunks;
      *(u32x4*)(lds + row * Bl::kPitch + c * 16) = reg[i];
    }
  }
};

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

// One column's running softmax over a block of kT score tiles (raw scores in st; p comes back in
// it), keys beyond `lim` left out.  m is the running maximum of score * scale * log2 e, l this
// lane's share of the denominator.  Returns the factor for what was accumulated before.
template <int kT>
__device__ __forceinline__ float softmax_step(f32x4* st, int key0, int lim, bool mask, float sl2, float& m, float& l) {
  const int g = (threadIdx.x & 63) >> 4;
  if (mask) {
#pragma unroll
    for (int t = 0; t < kT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) st[t][i] = key0 + t * 16 + g * 4 + i < lim ? st[t][i] : -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int t = 0; t < kT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, st[t][i]);
  mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
  const float mn = fmaxf(m, mx * sl2);
  const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: every p is exp2(-inf) = 0
  const float alpha = __builtin_amdgcn_exp2f(m - ref);
  float s = 0.f;
#pragma unroll
  for (int t = 0; t < kT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = __builtin_amdgcn_exp2f(fmaf(st[t][i], sl2, -ref));
      st[t][i] = p;
      s += p;
    }
  l = l * alpha + s;
  m = mn;
  return alpha;
}

// Forward: 4 waves of 16 kNT rows, key blocks through LDS, the next one's loads in flight meanwhile.
template <class Tr, int kDP, int kNT>
__global__ __launch_bounds__(256) void attn_kernel(AttnArgs a, int row_blocks) {
  using T = typename Tr::T;
  using V8 = typename Tr::V8;
  using Bl = Block<Tr, kDP>;
  constexpr int kKT = Bl::kBN / 16, kS = kDP / 32, kDT = kDP / 16, kRows = 64 * kNT;
  __shared__ __attribute__((aligned(16))) char lk[Bl::kBytesAll], lv[Bl::kBytesAll];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int item = xcd_item(blockIdx.x, gridDim.x);
  // long causal rows first
  const int bh = item / row_blocks, rb = a.causal ? row_blocks - 1 - (item - bh * row_blocks) : item - bh * row_blocks;
  const int b = bh / a.hk, hk = bh - b * a.hk;
  const Seq s = seq_of(a, b);
  const int r0 = rb * kRows;
  const T* kb = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vb = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
  const int last = (r0 + kRows < a.rows ? r0 + kRows : a.rows) - 1;
  // the last row in use of this block sees most
  int kend = s.klen;
  if (query_of(r0, a.group) >= s.qlen) {
    kend = 0;
  } else if (a.causal) {
    int i = query_of(last, a.group);
    i = i < s.qlen ? i : s.qlen - 1;
    kend = i + s.off + 1;
  }
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
  Stage<Tr, kDP> sk, sv;
  if (kend > 0) {
    sk.load_keys(kb, a.ks[1], 0, s.klen, a.d);
    sv.load_keys(vb, a.vs[1], 0, s.klen, a.d);
  }
  for (int k0 = 0; k0 < kend; k0 += Bl::kBN) {
    __syncthreads();
    sk.store(lk);
    sv.store(lv);
    __syncthreads();
    if (k0 + Bl::kBN < kend) {
      sk.load_keys(kb, a.ks[1], k0 + Bl::kBN, s.klen, a.d);
      sv.load_keys(vb, a.vs[1], k0 + Bl::kBN, s.klen, a.d);
    }
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
      const bool mask = __any(lim[j] < k0 + Bl::kBN);
      const float alpha = softmax_step<kKT>(st[j], k0, lim[j], mask, sl2, m[j], l[j]);
#pragma unroll
      for (int t = 0; t < kDT; ++t) acc[j][t] *= alpha;
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
  }
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    const int r = r0 + (wave * kNT + j) * 16 + l16;
    l[j] += __shfl_xor(l[j], 16, 64);
    l[j] += __shfl_xor(l[j], 32, 64);
    if (r >= a.rows) continue;
    const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
    T* o = row_ptr((T*)a.out, a.os, b, hk, a.group, r);
#pragma unroll
    for (int t = 0; t < kDT; ++t) store_out<Tr>(o, t * 16 + g * 4, a.d, acc[j][t] * inv);
    if (a.lse && g == 0) {
      const int i = query_of(r, a.group);
      a.lse[((int64_t)(b * a.hk + hk) * a.group + (r - i * a.group)) * a.nq + i] =
          l[j] == 0.f ? -INFINITY : fmaf(m[j], kLn2, logf(l[j]));
    }
  }
}

// Few rows, long keys: 16 rows per workgroup, whose waves walk different key blocks on their own
// (fragments of k straight from memory, v through a wave's own LDS), and blockIdx.y a range of
// keys.  The waves' sums meet in LDS; ranges go to scratch unless there is one.
template <class Tr, int kDP>
__global__ __launch_bounds__(256) void attn_split_kernel(AttnArgs a, int row_blocks) {
  using T = typename Tr::T;
  using V8 = typename Tr::V8;
  using Bl = Block<Tr, kDP>;
  constexpr int kKT = Bl::kBN / 16, kS = kDP / 32, kDT = kDP / 16, kVN = Bl::kN * 4;
  __shared__ __attribute__((aligned(16))) char lds[4 * Bl::kBytesAll];
  __shared__ float stat[4][2][16];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int bh = blockIdx.x / row_blocks, rb = blockIdx.x - bh * row_blocks;
  const int b = bh / a.hk, hk = bh - b * a.hk;
  const Seq s = seq_of(a, b);
  const int r = rb * 16 + l16;
  const int lim = key_limit(a, s, r);
  const T* kb = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vb = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
  // the range of this workgroup: whole key blocks
  const int blocks = (s.klen + Bl::kBN - 1) / Bl::kBN, per = (blocks + a.splits - 1) / a.splits;
  const int k_begin = blockIdx.y * per * Bl::kBN;
  int k_end = k_begin + per * Bl::kBN < s.klen ? k_begin + per * Bl::kBN : s.klen;
  V8 qf[kS];
#pragma unroll
  for (int c = 0; c < kS; ++c)
    qf[c] = load8<Tr>(row_ptr((const T*)a.q, a.qs, b, hk, a.group, r), (const T*)a.q, c * 32 + g * 8, a.d, lim > 0);
  float m = -INFINITY, l = 0.f;
  f32x4 acc[kDT];
#pragma unroll
  for (int t = 0; t < kDT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float sl2 = a.scale * kLog2e;
  char* lv = lds + wave * Bl::kBytesAll;
  for (int k0 = k_begin + wave * Bl::kBN; k0 < k_end; k0 += 4 * Bl::kBN) {
    V8 kf[kKT][kS];
    u32x4 vr[kVN];
#pragma unroll
    for (int t = 0; t < kKT; ++t)
#pragma unroll
      for (int c = 0; c < kS; ++c) {
        const int key = k0 + t * 16 + l16;
        kf[t][c] = load8<Tr>(kb + (int64_t)key * a.ks[1], kb, c * 32 + g * 8, a.d, key < k_end);
      }
#pragma unroll
    for (int i = 0; i < kVN; ++i) {
      const int j = i * 64 + lane, row = j / Bl::kRowChunks, c = (j % Bl::kRowChunks) * Bl::kEpc;
      vr[i] = load16_if<Tr>(vb + (int64_t)(k0 + row) * a.vs[1] + c, vb, a.d - c, k0 + row < k_end, a.d % Bl::kEpc == 0);
    }
    f32x4 st[kKT];
#pragma unroll
    for (int t = 0; t < kKT; ++t) {
      st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kS; ++c) st[t] = mma<Tr>(kf[t][c], qf[c], st[t]);
    }
    const int lim2 = lim < k_end ? lim : k_end;
    const float alpha = softmax_step<kKT>(st, k0, lim2, __any(lim2 < k0 + Bl::kBN), sl2, m, l);
#pragma unroll
    for (int t = 0; t < kDT; ++t) acc[t] *= alpha;
#pragma unroll
    for (int i = 0; i < kVN; ++i) {
      const int j = i * 64 + lane, row = j / Bl::kRowChunks, c = j % Bl::kRowChunks;
      *(u32x4*)(lv + row * Bl::kPitch + c * 16) = vr[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int u = 0; u < kKT / 2; ++u) {
      const V8 pf = pack8<Tr>(st[2 * u], st[2 * u + 1]);
#pragma unroll
      for (int t = 0; t < kDT; ++t) acc[t] = mma<Tr>(Bl::col_frag(lv, t, u, lane), pf, acc[t]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) {
    stat[wave][0][l16] = m;
    stat[wave][1][l16] = l;
  }
  __syncthreads();  // (also: every wave is done with its part of lds)
  float mm = stat[0][0][l16];
#pragma unroll
  for (int w = 1; w < 4; ++w) mm = fmaxf(mm, stat[w][0][l16]);
  const float ref = mm == -INFINITY ? 0.f : mm;
  const float f = __builtin_amdgcn_exp2f(m - ref);
  float ll = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) ll += stat[w][1][l16] * __builtin_amdgcn_exp2f(stat[w][0][l16] - ref);
  float* sum = (float*)lds;  // [4 waves][kDT][64 lanes][4]
#pragma unroll
  for (int t = 0; t < kDT; ++t) *(f32x4*)(sum + ((wave * kDT + t) * 64 + lane) * 4) = acc[t] * f;
  __syncthreads();
  if (r >= a.rows) return;
  const bool one = a.splits == 1;
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  float* part = one ? nullptr : a.part + (((int64_t)blockIdx.x * a.splits + blockIdx.y) * 16 + l16) * (kDP + 2);
  for (int t = wave; t < kDT; t += 4) {
    f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) v += *(const f32x4*)(sum + ((w * kDT + t) * 64 + lane) * 4);
    if (one) {
      store_out<Tr>(row_ptr((T*)a.out, a.os, b, hk, a.group, r), t * 16 + g * 4, a.d, v * inv);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) part[t * 16 + g * 4 + i] = v[i];
    }
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

// The ranges of one row joined in order: a wave per row, two elements of it per lane.
template <class Tr>
__global__ __launch_bounds__(64) void attn_join_kernel(AttnArgs a, int row_blocks, int dp) {
  using T = typename Tr::T;
  const int lane = threadIdx.x, bh = blockIdx.x / a.rows, r = blockIdx.x - bh * a.rows;
  const int b = bh / a.hk, hk = bh - b * a.hk;
  const float* p = a.part + (((int64_t)(bh * row_blocks + r / 16) * a.splits) * 16 + r % 16) * (dp + 2);
  const int64_t step = (int64_t)16 * (dp + 2);
  float mm = -INFINITY;
  for (int s = 0; s < a.splits; ++s) mm = fmaxf(mm, p[s * step + dp]);
  const float ref = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f, v0 = 0.f, v1 = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float* q = p + s * step;
    const float f = __builtin_amdgcn_exp2f(q[dp] - ref);
    ll += q[dp + 1] * f;
    if (lane < a.d) v0 += q[lane] * f;
    if (lane + 64 < a.d) v1 += q[lane + 64] * f;
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  T* o = row_ptr((T*)a.out, a.os, b, hk, a.group, r);
  if (lane < a.d) o[lane] = from_f32<Tr>(v0 * inv);
  if (lane + 64 < a.d) o[lane + 64] = from_f32<Tr>(v1 * inv);
  if (a.lse && lane == 0) {
    const int i = query_of(r, a.group);
    a.lse[((int64_t)(b * a.hk + hk) * a.group + (r - i * a.group)) * a.nq + i] = ll == 0.f ? -INFINITY : fmaf(mm, kLn2, logf(ll));
  }
}

// Row statistics of the backward pass in packed-row order: lse * log2 e (+infinity where a row has
// no key, which makes its P zero) and delta = sum over d of do o.  16 lanes per row.
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
  a.part[id] = lse == -INFINITY ? INFINITY : lse * kLog2e;
  a.part[all + id] = s;
}

// dk and dv: 4 waves of 16 kNT keys, blocks of packed rows (q, do) through LDS.
template <class Tr, int kDP, int kNT>
__global__ __launch_bounds__(256) void attn_dkv_kernel(AttnArgs a, int key_blocks) {
  using T = typename Tr::T;
  using V8 = typename Tr::V8;
  using Bl = Block<Tr, kDP>;
  constexpr int kRT = Bl::kBN / 16, kS = kDP / 32, kDT = kDP / 16, kKeys = 64 * kNT;
  __shared__ __attribute__((aligned(16))) char lq[Bl::kBytesAll], lo[Bl::kBytesAll];
  __shared__ __attribute__((aligned(16))) float stat[2][Bl::kBN];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const int bh = item / key_blocks, key0 = (item - bh * key_blocks) * kKeys;
  const int b = bh / a.hk, hk = bh - b * a.hk;
  const Seq s = seq_of(a, b);
  const int64_t all = (int64_t)a.b * a.hk * a.rows;
  const float* lse2 = a.part + (int64_t)bh * a.rows;
  V8 kf[kNT][kS], vf[kNT][kS];
  f32x4 dk[kNT][kDT], dv[kNT][kDT];
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
  const float sl2 = a.scale * kLog2e;
  Stage<Tr, kDP> sq, so;
  float st_lse = 0.f, st_delta = 0.f;
  auto fetch = [&](int r0) {
    sq.load_rows((const T*)a.q, a.qs, b, hk, a.group, r0, r_end, a.d);
    so.load_rows((const T*)a.go, a.gos, b, hk, a.group, r0, r_end, a.d);
    if (threadIdx.x < Bl::kBN) {
      const int r = r0 + threadIdx.x;
      st_lse = r < r_end ? lse2[r] : INFINITY;
      st_delta = r < r_end ? lse2[all + r] : 0.f;
    }
  };
  if (r_begin < r_end) fetch(r_begin);
  for (int r0 = r_begin; r0 < r_end; r0 += Bl::kBN) {
    __syncthreads();
    sq.store(lq);
    so.store(lo);
    if (threadIdx.x < Bl::kBN) {
      stat[0][threadIdx.x] = st_lse;
      stat[1][threadIdx.x] = st_delta;
    }
    __syncthreads();
    if (r0 + Bl::kBN < r_end) fetch(r0 + Bl::kBN);
    // the block's first query sees least
    const int sees = query_of(r0, a.group) + s.off;
    const bool mask = a.causal && key0 + kKeys - 1 > sees;
#pragma unroll
    for (int u = 0; u < kRT / 2; ++u) {
      f32x4 p[kNT][2], ds[kNT][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = 2 * u + h;
#pragma unroll
        for (int j = 0; j < kNT; ++j) p[j][h] = ds[j][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kS; ++c) {
          const V8 qf = Bl::row_frag(lq, t, c, lane), of = Bl::row_frag(lo, t, c, lane);
#pragma unroll
          for (int j = 0; j < kNT; ++j) {
            p[j][h] = mma<Tr>(qf, kf[j][c], p[j][h]);
            ds[j][h] = mma<Tr>(of, vf[j][c], ds[j][h]);
          }
        }
        const f32x4 ls = *(const f32x4*)&stat[0][t * 16 + g * 4], dl = *(const f32x4*)&stat[1][t * 16 + g * 4];
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          const int key = key0 + (wave * kNT + j) * 16 + l16;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float e = __builtin_amdgcn_exp2f(fmaf(p[j][h][i], sl2, -ls[i]));
            if (mask && key > query_of(r0 + t * 16 + g * 4 + i, a.group) + s.off) e = 0.f;
            p[j][h][i] = e;
            ds[j][h][i] = e * (ds[j][h][i] - dl[i]);
          }
        }
      }
      V8 pf[kNT], df[kNT];
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
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
  }
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    const int key = key0 + (wave * kNT + j) * 16 + l16;
    if (key >= a.nk) continue;
    const bool live = key < s.klen;  // a column behind the length holds P of zeros, not a gradient
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

// dq: 4 waves of 16 kNT rows, key blocks (k, v) through LDS.
template <class Tr, int kDP, int kNT>
__global__ __launch_bounds__(256) void attn_dq_kernel(AttnArgs a, int row_blocks) {
  using T = typename Tr::T;
  using V8 = typename Tr::V8;
  using Bl = Block<Tr, kDP>;
  constexpr int kKT = Bl::kBN / 16, kS = kDP / 32, kDT = kDP / 16, kRows = 64 * kNT;
  __shared__ __attribute__((aligned(16))) char lk[Bl::kBytesAll], lv[Bl::kBytesAll];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const int bh = item / row_blocks, rb = a.causal ? row_blocks - 1 - (item - bh * row_blocks) : item - bh * row_blocks;
  const int b = bh / a.hk, hk = bh - b * a.hk;
  const Seq s = seq_of(a, b);
  const int r0 = rb * kRows;
  const T* kb = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vb = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
  const int last = (r0 + kRows < a.rows ? r0 + kRows : a.rows) - 1;
  int kend = s.klen;
  if (query_of(r0, a.group) >= s.qlen) {
    kend = 0;
  } else if (a.causal) {
    int i = query_of(last, a.group);
    i = i < s.qlen ? i : s.qlen - 1;
    kend = i + s.off + 1;
  }
  const int64_t all = (int64_t)a.b * a.hk * a.rows;
  const float* lse2 = a.part + (int64_t)bh * a.rows;
  V8 qf[kNT][kS], of[kNT][kS];
  int lim[kNT];
  float ls[kNT], dl[kNT];
  f32x4 dq[kNT][kDT];
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
  Stage<Tr, kDP> sk, sv;
  if (kend > 0) {
    sk.load_keys(kb, a.ks[1], 0, s.klen, a.d);
    sv.load_keys(vb, a.vs[1], 0, s.klen, a.d);
  }
  for (int k0 = 0; k0 < kend; k0 += Bl::kBN) {
    __syncthreads();
    sk.store(lk);
    sv.store(lv);
    __syncthreads();
    if (k0 + Bl::kBN < kend) {
      sk.load_keys(kb, a.ks[1], k0 + Bl::kBN, s.klen, a.d);
      sv.load_keys(vb, a.vs[1], k0 + Bl::kBN, s.klen, a.d);
    }
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
          const bool mask = __any(lim[j] < k0 + Bl::kBN);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float e = __builtin_amdgcn_exp2f(fmaf(p[j][h][i], sl2, -ls[j]));
            if (mask && k0 + t * 16 + g * 4 + i >= lim[j]) e = 0.f;
            ds[j][h][i] = e * (ds[j][h][i] - dl[j]);
          }
        }
      }
      V8 df[kNT];
#pragma unroll
      for (int j = 0; j < kNT; ++j) df[j] = pack8<Tr>(ds[j][0], ds[j][1]);
#pragma unroll
      for (int t = 0; t < kDT; ++t) {
        const V8 kf = Bl::col_frag(lk, t, u, lane);
#pragma unroll
        for (int j = 0; j < kNT; ++j) dq[j][t] = mma<Tr>(kf, df[j], dq[j][t]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
    const int r = r0 + (wave * kNT + j) * 16 + l16;
    if (r >= a.rows) continue;
    T* p = row_ptr((T*)a.dq, a.dqs, b, hk, a.group, r);
    const bool live = lim[j] > 0;
#pragma unroll
    for (int t = 0; t < kDT; ++t)
      store_out<Tr>(p, t * 16 + g * 4, a.d, live ? dq[j][t] * a.scale : f32x4{0.f, 0.f, 0.f, 0.f});
  }
}

// ---- launch rules -----------------------------------------------------------------------------
constexpr int kCUs = 256;
inline int pad_d(int d) { return (d + 31) / 32 * 32; }
// The few-rows kernel pads 96 to 128: it is bound by its loads, and rows of 12 chunks cost it more
// lane masks than there are scalar registers
inline int split_pad(int d) { return pad_d(d) == 96 ? 128 : pad_d(d); }

// Row tiles per wave of the forward and dq kernels (a fragment read from LDS serves all of them):
// two for 16-bit heads while the workgroups still fill the chip
inline int row_tiles(int bytes, int64_t bh, int64_t rows) {
  return bytes == 2 && bh * cdiv(rows, 128) >= kCUs ? 2 : 1;
}
// Key ranges of the few-rows kernel; 0: the block kernel takes the call
inline int split_count(int bytes, int64_t bh, int64_t rows, int64_t nk) {
  const int64_t wgs = bh * cdiv(rows, 64), items = bh * cdiv(rows, 16);
  if (rows > 32 && (wgs >= kCUs / 2 || nk < 512)) return 0;
  int64_t s = cdiv(3 * kCUs, items);
  const int64_t most = cdiv(nk, 4 * (128 / bytes));
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

template <class Tr, int kDP>
void run_split(const AttnArgs& a, hipStream_t st) {
  const int64_t bh = (int64_t)a.b * a.hk;
  const int rb = (int)cdiv(a.rows, 16);
  hipLaunchKernelGGL((attn_split_kernel<Tr, kDP>), dim3((unsigned)(bh * rb), a.splits), dim3(256), 0, st, a, rb);
  if (a.splits > 1)
    hipLaunchKernelGGL(attn_join_kernel<Tr>, dim3((unsigned)(bh * a.rows)), dim3(64), 0, st, a, rb, kDP);
}

template <class Tr, int kDP>
void run_fwd(const AttnArgs& a, hipStream_t st) {
  const int64_t bh = (int64_t)a.b * a.hk;
  if (row_tiles(Tr::kBytes, bh, a.rows) == 2) {
    if constexpr (Tr::kBytes == 2) {
      const int rb = (int)cdiv(a.rows, 128);
      hipLaunchKernelGGL((attn_kernel<Tr, kDP, 2>), dim3((unsigned)(bh * rb)), dim3(256), 0, st, a, rb);
    }
  } else {
    const int rb = (int)cdiv(a.rows, 64);
    hipLaunchKernelGGL((attn_kernel<Tr, kDP, 1>), dim3((unsigned)(bh * rb)), dim3(256), 0, st, a, rb);
  }
}

template <class Tr, int kDP>
void run_bwd(const AttnArgs& a, hipStream_t st) {
  const int64_t bh = (int64_t)a.b * a.hk;
  hipLaunchKernelGGL(attn_delta_kernel<Tr>, dim3((unsigned)cdiv(bh * a.rows, 16)), dim3(256), 0, st, a);
  const int rb = (int)cdiv(a.rows, 64), kb = (int)cdiv(a.nk, 64);
  hipLaunchKernelGGL((attn_dkv_kernel<Tr, kDP, 1>), dim3((unsigned)(bh * kb)), dim3(256), 0, st, a, kb);
  hipLaunchKernelGGL((attn_dq_kernel<Tr, kDP, 1>), dim3((unsigned)(bh * rb)), dim3(256), 0, st, a, rb);
}

template <class Tr>
void run_attn(const AttnArgs& a, bool bwd, hipStream_t st) {
  if (!bwd && a.splits) {
    switch (split_pad(a.d)) {
      case 32: run_split<Tr, 32>(a, st); break;
      case 64: run_split<Tr, 64>(a, st); break;
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
  if (s > 1) *bytes = bh * cdiv(rows, 16) * s * 16 * (split_pad(a->d) + 2) * 4;
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
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == YK_ACT_F32) run_attn<F32>(k, false, st);
  else if (a->dtype == YK_ACT_BF16) run_attn<B16>(k, false, st);
  else run_attn<H16>(k, false, st);
  return launched("yk_attention");
}

int yk_attention_backward_workspace(const yk_attention_grad_args* a, int64_t* bytes) {
  YK_CHECK_ARG(a && bytes, "yk_attention_backward_workspace: NULL argument");
  if (const int rc = check_attn("yk_attention_backward_workspace", a)) return rc;
  *bytes = 2 * (int64_t)a->b * a->h_q * a->nq * 4;
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
  for (int i = 0; i < 3; ++i) k.gos[i] = a->go_stride[i], k.dqs[i] = a->dq_stride[i], k.dks[i] = a->dk_stride[i], k.dvs[i] = a->dv_stride[i];
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == YK_ACT_F32) run_attn<F32>(k, true, st);
  else if (a->dtype == YK_ACT_BF16) run_attn<B16>(k, true, st);
  else run_attn<H16>(k, true, st);
  return launched("yk_attention_backward");
}

}  // extern "C"
