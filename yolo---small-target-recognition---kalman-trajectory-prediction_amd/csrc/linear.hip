// Matrix product with bias, activation and residual in its epilogue, and its gradients
// (include/yk.h, yk_linear).
//
//   forward   y  = act(x w^T + bias) + res[m % res_rows]     [m][k] x [n][k]
//   backward  dz = dy act'(z);  dx = dz w;  dw = dz^T x;  dbias = column sums of dz;
//             dres[r] = sum of dy over the rows m % res_rows == r
//
// All three products are C[m][n] = sum over k of X(m, k) W(n, k), where either operand may lie
// transposed in memory (rows of k): forward (plain, plain), dx (plain, transposed), dw (both).  The W
// side is the MFMA's A operand, so a lane ends with 4 consecutive n of one m.
#include "token_common.h"

namespace yk {
namespace tok {

struct GemmArgs {
  const char* x;
  const char* w;
  const void* bias;
  const char* res;
  char* y;
  char* z;
  float* part;  // split sums: [splits][m][n] float32, or NULL
  int64_t x_stride, w_stride, res_stride, y_stride, z_stride;
  int m, n, k, res_rows, act, bias_f32, dtype;
  int tiles_m, tiles_n, k_split;  // k_split: K elements per blockIdx.y
};

// z, activation, residual and the stores of 8 consecutive n of one m, from sums that hold the bias
template <class Tr>
__device__ __forceinline__ void epilogue(const GemmArgs& a, int64_t m, int n, float* v) {
  using T = typename Tr::T;
  const int left = a.n - n;
  T* y = (T*)a.y + m * a.y_stride + n;
  T* z = a.z ? (T*)a.z + m * a.z_stride + n : nullptr;
  const T* res = a.res ? (const T*)a.res + (a.res_rows == a.m ? m : m % a.res_rows) * a.res_stride + n : nullptr;
  if (left >= 8) {
    if (z) store8<Tr>(z, v);
    if (a.act != YK_TOK_NONE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = act_f32(v[e], a.act);
    }
    if (res) add8<Tr>(res, v);
    store8<Tr>(y, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= left) continue;
      if (z) z[e] = from_f32<Tr>(v[e]);
      const float r = act_f32(v[e], a.act);
      y[e] = from_f32<Tr>(res ? r + to_f32<Tr>(res[e]) : r);
    }
  }
}
__device__ __forceinline__ void bias8(const GemmArgs& a, int n, float* b) {
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = 0.f;
  if (!a.bias) return;
  if (a.n - n >= 8) {
    if (a.bias_f32) add8<F32>((const float*)a.bias + n, b);
    else if (a.dtype == YK_ACT_BF16) add8<B16>((const unsigned short*)a.bias + n, b);
    else add8<H16>((const _Float16*)a.bias + n, b);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < a.n) b[e] = load_param(a.bias, n + e, a.bias_f32, a.dtype);
  }
}

// One 16-bit operand's tile in LDS: kRows rows (of m or n) x 128 bytes of K, as 16-byte chunks.
//   plain       [row][8 chunks of k]; chunk c of row r lies at c ^ (r & 7), so the 16 rows a
//               fragment read touches fall on different banks
//   transposed  [k][kRows]; the 16 rows of a fragment are one segment (32 bytes) of a k row;
//               segment s of k row kk lies at s ^ twist(kk), which spreads the k rows one read
//               touches over the banks; fragments come through ds_read_b64_tr_b16
template <class Tr, bool kTrans, int kRows>
struct Tile {
  using T = typename Tr::T;
  static_assert(Tr::kBytes == 2, "float32 operands: SplitTile");
  static constexpr int kK = 64;                       // K elements of a tile
  static constexpr int kEpc = 8;                      // elements of a chunk
  static constexpr int kChunks = kRows * 8;
  static constexpr int kPerRow = kTrans ? kRows / kEpc : 8;  // chunks of a stored row
  static constexpr int kSegs = kRows / 16;
  static constexpr int kSegChunks = 2;                // 16 elements = 32 bytes
  static constexpr int kBytesAll = kRows * 128;

  static __device__ __forceinline__ int twist(int kk) { return ((kk & 3) | ((kk >> 1) & 4)) & (kSegs - 1); }
  // stored row and first element of chunk j
  static __device__ __forceinline__ void locate(int j, int& row, int& col) {
    row = j / kPerRow;
    const int p = j % kPerRow;
    if constexpr (kTrans) col = (((p / kSegChunks) ^ twist(row)) * kSegChunks + p % kSegChunks) * kEpc;
    else col = (p ^ (row & 7)) * kEpc;
  }

  // K elements 32 * step + 8 * (lane / 16) .. + 7 of row 16 * t + lane % 16
  static __device__ __forceinline__ typename Tr::V8 frag(const char* lds, int t, int step, int lane) {
    const int l = lane & 15, g = lane >> 4;
    if constexpr (!kTrans) {
      return *(const typename Tr::V8*)(lds + (t * 16 + l) * 128 + (((step * 4 + g) ^ (l & 7)) << 4));
    } else {
      const int kk = step * 32 + g * 8 + (l >> 2);
      typedef __attribute__((address_space(3))) s16x4* lp;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lp)(lds + kk * (kRows * 2) + ((t ^ twist(kk)) << 5) + (l & 3) * 8));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lp)(lds + (kk + 4) * (kRows * 2) + ((t ^ twist(kk + 4)) << 5) + (l & 3) * 8));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// The loads of one operand's tiles by kThreads threads.  kAsync: straight from memory to LDS through a
// buffer descriptor, whose range check turns a chunk outside the matrix into zeros; needs 16-byte
// aligned rows and whole chunks.  Otherwise through registers, any alignment.
template <class Tr, bool kTrans, int kRows, int kThreads, bool kAsync>
struct Loader {
  using Tl = Tile<Tr, kTrans, kRows>;
  using T = typename Tr::T;
  static constexpr int kN = Tl::kChunks / kThreads;
  static constexpr unsigned kOut = 0x80000000u;  // past every descriptor's range
  const T* base;       // first stored row / column of this workgroup's tiles
  int64_t stride;
  int rows, cols;      // stored rows / columns left from there
  unsigned off[kAsync ? kN : 1];  // byte offset of each chunk, kOut where m (n) ends before it
  u32x4 reg[kAsync ? 1 : kN];

  __device__ __forceinline__ void init(const char* p, int64_t s, int r0, int m, int k0, int k1) {
    stride = s;
    if constexpr (kTrans) {
      base = (const T*)p + (int64_t)k0 * s + r0;
      rows = k1 - k0;
      cols = m - r0;
    } else {
      base = (const T*)p + (int64_t)r0 * s + k0;
      rows = m - r0;
      cols = k1 - k0;
    }
    if constexpr (kAsync) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        int row, col;
        Tl::locate(i * kThreads + threadIdx.x, row, col);
        off[i] = (kTrans ? col < cols : row < rows) ? (unsigned)((row * (int)stride + col) * Tr::kBytes) : kOut;
      }
    }
  }
  __device__ __forceinline__ void advance() {
    if constexpr (kTrans) {
      base += Tl::kK * stride;
      rows -= Tl::kK;
    } else {
      base += Tl::kK;
      cols -= Tl::kK;
    }
  }
  __device__ __forceinline__ void issue(char* lds) {
    const int tid = threadIdx.x;
    if constexpr (kAsync) {
      // (nothing left: every chunk lands as zeros)
      const int64_t span = rows > 0 && cols > 0 ? ((int64_t)(rows - 1) * stride + cols) * Tr::kBytes : 0;
      const int bytes = rfl((int)(span < 0x7ffffff0 ? span : 0x7ffffff0));
      const size_t b = (size_t)base;
      const size_t ub = ((size_t)(unsigned)rfl((int)(b >> 32)) << 32) | (unsigned)rfl((int)b);
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)ub, (short)0, bytes, 0x00020000);
      const bool tail = (kTrans ? rows : cols) < Tl::kK;  // K ends inside this tile
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        unsigned o = off[i];
        if (tail) {
          int row, col;
          Tl::locate(i * kThreads + tid, row, col);
          if ((kTrans ? row : col) >= (kTrans ? rows : cols)) o = kOut;
        }
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc, (__attribute__((address_space(3))) void*)(lds + (i * kThreads + rfl(tid & ~63)) * 16), 16, o, 0, 0, 0);
      }
    } else {
      const bool inside = rows >= (kTrans ? Tl::kK : kRows) && cols >= (kTrans ? kRows : Tl::kK);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        int row, col;
        Tl::locate(i * kThreads + tid, row, col);
        const T* p = base + row * stride + col;
        if (inside) reg[i] = *(const u32x4_any*)p;
        else reg[i] = row < rows ? load16<Tr>(p, cols - col) : u32x4{0, 0, 0, 0};
      }
    }
  }
  __device__ __forceinline__ void commit(char* lds) {
    if constexpr (!kAsync) {
#pragma unroll
      for (int i = 0; i < kN; ++i) *(u32x4*)(lds + (i * kThreads + threadIdx.x) * 16) = reg[i];
    }
  }
};

// A wave's accumulators pass through LDS 32 rows at a time (each wave in a part of its own), so that a lane
// finishes 8 neighbouring n and a row's stores and residual reads are whole lines.
template <int kFM, int kFN, int kWaves, int kLds>
struct Transit {
  static constexpr int kPass = 2, kPitch = kFN * 16 + 4, kCh = kFN * 2, kStepRows = 64 / kCh, kSteps = kPass * 16 / kStepRows;
  static_assert(kFM % kPass == 0 && kWaves * kPass * 16 * kPitch * 4 <= kLds, "the rows in transit fit the tiles' LDS");
  // body(j0): the rows 16 j0 .. + 31 are in buf
  template <class B>
  static __device__ __forceinline__ void run(const f32x4 (&acc)[kFN][kFM], float* buf, B&& body) {
    const int l = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j0 = 0; j0 < kFM; j0 += kPass) {
#pragma unroll
      for (int j = 0; j < kPass; ++j)
#pragma unroll
        for (int i = 0; i < kFN; ++i) *(f32x4*)(buf + (j * 16 + l) * kPitch + i * 16 + g * 4) = acc[i][j0 + j];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      body(j0);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
  static __device__ __forceinline__ void fetch(const float* buf, int row, int c, float* v) {
    const f32x4 lo = *(const f32x4*)(buf + row * kPitch + c * 8), hi = *(const f32x4*)(buf + row * kPitch + c * 8 + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
  }
};

// The epilogue of rows and columns that all exist, its activation known: addresses are a uniform base and a
// lane's 32-bit offset.
template <class Tr, int kAct, class X, int kFM, int kFN, class F>
__device__ __forceinline__ void finish_whole(const GemmArgs& a, const f32x4 (&acc)[kFN][kFM], float* buf, int m0, int n0, F&& mend) {
  using T = typename Tr::T;
  const int lane = threadIdx.x & 63, c = lane % X::kCh, r = lane / X::kCh;
  const unsigned yo = (unsigned)(r * (int)a.y_stride + c * 8), zo = (unsigned)(r * (int)a.z_stride + c * 8);
  float b[8];
  bias8(a, n0 + c * 8, b);
  X::run(acc, buf, [&](int j0) {
    // the residual's rows are on their way before the first store (which they might alias, for all the
    // compiler knows)
    u32x4 rv[X::kSteps][Tr::kBytes / 2];
    if (a.res) {
#pragma unroll
      for (int h = 0; h < X::kSteps; ++h) {
        const unsigned mr = (unsigned)(m0 + j0 * 16 + h * X::kStepRows + r);
        const T* p = (const T*)a.res + (int64_t)(a.res_rows == a.m ? mr : mr % (unsigned)a.res_rows) * a.res_stride + n0 + c * 8;
#pragma unroll
        for (int i = 0; i < Tr::kBytes / 2; ++i) rv[h][i] = *(const u32x4_any*)((const char*)p + i * 16);
      }
    }
    mend(buf, X::kPitch, m0 + j0 * 16);
#pragma unroll
    for (int h = 0; h < X::kSteps; ++h) {
      const int64_t m = (int64_t)m0 + j0 * 16 + h * X::kStepRows;  // (the first of the rows of this step)
      float v[8];
      X::fetch(buf, h * X::kStepRows + r, c, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += b[e];
      if (a.z) store8<Tr>((T*)a.z + m * a.z_stride + n0 + zo, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = act_f32(v[e], kAct);
      if (a.res) {
        T t[8];
        __builtin_memcpy(t, rv[h], sizeof t);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += to_f32<Tr>(t[e]);
      }
      store8<Tr>((T*)a.y + m * a.y_stride + n0 + yo, v);
    }
  });
}

// A wave's accumulators (rows m0 .., columns n0 ..) to memory: through the epilogue, or as a split's
// sums.  mend(buf, pitch, first row): may change the 32 rows in transit.
template <class Tr, int kFM, int kFN, int kWaves, int kLds, class F>
__device__ __forceinline__ void finish_tile(const GemmArgs& a, const f32x4 (&acc)[kFN][kFM], char* lds, int m0, int n0, F&& mend) {
  using X = Transit<kFM, kFN, kWaves, kLds>;
  float* buf = (float*)lds + rfl(threadIdx.x >> 6) * X::kPass * 16 * X::kPitch;
  constexpr int64_t kMaxStride = 1 << 24;
  if (!a.part && m0 + kFM * 16 <= a.m && n0 + kFN * 16 <= a.n && a.y_stride < kMaxStride && (!a.z || a.z_stride < kMaxStride)) {
    if (a.act == YK_TOK_GELU) finish_whole<Tr, YK_TOK_GELU, X>(a, acc, buf, m0, n0, mend);
    else if (a.act == YK_TOK_SILU) finish_whole<Tr, YK_TOK_SILU, X>(a, acc, buf, m0, n0, mend);
    else if (a.act == YK_TOK_RELU) finish_whole<Tr, YK_TOK_RELU, X>(a, acc, buf, m0, n0, mend);
    else finish_whole<Tr, YK_TOK_NONE, X>(a, acc, buf, m0, n0, mend);
    return;
  }
  const int lane = threadIdx.x & 63, c = lane % X::kCh, n = n0 + c * 8;
  float b[8];
  bias8(a, n, b);
  X::run(acc, buf, [&](int j0) {
    mend(buf, X::kPitch, m0 + j0 * 16);
#pragma unroll
    for (int h = 0; h < X::kSteps; ++h) {
      const int row = h * X::kStepRows + lane / X::kCh;
      const int64_t m = (int64_t)m0 + j0 * 16 + row;
      float v[8];
      X::fetch(buf, row, c, v);
      if (m >= a.m || n >= a.n) continue;
      if (a.part) {
        float* p = a.part + ((int64_t)blockIdx.y * a.m + m) * a.n + n;
        if (a.n - n >= 8) {
          store8<F32>(p, v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + e < a.n) p[e] = v[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += b[e];
        epilogue<Tr>(a, m, n, v);
      }
    }
  });
}

// Until this wave's loads but the last kLeft have landed, and its LDS reads are done; then until all
// waves are there.
template <int kLeft>
__device__ __forceinline__ void loads_landed() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLeft) : "memory");
  __builtin_amdgcn_s_barrier();
}

// kTM x kTN tile of C by kWM x kWN waves.  256-tiles, bf16: 8192^3 820-850 us (1290-1340 TFLOP/s; a wave's LDS reads
// and the loads into LDS take about the cycles its MFMAs do), 40960 x 4096 x 1024 313 us, of which some 65
// are first loads and epilogues that one workgroup per CU hides behind nothing; with GELU 365-385.  Three or four
// stages: 4096 x 1024 x 2048 in 128-tiles 26 -> 23 us, but the LDS they take leaves one workgroup
// per CU where two fit (10240 x 512 x 2048: 30 -> 40), and so do fragments read a half tile ahead: no gain.
// Rows that are not 16-byte aligned go through registers (4097 x 777 x 1111 fp16: 31 us), bound by the
// L1's rate for such loads.  kAsync: kStages - 1 tiles of K in flight, one barrier per
// tile; a buffer is filled again after the barrier that follows its last read.
template <class Tr, bool kXT, bool kWT, int kTM, int kTN, int kWM, int kWN, int kStages, bool kAsync>
__global__ __launch_bounds__(64 * kWM * kWN) void gemm_kernel(GemmArgs a) {
  using XTile = Tile<Tr, kXT, kTM>;
  using WTile = Tile<Tr, kWT, kTN>;
  constexpr int kThreads = 64 * kWM * kWN;
  constexpr int kFM = kTM / (16 * kWM), kFN = kTN / (16 * kWN);  // 16-wide fragments of a wave, per side
  constexpr int kSteps = XTile::kK / 32;
  // one array for both operands' tiles: with two, the compiler waits for every load in flight before
  // it reads either
  constexpr int kBuf = XTile::kBytesAll + WTile::kBytesAll;
  __shared__ __attribute__((aligned(16))) char lds[kStages][kBuf];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6);
  // tiles in groups of 8 along m, m fastest: a group's x tiles and the w tile in use stay in the XCD's L2
  const int item = xcd_item(blockIdx.x, a.tiles_m * a.tiles_n);
  const int per = 8 * a.tiles_n, grp = item / per, in = item - grp * per;
  const int gm = a.tiles_m - grp * 8 < 8 ? a.tiles_m - grp * 8 : 8;
  const int tn = in / gm, tm = grp * 8 + in - tn * gm;
  const int k0 = blockIdx.y * a.k_split, k1 = a.k - k0 < a.k_split ? a.k : k0 + a.k_split;
  Loader<Tr, kXT, kTM, kThreads, kAsync> lx;
  Loader<Tr, kWT, kTN, kThreads, kAsync> lw;
  lx.init(a.x, a.x_stride, tm * kTM, a.m, k0, k1);
  lw.init(a.w, a.w_stride, tn * kTN, a.n, k0, k1);
  const int wm = wave % kWM * kFM, wn = wave / kWM * kFN;  // first fragment of this wave
  f32x4 acc[kFN][kFM];
#pragma unroll
  for (int i = 0; i < kFN; ++i)
#pragma unroll
    for (int j = 0; j < kFM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int nk = (k1 - k0 + XTile::kK - 1) / XTile::kK;
  // one tile of K; `between`: the next tile's loads, behind the first LDS reads
  auto compute = [&](const char* buf, auto&& between) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      typename Tr::V8 wf[kFN], xf[kFM];
#pragma unroll
      for (int i = 0; i < kFN; ++i) wf[i] = WTile::frag(buf + XTile::kBytesAll, wn + i, s, lane);
#pragma unroll
      for (int j = 0; j < kFM; ++j) xf[j] = XTile::frag(buf, wm + j, s, lane);
      if (s == 0) between();
#pragma unroll
      for (int j = 0; j < kFM; ++j)
#pragma unroll
        for (int i = 0; i < kFN; ++i) acc[i][j] = mma<Tr>(wf[i], xf[j], acc[i][j]);
    }
  };
  if constexpr (kAsync) {
    constexpr int kLoads = decltype(lx)::kN + decltype(lw)::kN;
    auto issue = [&](int buf) {
      lx.issue(lds[buf]);
      lw.issue(lds[buf] + XTile::kBytesAll);
      lx.advance();
      lw.advance();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);
    int cur = 0, fill = kStages - 1;
    for (int kt = 0; kt < nk; ++kt) {
      loads_landed<(kStages - 2) * kLoads>();
      compute(lds[cur], [&] { issue(fill); });
      fill = cur;
      cur = cur + 1 == kStages ? 0 : cur + 1;
    }
    loads_landed<0>();
  } else {
    lx.issue(lds[0]);
    lw.issue(lds[0] + XTile::kBytesAll);
    lx.commit(lds[0]);
    lw.commit(lds[0] + XTile::kBytesAll);
    __syncthreads();
    for (int kt = 0; kt < nk; ++kt) {
      const int cur = kt & 1;
      if (kt + 1 < nk) {
        lx.advance();
        lw.advance();
        lx.issue(lds[cur ^ 1]);
        lw.issue(lds[cur ^ 1] + XTile::kBytesAll);
      }
      compute(lds[cur], [] {});
      if (kt + 1 < nk) {
        lx.commit(lds[cur ^ 1]);
        lw.commit(lds[cur ^ 1] + XTile::kBytesAll);
      }
      __syncthreads();
    }
  }

  finish_tile<Tr, kFM, kFN, kWM * kWN, kStages * kBuf>(a, acc, &lds[0][0], tm * kTM + wm * 16, tn * kTN + wn * 16,
                                                       [](float*, int, int) {});
}

// float32 on the bf16 matrix cores.  x = x0 + x1 + x2 exactly, three bf16 of 8 significant bits each
// (rounded to nearest, so |x1| <= 2^-9 |x| and |x2| <= 2^-18 |x|), and six of the nine products are
// summed: w0x0, w0x1, w1x0, w1x1, w0x2, w2x0.  bf16 products are exact in float32 and what is left out
// is below 2^-25 |w x|, less than one float32 rounding; six 16-cycle MFMAs per 32 of K replace eight
// 32-cycle float32 ones.  (A part below bf16's normal range, of an operand below some 2^-110, may be
// flushed.)  4096 x 1024 x 4096: 181-198 us, 267 on v_mfma_f32_16x16x4_f32.
//
// The parts are made once per tile, between the global loads' registers and LDS (three planes a
// side), not by every wave that reads them.  A tile is 32 of K:
//   plain       plane [row][4 chunks of 8 k], chunk c of row r at c ^ (r >> 2 & 3)
//   transposed  plane [k][kRows], segments of 16 rows twisted as in Tile
template <bool kTrans, int kRows>
struct SplitTile {
  using Tw = Tile<B16, kTrans, kRows>;
  static constexpr int kK = 32, kUnits = kRows * 4, kPerRow = kTrans ? kRows / 8 : 4, kPlane = kRows * 64;
  // stored row, first element and place of unit j (8 elements)
  static __device__ __forceinline__ void locate(int j, int& row, int& col, int& at) {
    row = j / kPerRow;
    const int c = j % kPerRow;
    col = c * 8;
    if constexpr (kTrans) at = row * (kRows * 2) + (((c >> 1) ^ Tw::twist(row)) << 5) + (c & 1) * 16;
    else at = row * 64 + ((c ^ ((row >> 2) & 3)) << 4);
  }
  static __device__ __forceinline__ s16x8 frag(const char* plane, int t, int lane) {
    const int l = lane & 15, g = lane >> 4;
    if constexpr (kTrans) return Tw::frag(plane, t, 0, lane);
    else return *(const s16x8*)(plane + (t * 16 + l) * 64 + ((g ^ (l >> 2)) << 4));
  }
};

// x rounded to bf16 (two at a time, v_cvt_pk_bf16_f32) and what that leaves
__device__ __forceinline__ unsigned split_pair(float& a, float& b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const unsigned u = __builtin_bit_cast(unsigned, bf16x2{(__bf16)a, (__bf16)b});
  a -= __uint_as_float(u << 16);
  b -= __uint_as_float(u & 0xffff0000u);
  return u;
}

template <bool kTrans, int kRows>
struct SplitLoader {
  using Tl = SplitTile<kTrans, kRows>;
  static constexpr int kN = Tl::kUnits / 256;
  const float* base;
  int64_t stride;
  int rows, cols;
  u32x4 reg[kN][2];
  __device__ __forceinline__ void init(const char* p, int64_t s, int r0, int m, int k0, int k1) {
    stride = s;
    base = (const float*)p + (kTrans ? (int64_t)k0 * s + r0 : (int64_t)r0 * s + k0);
    rows = kTrans ? k1 - k0 : m - r0;
    cols = kTrans ? m - r0 : k1 - k0;
  }
  __device__ __forceinline__ void advance() {
    base += kTrans ? Tl::kK * stride : Tl::kK;
    (kTrans ? rows : cols) -= Tl::kK;
  }
  __device__ __forceinline__ void issue() {
    const bool inside = rows >= (kTrans ? Tl::kK : kRows) && cols >= (kTrans ? kRows : Tl::kK);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      int row, col, at;
      Tl::locate(i * 256 + threadIdx.x, row, col, at);
      const float* p = base + row * stride + col;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (inside) reg[i][h] = *(const u32x4_any*)(p + 4 * h);
        else reg[i][h] = row < rows ? load16<F32>(p + 4 * h, cols - col - 4 * h) : u32x4{0, 0, 0, 0};
      }
    }
  }
  __device__ __forceinline__ void commit(char* lds) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      int row, col, at;
      Tl::locate(i * 256 + threadIdx.x, row, col, at);
      u32x4 part[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float a = __uint_as_float(reg[i][e >> 1][(e & 1) * 2]), b = __uint_as_float(reg[i][e >> 1][(e & 1) * 2 + 1]);
        part[0][e] = split_pair(a, b);
        part[1][e] = split_pair(a, b);
        part[2][e] = split_pair(a, b);
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) *(u32x4*)(lds + q * Tl::kPlane + at) = part[q];
    }
  }
};

template <bool kXT, bool kWT, int kTile>
__global__ __launch_bounds__(256, 2) void gemm_f32_kernel(GemmArgs a) {
  using XTile = SplitTile<kXT, kTile>;
  using WTile = SplitTile<kWT, kTile>;
  constexpr int kF = kTile / 32, kHalf = 3 * XTile::kPlane;
  __shared__ __attribute__((aligned(16))) char lds[2 * kHalf];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6);
  const int item = xcd_item(blockIdx.x, a.tiles_m * a.tiles_n);
  const int per = 8 * a.tiles_n, grp = item / per, in = item - grp * per;
  const int gm = a.tiles_m - grp * 8 < 8 ? a.tiles_m - grp * 8 : 8;
  const int tn = in / gm, tm = grp * 8 + in - tn * gm;
  const int k0 = blockIdx.y * a.k_split, k1 = a.k - k0 < a.k_split ? a.k : k0 + a.k_split;
  SplitLoader<kXT, kTile> lx;
  SplitLoader<kWT, kTile> lw;
  lx.init(a.x, a.x_stride, tm * kTile, a.m, k0, k1);
  lw.init(a.w, a.w_stride, tn * kTile, a.n, k0, k1);
  const int wm = (wave & 1) * kF, wn = (wave >> 1) * kF;
  f32x4 acc[kF][kF];
#pragma unroll
  for (int i = 0; i < kF; ++i)
#pragma unroll
    for (int j = 0; j < kF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int nk = (k1 - k0 + 31) / 32;
  lx.issue();
  lw.issue();
  for (int kt = 0; kt < nk; ++kt) {
    __syncthreads();
    lx.commit(lds);
    lw.commit(lds + kHalf);
    __syncthreads();
    if (kt + 1 < nk) {
      lx.advance();
      lw.advance();
      lx.issue();
      lw.issue();
    }
    s16x8 wf[kF][3];
#pragma unroll
    for (int i = 0; i < kF; ++i)
#pragma unroll
      for (int q = 0; q < 3; ++q) wf[i][q] = WTile::frag(lds + kHalf + q * WTile::kPlane, wn + i, lane);
#pragma unroll
    for (int j = 0; j < kF; ++j) {
      s16x8 xf[3];
#pragma unroll
      for (int q = 0; q < 3; ++q) xf[q] = XTile::frag(lds + q * XTile::kPlane, wm + j, lane);
      // (a pass over the wave's tiles per product: neighbouring MFMAs do not wait for each other)
      constexpr int kPair[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};
#pragma unroll
      for (int q = 0; q < 6; ++q)
#pragma unroll
        for (int i = 0; i < kF; ++i) acc[i][j] = mma<B16>(wf[i][kPair[q][0]], xf[kPair[q][1]], acc[i][j]);
    }
  }
  __syncthreads();
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kF; ++i)
#pragma unroll
    for (int j = 0; j < kF; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) bad = bad || acc[i][j][e] != acc[i][j][e];
  // An infinite operand, or one that bf16's range rounds to infinity, makes NaN of its parts: such
  // sums are taken again, plainly.  (Once a sum is NaN it stays one.)
  const bool any = __any(bad);
  auto mend = [&](float* buf, int pitch, int m0) {
    if (!any) return;
#pragma unroll 1
    for (int i = lane; i < 32 * kF * 16; i += 64) {
      const int row = i / (kF * 16), col = i % (kF * 16), m = m0 + row, n = tn * kTile + wn * 16 + col;
      if (buf[row * pitch + col] == buf[row * pitch + col] || m >= a.m || n >= a.n) continue;
      float s = 0.f;
#pragma unroll 1
      for (int64_t k = k0; k < k1 && s == s; ++k)
        s = fmaf(((const float*)a.x)[kXT ? k * a.x_stride + m : m * a.x_stride + k],
                 ((const float*)a.w)[kWT ? k * a.w_stride + n : n * a.w_stride + k], s);
      buf[row * pitch + col] = s;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  finish_tile<F32, kF, kF, 4, 2 * kHalf>(a, acc, lds, tm * kTile + wm * 16, tn * kTile + wn * 16, mend);
}

// Sum of the split products, then the epilogue: 8 consecutive n per kLanes threads, of which each adds
// every kLanes-th split, 4 loads in flight; their sums are joined in a fixed order.
template <class Tr, int kLanes>
__global__ __launch_bounds__(256) void split_sum_kernel(GemmArgs a, int splits) {
  __shared__ float lds[kLanes > 1 ? kLanes : 1][256 / kLanes][9];
  const int n8 = (a.n + 7) / 8, sub = threadIdx.x / (256 / kLanes), id = threadIdx.x % (256 / kLanes);
  const int64_t i = (int64_t)blockIdx.x * (256 / kLanes) + id;
  const int64_t m = i / n8;
  const int n = (int)(i - m * n8) * 8, left = a.n - n;
  float v[8] = {};
  if (m < a.m) {
    const int64_t step = (int64_t)a.m * a.n;
    const float* p = a.part + m * a.n + n;
    if (left >= 8) {
      for (int s0 = sub; s0 < splits; s0 += 4 * kLanes) {
        f32x4 t[4][2];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int s = s0 + q * kLanes;
          const float* r = p + (s < splits ? s : s0) * step;
          t[q][0] = load4<F32>(r);
          t[q][1] = load4<F32>(r + 4);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (s0 + q * kLanes >= splits) break;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += t[q][e >> 2][e & 3];
        }
      }
    } else {
      for (int s = sub; s < splits; s += kLanes) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) v[e] += p[s * step + e];
      }
    }
  }
  if constexpr (kLanes > 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) lds[sub][id][e] = v[e];
    __syncthreads();
    if (sub) return;
#pragma unroll
    for (int s = 1; s < kLanes; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += lds[s][id][e];
  }
  if (m >= a.m) return;
  float b[8];
  bias8(a, n, b);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += b[e];
  epilogue<Tr>(a, m, n, v);
}

// Few rows (m <= 16 kMT): the weight is read once, straight into fragments, by workgroups of 16
// output channels whose 8 waves split K 64 elements at a time; their sums meet in LDS.  Bound by the latency of
// launch and loads (8 x 2048 x 512 bf16: 4.0 us), for long K by the weight's bytes.
template <class Tr, int kMT>
__global__ __launch_bounds__(512) void rows_kernel(GemmArgs a) {
  using T = typename Tr::T;
  constexpr int kWaves = 8, kEpc = 16 / Tr::kBytes, kPer = 8 / kEpc;  // loads of a fragment
  __shared__ __attribute__((aligned(16))) float sum[kWaves][16 * kMT][20];
  const int lane = threadIdx.x & 63, wave = rfl(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const T* w = (const T*)a.w + (int64_t)(n0 + l) * a.w_stride;
  const bool wl = n0 + l < a.n;
  f32x4 acc[kMT];
#pragma unroll
  for (int j = 0; j < kMT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int k0 = wave * 64; k0 < a.k; k0 += kWaves * 64) {
    u32x4 wf[2][kPer], xf[kMT][2][kPer];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        const int k = k0 + s * 32 + g * 8 + p * kEpc;
        wf[s][p] = wl ? load16<Tr>(w + k, a.k - k) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < kMT; ++j) {
          const int m = j * 16 + l;
          xf[j][s][p] = m < a.m ? load16<Tr>((const T*)a.x + m * a.x_stride + k, a.k - k) : u32x4{0, 0, 0, 0};
        }
      }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < kMT; ++j)
        acc[j] = mma<Tr>(__builtin_bit_cast(typename Tr::V8, wf[s]), __builtin_bit_cast(typename Tr::V8, xf[j][s]), acc[j]);
  }
#pragma unroll
  for (int j = 0; j < kMT; ++j) *(f32x4*)&sum[wave][j * 16 + l][g * 4] = acc[j];
  __syncthreads();
  const int m = threadIdx.x >> 1, n = n0 + (threadIdx.x & 1) * 8;
  if (m >= a.m || n >= a.n) return;  // (m < 16 kMT: a.m is at most that)
  float v[8];
  bias8(a, n, v);
#pragma unroll
  for (int s = 0; s < kWaves; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += sum[s][m][n - n0 + e];
  epilogue<Tr>(a, m, n, v);
}

struct ColArgs {
  const char* dy;
  const char* z;   // with act: dz = dy act'(z) is stored and summed; else dy is summed
  char* dz;
  void* out;       // with one row group: the sums themselves
  float* part;     // [groups][r][n]
  int64_t dy_stride, z_stride, out_stride;
  int m, n, r, groups, act, out_f32, dtype, chunk_blocks;
  int r0;          // residue of the launch's first workgroups
};

// Sums over the rows m % r == residue, for each column; a workgroup holds 32 chunks of columns x 8
// rows of one residue, blockIdx.y a group of them.  Bound by HBM: dy and z in, dz out, 10240 x 2048 bf16 with
// GELU's slope 24 us, 5.2 TB/s (the activation known at run time only and no row read ahead: 35).
template <class Tr, int kAct>
__global__ __launch_bounds__(256) void cols_kernel(ColArgs a) {
  using T = typename Tr::T;
  constexpr int kEpc = 16 / Tr::kBytes;
  __shared__ float lds[8][32 * kEpc];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int sub_res = blockIdx.x / a.chunk_blocks, cb = blockIdx.x - sub_res * a.chunk_blocks, res = a.r0 + sub_res;
  const int c0 = (cb * 32 + lane) * kEpc;
  const int n = a.n - c0;
  float acc[kEpc];
#pragma unroll
  for (int e = 0; e < kEpc; ++e) acc[e] = 0.f;
  const int64_t step = (int64_t)gridDim.y * 8 * a.r;
  int64_t row = res + ((int64_t)blockIdx.y * 8 + sub) * a.r;
  if (n > 0 && row < a.m) {
    u32x4 u, uz;  // the row after the one worked on is on its way
    auto load = [&](int64_t at) {
      u = load16<Tr>((const T*)a.dy + at * a.dy_stride + c0, n);
      if constexpr (kAct != YK_TOK_NONE) uz = load16<Tr>((const T*)a.z + at * a.z_stride + c0, n);
    };
    load(row);
    for (; row < a.m; row += step) {
      T d[kEpc], zv[kEpc];
      __builtin_memcpy(d, &u, 16);
      if constexpr (kAct != YK_TOK_NONE) __builtin_memcpy(zv, &uz, 16);
      if (row + step < a.m) load(row + step);
      if constexpr (kAct != YK_TOK_NONE) {
        // dz is rounded to the operands' type: it is an operand of two matrix products
#pragma unroll
        for (int e = 0; e < kEpc; ++e) {
          const float f = to_f32<Tr>(d[e]) * act_slope(to_f32<Tr>(zv[e]), kAct);
          acc[e] += f;
          d[e] = from_f32<Tr>(f);
        }
        T* o = (T*)a.dz + row * a.n + c0;
        if (n >= kEpc) {
          u32x4 v;
          __builtin_memcpy(&v, d, 16);
          *(u32x4_any*)o = v;
        } else {
          for (int e = 0; e < n; ++e) o[e] = d[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < kEpc; ++e) acc[e] += to_f32<Tr>(d[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < kEpc; ++e) lds[sub][lane * kEpc + e] = acc[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * kEpc; i += 256) {
    const int c = cb * 32 * kEpc + i;
    if (c >= a.n) continue;
    float v = 0.f;
#pragma unroll
    for (int s = 0; s < 8; ++s) v += lds[s][i];
    if (a.part) a.part[((int64_t)blockIdx.y * a.r + res) * a.n + c] = v;
    else if (a.out) store_param(a.out, res * a.out_stride + c, v, a.out_f32, a.dtype);
  }
}

// The row groups' sums added in order: 64 (residue, column) pairs x 16 group ranges.
__global__ __launch_bounds__(1024) void cols_sum_kernel(ColArgs a) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t all = (int64_t)a.r * a.n, i = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (i < all)
    for (int p = g; p < a.groups; p += 16) s += a.part[p * all + i];
  lds[g][lane] = s;
  __syncthreads();
  if (g == 0 && i < all) {
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) v += lds[j][lane];
    const int64_t row = i / a.n;
    store_param(a.out, row * a.out_stride + (i - row * a.n), v, a.out_f32, a.dtype);
  }
}

// ---- launch rules -----------------------------------------------------------------------------
struct Plan {
  int tile, splits, k_split;
};
constexpr int kCUs = 256;

// Time of a product by tile size, from sweeps of tile and split on this card (microseconds; a step
// is 64 of K for the 16-bit types, 32 for float32): `alone` per step for the only workgroup of
// its CU (its loads' latency), `shared` per step and workgroup where `per_cu` of them share it
// (the CU's load rate; the MFMAs and the splitting for float32), `ends` / `ends_shared` for the first loads and the
// epilogue.  16-bit (m x n x k), tiles of 64 / 128 / 256: 1000^3 9.0 / 18.8 / 24 us; 4096 x 1024 x 1024 16.7 /
// 14.3 / 28; 4096 x 4096 x 1024 60 / 41 / 35; 40960 x 4096 x 1024 548 / 379 / 320.  float32
// 10240 x 2048 x 512: 186 / 203 (64 / 128).
struct TileTime {
  int tile, per_cu;
  double alone, shared, ends, ends_shared;
};
constexpr TileTime kTimes16[] = {{256, 1, 1.5, 1.5, 9, 9}, {128, 2, 0.7, 0.44, 3.5, 2.6}, {64, 4, 0.35, 0.19, 2.5, 0.8}};
constexpr TileTime kTimes32[] = {{128, 2, 1.75, 1.34, 5, 3.5}, {64, 4, 0.85, 0.455, 3, 1.2}};

// The tile and the split of K that the table says are fastest.  trans: operands that lie transposed
// (their fragments take twice the LDS reads, which shows where a 16-bit workgroup is alone: 2048 x 512
// x 10240, both transposed, 256 64-tiles: 103 us, split in 4: 45).  A split costs a launch and its
// float32 sums once written and once read.
inline Plan plan_gemm(int64_t m, int64_t n, int64_t k, int bytes, int trans, bool async) {
  const int64_t kk = 128 / bytes, steps = cdiv(k, kk);
  Plan best{64, 1, 0};
  double best_t = 1e30;
  const TileTime* times = bytes == 2 ? kTimes16 : kTimes32;
  for (int i = bytes == 2 && !async ? 1 : 0; i < (bytes == 2 ? 3 : 2); ++i) {  // (256: no variant through registers)
    const TileTime& t = times[i];
    const int64_t tiles = cdiv(m, t.tile) * cdiv(n, t.tile);
    if (tiles > most_groups(t.tile == 256 ? 512 : 256)) continue;  // (128-tiles are never: check_linear)
    for (int64_t s = 1; s == 1 || (s <= 64 && steps >= 4 * s && tiles * s <= kCUs * t.per_cu); s += s < 4 ? 1 : s / 2) {
      const int64_t per = cdiv(steps, s), wgs = cdiv(tiles * cdiv(steps, per), kCUs);
      auto turn = [&](int64_t r) {  // r workgroups at once on a CU
        return r == 0 ? 0.0 : per * fmax(t.alone * (bytes == 2 ? 1 + 0.4 * trans : 1), r * t.shared) + fmax(t.ends, r * t.ends_shared);
      };
      double us = (wgs / t.per_cu) * turn(t.per_cu) + turn(wgs % t.per_cu);
      if (s > 1) us += 4 + (double)m * n * s * 8 / 8e6;
      if (us < best_t) {
        best_t = us;
        best = Plan{t.tile, (int)cdiv(steps, per), (int)(per * kk)};
      }
    }
  }
  return best;
}
inline int64_t gemm_scratch(int64_t m, int64_t n, int64_t k, int bytes, int trans) {
  int64_t need = 0;  // whether the rows are aligned is known with the pointers only
  for (int async = 0; async < 2; ++async) {
    const Plan p = plan_gemm(m, n, k, bytes, trans, async);
    const int64_t b = p.splits > 1 ? (int64_t)p.splits * m * n * 4 : 0;
    need = b > need ? b : need;
  }
  return need;
}
constexpr int kFewRows = 64;

template <class Tr, bool kXT, bool kWT, bool kAsync>
void launch_tiles(const GemmArgs& a, int tile, int splits, hipStream_t st) {
  const dim3 grid((unsigned)(a.tiles_m * a.tiles_n), (unsigned)splits);
  if constexpr (Tr::kBytes == 4) {
    if (tile == 128) launch((gemm_f32_kernel<kXT, kWT, 128>), grid, dim3(256), 0, st, a);
    else launch((gemm_f32_kernel<kXT, kWT, 64>), grid, dim3(256), 0, st, a);
    return;
  } else {
  if constexpr (kAsync) {
    if (tile == 256) {
      launch((gemm_kernel<Tr, kXT, kWT, 256, 256, 2, 4, 2, true>), grid, dim3(512), 0, st, a);
      return;
    }
  }
  if (tile == 128) launch((gemm_kernel<Tr, kXT, kWT, 128, 128, 2, 2, 2, kAsync>), grid, dim3(256), 0, st, a);
  else launch((gemm_kernel<Tr, kXT, kWT, 64, 64, 2, 2, 2, kAsync>), grid, dim3(256), 0, st, a);
  }
}

// rows of 16-byte chunks whose offsets inside a tile stay below 2^31 (256 rows of less than 2^23 bytes)
inline bool aligned_rows(const void* p, int64_t stride, int64_t cols, int bytes) {
  return (uintptr_t)p % 16 == 0 && stride * bytes % 16 == 0 && cols * bytes % 16 == 0 && stride * bytes < (1 << 23);
}

template <class Tr, bool kXT, bool kWT>
Plan plan_for(const GemmArgs& a, bool& async) {
  async = aligned_rows(a.x, a.x_stride, kXT ? a.m : a.k, Tr::kBytes) &&
          aligned_rows(a.w, a.w_stride, kWT ? a.n : a.k, Tr::kBytes);
  return plan_gemm(a.m, a.n, a.k, Tr::kBytes, kXT + kWT, async);
}

// part: `room` bytes of scratch; without enough of it K is not split, and the tile stays the one planned with
// the split (float32 2560 x 512 x 2048: 47 us, without scratch 116; 320 x 320 x 1024: 13 and 28)
template <class Tr, bool kXT, bool kWT>
void launch_gemm(GemmArgs a, void* part, int64_t room, hipStream_t st) {
  bool async;
  Plan p = plan_for<Tr, kXT, kWT>(a, async);
  if (p.splits > 1 && (!part || room < (int64_t)p.splits * a.m * a.n * 4)) p.splits = 1;
  if (p.splits == 1) p.k_split = a.k;
  a.part = p.splits > 1 ? (float*)part : nullptr;
  a.k_split = p.k_split;
  a.tiles_m = (int)cdiv(a.m, p.tile);
  a.tiles_n = (int)cdiv(a.n, p.tile);
  if (async && Tr::kBytes == 2) launch_tiles<Tr, kXT, kWT, true>(a, p.tile, p.splits, st);
  else launch_tiles<Tr, kXT, kWT, false>(a, p.tile, p.splits, st);
  if (p.splits > 1) {
    const int64_t items = (int64_t)a.m * cdiv(a.n, 8);
    if (p.splits >= 8) launch((split_sum_kernel<Tr, 8>), dim3((unsigned)cdiv(items, 32)), dim3(256), 0, st, a, p.splits);
    else launch((split_sum_kernel<Tr, 1>), dim3((unsigned)cdiv(items, 256)), dim3(256), 0, st, a, p.splits);
  }
}

template <class Tr>
void run_linear(const GemmArgs& a, void* part, int64_t room, hipStream_t st) {
  if (a.m <= kFewRows && cdiv(a.n, 16) <= most_groups(512)) {
    const dim3 grid((unsigned)cdiv(a.n, 16));
    if (a.m <= 16) launch((rows_kernel<Tr, 1>), grid, dim3(512), 0, st, a);
    else if (a.m <= 32) launch((rows_kernel<Tr, 2>), grid, dim3(512), 0, st, a);
    else launch((rows_kernel<Tr, 4>), grid, dim3(512), 0, st, a);
    return;
  }
  launch_gemm<Tr, false, false>(a, part, room, st);
}

// Row groups of the column sums: enough workgroups for the chip, at least 32 rows each
inline int col_groups(int64_t m, int64_t n, int64_t r, int bytes) {
  const int64_t wgs = r * cdiv(n, 32 * (16 / bytes)), rows = cdiv(m, r);
  int64_t g = cdiv(4 * kCUs, wgs);
  if (g > cdiv(rows, 32)) g = cdiv(rows, 32);
  return (int)(g < 1 ? 1 : g > 512 ? 512 : g);
}
template <class Tr>
void run_cols(ColArgs c, float* part, hipStream_t st) {
  c.groups = col_groups(c.m, c.n, c.r, Tr::kBytes);
  c.chunk_blocks = (int)cdiv(c.n, 32 * (16 / Tr::kBytes));
  c.part = c.out && c.groups > 1 ? part : nullptr;
  const int64_t per = most_groups(256) / c.chunk_blocks;  // residues of a launch
  for (int64_t r0 = 0; r0 < c.r; r0 += per) {
    c.r0 = (int)r0;
    const dim3 grid((unsigned)(c.chunk_blocks * (c.r - r0 < per ? c.r - r0 : per)), (unsigned)c.groups);
    switch (c.act) {
      case YK_TOK_GELU: launch((cols_kernel<Tr, YK_TOK_GELU>), grid, dim3(256), 0, st, c); break;
      case YK_TOK_SILU: launch((cols_kernel<Tr, YK_TOK_SILU>), grid, dim3(256), 0, st, c); break;
      case YK_TOK_RELU: launch((cols_kernel<Tr, YK_TOK_RELU>), grid, dim3(256), 0, st, c); break;
      default: launch((cols_kernel<Tr, YK_TOK_NONE>), grid, dim3(256), 0, st, c);
    }
  }
  if (c.part)
    launch(cols_sum_kernel, dim3((unsigned)cdiv((int64_t)c.r * c.n, 64)), dim3(1024), 0, st, c);
}

template <class Tr>
void run_linear_grad(const yk_linear_grad_args& g, hipStream_t st) {
  const bool act = g.act != YK_TOK_NONE;
  char* ws = (char*)g.ws;
  char* dz = (char*)g.dy;
  int64_t dz_stride = g.dy_stride;
  if (act) {
    dz = ws;
    dz_stride = g.n;
    ws += cdiv(g.m * g.n * Tr::kBytes, 16) * 16;
  }
  float* part = (float*)ws;  // one region: the kernels that use it follow each other on the stream
  const int64_t room = g.ws ? g.ws_bytes - (ws - (char*)g.ws) : 0;
  if (act || g.dbias) {
    ColArgs c{(const char*)g.dy, (const char*)g.z, dz, g.dbias, nullptr, g.dy_stride, g.z_stride, g.n, (int)g.m,
              (int)g.n, 1, 1, g.act, g.bias_f32 || Tr::kBytes == 4, g.dtype, 1};
    run_cols<Tr>(c, part, st);
  }
  if (g.dres) {
    ColArgs c{(const char*)g.dy, nullptr, nullptr, g.dres, nullptr, g.dy_stride, 0, g.dres_stride, (int)g.m,
              (int)g.n, (int)g.res_rows, 1, YK_TOK_NONE, Tr::kBytes == 4, g.dtype, 1};
    run_cols<Tr>(c, part, st);
  }
  if (g.dx) {
    GemmArgs a{};
    a.x = dz, a.x_stride = dz_stride;
    a.w = (const char*)g.w, a.w_stride = g.w_stride;
    a.y = (char*)g.dx, a.y_stride = g.dx_stride;
    a.m = (int)g.m, a.n = (int)g.k, a.k = (int)g.n, a.dtype = g.dtype;
    launch_gemm<Tr, false, true>(a, part, room, st);
  }
  if (g.dw) {
    GemmArgs a{};
    a.x = dz, a.x_stride = dz_stride;
    a.w = (const char*)g.x, a.w_stride = g.x_stride;
    a.y = (char*)g.dw, a.y_stride = g.dw_stride;
    a.m = (int)g.n, a.n = (int)g.k, a.k = (int)g.m, a.dtype = g.dtype;
    launch_gemm<Tr, true, true>(a, part, room, st);
  }
}

int check_linear(const char* fn, int dtype, int act, int64_t m, int64_t n, int64_t k) {
  YK_CHECK_ARG(tok_bytes(dtype), std::string(fn) + ": dtype must be YK_ACT_BF16, YK_ACT_F32 or YK_ACT_F16");
  YK_CHECK_ARG(act >= YK_TOK_NONE && act <= YK_TOK_RELU, std::string(fn) + ": bad activation");
  YK_CHECK_ARG(m >= 0 && m < (1 << 30) && n >= 1 && n < (1 << 30) && k >= 1 && k < (1 << 30),
               std::string(fn) + ": sizes out of range (m in [0, 2^30), n and k in [1, 2^30))");
  YK_CHECK_ARG(cdiv(m, 128) * cdiv(n, 128) <= most_groups(256) && cdiv(m, 128) * cdiv(k, 128) <= most_groups(256) &&
                   cdiv(n, 128) * cdiv(k, 128) <= most_groups(256),
               std::string(fn) + ": more tiles than a launch holds");
  return YK_OK;
}

}  // namespace tok
}  // namespace yk

using namespace yk::tok;

extern "C" {

int yk_linear_workspace(const yk_linear_args* a, int64_t* bytes) {
  YK_CHECK_ARG(a && bytes, "yk_linear_workspace: NULL argument");
  if (const int rc = check_linear("yk_linear_workspace", a->dtype, a->act, a->m, a->n, a->k)) return rc;
  *bytes = a->m <= kFewRows ? 0 : gemm_scratch(a->m, a->n, a->k, tok_bytes(a->dtype), 0);
  return YK_OK;
}

int yk_linear(yk_ctx* ctx, const yk_linear_args* a, void* stream) {
  YK_CHECK_ARG(ctx && a, "yk_linear: NULL argument");
  if (const int rc = check_linear("yk_linear", a->dtype, a->act, a->m, a->n, a->k)) return rc;
  if (a->m == 0) return YK_OK;
  YK_CHECK_ARG(a->x && a->w && a->y, "yk_linear: x, w and y must be set");
  YK_CHECK_ARG(!a->res || (a->res_rows >= 1 && a->res_rows <= a->m), "yk_linear: res_rows must be in [1, m]");
  YK_CHECK_ARG(a->x_stride >= 0 && a->w_stride >= 0 && (!a->res || a->res_stride >= 0) &&
                   (a->m == 1 || (a->y_stride >= a->n && (!a->z || a->z_stride >= a->n))),
               "yk_linear: a negative row stride, or an output's is shorter than its row");
  YK_CHECK_ARG(!a->ws || (a->ws_bytes >= 0 && (uintptr_t)a->ws % 16 == 0),
               "yk_linear: ws must be 16-byte aligned (NULL or too short: K is not split)");
  yk::DeviceGuard g(ctx->device);
  GemmArgs k{(const char*)a->x, (const char*)a->w, a->bias, (const char*)a->res, (char*)a->y, (char*)a->z, nullptr,
             a->x_stride, a->w_stride, a->res_stride, a->y_stride, a->z_stride, (int)a->m, (int)a->n, (int)a->k,
             (int)a->res_rows, a->act, a->bias_f32 || a->dtype == YK_ACT_F32, a->dtype, 0, 0, 0};
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == YK_ACT_F32) run_linear<F32>(k, a->ws, a->ws_bytes, st);
  else if (a->dtype == YK_ACT_BF16) run_linear<B16>(k, a->ws, a->ws_bytes, st);
  else run_linear<H16>(k, a->ws, a->ws_bytes, st);
  return launched("yk_linear");
}

int yk_linear_backward_workspace(const yk_linear_grad_args* a, int64_t* bytes) {
  YK_CHECK_ARG(a && bytes, "yk_linear_backward_workspace: NULL argument");
  if (const int rc = check_linear("yk_linear_backward_workspace", a->dtype, a->act, a->m, a->n, a->k)) return rc;
  YK_CHECK_ARG(!a->dres || (a->res_rows >= 1 && a->res_rows <= a->m), "yk_linear_backward_workspace: res_rows must be in [1, m]");
  const int e = tok_bytes(a->dtype);
  int64_t part = 0;
  auto grow = [&](int64_t b) { part = b > part ? b : part; };
  if (a->m) {
    if (a->dbias) grow(col_groups(a->m, a->n, 1, e) * a->n * 4);
    if (a->dres) grow((int64_t)col_groups(a->m, a->n, a->res_rows, e) * a->res_rows * a->n * 4);
    if (a->dx) grow(gemm_scratch(a->m, a->k, a->n, e, 1));
    if (a->dw) grow(gemm_scratch(a->n, a->k, a->m, e, 2));
    if (a->act != YK_TOK_NONE) part += cdiv(a->m * a->n * e, 16) * 16;
  }
  *bytes = part;
  return YK_OK;
}

int yk_linear_backward(yk_ctx* ctx, const yk_linear_grad_args* a, void* stream) {
  YK_CHECK_ARG(ctx && a, "yk_linear_backward: NULL argument");
  if (const int rc = check_linear("yk_linear_backward", a->dtype, a->act, a->m, a->n, a->k)) return rc;
  if (!a->dx && !a->dw && !a->dbias && !a->dres) return YK_OK;
  YK_CHECK_ARG(a->m >= 1, "yk_linear_backward: m must be >= 1");
  YK_CHECK_ARG(a->dy && (a->act == YK_TOK_NONE || a->z) && (!a->dx || a->w) && (!a->dw || a->x),
               "yk_linear_backward: an input that the requested gradients need is NULL");
  YK_CHECK_ARG(a->dy_stride >= 0 && a->x_stride >= 0 && a->w_stride >= 0 && a->z_stride >= 0 &&
                   (!a->dx || a->m == 1 || a->dx_stride >= a->k) && (!a->dw || a->n == 1 || a->dw_stride >= a->k) &&
                   (!a->dres || a->res_rows == 1 || a->dres_stride >= a->n),
               "yk_linear_backward: a negative row stride, or an output's is shorter than its row");
  int64_t need = 0;
  if (const int rc = yk_linear_backward_workspace(a, &need)) return rc;
  YK_CHECK_ARG(need == 0 || (a->ws && a->ws_bytes >= need && (uintptr_t)a->ws % 16 == 0),
               "yk_linear_backward: ws must be yk_linear_backward_workspace bytes, 16-byte aligned");
  yk::DeviceGuard g(ctx->device);
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == YK_ACT_F32) run_linear_grad<F32>(*a, st);
  else if (a->dtype == YK_ACT_BF16) run_linear_grad<B16>(*a, st);
  else run_linear_grad<H16>(*a, st);
  return launched("yk_linear_backward");
}

}  // extern "C"
