// Tiled matrix products on the 16-bit matrix cores (CDNA4, gfx950) with the epilogue left to the
// caller: the main loop of the vocabulary head's loss (linear_xent.hip) and of the Linear layer
// with an 8-bit input checkpoint (act8.hip).
//
//   C[i][j] = sum_k I(i, k) J(j, k)        fp32 accumulators, 16-bit operands
//
//  * An operand is "row" (k contiguous: I[i][k]) or "col" (k outermost: I[k][i]).  A row operand's
//    stage is kept as rows of BK elements, their 16-byte chunks XOR-swizzled, and read with
//    ds_read_b128; a col operand's as panels of 128 columns, read with the transposing
//    ds_read_b64_tr_b16.  So x w^T (row, row), dy w (row, col) and dy^T x (col, col) share one loop
//    and nothing is transposed in memory.
//  * v_mfma_f32_32x32x16 with J as its first operand: a lane then holds ONE row i (lane & 31) and
//    four consecutive columns j in each register quad, so a softmax over j is nearly all in-lane and
//    a store moves 8 or 16 bytes.
//  * Stages of BK reduction steps arrive in a ring of ST LDS buffers by 16-byte LDS-DMA (no staging
//    registers), one barrier a stage.  The barrier stands in front of a stage's last products: their
//    fragments are in registers, so the buffer is refilled (one DMA instruction between two products)
//    and the next stage's first fragments are read while they run.  Chunks past the reduction's end
//    read a zero chunk; rows past an operand's end read its last row (never stored).
//  * fp32 operands run as three bf16 planes, x = hi + mid + lo exactly: each is what the planes before it
//    leave, rounded to bf16, and 3 x 8 bits are fp32's 24.  bf16 has fp32's exponents, so the planes hold an
//    element by itself, whatever else its row or tensor holds (down to 2^-110, below which lo, then
//    mid, run out of exponents).  Six products, the smallest first: mid.lo, lo.mid (2^-27 of the result each)
//    and lo.lo are left out.  Two fp16 planes would do with three products, but hold an element only to
//    2^-50 of the largest that shares its scale: one row of 1e16 in a tensor, and the others are gone.
#pragma once

#include "common.h"

#include <algorithm>
#include <type_traits>

namespace voda {
namespace gt {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4_v __attribute__((__vector_size__(4 * sizeof(__bf16))));
typedef __attribute__((address_space(3))) bf16x4_v lds_bf16x4;
typedef __attribute__((address_space(3))) void lds_void;

// what chunks past a reduction's end read
static __device__ __attribute__((aligned(16))) uint32_t zero_chunk[4];

struct Operand {
  const uint16_t* p;
  int64_t ld;     // elements between rows (row operand: between i; col operand: between k)
  int64_t plane;  // elements between two planes
  int n;          // rows i (>= 1)
};

// LDS[m0 + 16 * lane] = global[gptr].  s_nop: the load may read M0 one wait state after its write, and in here
// the compiler puts none.
__device__ __forceinline__ void dma16(const void* gptr, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(gptr), "s"(lds_addr) : "memory", "m0");
}

template <int N>
__device__ __forceinline__ void wait_vm_barrier() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// byte offset of 16-byte chunk ``ch`` (0..15) of row ``r`` of a 128-column panel (col operands)
__device__ __forceinline__ int panel_off(int r, int ch) {
  return r * 256 + 16 * (ch ^ (((r & 3) << 2) | ((r >> 2) & 3)));
}

__device__ __forceinline__ uint2 tr_read(const uint8_t* base, int off) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(base + off)));
}

__device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// sum of a fragment's eight elements, in fp32
__device__ __forceinline__ float sum8(uint4 f) {
  const uint32_t u[4] = {f.x, f.y, f.z, f.w};
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u[e]), bf16x2{1, 1}, s, false);
  return s;
}

// One operand's stage in LDS: EXT rows i x BK reduction steps, filled by NW waves, read by waves
// whose sub-tile is T 32-row tiles from row ``sub`` on.
template <bool COL, int EXT, int BK, int NW, int T>
struct Stage {
  static constexpr int kBytes = EXT * BK * 2;
  static constexpr int kInstr = kBytes / 1024;  // 1 KB wave-instructions
  static constexpr int kPer = kInstr / NW;      // per wave
  static_assert(kInstr % NW == 0, "a stage is whole wave-instructions for every wave");
  static_assert(!COL || EXT % 128 == 0, "col operands come in panels of 128");
  static constexpr int CPR = BK / 8;            // row operands: chunks a row
  static constexpr int RPI = 64 / CPR;          // rows a wave-instruction

  const uint16_t* src[kPer];
  int off[COL ? 2 * T : BK / 16];

  // The LDS serves 16 lanes of 16 bytes a clock, 256 bytes: the rows that share a place in 256 bytes
  // differ in their swizzle among any 16 neighbouring rows
  static_assert(CPR <= 16, "rows of at most 256 bytes");
  static __device__ __forceinline__ int swz(int row) { return (row / (16 / CPR)) & (CPR - 1); }

  // place of this lane's chunk in wave-instruction q: its row / column and k inside the stage
  static __device__ __forceinline__ void place(int q, int lane, int& r, int& k) {
    if constexpr (COL) {
      const int panel = q / (BK / 4), rq = q % (BK / 4);
      k = 4 * rq + (lane >> 4);
      r = panel * 128 + 8 * ((lane & 15) ^ (((k & 3) << 2) | ((k >> 2) & 3)));
    } else {
      const int row = q * RPI + lane / CPR;
      r = row;
      k = 8 * ((lane % CPR) ^ swz(row));
    }
  }

  __device__ __forceinline__ void init(const Operand& o, int r0, int k0, int wave, int lane, int sub) {
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      int r, k;
      place(wave * kPer + u, lane, r, k);
      if constexpr (COL)  // chunks of 8 columns past the last one read that one, never stored
        src[u] = o.p + int64_t(k0 + k) * o.ld + min(r0 + r, (o.n - 1) & ~7);
      else
        src[u] = o.p + int64_t(min(r0 + r, o.n - 1)) * o.ld + k0 + k;
    }
    const int h = lane >> 5;
    if constexpr (COL) {
      const int g = lane >> 4, q = (lane & 15) >> 2, pp = lane & 3;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const int c = sub + 32 * t;  // first column of the tile inside the stage
        const int base = (c >> 7) * (BK * 256) + 8 * (pp & 1);
        const int ch = ((c & 127) >> 3) + 2 * (g & 1) + (pp >> 1);
        off[2 * t] = base + panel_off(8 * h + q, ch);
        off[2 * t + 1] = base + panel_off(8 * h + q + 4, ch);
      }
    } else {
      const int row = sub + (lane & 31);
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk) off[kk] = row * (BK * 2) + 16 * ((2 * kk + h) ^ swz(row));
    }
  }

  // this wave's instruction u: ``shift`` elements from the first stage's addresses, ``left`` reduction
  // steps remain
  __device__ __forceinline__ void issue(int u, uint8_t* lds, int64_t shift, int left, int wave, int lane) const {
    const int q = wave * kPer + u;
    int r, k;
    place(q, lane, r, k);
    dma16(k < left ? static_cast<const void*>(src[u] + shift) : zero_chunk,
          __builtin_amdgcn_readfirstlane(uint32_t(size_t((lds_void*)(lds + 1024 * q)))));
  }

  __device__ __forceinline__ uint4 frag(const uint8_t* lds, int t, int kk) const {
    if constexpr (COL) {
      const uint2 lo = tr_read(lds + 4096 * kk, off[2 * t]), hi = tr_read(lds + 4096 * kk, off[2 * t + 1]);
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else {
      return *reinterpret_cast<const uint4*>(lds + off[kk] + t * (64 * BK));
    }
  }
};

// Tile of WJ x WI waves, each TJ x TI 32 x 32 blocks: BJ = 32 WJ TJ columns, BI = 32 WI TI rows.
// NP products: 1 (plain 16-bit operands), 2 or 3 (I in that many planes, J in one), 6 (both in three).
template <int NP, bool IT, bool JT, int WJ_, int WI_, int TJ_, int TI_, int BK_, int ST_>
struct Tile {
  static constexpr int WJ = WJ_, WI = WI_, TJ = TJ_, TI = TI_, BK = BK_, ST = ST_;
  static constexpr int NW = WJ * WI, kThreads = 64 * NW;
  static constexpr int BJ = 32 * WJ * TJ, BI = 32 * WI * TI;
  using SI = Stage<IT, BI, BK, NW, TI>;
  using SJ = Stage<JT, BJ, BK, NW, TJ>;
  static constexpr int kStage = SI::kBytes + SJ::kBytes;
  static constexpr int kLds = ST * kStage;
  static constexpr int kPer = SI::kPer + SJ::kPer;
  static_assert(NP == 1 || NP == 2 || NP == 3 || NP == 6, "products");
  static_assert(ST >= 2 && (ST - 1) * kPer < 64 && BK % 32 == 0, "ring depth");

  // planes of product p: (2 0) (0 2) (1 1) (1 0) (0 1) (0 0), or I's from the last on
  static __device__ __forceinline__ int plane_i(int p) { return NP == 6 ? (0x52 >> (2 * p)) & 3 : NP - 1 - p; }
  static __device__ __forceinline__ int plane_j(int p) { return NP == 6 ? (0x118 >> (2 * p)) & 3 : 0; }

  struct Where {
    int lane, wave, h, il, wi, wj;
    __device__ __forceinline__ Where() {
      lane = threadIdx.x & 63;
      wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
      h = lane >> 5;
      il = lane & 31;
      wj = wave % WJ;
      wi = wave / WJ;
    }
    // row i of block ti and first column of register quad g of block tj, inside the tile
    __device__ __forceinline__ int i(int ti) const { return (wi * TI + ti) * 32 + il; }
    __device__ __forceinline__ int j(int tj, int g) const { return (wj * TJ + tj) * 32 + 8 * g + 4 * h; }
  };

  // acc[tj][ti] = the tile's products over k in [k0, k1).  SUM and ``want``: also the sums of I over k
  // (all its planes) for this lane's rows i; half h of the wave holds half of them.
  template <bool SUM>
  static __device__ __forceinline__ void run(uint8_t* smem, const Operand& I, const Operand& J, int i0, int j0, int k0,
                                             int k1, f32x16 (&acc)[TJ][TI], float (&isum)[TI], bool want = false) {
    const Where w;
    SI si;
    SJ sj;
    si.init(I, i0, k0, w.wave, w.lane, w.wi * TI * 32);
    sj.init(J, j0, k0, w.wave, w.lane, w.wj * TJ * 32);
#pragma unroll
    for (int a = 0; a < TJ; ++a)
#pragma unroll
      for (int b = 0; b < TI; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
#pragma unroll
    for (int b = 0; b < TI; ++b) isum[b] = 0.f;
    const int steps = k1 > k0 ? (k1 - k0 + BK - 1) / BK : 0;
    const int total = NP * steps;
    const int64_t stepi = IT ? BK * I.ld : BK, stepj = JT ? BK * J.ld : BK;
    int at = 0, prod = 0;  // next stage to issue: its step and product
    // instruction u of the next stage into ``lds``
    int64_t shi = 0, shj = 0;
    int left = 0;
    auto aim = [&] {
      left = k1 - k0 - at * BK;
      shi = at * stepi + plane_i(prod) * I.plane;
      shj = at * stepj + plane_j(prod) * J.plane;
      if (++at >= steps) { at = 0; ++prod; }
    };
    auto issue = [&](int u, uint8_t* lds) {
      if (u < SI::kPer) si.issue(u, lds, shi, left, w.wave, w.lane);
      else sj.issue(u - SI::kPer, lds + SI::kBytes, shj, left, w.wave, w.lane);
    };
#pragma unroll
    for (int s = 0; s < ST; ++s) {
      if (s >= total) break;
      aim();
#pragma unroll
      for (int u = 0; u < kPer; ++u) issue(u, smem + s * kStage);
    }
    uint4 fi[2][TI], fj[2][TJ];
    auto fetch = [&](int buf, int kk, int set) {
      const uint8_t* li = smem + buf * kStage;
#pragma unroll
      for (int b = 0; b < TI; ++b) fi[set][b] = si.frag(li, b, kk);
#pragma unroll
      for (int a = 0; a < TJ; ++a) fj[set][a] = sj.frag(li + SI::kBytes, a, kk);
    };
    // until at most n stages are on their way, then the barrier
    auto wait_stages = [](int n) {
      if (ST > 3 && n >= 3) wait_vm_barrier<(ST > 3 ? 3 * kPer : 0)>();
      else if (ST > 2 && n >= 2) wait_vm_barrier<(ST > 2 ? 2 * kPer : 0)>();
      else if (n >= 1) wait_vm_barrier<kPer>();
      else wait_vm_barrier<0>();
    };
    wait_stages(total - 1);
    fetch(0, 0, 0);
    int buf = 0, st = 0;
    int sum_prod = 0, sum_at = 0;  // SUM: product and step of the stage that runs
    constexpr int mf = TI * TJ;
    // one stage; ``more``: a stage is left to issue into the buffer that it frees
    auto stage = [&](auto more) {
      const int next = buf + 1 == ST ? 0 : buf + 1;
#pragma unroll
      for (int kk = 0; kk < BK / 16; ++kk) {
        const bool tail = kk + 1 == BK / 16;
        if (tail) {
          if constexpr (more.value) {
            wait_vm_barrier<(ST - 2) * kPer>();
            aim();
          } else {
            wait_stages(total - 2 - st);
          }
          fetch(next, 0, 0);  // past the last stage: never used
        }
        if constexpr (SUM) {
          // each of I's planes once, where it runs with J's first
          if (want && plane_j(sum_prod) == 0) {
#pragma unroll
            for (int b = 0; b < TI; ++b) isum[b] += sum8(fi[kk & 1][b]);
          }
        }
#pragma unroll
        for (int x = 0; x < mf; ++x) {
          acc[x / TI][x % TI] = mfma(fj[kk & 1][x / TI], fi[kk & 1][x % TI], acc[x / TI][x % TI]);
          // between two products: a DMA instruction or two of the refill, or a fragment of the next step
          if (tail) {
            if constexpr (more.value) {
              constexpr int per = (kPer + mf - 1) / mf;
#pragma unroll
              for (int y = x * per; y < (x + 1) * per && y < kPer; ++y) issue(y, smem + buf * kStage);
            }
          } else {
            constexpr int nf = TI + TJ;
            const uint8_t* li = smem + buf * kStage;
#pragma unroll
            for (int y = 0; y < nf; ++y)
              if (y * mf / nf == x) {
                if (y < TI) fi[(kk + 1) & 1][y] = si.frag(li, y, kk + 1);
                else fj[(kk + 1) & 1][y - TI] = sj.frag(li + SI::kBytes, y - TI, kk + 1);
              }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      buf = next;
      if (SUM && ++sum_at == steps) { sum_at = 0; ++sum_prod; }
    };
    for (; st + ST < total; ++st) stage(std::true_type{});
    for (; st < total; ++st) stage(std::false_type{});
    wait_vm_barrier<0>();
  }
};

// Tiles in the order that an XCD's L2 serves best: workgroups are dealt to the 8 XCDs in turn, so
// each XCD gets one run of the order; inside it, groups of ``gi`` row tiles stay while the column
// tiles go by.  The order covers the live tiles only (a device count decides how many there are), so
// that the work is spread over the XCDs whatever their number.
__device__ __forceinline__ void tile_at(int bid, int live, int ti, int tj, int gi, int& i, int& j, int& s) {
  const int x = bid & 7, q = live >> 3, r = live & 7;
  const int t = x * q + min(x, r) + (bid >> 3);
  const int tiles = ti * tj;
  s = t / tiles;
  const int u = t - s * tiles;
  const int per = gi * tj, grp = u / per, v = u - grp * per;
  const int rows = min(gi, ti - grp * gi);
  j = v / rows;
  i = grp * gi + (v - j * rows);
}

constexpr int kGroup = 8;  // row tiles a group

// Splits of a reduction: as many as fill the chip's ``slots`` workgroups once, each at least ``least``
// steps long, ``most`` at most.  The same on the host and on the device, where the sizes may be known
// only there.
struct Split {
  int slots, least, most = 64;
  __host__ __device__ int of(int64_t tiles, int64_t nk) const {
    int64_t s = slots / (tiles < 1 ? 1 : tiles);
    s = s < nk / least ? s : nk / least;
    return int(s < 1 ? 1 : s > most ? most : s);
  }
};

// fp32 -> its three planes.  A finite x that would round past bf16's largest takes that one; an infinite or
// NaN x is hi alone.
__device__ __forceinline__ void split3(float x, uint16_t& hi, uint16_t& mid, uint16_t& lo) {
  const bool finite = fabsf(x) <= 3.4028235e38f;
  hi = f2bf(x);
  if (finite && (hi & 0x7fff) == 0x7f80) --hi;
  const float r = x - bf2f(hi);  // exact, as is what follows
  mid = f2bf(r);
  lo = f2bf(r - bf2f(mid));
  if (!finite) mid = lo = 0;
}

// ---- stores -----------------------------------------------------------------------------------

// What becomes of a product: out = (sum of its splits) * factor [* gelu'(checkpoint)] [+ bias]
// [+ out], in fp32 until the one rounding to out's type.
struct Emit {
  void* out;
  int64_t ldo;
  int bf16;                 // out's type: bf16 or fp32
  int nj;                   // columns
  int vec;                  // rows start 16-byte aligned: eights go out in whole vectors
  int accumulate;           // add to what out holds
  const void* bias;         // [nj], or null
  int bias_bf16;
  const uint8_t* q;         // e4m3 checkpoint [i][ldq] whose gelu' multiplies, or null
  const uint8_t* qs;        // its scales [i][ldq / 32]
  int64_t ldq;
  // the factor: *gl / max(*gn, 1), or 1 without them
  const float* gl;
  const int* gn;

  // what a kernel reads once: the factor and the bias of a lane's eight columns
  struct Once {
    float a;
    float bias[8];
  };
  __device__ __forceinline__ Once once(int j) const {
    Once o;
    o.a = gl ? *gl / float(max(*gn, 1)) : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      o.bias[e] = !bias || j + e >= nj ? 0.f
                  : bias_bf16          ? bf2f(static_cast<const uint16_t*>(bias)[j + e])
                                       : static_cast<const float*>(bias)[j + e];
    return o;
  }
  // the checkpoint of columns j .. j+7 of row i
  struct Check {
    uint2 u;
    uint32_t s;
  };
  __device__ __forceinline__ Check check(int i, int j) const {
    Check c = {make_uint2(0, 0), 0};
    if (q && j < nj) {  // ldq % 32 == 0
      c.u = *reinterpret_cast<const uint2*>(q + int64_t(i) * ldq + j);
      c.s = qs[int64_t(i) * (ldq >> 5) + (j >> 5)];
    }
    return c;
  }
  // columns j .. j+7 of row i (j % 8 == 0); ``keep`` false: the row is zero whatever the factor is
  __device__ __forceinline__ void eight(const Once& o, const Check& c, int i, int j, float (&v)[8], bool keep = true) const {
    if (j >= nj) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = !keep ? 0.f : v[e] * o.a;
    if (q) {
      const uint2 u = c.u;
      const float s = __uint_as_float(c.s << 23);
      v[0] *= gelu_tanh_grad(__builtin_amdgcn_cvt_f32_fp8(u.x, 0) * s);
      v[1] *= gelu_tanh_grad(__builtin_amdgcn_cvt_f32_fp8(u.x, 1) * s);
      v[2] *= gelu_tanh_grad(__builtin_amdgcn_cvt_f32_fp8(u.x, 2) * s);
      v[3] *= gelu_tanh_grad(__builtin_amdgcn_cvt_f32_fp8(u.x, 3) * s);
      v[4] *= gelu_tanh_grad(__builtin_amdgcn_cvt_f32_fp8(u.y, 0) * s);
      v[5] *= gelu_tanh_grad(__builtin_amdgcn_cvt_f32_fp8(u.y, 1) * s);
      v[6] *= gelu_tanh_grad(__builtin_amdgcn_cvt_f32_fp8(u.y, 2) * s);
      v[7] *= gelu_tanh_grad(__builtin_amdgcn_cvt_f32_fp8(u.y, 3) * s);
    }
    if (bias) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += o.bias[e];
    }
    put(i, j, v);
  }
  __device__ __forceinline__ void put(int i, int j, const float (&v)[8]) const {
    const bool whole = vec && j + 8 <= nj;
    if (bf16) {
      uint16_t* o = static_cast<uint16_t*>(out) + int64_t(i) * ldo + j;
      if (whole) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (accumulate) u = *reinterpret_cast<const uint4*>(o);
        auto two = [&](uint32_t old, float x, float y) {
          return uint32_t(f2bf(x + bf2f(old & 0xffff))) | (uint32_t(f2bf(y + bf2f(old >> 16))) << 16);
        };
        *reinterpret_cast<uint4*>(o) =
            make_uint4(two(u.x, v[0], v[1]), two(u.y, v[2], v[3]), two(u.z, v[4], v[5]), two(u.w, v[6], v[7]));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (j + e < nj) o[e] = f2bf(v[e] + (accumulate ? bf2f(o[e]) : 0.f));
      }
    } else {
      float* o = static_cast<float*>(out) + int64_t(i) * ldo + j;
      if (whole) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
        if (accumulate) {
          a = *reinterpret_cast<const float4*>(o);
          b = *reinterpret_cast<const float4*>(o + 4);
        }
        *reinterpret_cast<float4*>(o) = make_float4(v[0] + a.x, v[1] + a.y, v[2] + a.z, v[3] + a.w);
        *reinterpret_cast<float4*>(o + 4) = make_float4(v[4] + b.x, v[5] + b.y, v[6] + b.z, v[7] + b.w);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (j + e < nj) o[e] = v[e] + (accumulate ? o[e] : 0.f);
      }
    }
  }
};

// A wave's block of 32 rows x 32 TJ columns goes through its own part of the LDS, fp32, so that the
// stores move whole lines: straight from the accumulators a store would scatter 32 rows' worth of 16
// or 32 bytes.  Chunks of 16 bytes are XOR-swizzled by the row: no bank conflicts either way.
// ``g(i, j, v)`` gets eight columns of a row at a time, a lane the same columns each time.
template <class T, class G>
__device__ __forceinline__ void through_lds(uint8_t* smem, const typename T::Where& w, const f32x16 (&acc)[T::TJ][T::TI],
                                            int b, G&& g) {
  constexpr int CH = 8 * T::TJ;  // chunks a row
  static_assert(T::kLds / T::NW >= 32 * CH * 16, "a wave's block fits its part of the LDS");
  uint8_t* mine = smem + w.wave * (T::kLds / T::NW / 16 * 16);
  uint8_t* row = mine + w.il * (CH * 16);
  const int sw = 16 * (w.il & (CH - 1)) ^ (16 * w.h);
#pragma unroll
  for (int a = 0; a < T::TJ; ++a)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      *reinterpret_cast<float4*>(row + ((16 * (8 * a + 2 * q)) ^ sw)) =
          make_float4(acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]);
    }
  __builtin_amdgcn_wave_barrier();
  constexpr int EI = CH / 2;     // eights a row
  constexpr int RP = 64 / EI;    // rows a pass
  const int e = w.lane % EI;
#pragma unroll 2
  for (int r = w.lane / EI; r < 32; r += RP) {
    const uint8_t* from = mine + r * (CH * 16);
    const int x = 16 * ((2 * e) ^ (r & (CH - 1)));
    const float4 lo = *reinterpret_cast<const float4*>(from + x), hi = *reinterpret_cast<const float4*>(from + (x ^ 16));
    float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    g((w.wi * T::TI + b) * 32 + r, w.wj * T::TJ * 32 + 8 * e, v);
  }
  __builtin_amdgcn_wave_barrier();
}

struct GemmArgs {
  Operand I, J;
  const int* ni_dev;     // rows in use (<= I.n), or null: all
  const int* nk_dev;     // reduction length in use (<= nk), or null: all
  int nk;
  Split split;
  int nk_split;          // length that the number of splits goes by
  // fp32 partial results [split][rows in use][lds] (``add``: onto what is there), or null: one split
  float* slab;
  int64_t lds;
  int add;
  float* bslab;          // [split][I.n] partial sums of I over k (col I), or null
  void* bout;            // their result when there is no slab
  int bout_bf16;
  Emit e;

  __device__ __forceinline__ int rows() const { return ni_dev ? min(I.n, *ni_dev) : I.n; }
  __device__ __forceinline__ int length() const { return nk_dev ? min(nk, *nk_dev) : nk; }
  __device__ __forceinline__ int splits(int64_t tiles) const {
    return slab ? split.of(tiles, nk_dev ? length() : nk_split) : 1;
  }
};

// one split's reduction range: whole stages, as even as they go
__device__ __forceinline__ void split_range(int nk, int splits, int s, int bk, int& k0, int& k1) {
  const int steps = (nk + bk - 1) / bk, per = (steps + splits - 1) / splits;
  k0 = min(nk, s * per * bk);
  k1 = min(nk, k0 + per * bk);
}

// a sum over I alone
__device__ __forceinline__ void emit_sum(const Emit& e, const Emit::Once& o, void* out, bool bf16, int i, float v) {
  v = v * o.a;
  if (bf16) {
    uint16_t* o = static_cast<uint16_t*>(out) + i;
    *o = f2bf(v + (e.accumulate ? bf2f(*o) : 0.f));
  } else {
    float* o = static_cast<float*>(out) + i;
    *o = v + (e.accumulate ? *o : 0.f);
  }
}

template <class T, bool SUM>
__global__ __launch_bounds__(T::kThreads, 2) void gemm_kernel(GemmArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[T::kLds];
  Operand I = p.I;
  I.n = p.rows();
  const int ni = (I.n + T::BI - 1) / T::BI, nj = (p.e.nj + T::BJ - 1) / T::BJ;
  const int splits = p.splits(int64_t(ni) * nj), live = ni * nj * splits;
  if (int(blockIdx.x) >= live) return;
  int ti, tj, s, k0, k1;
  tile_at(blockIdx.x, live, ni, nj, kGroup, ti, tj, s);
  const int i0 = ti * T::BI, j0 = tj * T::BJ;
  split_range(p.length(), splits, s, T::BK, k0, k1);
  const typename T::Where w;
  const bool want = SUM && (p.bslab || p.bout) && tj == 0 && w.wj == 0;
  f32x16 acc[T::TJ][T::TI];
  float isum[T::TI];
  T::template run<SUM>(smem, I, p.J, i0, j0, k0, k1, acc, isum, want);
  // through_lds gives a lane the same columns each time
  const int once_j = j0 + w.wj * T::TJ * 32 + 8 * (w.lane % (4 * T::TJ));
  const Emit::Once once = p.e.once(once_j);
  Emit o = p.e;
  if (p.slab) {
    o.out = p.slab + int64_t(s) * I.n * p.lds;
    o.ldo = o.nj = int(p.lds);
    o.bf16 = 0;
    o.vec = 1;
    o.accumulate = p.add;
  }
  // a lane's rows, RP apart from one call to the next: each row's checkpoint is read a call ahead
  constexpr int RP = 16 / T::TJ;
  auto ahead = [&](int r) { return p.slab ? Emit::Check{} : p.e.check(min(i0 + r, I.n - 1), once_j); };
  Emit::Check next = ahead(w.wi * T::TI * 32 + w.lane / (4 * T::TJ));
#pragma unroll
  for (int b = 0; b < T::TI; ++b) {
    const int i = i0 + w.i(b);
    if constexpr (SUM) {
      if (want) {
        const float tot = isum[b] + __shfl_xor(isum[b], 32, 64);
        if (w.h == 0 && i < I.n) {
          if (p.bslab) p.bslab[int64_t(s) * p.I.n + i] = tot;
          else emit_sum(p.e, once, p.bout, p.bout_bf16, i, tot);
        }
      }
    }
    through_lds<T>(smem, w, acc, b, [&](int r, int c, float(&v)[8]) {
      const Emit::Check now = next;
      next = ahead(r + RP);
      if (i0 + r >= I.n) return;
      if (p.slab) o.put(i0 + r, j0 + c, v);
      else o.eight(once, now, i0 + r, j0 + c, v);
    });
  }
}

// Sums of ``parts`` partial sums a column (rows_dev: of ``per`` for each ``bi`` rows in use instead).
struct ColumnSums {
  const float* part;  // [parts][ld], or null: none
  int64_t ld;
  int n, parts;
  const int* rows_dev;
  int bi, per;
  void* out;
  int bf16;
  Emit e;             // the factor and whether to add
};

// Sums the splits of a product's slab and stores the result; ``inv`` (or null) maps an output row to its
// row of the slab, -1 where the row is zero.  LANES threads take eight columns together, each every
// LANES-th split; behind them one thread a column sum.
struct FinishArgs {
  GemmArgs g;
  int bi, bj;   // the product's tile
  int rows;     // 0: column sums alone
  const int* inv;
  ColumnSums c;
};

template <int LANES>
static __global__ __launch_bounds__(256) void finish_kernel(FinishArgs p) {
  const int eights = (p.g.e.nj + 7) >> 3;
  const int64_t n = int64_t(p.rows) * eights;
  const int64_t t = (int64_t(blockIdx.x) * 256 + threadIdx.x) / LANES;
  const int part = threadIdx.x % LANES;
  if (t < n) {
    const int used = p.g.rows();
    const int splits = p.g.splits(int64_t((used + p.bi - 1) / p.bi) * ((p.g.e.nj + p.bj - 1) / p.bj));
    const int i = int(t / eights), j = 8 * int(t - int64_t(i) * eights);
    const int src = p.inv ? p.inv[i] : i;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (src >= 0) {
      const float* a = p.g.slab + int64_t(src) * p.g.lds + j;
#pragma unroll 4
      for (int s = part; s < splits; s += LANES) {
        const float* b = a + int64_t(s) * used * p.g.lds;
        const float4 x = *reinterpret_cast<const float4*>(b), y = *reinterpret_cast<const float4*>(b + 4);
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
      }
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += __shfl_xor(v[e], o, 64);
    if (part == 0) p.g.e.eight(p.g.e.once(j), p.g.e.check(i, j), i, j, v, src >= 0);
  } else if (p.c.part && t - n < p.c.n && part == 0) {
    const int i = int(t - n);
    const int parts = p.c.rows_dev ? (*p.c.rows_dev + p.c.bi - 1) / p.c.bi * p.c.per : p.c.parts;
    float v = 0.f;
#pragma unroll 8
    for (int s = 0; s < parts; ++s) v += p.c.part[int64_t(s) * p.c.ld + i];
    emit_sum(p.c.e, p.c.e.once(p.c.e.nj), p.c.out, p.c.bf16, i, v);
  }
}

// ---- fp32 -> planes ----------------------------------------------------------------------------

struct Rows {
  const float* p;
  int64_t ld;
  int n, width;
};

__device__ __forceinline__ uint2 pack4(const uint16_t (&v)[4]) {
  return make_uint2(v[0] | (uint32_t(v[1]) << 16), v[2] | (uint32_t(v[3]) << 16));
}

// x's rows as three planes [n][kp] (zeros from width to kp), one quad a thread
static __global__ __launch_bounds__(256) void split_kernel(Rows x, uint16_t* __restrict__ out, int kp, int64_t plane) {
  const int quads = kp >> 2;
  const bool vec = (x.ld & 3) == 0 && (x.width & 3) == 0 && (reinterpret_cast<uintptr_t>(x.p) & 15) == 0;
  const int64_t n = int64_t(x.n) * quads;
  for (int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x; t < n; t += int64_t(gridDim.x) * 256) {
    const int64_t r = t / quads;
    const int c = 4 * int(t - r * quads);
    const float* row = x.p + r * x.ld + c;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (vec) {
      if (c < x.width) {
        const float4 u = *reinterpret_cast<const float4*>(row);
        v[0] = u.x;
        v[1] = u.y;
        v[2] = u.z;
        v[3] = u.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < x.width) v[e] = row[e];
    }
    uint16_t hi[4], mid[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split3(v[e], hi[e], mid[e], lo[e]);
    *reinterpret_cast<uint2*>(out + 4 * t) = pack4(hi);
    *reinterpret_cast<uint2*>(out + plane + 4 * t) = pack4(mid);
    *reinterpret_cast<uint2*>(out + 2 * plane + 4 * t) = pack4(lo);
  }
}

// the planes in ``out`` [3][n][kp], as an operand
inline Operand split(const Rows& x, uintptr_t out, int kp, hipStream_t st) {
  uint16_t* o = reinterpret_cast<uint16_t*>(out);
  const int64_t plane = int64_t(x.n) * kp;
  hipLaunchKernelGGL(split_kernel, dim3(stream_grid(int64_t(x.n) * (kp >> 2), 256, 8192)), dim3(256), 0, st, x, o, kp, plane);
  check_launch();
  return {o, kp, plane, x.n};
}

// ---- choices shared by the operators -------------------------------------------------------------

inline int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

inline int whole_rows(uintptr_t p, int64_t ld, bool bf16) { return p % 16 == 0 && ld % (bf16 ? 8 : 4) == 0; }

// Tiles (columns x rows).  A CU is bound by the rate at which lines reach its LDS, so the tile should be
// as large as the product fills the chip with:
//   kWide 256 x 256, one workgroup of 8 waves a CU (four waves of 128 x 128 read a third less from the
//         LDS and ran 8192 x 2048 x 32768 at 1170 TFLOP/s against 1100, but one wave a SIMD lost as
//         much again in every epilogue that computes);
//   kBig  256 x 128, two workgroups a CU: one's epilogue runs beside the other's products;
//   kSq   128 x 128, two a CU;
//   kDeep 128 x 128, one a CU on a ring twice as deep, where there are not two: nothing else hides the
//         loads' latency (2 us a stage) then.  [1001 x 331] . [331 x 1348] in fp32 36 -> 23 us, but
//         [8192 x 2304]^T . [8192 x 768] in bf16, which splits into two a CU, 50 -> 64;
//   kFew  128 x 32 (row operands), for a handful of rows, whose products only stream the weights.
template <int NP, bool IT, bool JT> using Wide = Tile<NP, IT, JT, 2, 4, 4, 2, 64, 2>;
template <int NP, bool IT, bool JT> using Big = Tile<NP, IT, JT, 2, 2, 4, 2, 32, 3>;
template <int NP, bool IT, bool JT> using Sq = Tile<NP, IT, JT, 2, 2, 2, 2, 64, 2>;
template <int NP, bool IT, bool JT> using Deep = Tile<NP, IT, JT, 2, 2, 2, 2, 64, 4>;
template <int NP, bool IT, bool JT> using Few = Tile<NP, IT, JT, 4, 1, 1, 1, 64, 3>;

enum { kWide = 0, kBig = 1, kSq = 2, kDeep = 3, kFew = 4 };
inline int tile_bj(int t) { return t <= kBig ? 256 : 128; }
inline int tile_bi(int t) { return t == kWide ? 256 : t == kFew ? 32 : 128; }
inline int tile_slots(int t) { return t == kWide || t == kDeep ? 256 : 512; }  // workgroups that the chip holds

inline int64_t tiles_of(int tile, int64_t ni, int64_t nj) {
  return ((ni + tile_bi(tile) - 1) / tile_bi(tile)) * ((nj + tile_bj(tile) - 1) / tile_bj(tile));
}

// least reduction steps a split; short ones where there are few workgroups
inline int tile_least(int t) { return t >= kDeep ? 128 : 256; }

inline Split split_of(int tile) { return {tile_slots(tile), tile_least(tile)}; }

// Tile of a product of reduction length nk in np passes, which ``split``s over its reduction or not.
inline int choose_tile(int64_t ni, int64_t nj, int64_t nk, int np, bool col_i, bool split) {
  if (ni <= 32 && !col_i) return kFew;
  const int64_t w = tiles_of(kWide, ni, nj), b = tiles_of(kBig, ni, nj), q = tiles_of(kSq, ni, nj);
  // the busiest CU's work: a kBig tile is half a kWide one at 0.84 of its rate (850 against 1000 TFLOP/s
  // over a long reduction); over a short one kWide's epilogue, which nothing hides, costs more than that
  if (w >= 192 && nk * np >= 1536 && (w + 255) / 256 * 10 <= (b + 255) / 256 * 6) return kWide;
  if (b >= 256) return kBig;
  // a split reduction fills the chip with the largest tile too, at twice kSq's slabs: with 1820 to 6912 steps
  // a split it won ([8704 x 15000]^T . [8704 x 256] in bf16 and qkv's gradients in fp32, 448 -> 438 and 615 ->
  // 565 us a pass), with 900 to 1150 it lost (qkv's in bf16, 164 -> 172)
  if (split) {
    const int64_t s = split_of(kWide).of(w, nk);
    if (w * s >= 192 && nk / s * np >= 1536) return kWide;
  }
  return q * (split ? split_of(kSq).of(q, nk) : 1) > 256 ? kSq : kDeep;
}

// Largest grid and slab (in rows) of a product whose rows in use are known on the device only: any
// number up to ni.
struct Extent {
  int64_t grid, slab_rows;
};
inline Extent extent_of(int tile, int64_t ni, int64_t nj, const Split& split, int64_t nk) {
  Extent x{1, 1};
  const int64_t n = tiles_of(tile, ni, 1), tj = tiles_of(tile, 1, nj);
  auto add = [&](int64_t t) {
    const int64_t s = split.of(t * tj, nk);
    x.grid = std::max(x.grid, t * tj * s);
    x.slab_rows = std::max(x.slab_rows, s * std::min(ni, t * tile_bi(tile)));
  };
  for (int64_t t = 1; t < n && t * tj <= split.slots; ++t) add(t);  // past the slots there is one split
  add(n);
  return x;
}

template <class T, bool SUM>
inline void launch_gemm(const GemmArgs& p, int64_t grid, hipStream_t st) {
  hipLaunchKernelGGL((gemm_kernel<T, SUM>), dim3(unsigned(grid)), dim3(T::kThreads), 0, st, p);
  check_launch();
}

template <int NP, bool IT, bool JT, bool SUM>
inline void gemm(int tile, const GemmArgs& p, int64_t grid, hipStream_t st) {
  if (tile == kWide) launch_gemm<Wide<NP, IT, JT>, SUM>(p, grid, st);
  else if (tile == kBig) launch_gemm<Big<NP, IT, JT>, SUM>(p, grid, st);
  else if (tile == kSq) launch_gemm<Sq<NP, IT, JT>, SUM>(p, grid, st);
  else if (tile == kDeep) launch_gemm<Deep<NP, IT, JT>, SUM>(p, grid, st);
  else if constexpr (!IT) launch_gemm<Few<NP, IT, JT>, SUM>(p, grid, st);
}

inline void finish(int tile, const GemmArgs& g, int rows, const int* inv, const ColumnSums& c, hipStream_t st) {
  const FinishArgs p = {g, tile_bi(tile), tile_bj(tile), rows, inv, c};
  const int64_t n = int64_t(rows) * ((g.e.nj + 7) / 8) + (c.part ? c.n : 0);
  if (n == 0) return;
  // few outputs: eight lanes on each keep the loads of many splits in flight (20 x 256 of 58 splits 11 ->
  // 6 us); with enough threads they would only divide the lines between them
  if (n <= 16384) hipLaunchKernelGGL((finish_kernel<8>), dim3(unsigned((n * 8 + 255) / 256)), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((finish_kernel<1>), dim3(unsigned((n + 255) / 256)), dim3(256), 0, st, p);
  check_launch();
}

}  // namespace gt
}  // namespace voda
