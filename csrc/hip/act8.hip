// Linear layer whose backward works from an 8-bit checkpoint of its input (CDNA4, gfx950).
//
//   y  = act(x) w^T + b             act: identity or gelu_tanh; from x itself
//   c  = what the checkpoint of x stands for
//   dx = (dy w) act'(c)     dw = dy^T act(c)     db = sum dy
//
// Checkpoint: blocks of 32 features of one row, each e4m3 times the smallest power of two 2^e,
// e >= -126, with the block's largest finite |x| <= 448 2^e.  The scaling is exact, so the one rounding
// is e4m3's (at most 2^-4 of the value, or 2^(e-10) for the smallest); only what would round past fp32's
// own range stays at 240 2^120, within 2^-4 too.  Infinite and NaN elements are held as NaN.  33 bytes
// for 32 features against 64 (bf16) or 128 (fp32).
//
//  * act8_pack reads x once and writes the checkpoint and, where the product cannot take x as it is,
//    act(x) as the product's operand (bf16, or the three planes of fp32).  It moves 8 features a
//    thread; a block's maximum is two shuffles inside a quad of lanes.
//  * act8_unpack writes act(c) for dw's product: the GELU is then computed once an element, not once
//    for each of dw's row tiles.  bf16 holds an identity c exactly (four significant bits).
//  * The three products are gemm_tile.h's; gelu'(c) is applied in dx's epilogue from the checkpoint.
//    fp32: x, w and dy as three bf16 planes, six 16-bit products; an identity c is exact in one plane, so
//    its dw takes three.
#include "gemm_tile.h"
#include "ops.h"

namespace voda {

namespace {

using namespace gt;

struct PackArgs {
  const void* x;
  int64_t ldx;
  int rows, width, vec, gelu;
  uint8_t* q;       // [rows][kq], kq = width up to whole blocks of 32; null: no checkpoint
  uint8_t* qs;      // [rows][kq / 32]
  int kq;
  uint16_t* o;      // act(x): [rows][kq] bf16, or three planes; or null
  int64_t plane;
};

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.4028235e38f; }

__device__ __forceinline__ void load8(const PackArgs& p, bool f32, int64_t r, int c, float (&v)[8]) {
  if (f32) {
    const float* row = static_cast<const float*>(p.x) + r * p.ldx + c;
    if (p.vec && c < p.width) {
      const float4 a = *reinterpret_cast<const float4*>(row), b = *reinterpret_cast<const float4*>(row + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < p.width ? row[e] : 0.f;
    }
  } else {
    const uint16_t* row = static_cast<const uint16_t*>(p.x) + r * p.ldx + c;
    if (p.vec && c < p.width) {
      const uint4 u = *reinterpret_cast<const uint4*>(row);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = bf2f(w[e] & 0xffff);
        v[2 * e + 1] = bf2f(w[e] >> 16);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < p.width ? bf2f(row[e]) : 0.f;
    }
  }
}

__device__ __forceinline__ uint4 pack8_bf16(const float (&v)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = uint32_t(f2bf(v[2 * e])) | (uint32_t(f2bf(v[2 * e + 1])) << 16);
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// the three planes of 8 values
__device__ __forceinline__ void store8_planes(const float (&v)[8], uint16_t* o, int64_t plane) {
  uint16_t q[3][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) split3(v[e], q[0][e], q[1][e], q[2][e]);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const uint16_t* a = q[k];
    *reinterpret_cast<uint4*>(o + k * plane) =
        make_uint4(a[0] | (uint32_t(a[1]) << 16), a[2] | (uint32_t(a[3]) << 16), a[4] | (uint32_t(a[5]) << 16),
                   a[6] | (uint32_t(a[7]) << 16));
  }
}

template <bool F32>
__global__ __launch_bounds__(256) void act8_pack_kernel(PackArgs p) {
  const int eights = p.kq >> 3;  // a multiple of 4: a quad of lanes is one block of 32
  const int64_t n = int64_t(p.rows) * eights;
  const int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (t >= n) return;
  const int64_t r = t / eights;
  const int c = 8 * int(t - r * eights);
  float v[8];
  load8(p, F32, r, c, v);
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, finite(v[e]) ? fabsf(v[e]) : 0.f);
  m = fmaxf(m, __shfl_xor(m, 1, 64));
  m = fmaxf(m, __shfl_xor(m, 2, 64));
  // m = 1.f 2^E <= 1.75 2^8 2^e
  const uint32_t bits = __float_as_uint(m);
  const int ex = max(int(bits >> 23) - 127 - 8 + int((bits & 0x7fffff) > 0x600000), -126);
  const float inv = __uint_as_float(uint32_t(127 - ex) << 23);
  const float most = ex == 120 ? 240.f : 448.f;  // 256 2^120 is past fp32
  float w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = finite(v[e]) ? fminf(fmaxf(v[e] * inv, -most), most) : NAN;
  uint32_t q0 = 0, q1 = 0;
  q0 = __builtin_amdgcn_cvt_pk_fp8_f32(w[0], w[1], q0, false);
  q0 = __builtin_amdgcn_cvt_pk_fp8_f32(w[2], w[3], q0, true);
  q1 = __builtin_amdgcn_cvt_pk_fp8_f32(w[4], w[5], q1, false);
  q1 = __builtin_amdgcn_cvt_pk_fp8_f32(w[6], w[7], q1, true);
  if (p.q) {
    *reinterpret_cast<uint2*>(p.q + 8 * t) = make_uint2(q0, q1);
    if ((c & 31) == 0) p.qs[t >> 2] = uint8_t(ex + 127);
  }
  if (!p.o) return;
  if (p.gelu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = gelu_tanh_f(v[e]);
  }
  if constexpr (F32) store8_planes(v, p.o + 8 * t, p.plane);
  else *reinterpret_cast<uint4*>(p.o + 8 * t) = pack8_bf16(v);
}

struct UnpackArgs {
  const uint8_t* q;
  const uint8_t* qs;
  int64_t n;       // groups of 8
  int gelu;
  uint16_t* o;     // act(c): bf16, or (fp32 with the GELU) three planes
  int64_t plane;
};

__device__ __forceinline__ void unpack8(const uint8_t* q, const uint8_t* qs, int64_t t, float (&v)[8]) {
  const uint2 u = *reinterpret_cast<const uint2*>(q + 8 * t);
  const float s = __uint_as_float(uint32_t(qs[t >> 2]) << 23);
  v[0] = __builtin_amdgcn_cvt_f32_fp8(u.x, 0) * s;
  v[1] = __builtin_amdgcn_cvt_f32_fp8(u.x, 1) * s;
  v[2] = __builtin_amdgcn_cvt_f32_fp8(u.x, 2) * s;
  v[3] = __builtin_amdgcn_cvt_f32_fp8(u.x, 3) * s;
  v[4] = __builtin_amdgcn_cvt_f32_fp8(u.y, 0) * s;
  v[5] = __builtin_amdgcn_cvt_f32_fp8(u.y, 1) * s;
  v[6] = __builtin_amdgcn_cvt_f32_fp8(u.y, 2) * s;
  v[7] = __builtin_amdgcn_cvt_f32_fp8(u.y, 3) * s;
}

template <bool PLANES>
__global__ __launch_bounds__(256) void act8_unpack_kernel(UnpackArgs p) {
  const int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (t >= p.n) return;
  float v[8];
  unpack8(p.q, p.qs, t, v);
  if (p.gelu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = gelu_tanh_f(v[e]);
  }
  if constexpr (PLANES) store8_planes(v, p.o + 8 * t, p.plane);
  else *reinterpret_cast<uint4*>(p.o + 8 * t) = pack8_bf16(v);
}

// checkpoint -> values in dt, [rows][width] contiguous
template <bool F32>
__global__ __launch_bounds__(256) void act8_values_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ qs,
                                                          int64_t n, int kq, int width, void* __restrict__ out) {
  const int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (t >= n) return;
  float v[8];
  unpack8(q, qs, t, v);
  const int eights = kq >> 3;
  const int64_t r = t / eights;
  const int c = 8 * int(t - r * eights);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (c + e >= width) break;
    if constexpr (F32) static_cast<float*>(out)[r * width + c + e] = v[e];
    else static_cast<uint16_t*>(out)[r * width + c + e] = f2bf(v[e]);
  }
}

unsigned blocks(int64_t threads) { return unsigned((threads + 255) / 256); }

struct Act8Plan {
  int kq, np8, kp;               // features up to 32, outputs up to 8, features up to 8
  int y_tile, dx_tile, dw_tile;
  Split y_split, dx_split, dw_split;
  int y_s, dx_s, dw_s;
  bool copy;                     // the forward's product reads a copy that act8_pack writes
  // forward workspace: x's operand, slab
  int64_t f_x, f_slab, fwd;
  // backward workspace: dy's planes, act(c), slabs
  int64_t b_dy, b_c, b_dx, b_dw, b_db, bwd;
};

Act8Plan act8_plan(int64_t rows, int64_t width, int64_t out, bool f32, bool gelu, bool copy) {
  Act8Plan q{};
  q.kq = int(up(width, 32));
  q.kp = int(up(width, 8));
  q.np8 = int(up(out, 8));
  q.copy = copy;
  const int np = f32 ? 6 : 1;
  q.y_tile = choose_tile(rows, out, width, np, false, true);
  q.dx_tile = choose_tile(rows, width, out, np, false, true);
  q.dw_tile = choose_tile(out, width, rows, f32 && !gelu ? 3 : np, true, true);
  q.y_split = split_of(q.y_tile);
  q.dx_split = split_of(q.dx_tile);
  q.dw_split = split_of(q.dw_tile);
  q.y_s = q.y_split.of(tiles_of(q.y_tile, rows, out), q.kp);
  q.dx_s = q.dx_split.of(tiles_of(q.dx_tile, rows, width), out);
  q.dw_s = q.dw_split.of(tiles_of(q.dw_tile, out, width), rows);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at = up(at + bytes, 256);
    return o;
  };
  q.f_x = take(copy ? rows * q.kq * (f32 ? 6 : 2) : 0);
  q.f_slab = take(q.y_s > 1 ? q.y_s * rows * up(out, 8) * 4 : 0);
  q.fwd = at;
  at = 0;
  q.b_dy = take(f32 ? rows * q.np8 * 6 : 0);
  q.b_c = take(rows * q.kq * (f32 && gelu ? 6 : 2));
  q.b_dx = take(q.dx_s > 1 ? q.dx_s * rows * q.kp * 4 : 0);
  q.b_dw = take(q.dw_s > 1 ? q.dw_s * out * q.kp * 4 : 0);
  q.b_db = take(q.dw_s > 1 ? q.dw_s * out * 4 : 0);
  q.bwd = at;
  return q;
}

void check_act8(int64_t rows, int64_t width, int64_t out, int dt) {
  VODA_CHECK(rows > 0 && rows < (1 << 30) && width > 0 && width <= (1 << 20) && out > 0 && out <= (1 << 20),
             "linear_act8: sizes out of range");
  // a launch holds less than 2^32 threads: 256 x 128 a workgroup of 256, eight features a thread of the packing
  VODA_CHECK(up(rows, 128) / 128 * (up(width > out ? width : out, 256) / 256) < (1 << 24) &&
                 rows * up(width, 32) <= (int64_t(1) << 34),
             "linear_act8: rows x features too large");
  VODA_CHECK(dt == kF32 || dt == kBF16, "linear_act8: fp32 or bf16");
}

}  // namespace

// (forward workspace, backward workspace) bytes, features up to 32, outputs up to 8
std::vector<int64_t> linear_act8_sizes(int64_t rows, int64_t width, int64_t out, int dt, bool copy, bool gelu) {
  check_act8(rows, width, out, dt);
  const Act8Plan q = act8_plan(rows, width, out, dt == kF32, gelu, copy);
  return {q.fwd, q.bwd, q.kq, q.np8};
}

void act8_pack(uintptr_t x, int64_t ldx, int64_t rows, int64_t width, int dt, uintptr_t qp, uintptr_t qs,
               uintptr_t stream) {
  check_act8(rows, width, 1, dt);
  VODA_CHECK(qp % 16 == 0, "act8: checkpoint must be 16-byte aligned");
  PackArgs p{};
  p.x = reinterpret_cast<const void*>(x);
  p.ldx = ldx;
  p.rows = int(rows);
  p.width = int(width);
  p.vec = x % 16 == 0 && ldx % 8 == 0 && width % 8 == 0;
  p.q = reinterpret_cast<uint8_t*>(qp);
  p.qs = reinterpret_cast<uint8_t*>(qs);
  p.kq = int(up(width, 32));
  const dim3 grid(blocks(rows * (p.kq >> 3)));
  if (dt == kF32) hipLaunchKernelGGL((act8_pack_kernel<true>), grid, dim3(256), 0, as_stream(stream), p);
  else hipLaunchKernelGGL((act8_pack_kernel<false>), grid, dim3(256), 0, as_stream(stream), p);
  check_launch();
}

void act8_values(uintptr_t qp, uintptr_t qs, int64_t rows, int64_t width, int dt, uintptr_t out, uintptr_t stream) {
  check_act8(rows, width, 1, dt);
  VODA_CHECK(qp % 16 == 0, "act8: checkpoint must be 16-byte aligned");
  const int kq = int(up(width, 32));
  const int64_t n = rows * (kq >> 3);
  if (dt == kF32)
    hipLaunchKernelGGL((act8_values_kernel<true>), dim3(blocks(n)), dim3(256), 0, as_stream(stream),
                       reinterpret_cast<const uint8_t*>(qp), reinterpret_cast<const uint8_t*>(qs), n, kq, int(width),
                       reinterpret_cast<void*>(out));
  else
    hipLaunchKernelGGL((act8_values_kernel<false>), dim3(blocks(n)), dim3(256), 0, as_stream(stream),
                       reinterpret_cast<const uint8_t*>(qp), reinterpret_cast<const uint8_t*>(qs), n, kq, int(width),
                       reinterpret_cast<void*>(out));
  check_launch();
}

// y [rows][out] contiguous; the checkpoint (q, qs) is written where q is not null; ``wp`` (fp32):
// workspace for w's planes, [3][out][width up to 8].
void linear_act8_fwd(uintptr_t x, int64_t ldx, uintptr_t w, int64_t ldw, uintptr_t bias, int bias_dt, uintptr_t y,
                     uintptr_t qp, uintptr_t qs, int64_t rows, int64_t width, int64_t out, int dt, bool gelu, bool copy,
                     uintptr_t wp, uintptr_t ws, uintptr_t stream) {
  check_act8(rows, width, out, dt);
  const bool f32 = dt == kF32;
  VODA_CHECK(f32 || (w % 16 == 0 && ldw % 8 == 0 && ldw >= up(width, 8)),
             "linear_act8: bf16 weight rows must be 16-byte aligned and whole 16-byte vectors");
  VODA_CHECK(copy || (!f32 && !gelu && x % 16 == 0 && ldx % 8 == 0 && width % 8 == 0),
             "linear_act8: this input needs a copy");
  VODA_CHECK(qp % 16 == 0 && ws % 256 == 0 && wp % 16 == 0 && (wp || !f32), "linear_act8: workspaces must be aligned");
  const Act8Plan q = act8_plan(rows, width, out, f32, gelu, copy);
  hipStream_t st = as_stream(stream);
  uint8_t* base = reinterpret_cast<uint8_t*>(ws);
  PackArgs p{};
  p.x = reinterpret_cast<const void*>(x);
  p.ldx = ldx;
  p.rows = int(rows);
  p.width = int(width);
  p.vec = x % 16 == 0 && ldx % 8 == 0 && width % 8 == 0;
  p.gelu = gelu;
  p.q = reinterpret_cast<uint8_t*>(qp);
  p.qs = reinterpret_cast<uint8_t*>(qs);
  p.kq = q.kq;
  p.o = copy ? reinterpret_cast<uint16_t*>(base + q.f_x) : nullptr;
  p.plane = rows * q.kq;
  if (p.q || p.o) {
    const dim3 grid(blocks(rows * (q.kq >> 3)));
    if (f32) hipLaunchKernelGGL((act8_pack_kernel<true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((act8_pack_kernel<false>), grid, dim3(256), 0, st, p);
    check_launch();
  }
  GemmArgs a{};
  a.I = copy ? Operand{p.o, q.kq, p.plane, int(rows)} : Operand{reinterpret_cast<const uint16_t*>(x), ldx, 0, int(rows)};
  a.J = {reinterpret_cast<const uint16_t*>(w), ldw, 0, int(out)};
  if (f32) a.J = split({reinterpret_cast<const float*>(w), ldw, int(out), int(width)}, wp, q.kp, st);
  a.nk = q.kp;
  a.split = q.y_split;
  a.nk_split = a.nk;
  a.e.out = reinterpret_cast<void*>(y);
  a.e.ldo = out;
  a.e.bf16 = !f32;
  a.e.nj = int(out);
  a.e.vec = whole_rows(y, out, !f32);
  a.e.bias = reinterpret_cast<const void*>(bias);
  a.e.bias_bf16 = bias_dt == kBF16;
  if (q.y_s > 1) {
    a.slab = reinterpret_cast<float*>(base + q.f_slab);
    a.lds = up(out, 8);
  }
  const int64_t grid_y = tiles_of(q.y_tile, rows, out) * q.y_s;
  if (f32) gemm<6, false, false, false>(q.y_tile, a, grid_y, st);
  else gemm<1, false, false, false>(q.y_tile, a, grid_y, st);
  if (a.slab) finish(q.y_tile, a, int(rows), nullptr, {}, st);
}

// dx [rows][width] in x's type (added to when ``dx_add``); dw [out][ldd] in ``grad_dt`` and db [out] in
// ``db_dt`` (added to when ``accumulate``); dx, db, or dw and db may be null, and the checkpoint where
// neither dw nor the GELU asks for it.  dy: bf16 rows of whole 16-byte vectors.
void linear_act8_bwd(uintptr_t dy, int64_t ldy, uintptr_t w, int64_t ldw, uintptr_t qp, uintptr_t qs, uintptr_t dx,
                     bool dx_add, uintptr_t dw, int64_t ldd, uintptr_t db, int grad_dt, int db_dt, bool accumulate,
                     int64_t rows, int64_t width, int64_t out, int dt, bool gelu, uintptr_t wp, uintptr_t ws, uintptr_t stream) {
  check_act8(rows, width, out, dt);
  const bool f32 = dt == kF32;
  VODA_CHECK((grad_dt == kF32 || grad_dt == kBF16) && (db_dt == kF32 || db_dt == kBF16),
             "linear_act8: weight and bias gradients must be fp32 or bf16");
  VODA_CHECK(f32 || (w % 16 == 0 && ldw % 8 == 0 && ldw >= up(width, 8)),
             "linear_act8: bf16 weight rows must be 16-byte aligned and whole 16-byte vectors");
  VODA_CHECK(f32 || (dy % 16 == 0 && ldy % 8 == 0 && ldy >= up(out, 8)),
             "linear_act8: bf16 gradient rows must be 16-byte aligned and whole 16-byte vectors");
  VODA_CHECK(qp % 16 == 0 && ws % 256 == 0 && wp % 16 == 0 && (wp || !f32 || !dx), "linear_act8: workspaces must be aligned");
  VODA_CHECK((qp && qs) || (!dw && !gelu), "linear_act8: the backward needs the checkpoint");
  const Act8Plan q = act8_plan(rows, width, out, f32, gelu, true);
  hipStream_t st = as_stream(stream);
  uint8_t* base = reinterpret_cast<uint8_t*>(ws);
  const uint8_t* q8 = reinterpret_cast<const uint8_t*>(qp);
  const uint8_t* s8 = reinterpret_cast<const uint8_t*>(qs);
  Operand DY = {reinterpret_cast<const uint16_t*>(dy), ldy, 0, int(rows)};
  Operand W = {reinterpret_cast<const uint16_t*>(w), ldw, 0, int(out)};
  if (f32) {
    DY = split({reinterpret_cast<const float*>(dy), ldy, int(rows), int(out)}, reinterpret_cast<uintptr_t>(base + q.b_dy), q.np8, st);
    if (dx) W = split({reinterpret_cast<const float*>(w), ldw, int(out), int(width)}, wp, q.kp, st);
  }
  if (dx) {
    GemmArgs a{};
    a.I = DY;
    a.J = W;
    a.J.n = q.kp;  // columns: W is read down its rows
    a.nk = int(out);
    a.split = q.dx_split;
    a.nk_split = a.nk;
    a.e.out = reinterpret_cast<void*>(dx);
    a.e.ldo = width;
    a.e.bf16 = !f32;
    a.e.nj = int(width);
    a.e.vec = whole_rows(dx, width, !f32);
    a.e.accumulate = dx_add;
    if (gelu) {
      a.e.q = q8;
      a.e.qs = s8;
      a.e.ldq = q.kq;
    }
    if (q.dx_s > 1) {
      a.slab = reinterpret_cast<float*>(base + q.b_dx);
      a.lds = q.kp;
    }
    const int64_t grid_x = tiles_of(q.dx_tile, rows, width) * q.dx_s;
    if (f32) gemm<6, false, true, false>(q.dx_tile, a, grid_x, st);
    else gemm<1, false, true, false>(q.dx_tile, a, grid_x, st);
    if (a.slab) finish(q.dx_tile, a, int(rows), nullptr, {}, st);
  }
  if (!dw) return;
  UnpackArgs u{};
  u.q = q8;
  u.qs = s8;
  u.n = rows * (q.kq >> 3);
  u.gelu = gelu;
  u.o = reinterpret_cast<uint16_t*>(base + q.b_c);
  u.plane = rows * q.kq;
  if (f32 && gelu) hipLaunchKernelGGL((act8_unpack_kernel<true>), dim3(blocks(u.n)), dim3(256), 0, st, u);
  else hipLaunchKernelGGL((act8_unpack_kernel<false>), dim3(blocks(u.n)), dim3(256), 0, st, u);
  check_launch();
  GemmArgs a{};
  a.I = DY;
  a.I.n = int(out);
  a.J = {u.o, q.kq, u.plane, q.kq};
  a.nk = int(rows);
  a.split = q.dw_split;
  a.nk_split = a.nk;
  a.e.out = reinterpret_cast<void*>(dw);
  a.e.ldo = ldd;
  a.e.bf16 = grad_dt == kBF16;
  a.e.nj = int(width);
  a.e.vec = whole_rows(dw, ldd, a.e.bf16);
  a.e.accumulate = accumulate;
  a.bout = reinterpret_cast<void*>(db);
  a.bout_bf16 = db_dt == kBF16;
  if (q.dw_s > 1) {
    a.slab = reinterpret_cast<float*>(base + q.b_dw);
    a.lds = q.kp;
    a.bslab = db ? reinterpret_cast<float*>(base + q.b_db) : nullptr;
  }
  const int64_t grid_w = tiles_of(q.dw_tile, out, width) * q.dw_s;
  if (f32 && gelu) gemm<6, true, true, true>(q.dw_tile, a, grid_w, st);
  else if (f32) gemm<3, true, true, true>(q.dw_tile, a, grid_w, st);
  else gemm<1, true, true, true>(q.dw_tile, a, grid_w, st);
  if (a.slab) {
    ColumnSums c{};
    c.part = a.bslab;
    c.ld = c.n = int(out);
    c.parts = q.dw_s;
    c.out = a.bout;
    c.bf16 = a.bout_bf16;
    c.e = a.e;
    finish(q.dw_tile, a, int(out), nullptr, c, st);
  }
}

}  // namespace voda
