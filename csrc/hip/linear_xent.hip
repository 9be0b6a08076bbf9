// Softmax cross-entropy of a vocabulary head without its logits (CDNA4, gfx950).
//
//   z[r][v]  = sum_k x[r][k] w[v][k] + b[v]           v < C (classes), r over the labelled rows
//   loss     = 1/n sum_r (lse_r - z[r][y_r])          lse_r = log sum_v exp z[r][v]
//   G[r][v]  = exp(z[r][v] - lse_r) - [v == y_r]
//   dx = g/n G w     dw = g/n G^T x     db = g/n sum_r G     (g: the loss's own gradient)
//
// The logits of a tile live in the accumulators only.  Forward: one product x w^T whose epilogue
// leaves a (max, sum exp) pair a row for each 32 * TJ columns of the vocabulary, joined by
// xent_join.  Backward: piece by piece of the vocabulary the product runs again and leaves G of the
// piece in a workspace (16 bits; fp32 inputs: three bf16 planes), which the two gradient products read.
// So 8 n C K operations instead of 6, and no memory that grows with n C.
//
// Rows whose label is ignored (or lies outside [0, C)) are left out at the start: xent_gather copies
// the labelled rows together, all later kernels work on those n rows (n stays on the device, the
// launches are sized for all rows and the workgroups behind n end at once).  An ignored row costs
// nothing, its dx is exactly zero and nothing that it holds, NaN included, reaches any output.
//
// bf16 inputs: G is rounded once to bf16 for the two products (at most 2^-8 of each element, random in
// sign, against the same rounding of the sums to bf16 at the end), up to 128 rows kept in two planes;
// the one-hot part is subtracted before that rounding and g/n multiplied after the sums.  db sums G as it
// was before.  fp32 inputs: three bf16 planes an operand (gemm_tile.h), G too.
// Sums over rows and splits have a fixed order: the same call gives the same bits.
#include "gemm_tile.h"
#include "ops.h"

#include <algorithm>
#include <type_traits>

namespace voda {

namespace {

using namespace gt;

// Exponents go as (z - max) log2(e): 0 where z is the largest, whatever its size, and the subtraction is
// exact near it.  One fma, z log2(e) - c with c = max log2(e), would save an instruction an element and 2 % of
// a pass, but c's own rounding, |c| 2^-24, would be in every exponent: a sum that misses 1, a negative loss
// from |max| near 30 on, and infinite sums of a slot whose classes are masked by -1e10.
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kGatherRows = 32;   // rows a gather workgroup

// device scalars of one call
struct XentDev {
  int n;           // labelled rows
  int done;        // workgroups of xent_join that are through
};

__device__ __forceinline__ bool labelled(int64_t y, int64_t ignore, int classes) {
  return y != ignore && y >= 0 && y < classes;
}

struct GatherArgs {
  const void* x;
  int64_t ldx;
  int rows, width, classes, vec;
  const int64_t* labels;
  int64_t ignore;
  uint16_t* xc;      // [rows][kp] (fp32: three planes)
  int kp;
  int64_t plane;
  int* inv;          // [rows]: place among the labelled rows, or -1
  int* lab;          // [rows]: labels of the labelled rows
  XentDev* dev;
  int64_t* n_out;
  const void* bias;  // [classes] or null
  int bias_bf16;
  float* bias32;     // [bias_n]: bias, 0 where there is none, -inf from classes on
  int bias_n;
  int gather_blocks;
  const int* counts; // labelled rows of each kCountRows, or null: count them here
};

// Many rows: how many of each 1024 are labelled.
constexpr int kCountRows = 1024;
__global__ __launch_bounds__(256) void xent_count_kernel(const int64_t* __restrict__ labels, int rows, int64_t ignore,
                                                         int classes, int* __restrict__ counts) {
  __shared__ int cnt[4];
  int c = 0;
#pragma unroll
  for (int k = 0; k < kCountRows / 256; ++k) {
    const int r = blockIdx.x * kCountRows + 256 * k + threadIdx.x;
    c += r < rows && labelled(labels[r], ignore, classes);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
  if ((threadIdx.x & 63) == 0) cnt[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = cnt[0] + cnt[1] + cnt[2] + cnt[3];
}

// Labelled rows of x together, and what goes with them; then the bias in fp32.
template <bool F32>
__global__ __launch_bounds__(256) void xent_gather_kernel(GatherArgs p) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  if (int(blockIdx.x) >= p.gather_blocks) {
    const int v = (blockIdx.x - p.gather_blocks) * 256 + t;
    if (v < p.bias_n)
      p.bias32[v] = v >= p.classes ? -INFINITY
                    : !p.bias      ? 0.f
                    : p.bias_bf16  ? bf2f(static_cast<const uint16_t*>(p.bias)[v])
                                   : static_cast<const float*>(p.bias)[v];
    return;
  }
  __shared__ int cnt[4];
  __shared__ int place[kGatherRows];
  // labelled rows in front of this workgroup's: every workgroup counts them itself (8 bytes a row
  // out of the L2), cheaper than a second launch up to some thousand rows, or from the counts
  const int r0 = blockIdx.x * kGatherRows;
  int c = 0, from = 0;
  if (p.counts) {
    const int segs = r0 / kCountRows;
#pragma unroll 8
    for (int k = t; k < segs; k += 256) c += p.counts[k];
    from = segs * kCountRows;
  }
#pragma unroll 8
  for (int r = from + t; r < r0; r += 256) c += labelled(p.labels[r], p.ignore, p.classes);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
  if (lane == 0) cnt[wave] = c;
  __syncthreads();
  if (wave == 0) {
    const int base = cnt[0] + cnt[1] + cnt[2] + cnt[3];
    const int r = r0 + lane;
    const bool mine = lane < kGatherRows && r < p.rows;
    const int64_t y = mine ? p.labels[r] : -1;
    const bool ok = mine && labelled(y, p.ignore, p.classes);
    const uint64_t all = __ballot(ok);
    const int at = base + __popcll(all & ((uint64_t(1) << lane) - 1));
    if (mine) {
      p.inv[r] = ok ? at : -1;
      place[lane] = ok ? at : -1;
      if (ok) p.lab[at] = int(y);
    }
    if (lane == 0 && r0 + kGatherRows >= p.rows) {
      p.dev->n = base + __popcll(all);
      p.dev->done = 0;
      *p.n_out = base + __popcll(all);
    }
  }
  __syncthreads();
  for (int u = wave; u < kGatherRows && r0 + u < p.rows; u += 4) {
    const int at = place[u];
    if (at < 0) continue;
    uint16_t* o = p.xc + int64_t(at) * p.kp;
    if constexpr (F32) {
      const float* row = static_cast<const float*>(p.x) + int64_t(r0 + u) * p.ldx;
      if (p.vec) {
        for (int k = 4 * lane; k < p.kp; k += 256) {
          float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
          if (k < p.width) f = *reinterpret_cast<const float4*>(row + k);
          const float v[4] = {f.x, f.y, f.z, f.w};
          uint16_t hi[4], mid[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) split3(v[e], hi[e], mid[e], lo[e]);
          *reinterpret_cast<uint2*>(o + k) = pack4(hi);
          *reinterpret_cast<uint2*>(o + p.plane + k) = pack4(mid);
          *reinterpret_cast<uint2*>(o + 2 * p.plane + k) = pack4(lo);
        }
      } else {
        for (int k = lane; k < p.kp; k += 64) {
          uint16_t hi, mid, lo;
          split3(k < p.width ? row[k] : 0.f, hi, mid, lo);
          o[k] = hi;
          o[p.plane + k] = mid;
          o[2 * p.plane + k] = lo;
        }
      }
    } else {
      const uint16_t* row = static_cast<const uint16_t*>(p.x) + int64_t(r0 + u) * p.ldx;
      if (p.vec) {
        for (int k = 8 * lane; k < p.kp; k += 512)
          *reinterpret_cast<uint4*>(o + k) = *reinterpret_cast<const uint4*>(row + k);
      } else {
        for (int k = lane; k < p.kp; k += 64) o[k] = k < p.width ? row[k] : uint16_t(0);
      }
    }
  }
}

struct LogitArgs {
  Operand X, W;
  int width, tj;
  int v0, v1;           // vocabulary columns of this launch
  const float* bias32;
  const XentDev* dev;
  const int* lab;
  // forward: partial (max, sum exp) [slot][rows], a slot 32 TJ columns; the label's logit and whether
  // an earlier column of its slot equals it
  float2* part;
  float* zlab;
  int* tie;
  // backward: (max, 1 / sum exp) of each row; G [rows][ldg] (fp32 inputs: three planes)
  const float2* stat;
  uint16_t* G;
  int64_t ldg, gplane;
  float* sums;          // sums of G over a wave's rows [tile, wave][sums_ld], or null
  int64_t sums_ld;
};

// Rows are the tile's i, vocabulary columns its j.  The epilogue is vector work that the matrix cores
// wait for unless another workgroup of the CU is in its main loop: two workgroups a CU (72 KB of LDS each).
// PL: planes of G.
template <class T, bool BWD, int PL>
__global__ __launch_bounds__(T::kThreads, 2) void xent_logits_kernel(LogitArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[T::kLds];
  Operand X = p.X;
  X.n = min(X.n, p.dev->n);
  const int ni = (X.n + T::BI - 1) / T::BI, live = ni * p.tj;
  if (int(blockIdx.x) >= live) return;
  int ti, tj, s;
  tile_at(blockIdx.x, live, ni, p.tj, kGroup, ti, tj, s);
  const int i0 = ti * T::BI, j0 = p.v0 + tj * T::BJ;
  const typename T::Where w;
  // of this lane's rows, on their way while the products run (the forward, which needs the label alone,
  // has no register for it)
  int lab[T::TI];
  float2 stat[T::TI];
#pragma unroll
  for (int c = 0; c < (BWD ? T::TI : 0); ++c) {
    const int i = min(i0 + w.i(c), X.n - 1);
    lab[c] = p.lab[i];
    stat[c] = p.stat[i];
  }
  f32x16 acc[T::TJ][T::TI];
  float unused[T::TI];
  T::template run<false>(smem, X, p.W, i0, j0, 0, p.width, acc, unused);
  // z = products + bias; columns past the classes get the bias's -inf
#pragma unroll
  for (int a = 0; a < (BWD ? 0 : T::TJ); ++a) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 b4 = *reinterpret_cast<const float4*>(p.bias32 + j0 + w.j(a, g));
      const float b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int c = 0; c < T::TI; ++c) acc[a][c][4 * g + e] += b[e];
    }
  }
  float sums[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // BWD: of this lane's columns
#pragma unroll
  for (int c = 0; c < T::TI; ++c) {
    if constexpr (!BWD) {
      const int i = i0 + w.i(c);
      const bool live = i < X.n;
      const int y = live ? p.lab[i] : -1;
      float m = -INFINITY;
#pragma unroll
      for (int a = 0; a < T::TJ; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[a][c][r]);
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float ms = m == -INFINITY ? 0.f : m;  // all -inf: a sum of zeros
      float sum = 0.f;
#pragma unroll
      for (int a = 0; a < T::TJ; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f((acc[a][c][r] - ms) * kLog2e);
      sum += __shfl_xor(sum, 32, 64);
      const int slot = tj * T::WJ + w.wj;
      if (live && w.h == 0) p.part[int64_t(slot) * p.X.n + i] = make_float2(m, sum);
      // the label's logit, from the one wave whose columns hold it
      const int jw = j0 + w.wj * T::TJ * 32;
      const bool here = y >= jw && y < jw + T::TJ * 32;
      if (__ballot(here)) {
        float z = -INFINITY;
        bool has = false;
#pragma unroll
        for (int a = 0; a < T::TJ; ++a)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (j0 + w.j(a, r >> 2) + (r & 3) == y) {
              z = acc[a][c][r];
              has = true;
            }
        const float z2 = __shfl_xor(z, 32, 64);
        if (!has) z = z2;
        int t = 0;
        if (__ballot(here && z == m)) {  // only then can the label be the row's first maximum
#pragma unroll
          for (int a = 0; a < T::TJ; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) t |= int(j0 + w.j(a, r >> 2) + (r & 3) < y && acc[a][c][r] == z);
          t |= __shfl_xor(t, 32, 64);
        }
        if (here && w.h == 0) {
          p.zlab[i] = z;
          p.tie[i] = t;
        }
      }
    } else {
      float bias[8];
      bool have = false;
      through_lds<T>(smem, w, acc, c, [&](int r, int j, float(&v)[8]) {
        const float sm = __shfl(stat[c].x, r & 31, 64), sy = __shfl(stat[c].y, r & 31, 64);
        const int y = __shfl(lab[c], r & 31, 64) - (j0 + j);
        if (i0 + r >= X.n) return;
        if (!have) {  // a lane's columns stay the same
          const float* b = p.bias32 + j0 + j;
          const float4 x = *reinterpret_cast<const float4*>(b), y = *reinterpret_cast<const float4*>(b + 4);
          bias[0] = x.x; bias[1] = x.y; bias[2] = x.z; bias[3] = x.w;
          bias[4] = y.x; bias[5] = y.y; bias[6] = y.z; bias[7] = y.w;
          have = true;
        }
        uint16_t* g = p.G + int64_t(i0 + r) * p.ldg + (j0 - p.v0) + j;
        float d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = __builtin_amdgcn_exp2f((v[e] + bias[e] - sm) * kLog2e) * sy;
        if (__ballot(unsigned(y) < 8u)) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e == y) d[e] -= 1.f;
        }
        uint16_t q[PL][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sums[e] += d[e];
#pragma unroll
          for (int k = 0; k < PL; ++k) {  // each plane what those before it leave
            q[k][e] = f2bf(d[e]);
            d[e] -= bf2f(q[k][e]);
          }
        }
        auto eight = [](const uint16_t(&a)[8]) {
          return make_uint4(a[0] | (uint32_t(a[1]) << 16), a[2] | (uint32_t(a[3]) << 16), a[4] | (uint32_t(a[5]) << 16),
                            a[6] | (uint32_t(a[7]) << 16));
        };
#pragma unroll
        for (int k = 0; k < PL; ++k) *reinterpret_cast<uint4*>(g + k * p.gplane) = eight(q[k]);
      });
    }
  }
  if constexpr (BWD) {
    if (p.sums) {
      // db from G as it is, not as it was rounded for the products: its terms cancel
      constexpr int EI = 4 * T::TJ;  // lanes with columns of their own
#pragma unroll
      for (int o = EI; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[e] += __shfl_xor(sums[e], o, 64);
      if (w.lane < EI) {
        float* o = p.sums + int64_t(ti * T::WI + w.wi) * p.sums_ld + (j0 - p.v0) + w.wj * T::TJ * 32 + 8 * w.lane;
        *reinterpret_cast<float4*>(o) = make_float4(sums[0], sums[1], sums[2], sums[3]);
        *reinterpret_cast<float4*>(o + 4) = make_float4(sums[4], sums[5], sums[6], sums[7]);
      }
    }
  }
}

// Joins the slots of ROWS rows a workgroup: 1024 / ROWS groups of ROWS threads each take every so-manieth
// slot.  The last workgroup to finish adds the workgroups' sums up, in their order.  16 rows where
// there are few (their slots are read by 64 groups at once: 20 rows of 469 slots 14.6 -> 5.8 us, 1280 of
// 239 8.0 -> 7.1), 64 otherwise (a fourth of the workgroups for the count that finds the last one: 10240
// rows of 118 slots 21.6 -> 10.9).
constexpr int kJoinWaves = 16;
template <int kJoinRows>
__global__ __launch_bounds__(64 * kJoinWaves) void xent_join_kernel(const float2* __restrict__ part, int slots, int cap,
                                                                    int slot_cols, const float* __restrict__ zlab,
                                                                    const int* __restrict__ tie,
                                                                    const int* __restrict__ lab, XentDev* dev,
                                                                    float2* __restrict__ stat,
                                                                    double* __restrict__ lsum,
                                                                    int* __restrict__ csum, float* __restrict__ loss,
                                                                    int64_t* __restrict__ correct) {
  constexpr int kJoinGroups = 64 * kJoinWaves / kJoinRows, kQ = 64 / kJoinRows;
  __shared__ float sm[kJoinGroups][kJoinRows], ss[kJoinGroups][kJoinRows];
  __shared__ int sl[kJoinGroups][kJoinRows];
  __shared__ int last;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = threadIdx.x % kJoinRows, grp = threadIdx.x / kJoinRows;
  const int n = dev->n;
  const int i = blockIdx.x * kJoinRows + row;
  const bool live = i < n;
  const int yslot = live ? lab[i] / slot_cols : 0;
  const float z = live ? zlab[i] : 0.f;
  float m = -INFINITY, s = 0.f;
  int beaten = 0;  // a slot in front of the label's holds a logit as large
  if (live) {
#pragma unroll 4
    for (int k = grp; k < slots; k += kJoinGroups) {
      const float2 v = part[int64_t(k) * cap + i];
      const float nm = fmaxf(m, v.x);
      const float at = nm == -INFINITY ? 0.f : nm;
      s = s * __builtin_amdgcn_exp2f((m - at) * kLog2e) + v.y * __builtin_amdgcn_exp2f((v.x - at) * kLog2e);
      m = nm;
      beaten |= k < yslot && v.x >= z;
    }
  }
  sm[grp][row] = m;
  ss[grp][row] = s;
  sl[grp][row] = beaten;
  __syncthreads();
  if (wave == 0) {
    // kQ lanes a row, each a share of the groups
    const int q = lane / kJoinRows;
    m = -INFINITY;
    beaten = 0;
#pragma unroll
    for (int k = 0; k < kJoinGroups / kQ; ++k) {
      m = fmaxf(m, sm[kQ * k + q][row]);
      beaten |= sl[kQ * k + q][row];
    }
#pragma unroll
    for (int o = kJoinRows; o < 64; o <<= 1) {
      m = fmaxf(m, __shfl_xor(m, o, 64));
      beaten |= __shfl_xor(beaten, o, 64);
    }
    const float at = m == -INFINITY ? 0.f : m;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < kJoinGroups / kQ; ++k)
      s += ss[kQ * k + q][row] * __builtin_amdgcn_exp2f((sm[kQ * k + q][row] - at) * kLog2e);
#pragma unroll
    for (int o = kJoinRows; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
    double l = 0.0;
    int ok = 0;
    if (live && q == 0) {
      stat[i] = make_float2(m, 1.f / s);
      // (max - z) first: exact where the label's logit is the largest or near it
      l = double(m - z) + double(logf(s));
      ok = z == m && !beaten && !tie[i] && s == s;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      l += __shfl_xor(l, o, 64);
      ok += __shfl_xor(ok, o, 64);
    }
    if (lane == 0) {
      __hip_atomic_store(lsum + blockIdx.x, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(csum + blockIdx.x, ok, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = __hip_atomic_fetch_add(&dev->done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == int(gridDim.x) - 1;
    }
  }
  __syncthreads();
  if (!last || wave != 0) return;
  double l = 0.0;
  int64_t ok = 0;
  for (unsigned b = lane; b < gridDim.x; b += 64) {
    l += __hip_atomic_load(lsum + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    ok += __hip_atomic_load(csum + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    l += __shfl_xor(l, o, 64);
    ok += __shfl_xor(ok, o, 64);
  }
  if (lane == 0) {
    *loss = n > 0 ? float(l / n) : 0.f;
    *correct = ok;
  }
}

// waves down a tile's rows
int tile_wi(int t) { return t == kWide ? 4 : t == kFew ? 1 : 2; }
// columns of one (max, sum) slot: a wave's part of the tile
int tile_slot(int t) { return t <= kBig ? 128 : t == kFew ? 32 : 64; }

// NP products a logit (gemm_tile.h), PL planes of G
template <int NP, bool BWD, int PL>
void launch_logits(LogitArgs& p, int tile, hipStream_t st) {
  p.tj = (p.v1 - p.v0 + tile_bj(tile) - 1) / tile_bj(tile);
  const dim3 grid(unsigned(tiles_of(tile, p.X.n, p.v1 - p.v0)));
  auto go = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL((xent_logits_kernel<T, BWD, PL>), grid, dim3(T::kThreads), 0, st, p);
    check_launch();
  };
  // bf16's G has two planes with few rows only, one with more than kFew and kSq are for
  constexpr bool few = !(BWD && PL == 1), large = !(BWD && PL == 2);
  if constexpr (few)
    if (tile == kFew) return go(static_cast<Few<NP, false, false>*>(nullptr));
  if constexpr (large) {
    if (tile == kBig) return go(static_cast<Big<NP, false, false>*>(nullptr));
    if (tile == kDeep) return go(static_cast<Deep<NP, false, false>*>(nullptr));
    if (tile == kWide) return go(static_cast<Wide<NP, false, false>*>(nullptr));
  }
  go(static_cast<Sq<NP, false, false>*>(nullptr));
}

}  // namespace

// ---- host --------------------------------------------------------------------------------------

namespace {

struct XentPlan {
  int kp, vpad, piece, tile, slots, gtile, dx_tile, dw_tile, dw_splits;
  int planes;             // of G
  Split dx_split, dw_split;
  Extent dx;
  int64_t fwd_bytes, bwd_bytes;
  // offsets into the forward's workspace
  int64_t o_part, o_zlab, o_tie, o_lsum, o_csum, o_counts;
  // offsets into the backward's
  int64_t b_g, b_dx, b_dw, b_db;
};

constexpr int kTwoRows = 128;
// rows from which xent_count runs: the gather takes 6.2 / 9.2 / 15.9 / 42 us without it at 8192 / 16384 /
// 32768 / 65536 rows of 64, 4.8 / 5.3 / 6.3 / 8.8 with it, and it takes 2.8 and a launch
constexpr int kCountFrom = 12288;

// g_bytes: most for G of one piece of the vocabulary (one piece has 256 columns at least)
XentPlan xent_plan(int rows, int width, int classes, bool f32, int64_t g_bytes) {
  XentPlan q{};
  const int np = f32 ? 6 : 1;
  // bf16: one rounding of G to bf16 is one more of the same size as the gradients' own, and over many
  // rows their errors add up to 1.2 times that one's; with a few rows one element can make up a
  // gradient, and the sum reaches twice.  There the products only stream the weights, and a second plane
  // costs nothing.
  q.planes = f32 ? 3 : rows <= kTwoRows ? 2 : 1;
  q.kp = int(up(width, 8));
  q.vpad = int(up(classes, 256));
  auto tile = [&](int cols) { return rows > 32 && rows <= kTwoRows ? kSq : choose_tile(rows, cols, width, np, false, false); };
  q.tile = tile(classes);
  q.slots = int(up(classes, tile_bj(q.tile)) / tile_slot(q.tile));
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at = up(at + bytes, 256);
    return o;
  };
  q.o_part = take(int64_t(q.slots) * rows * 8);
  q.o_zlab = take(int64_t(rows) * 4);
  q.o_tie = take(int64_t(rows) * 4);
  const int64_t jb = (rows + 15) / 16;
  q.o_lsum = take(jb * 8);
  q.o_csum = take(jb * 4);
  q.o_counts = take(rows > kCountFrom ? (rows + kCountRows - 1) / kCountRows * int64_t(4) : 0);
  q.fwd_bytes = at;
  at = 0;
  // pieces of equal width, so that none of them is a remainder that fills a few CUs
  const int64_t row_bytes = int64_t(rows) * 2 * q.planes;
  const int64_t most = std::max<int64_t>(256, g_bytes / row_bytes / 256 * 256);
  const int64_t pieces = (q.vpad + most - 1) / most;
  q.piece = int(up((q.vpad + pieces - 1) / pieces, 256));
  q.gtile = tile(q.piece);
  q.b_g = take(row_bytes * q.piece);
  // dx: few tiles and a long reduction (the piece), so as large a tile as the rows fill: its slabs'
  // traffic grows with the splits
  q.dx_tile = rows <= 32 ? kFew : rows < 1024 ? kSq : kWide;
  q.dx_split = split_of(q.dx_tile);
  q.dx = extent_of(q.dx_tile, rows, width, q.dx_split, q.piece);
  q.b_dx = take(q.dx.slab_rows * q.kp * 4);
  const int64_t wi = std::min(q.piece, classes);
  q.dw_tile = rows <= kTwoRows ? kSq : choose_tile(wi, width, rows, np, true, true);
  q.dw_split = split_of(q.dw_tile);
  q.dw_splits = q.dw_split.of(tiles_of(q.dw_tile, wi, width), rows);
  q.dw_split.most = q.dw_splits;  // a narrower last piece has no room for more
  q.b_dw = take(q.dw_splits > 1 ? int64_t(q.dw_splits) * q.piece * q.kp * 4 : 0);
  q.b_db = take((rows + tile_bi(q.gtile) - 1) / tile_bi(q.gtile) * int64_t(tile_wi(q.gtile)) * q.piece * 4);
  q.bwd_bytes = at;
  return q;
}

void check_xent(int64_t rows, int64_t width, int64_t classes, int64_t vocab, int64_t g_bytes) {
  VODA_CHECK(rows > 0 && rows <= (1 << 24), "linear_xent: 1 to 2^24 rows");
  VODA_CHECK(width > 0 && width <= (1 << 20), "linear_xent: width 1 to 2^20");
  VODA_CHECK(classes > 0 && classes <= vocab && vocab <= (1 << 24), "linear_xent: 1 <= classes <= vocabulary <= 2^24");
  // a launch holds less than 2^32 threads: 256 x 128 a workgroup of 256, eight outputs a thread of the finish
  VODA_CHECK(up(rows, 128) / 128 * (up(classes, 256) / 256) < (1 << 24), "linear_xent: rows x vocabulary too large");
  VODA_CHECK(rows * up(width, 8) <= (int64_t(1) << 34), "linear_xent: rows x width too large");
  VODA_CHECK(g_bytes >= 0, "linear_xent: the workspace's limit is negative");
}

}  // namespace

namespace {

// G w, on one of the tiles that the plan takes for dx: kFew needs 32 rows at most, where bf16's G has two
// planes, kWide 1024 at least, where it has one
template <int NP>
void dx_gemm(int tile, const GemmArgs& p, int64_t grid, hipStream_t st) {
  if constexpr (NP != 1)
    if (tile == kFew) return launch_gemm<Few<NP, false, true>, false>(p, grid, st);
  if constexpr (NP != 2)
    if (tile == kWide) return launch_gemm<Wide<NP, false, true>, false>(p, grid, st);
  launch_gemm<Sq<NP, false, true>, false>(p, grid, st);
}

}  // namespace

// bytes of (forward workspace, backward workspace), and the widths of x's compact rows and of the
// padded fp32 bias
std::vector<int64_t> linear_xent_sizes(int64_t rows, int64_t width, int64_t classes, int64_t vocab, bool f32, int64_t g_bytes) {
  check_xent(rows, width, classes, vocab, g_bytes);
  const XentPlan q = xent_plan(int(rows), int(width), int(classes), f32, g_bytes);
  return {q.fwd_bytes, q.bwd_bytes, q.kp, q.vpad, int64_t(sizeof(XentDev))};
}

// What the backward needs (x's compact rows xc, bias32, inv, lab, stat, dev), each its own allocation of the
// caller.  ``wp`` (fp32): workspace for w's planes, [3][classes][width up to 8].
void linear_xent_fwd(uintptr_t x, int64_t ldx, uintptr_t w, int64_t ldw, uintptr_t bias, int bias_dt, uintptr_t labels,
                     int64_t ignore, int64_t rows, int64_t width, int64_t classes, int64_t vocab, int dt, uintptr_t ws,
                     uintptr_t xc, uintptr_t bias32, uintptr_t inv, uintptr_t lab, uintptr_t stat, uintptr_t dev,
                     uintptr_t wp, uintptr_t loss, uintptr_t correct, uintptr_t n_out, uintptr_t stream) {
  check_xent(rows, width, classes, vocab, 0);
  VODA_CHECK(dt == kF32 || dt == kBF16, "linear_xent: x must be fp32 or bf16");
  const bool f32 = dt == kF32;
  VODA_CHECK(f32 || (w % 16 == 0 && ldw % 8 == 0 && ldw >= up(width, 8)),
             "linear_xent: bf16 weight rows must be 16-byte aligned and whole 16-byte vectors");
  VODA_CHECK(xc % 16 == 0 && ws % 256 == 0 && wp % 16 == 0 && (wp || !f32), "linear_xent: workspaces must be aligned");
  const XentPlan q = xent_plan(int(rows), int(width), int(classes), f32, 0);
  hipStream_t st = as_stream(stream);
  uint8_t* base = reinterpret_cast<uint8_t*>(ws);
  XentDev* d = reinterpret_cast<XentDev*>(dev);
  GatherArgs g{};
  g.x = reinterpret_cast<const void*>(x);
  g.ldx = ldx;
  g.rows = int(rows);
  g.width = int(width);
  g.classes = int(classes);
  g.vec = f32 ? x % 16 == 0 && ldx % 4 == 0 && width % 4 == 0 : x % 16 == 0 && ldx % 8 == 0 && width % 8 == 0;
  g.labels = reinterpret_cast<const int64_t*>(labels);
  g.ignore = ignore;
  g.xc = reinterpret_cast<uint16_t*>(xc);
  g.kp = q.kp;
  g.plane = rows * q.kp;
  g.inv = reinterpret_cast<int*>(inv);
  g.lab = reinterpret_cast<int*>(lab);
  g.dev = d;
  g.n_out = reinterpret_cast<int64_t*>(n_out);
  g.bias = reinterpret_cast<const void*>(bias);
  g.bias_bf16 = bias_dt == kBF16;
  g.bias32 = reinterpret_cast<float*>(bias32);
  g.bias_n = q.vpad;
  g.gather_blocks = int((rows + kGatherRows - 1) / kGatherRows);
  if (rows > kCountFrom) {
    int* counts = reinterpret_cast<int*>(base + q.o_counts);
    hipLaunchKernelGGL(xent_count_kernel, dim3(unsigned((rows + kCountRows - 1) / kCountRows)), dim3(256), 0, st, g.labels,
                       int(rows), ignore, int(classes), counts);
    check_launch();
    g.counts = counts;
  }
  const dim3 gg(unsigned(g.gather_blocks + (q.vpad + 255) / 256));
  if (f32) hipLaunchKernelGGL((xent_gather_kernel<true>), gg, dim3(256), 0, st, g);
  else hipLaunchKernelGGL((xent_gather_kernel<false>), gg, dim3(256), 0, st, g);
  check_launch();
  LogitArgs p{};
  p.X = {g.xc, q.kp, g.plane, int(rows)};
  p.W = {reinterpret_cast<const uint16_t*>(w), ldw, 0, int(classes)};
  if (f32) p.W = split({reinterpret_cast<const float*>(w), ldw, int(classes), int(width)}, wp, q.kp, st);
  p.width = q.kp;
  p.v0 = 0;
  p.v1 = int(classes);
  p.bias32 = g.bias32;
  p.dev = d;
  p.lab = g.lab;
  p.part = reinterpret_cast<float2*>(base + q.o_part);
  p.zlab = reinterpret_cast<float*>(base + q.o_zlab);
  p.tie = reinterpret_cast<int*>(base + q.o_tie);
  if (f32) launch_logits<6, false, 1>(p, q.tile, st);
  else launch_logits<1, false, 1>(p, q.tile, st);
  auto join = [&](auto kernel, int per) {
    hipLaunchKernelGGL(kernel, dim3(unsigned((rows + per - 1) / per)), dim3(64 * kJoinWaves), 0, st, p.part, q.slots, int(rows),
                       tile_slot(q.tile), p.zlab, p.tie, g.lab, d, reinterpret_cast<float2*>(stat),
                       reinterpret_cast<double*>(base + q.o_lsum), reinterpret_cast<int*>(base + q.o_csum),
                       reinterpret_cast<float*>(loss), reinterpret_cast<int64_t*>(correct));
  };
  if (rows <= 1024) join(xent_join_kernel<16>, 16);
  else join(xent_join_kernel<64>, 64);
  check_launch();
}

// dx [rows][width] contiguous in x's type; rows [0, classes) of dw [..][ldd] in ``grad_dt`` and of db in
// ``db_dt`` (added to when ``accumulate``); each of dx, dw and db may be null.  ``g_bytes`` as in the
// sizes.
void linear_xent_bwd(uintptr_t w, int64_t ldw, int64_t rows, int64_t width, int64_t classes, int64_t vocab, int dt,
                     uintptr_t ws, uintptr_t xc, uintptr_t bias32, uintptr_t inv, uintptr_t lab, uintptr_t stat,
                     uintptr_t dev, uintptr_t wp, uintptr_t gloss, uintptr_t dx, uintptr_t dw, int64_t ldd,
                     uintptr_t db, int grad_dt, int db_dt, bool accumulate, int64_t g_bytes, uintptr_t stream) {
  check_xent(rows, width, classes, vocab, g_bytes);
  VODA_CHECK(dt == kF32 || dt == kBF16, "linear_xent: x must be fp32 or bf16");
  VODA_CHECK((grad_dt == kF32 || grad_dt == kBF16) && (db_dt == kF32 || db_dt == kBF16),
             "linear_xent: weight and bias gradients must be fp32 or bf16");
  const bool f32 = dt == kF32;
  VODA_CHECK(f32 || (w % 16 == 0 && ldw % 8 == 0 && ldw >= up(width, 8)),
             "linear_xent: bf16 weight rows must be 16-byte aligned and whole 16-byte vectors");
  VODA_CHECK(xc % 16 == 0 && ws % 256 == 0 && wp % 16 == 0 && (wp || !f32), "linear_xent: workspaces must be aligned");
  const XentPlan q = xent_plan(int(rows), int(width), int(classes), f32, g_bytes);
  hipStream_t st = as_stream(stream);
  uint8_t* base = reinterpret_cast<uint8_t*>(ws);
  XentDev* d = reinterpret_cast<XentDev*>(dev);
  LogitArgs p{};
  p.X = {reinterpret_cast<const uint16_t*>(xc), q.kp, rows * q.kp, int(rows)};
  p.W = {reinterpret_cast<const uint16_t*>(w), ldw, 0, int(classes)};
  if (f32) p.W = split({reinterpret_cast<const float*>(w), ldw, int(classes), int(width)}, wp, q.kp, st);
  p.width = q.kp;
  p.bias32 = reinterpret_cast<const float*>(bias32);
  p.dev = d;
  p.lab = reinterpret_cast<const int*>(lab);
  p.stat = reinterpret_cast<const float2*>(stat);
  p.G = reinterpret_cast<uint16_t*>(base + q.b_g);
  p.ldg = q.piece;
  p.gplane = rows * q.piece;
  p.sums = db ? reinterpret_cast<float*>(base + q.b_db) : nullptr;
  p.sums_ld = q.piece;
  Emit e{};
  e.gl = reinterpret_cast<const float*>(gloss);
  e.gn = &d->n;
  const int gsz = grad_dt == kF32 ? 4 : 2;
  GemmArgs x{};
  x.I = {p.G, q.piece, p.gplane, int(rows)};
  x.ni_dev = &d->n;
  x.split = q.dx_split;
  x.nk_split = q.piece;
  x.slab = reinterpret_cast<float*>(base + q.b_dx);
  x.lds = q.kp;
  x.e = e;
  x.e.out = reinterpret_cast<void*>(dx);
  x.e.ldo = width;
  x.e.bf16 = !f32;
  x.e.nj = int(width);
  x.e.vec = whole_rows(dx, width, !f32);
  ColumnSums c{};  // db of a piece
  if (db) {
    c.part = p.sums;
    c.ld = q.piece;
    c.rows_dev = &d->n;
    c.bi = tile_bi(q.gtile);
    c.per = tile_wi(q.gtile);
    c.bf16 = db_dt == kBF16;
    c.e.gl = e.gl;
    c.e.gn = e.gn;
    c.e.accumulate = accumulate;
  }
  for (int v0 = 0; v0 < classes; v0 += q.piece) {
    const int v1 = int(std::min<int64_t>(classes, v0 + q.piece));
    p.v0 = v0;
    p.v1 = v1;
    if (f32) launch_logits<6, true, 3>(p, q.gtile, st);
    else if (q.planes == 2) launch_logits<1, true, 2>(p, q.gtile, st);
    else launch_logits<1, true, 1>(p, q.gtile, st);
    if (dx) {
      x.J = {p.W.p + int64_t(v0) * p.W.ld, p.W.ld, p.W.plane, int(up(width, 8))};
      x.nk = v1 - v0;
      x.add = v0 > 0;
      if (f32) dx_gemm<6>(q.dx_tile, x, q.dx.grid, st);
      else if (q.planes == 1) dx_gemm<1>(q.dx_tile, x, q.dx.grid, st);
      else dx_gemm<2>(q.dx_tile, x, q.dx.grid, st);
    }
    if (dw) {
      GemmArgs a{};
      a.I = {p.G, q.piece, p.gplane, v1 - v0};
      a.J = {p.X.p, p.X.ld, p.X.plane, int(up(width, 8))};
      a.nk_dev = &d->n;
      a.nk = int(rows);
      a.split = q.dw_split;
      a.e = e;
      a.e.out = reinterpret_cast<void*>(dw + uintptr_t(int64_t(v0) * ldd * gsz));
      a.e.ldo = ldd;
      a.e.bf16 = grad_dt == kBF16;
      a.e.nj = int(width);
      a.e.vec = whole_rows(dw, ldd, a.e.bf16);
      a.e.accumulate = accumulate;
      if (q.dw_splits > 1) {
        a.slab = reinterpret_cast<float*>(base + q.b_dw);
        a.lds = q.kp;
      }
      const int64_t grid = tiles_of(q.dw_tile, v1 - v0, width) * q.dw_splits;
      if (f32) gemm<6, true, true, false>(q.dw_tile, a, grid, st);
      else if (q.planes == 2) launch_gemm<Sq<2, true, true>, false>(a, grid, st);
      else gemm<1, true, true, false>(q.dw_tile, a, grid, st);
      if (a.slab) finish(q.dw_tile, a, a.I.n, nullptr, {}, st);
    }
    c.n = v1 - v0;
    c.out = reinterpret_cast<void*>(db + uintptr_t(v0) * (db_dt == kF32 ? 4 : 2));
    // dx is whole after the last piece
    finish(q.dx_tile, x, dx && v1 == classes ? int(rows) : 0, reinterpret_cast<const int*>(inv), c, st);
  }
}

}  // namespace voda
