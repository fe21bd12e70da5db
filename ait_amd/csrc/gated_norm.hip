// ait_amd/csrc/gated_norm.hip -- ait_gated_norm_fwd / _bwd: the norm behind a block, its gate and residual scale, the residual
// and the norm in front of the next block, one pass over the rows.
//
//   m = norm(f) w_post (+ b_post),   y = x + scale * gate * m,   h = norm(y) w_pre (+ b_pre)
//   norm(t) = (t - mean) / sqrt(mean((t - mean)^2) + eps), or without the means
//
// Bound by memory: x, f and the gate are read once, y and h written once; a row lives in the registers of its G waves between
// the two norms (all sums f32, the variance from the centred values).  The backward reads x, f, gate, dy, dh and forms the row
// again from them and the four saved statistics, in f32 -- y as it was before it was rounded -- and keeps the column sums (the
// parameters' gradients) in registers over the rows of a workgroup; the workgroups' parts are added in order by a second
// kernel, so results repeat bit for bit.
//
// What bounds it: memory.  58800 rows of 512 in f32, LayerNorm: forward 482 MB in 98 us (4.9 TB/s, a large copy's rate here),
// backward 722 MB in 149 (4.8).  About 12600 packed rows of 5120, f32 stream and bf16 branch, a gate a sequence: forward 774 MB
// in 162 to 180 us (4.8 to 4.3), backward 1162 MB in 240 to 250 (4.8 to 4.6).  What it took in the backward, where one workgroup
// of ten waves fits a CU and its phases meet at barriers: a row's loads without branches around them, so that they are in flight
// together, sums over the lanes without trips to shared memory, and parameters held (335 us before the three).  Five rows of
// 4096: 3.8 us, a launch and three dependent trips to memory.
#include "common.h"

#include <type_traits>

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct NormArgs {
  const void* x;
  const void* f;
  const void* gate;
  const float* w_post;
  const float* b_post;
  const float* w_pre;
  const float* b_pre;
  const float* scale;
  const int* cu;
  long long x_row, f_row, g_row, y_row, h_row;
  int rows, width, layer, gate_kind, n_seq;      // gate_kind: 0 none, 1 a row's own, 2 its sequence's
  float eps;
  void* y;
  void* h;
  float* stats;        // [rows][4]: mean of f, 1 / deviation of f, mean of y, 1 / deviation of y
  // backward
  const void* dy;
  const void* dh;
  long long dy_row, dh_row, dx_row, df_row, dg_row;
  void* dx;
  void* df;
  void* dgate;
  float* parts;        // [blocks][n_parts][width] of the parameters, then [units + n_seq][width] of the sequences' gates
  int units, per, blocks, n_parts;      // a unit: a group of waves and its `per` consecutive rows; blocks: workgroups
  int zero_rest;
};
// which parts there are: w_post, w_pre, then scale, b_post, b_pre where given

template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T* row, int at, int width, float* v) {
  if constexpr (VEC) {
    if (at < width) {
      if constexpr (sizeof(T) == 2) {
        const bf16x8 t = *reinterpret_cast<const bf16x8*>(row + at);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)t[e];
      } else {
        const f32x4 a = *reinterpret_cast<const f32x4*>(row + at), b = *reinterpret_cast<const f32x4*>(row + at + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) { v[e] = a[e]; v[4 + e] = b[e]; }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = at + e < width ? (float)row[at + e] : 0.f;
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* row, int at, int width, const float* v) {
  if constexpr (VEC) {
    if (at >= width) return;
    if constexpr (sizeof(T) == 2) {
      bf16x8 t;
#pragma unroll
      for (int e = 0; e < 8; e++) t[e] = (__bf16)v[e];
      *reinterpret_cast<bf16x8*>(row + at) = t;
    } else {
      f32x4 a, b;
#pragma unroll
      for (int e = 0; e < 4; e++) { a[e] = v[e]; b[e] = v[4 + e]; }
      *reinterpret_cast<f32x4*>(row + at) = a;
      *reinterpret_cast<f32x4*>(row + at + 4) = b;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (at + e < width) row[at + e] = (T)v[e];
  }
}

// Eight values of a row on their way: loads without a branch around them (behind the row's end its last ones are loaded, and not
// taken), so that all of a row's loads are in flight together.  In a branch each is waited for before the next one is issued.
template <bool VEC, typename T> struct In;
template <> struct In<true, __bf16> {
  bf16x8 t;
  __device__ __forceinline__ void load(const __bf16* row, int at, int width) { t = *reinterpret_cast<const bf16x8*>(row + min(at, width - 8)); }
  __device__ __forceinline__ void get(float* v, bool there) const {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = there ? (float)t[e] : 0.f;
  }
};
template <> struct In<true, float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float* row, int at, int width) {
    const float* p = row + min(at, width - 8);
    a = *reinterpret_cast<const f32x4*>(p);
    b = *reinterpret_cast<const f32x4*>(p + 4);
  }
  __device__ __forceinline__ void get(float* v, bool there) const {
#pragma unroll
    for (int e = 0; e < 4; e++) { v[e] = there ? a[e] : 0.f; v[4 + e] = there ? b[e] : 0.f; }
  }
};
template <typename T> struct In<false, T> {
  float t[8];
  __device__ __forceinline__ void load(const T* row, int at, int width) { load8<false>(row, at, width, t); }
  __device__ __forceinline__ void get(float* v, bool there) const {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = there ? t[e] : 0.f;
  }
};

template <bool VEC>
__device__ __forceinline__ bool inside(int at, int e, int width) { return VEC ? at < width : at + e < width; }

// the sum of a wave's lanes, in every lane: inside 16 lanes, over the 16s, from the last lane (no trip to shared memory)
__device__ __forceinline__ float lane_sum(float v) {
#define AIT_DPP_ADD(ctrl, rows) \
  v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xf, true))
  AIT_DPP_ADD(0x111, 0xf);
  AIT_DPP_ADD(0x112, 0xf);
  AIT_DPP_ADD(0x114, 0xf);
  AIT_DPP_ADD(0x118, 0xf);
  AIT_DPP_ADD(0x142, 0xa);
  AIT_DPP_ADD(0x143, 0xc);
#undef AIT_DPP_ADD
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// sums over the G waves of a row, two at a time; every lane gets them.  `slot` alternates so that one barrier a sum is enough
template <int G>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* lds, int& slot, int group_wave, int wave) {
  a = lane_sum(a);
  b = lane_sum(b);
  if constexpr (G > 1) {
    float* p = lds + (slot & 1) * 32;
    slot++;
    if ((threadIdx.x & 63) == 0) { p[2 * wave] = a; p[2 * wave + 1] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < G; w++) { a += p[2 * (group_wave + w)]; b += p[2 * (group_wave + w) + 1]; }
  }
}

__device__ __forceinline__ int clamp_row(const int* cu, int i, int rows) {
  const int v = cu[i];
  return v < 0 ? 0 : v > rows ? rows : v;
}
// the sequence of a row, n_seq behind the last one
__device__ __forceinline__ int seq_of(const int* cu, int n_seq, int rows, int row) {
  if (row >= clamp_row(cu, n_seq, rows)) return n_seq;
  int lo = 0, hi = n_seq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (clamp_row(cu, mid, rows) <= row) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// G waves a row, V blocks of eight values a lane: a row has up to 64 G * 8 V values.  NT threads: NT / 64 / G rows at a time
template <int G> struct Block { static constexpr int kRows = G == 1 ? 4 : G == 2 ? 2 : 1, kWaves = G * kRows, kThreads = kWaves * 64; };

template <typename X, typename F, int G, int V, bool VEC>
__global__ __launch_bounds__(Block<G>::kThreads) void gated_norm_fwd_kernel(const NormArgs a) {
  __shared__ float lds[64];
  const int wave = threadIdx.x >> 6, group = wave / G, gl = threadIdx.x - group * G * 64;
  const int row = blockIdx.x * Block<G>::kRows + group, W = a.width;
  int slot = 0;
  const bool there = row < a.rows;
  const int rc = there ? row : a.rows - 1;
  const float inv_w = 1.f / W;
  const int seq = a.gate_kind == 2 ? seq_of(a.cu, a.n_seq, a.rows, rc) : 0;
  const bool dead = a.gate_kind == 2 && seq == a.n_seq;          // behind the last sequence: left as it is, or set to zero
  const bool write = there && (!dead || a.zero_rest);
  float f[V][8], x[V][8];
  {
    In<VEC, F> rf[V];
    In<VEC, X> rx[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
      rf[v].load(reinterpret_cast<const F*>(a.f) + rc * a.f_row, (gl + v * G * 64) * 8, W);
      rx[v].load(reinterpret_cast<const X*>(a.x) + rc * a.x_row, (gl + v * G * 64) * 8, W);
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
      const bool in = !VEC || (gl + v * G * 64) * 8 < W;
      rf[v].get(f[v], in);
      rx[v].get(x[v], in);
    }
  }
  float mean = 0.f, s1 = 0.f, s2 = 0.f;
  if (a.layer) {
#pragma unroll
    for (int v = 0; v < V; v++)
#pragma unroll
      for (int e = 0; e < 8; e++) s1 += f[v][e];
    row_sum2<G>(s1, s2, lds, slot, group * G, wave);
    mean = s1 * inv_w;
  }
  s1 = s2 = 0.f;
#pragma unroll
  for (int v = 0; v < V; v++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      f[v][e] -= inside<VEC>((gl + v * G * 64) * 8, e, W) ? mean : 0.f;
      s1 = __builtin_fmaf(f[v][e], f[v][e], s1);
    }
  row_sum2<G>(s1, s2, lds, slot, group * G, wave);
  const float r = 1.f / __builtin_sqrtf(s1 * inv_w + a.eps), fmean = mean;
  s1 = s2 = 0.f;
#pragma unroll
  for (int v = 0; v < V; v++) {
    const int at = (gl + v * G * 64) * 8;
    float p[8];
    load8<VEC>(a.w_post, at, W, p);
#pragma unroll
    for (int e = 0; e < 8; e++) f[v][e] = f[v][e] * r * p[e];
    if (a.b_post) {
      load8<VEC>(a.b_post, at, W, p);
#pragma unroll
      for (int e = 0; e < 8; e++) f[v][e] += p[e];
    }
    if (a.gate_kind) {
      load8<VEC>(reinterpret_cast<const F*>(a.gate) + (a.gate_kind == 2 ? (dead ? 0 : seq) : rc) * a.g_row, at, W, p);
#pragma unroll
      for (int e = 0; e < 8; e++) f[v][e] *= p[e];
    }
    if (a.scale) {
      load8<VEC>(a.scale, at, W, p);
#pragma unroll
      for (int e = 0; e < 8; e++) f[v][e] *= p[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
      x[v][e] += f[v][e];
      s1 += x[v][e];
    }
    if (dead) {
#pragma unroll
      for (int e = 0; e < 8; e++) x[v][e] = 0.f;
    }
    if (write) store8<VEC>(reinterpret_cast<X*>(a.y) + rc * a.y_row, at, W, x[v]);
  }
  mean = 0.f;
  if (a.layer) {
    row_sum2<G>(s1, s2, lds, slot, group * G, wave);
    mean = s1 * inv_w;
  }
  s1 = s2 = 0.f;
#pragma unroll
  for (int v = 0; v < V; v++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      x[v][e] -= inside<VEC>((gl + v * G * 64) * 8, e, W) ? mean : 0.f;
      s1 = __builtin_fmaf(x[v][e], x[v][e], s1);
    }
  row_sum2<G>(s1, s2, lds, slot, group * G, wave);
  const float ry = 1.f / __builtin_sqrtf(s1 * inv_w + a.eps);
#pragma unroll
  for (int v = 0; v < V; v++) {
    const int at = (gl + v * G * 64) * 8;
    float p[8];
    load8<VEC>(a.w_pre, at, W, p);
#pragma unroll
    for (int e = 0; e < 8; e++) x[v][e] = x[v][e] * ry * p[e];
    if (a.b_pre) {
      load8<VEC>(a.b_pre, at, W, p);
#pragma unroll
      for (int e = 0; e < 8; e++) x[v][e] += p[e];
    }
    if (dead) {
#pragma unroll
      for (int e = 0; e < 8; e++) x[v][e] = 0.f;
    }
    if (write) store8<VEC>(reinterpret_cast<F*>(a.h) + rc * a.h_row, at, W, x[v]);
  }
  if (a.stats && there && gl == 0) {
    f32x4 s;
    s[0] = fmean; s[1] = r; s[2] = mean; s[3] = ry;
    *reinterpret_cast<f32x4*>(a.stats + 4ll * row) = s;
  }
}

// one workgroup: `per` rows, one behind another per group of waves (a workgroup's groups take them in turn)
// SUMS_B: also the biases' gradients
template <typename X, typename F, int G, int V, bool VEC, bool SUMS_B>
__global__ __launch_bounds__(Block<G>::kThreads) void gated_norm_bwd_kernel(const NormArgs a) {
  constexpr int R = Block<G>::kRows;
  __shared__ float lds[64];
  const int wave = threadIdx.x >> 6, group = wave / G, gl = threadIdx.x - group * G * 64, W = a.width;
  const float inv_w = 1.f / W;
  int slot = 0;
  // column sums: [part][value]; a group's rows are `per` / R consecutive ones
  float cp[V][8], cq[V][8], cs[V][8], bp[V][8], bq[V][8], cg[V][8];
#pragma unroll
  for (int v = 0; v < V; v++)
#pragma unroll
    for (int e = 0; e < 8; e++) cp[v][e] = cq[v][e] = cs[v][e] = bp[v][e] = bq[v][e] = cg[v][e] = 0.f;
  const int unit = blockIdx.x * R + group, first = unit * a.per, last = min(first + a.per, a.rows);
  float* gate_parts = a.parts + (size_t)a.blocks * a.n_parts * W;
  // The parameters of a lane's values are held over all rows where a lane has one block of eight: in registers up to eight waves,
  // in shared memory for more, whose 168 registers a lane are too few for both (with biases 12 to 48 bytes a lane spill even so).
  // Two blocks a lane (rows over 6144, unaligned ones over 4096) read them in place and spill: 12 to 36 bytes a lane without biases,
  // 164 to 204 with, 208 to 476 unaligned.  (The next row's loads issued under this one's arithmetic gain nothing where registers
  // allow it, 150 us against 149, and spill in ten waves: 280 against 241.)
  constexpr bool HELD = V == 1 && G <= 8, LDSP = V == 1 && !HELD;
  __shared__ __attribute__((aligned(16))) float wl[LDSP ? (SUMS_B ? 4 : 3) : 1][LDSP ? G * 512 : 4];
  const float* from[4] = {a.w_post, a.w_pre, a.scale, a.b_post};
  float w[HELD ? 4 : 1][8];
  if constexpr (V == 1) {
#pragma unroll
    for (int i = 0; i < (SUMS_B ? 4 : 3); i++) {
      float t[8];
#pragma unroll
      for (int e = 0; e < 8; e++) t[e] = i == 2 ? 1.f : 0.f;
      if (from[i]) load8<VEC>(from[i], gl * 8, W, t);
      if constexpr (HELD) {
#pragma unroll
        for (int e = 0; e < 8; e++) w[i][e] = t[e];
      } else {      // (a lane reads what it wrote itself: no barrier)
        store8<true>(&wl[i][0], gl * 8, G * 512, t);
      }
    }
  }
  auto parameter = [&](auto which, int at, float* to) {      // 0 w_post, 1 w_pre, 2 scale or 1, 3 b_post or 0
    constexpr int i = decltype(which)::value;
    if constexpr (HELD) {
#pragma unroll
      for (int e = 0; e < 8; e++) to[e] = w[i][e];
    } else if constexpr (LDSP) {
      load8<true>(&wl[i][0], gl * 8, G * 512, to);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) to[e] = i == 2 ? 1.f : 0.f;
      if (i < 2 || from[i]) load8<VEC>(from[i], at, W, to);
    }
  };
  constexpr std::integral_constant<int, 0> kPost{};
  constexpr std::integral_constant<int, 1> kPre{};
  constexpr std::integral_constant<int, 2> kScale{};
  constexpr std::integral_constant<int, 3> kPostBias{};
  In<VEC, F> rf[V], rd[V], rg[V];
  In<VEC, X> ry[V], rt[V];
  f32x4 rs;
  auto fetch = [&](int row) {
    const long long rc = min(row, a.rows - 1);
    rs = *reinterpret_cast<const f32x4*>(a.stats + 4 * rc);
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int at = (gl + v * G * 64) * 8;
      rf[v].load(reinterpret_cast<const F*>(a.f) + rc * a.f_row, at, W);
      ry[v].load(reinterpret_cast<const X*>(a.x) + rc * a.x_row, at, W);
      rd[v].load(reinterpret_cast<const F*>(a.dh) + rc * a.dh_row, at, W);
      rt[v].load(reinterpret_cast<const X*>(a.dy) + rc * a.dy_row, at, W);
      if (a.gate_kind == 1) rg[v].load(reinterpret_cast<const F*>(a.gate) + rc * a.g_row, at, W);
    }
  };
  auto fetch_gate = [&](int s) {
#pragma unroll
    for (int v = 0; v < V; v++) rg[v].load(reinterpret_cast<const F*>(a.gate) + (s < a.n_seq ? s : 0) * a.g_row, (gl + v * G * 64) * 8, W);
  };
  int seq = 0;
  if (a.gate_kind == 2) {
    if (first < a.rows) seq = seq_of(a.cu, a.n_seq, a.rows, first);
    if (a.n_seq > 0) fetch_gate(seq);
  }
  for (int i = 0; i < a.per; i++) {          // (every group makes every turn: the sums meet at barriers)
    const int row = first + i;
    const bool there = row < last;
    const int rc = there ? row : a.rows - 1;
    if (a.gate_kind == 2 && there && seq < a.n_seq && row >= clamp_row(a.cu, seq + 1, a.rows)) {
      // the sequence's share of this workgroup is complete: units and sequences only ever go up together, so unit + sequence
      // numbers the pairs that meet without a clash
#pragma unroll
      for (int v = 0; v < V; v++) {
        store8<VEC>(gate_parts + (size_t)(unit + seq) * W, (gl + v * G * 64) * 8, W, cg[v]);
#pragma unroll
        for (int e = 0; e < 8; e++) cg[v][e] = 0.f;
      }
      seq = seq_of(a.cu, a.n_seq, a.rows, row);
      fetch_gate(seq);
    }
    const bool dead = !there || (a.gate_kind == 2 && seq == a.n_seq);
    const bool write = there && (!dead || a.zero_rest);
    fetch(row);
    // a dead row is a row of zeros, whatever memory holds
    f32x4 st = rs;
    if (dead) st[0] = st[1] = st[2] = st[3] = 0.f;
    float f[V][8], y[V][8], d[V][8], t[V][8], gate[V][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < V; v++) {
      const bool in = !dead && (!VEC || (gl + v * G * 64) * 8 < W);
      rf[v].get(f[v], in);
      ry[v].get(y[v], in);
      rd[v].get(d[v], in);
      rt[v].get(t[v], in);
#pragma unroll
      for (int e = 0; e < 8; e++) gate[v][e] = 1.f;
      if (a.gate_kind) rg[v].get(gate[v], in);
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int at = (gl + v * G * 64) * 8;
      float p[8], q[8], m[8];
      parameter(kPost, at, p);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        f[v][e] = inside<VEC>(at, e, W) ? (f[v][e] - st[0]) * st[1] : 0.f;       // norm(f)
        m[e] = f[v][e] * p[e];
      }
      if constexpr (SUMS_B) {
        parameter(kPostBias, at, p);
#pragma unroll
        for (int e = 0; e < 8; e++) m[e] += p[e];
      }
      parameter(kScale, at, q);
#pragma unroll
      for (int e = 0; e < 8; e++) y[v][e] = inside<VEC>(at, e, W) ? (y[v][e] + m[e] * gate[v][e] * q[e] - st[2]) * st[3] : 0.f;      // norm(y)
      parameter(kPre, at, p);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        cq[v][e] = __builtin_fmaf(d[v][e], y[v][e], cq[v][e]);
        if (SUMS_B) bq[v][e] += d[v][e];
        d[v][e] *= p[e];
        s1 = __builtin_fmaf(d[v][e], y[v][e], s1);
        s2 += d[v][e];
      }
    }
    row_sum2<G>(s1, s2, lds, slot, group * G, wave);
    s1 *= inv_w;
    s2 = a.layer ? s2 * inv_w : 0.f;
    float t1 = 0.f, t2 = 0.f;
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int at = (gl + v * G * 64) * 8;
      float q[8], m[8], b[8];
      float* u = t[v];
#pragma unroll
      for (int e = 0; e < 8; e++) u[e] = u[e] + st[3] * (d[v][e] - s2 - y[v][e] * s1);        // d y
      if (write) store8<VEC>(reinterpret_cast<X*>(a.dx) + rc * a.dx_row, at, W, u);
      parameter(kScale, at, q);
      parameter(kPost, at, m);
#pragma unroll
      for (int e = 0; e < 8; e++) b[e] = 0.f;
      if constexpr (SUMS_B) parameter(kPostBias, at, b);
      float k[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float um = u[e] * (f[v][e] * m[e] + b[e]);
        cs[v][e] = __builtin_fmaf(um, gate[v][e], cs[v][e]);
        k[e] = um * q[e];                                            // d gate
        cg[v][e] += k[e];
        u[e] *= gate[v][e] * q[e];                                         // d m
        if (SUMS_B) bp[v][e] += u[e];
        cp[v][e] = __builtin_fmaf(u[e], f[v][e], cp[v][e]);
      }
      if (a.gate_kind == 1 && there) store8<VEC>(reinterpret_cast<F*>(a.dgate) + rc * a.dg_row, at, W, k);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        d[v][e] = u[e] * m[e];
        t1 = __builtin_fmaf(d[v][e], f[v][e], t1);
        t2 += d[v][e];
      }
    }
    row_sum2<G>(t1, t2, lds, slot, group * G, wave);
    t1 *= inv_w;
    t2 = a.layer ? t2 * inv_w : 0.f;
#pragma unroll
    for (int v = 0; v < V; v++) {
#pragma unroll
      for (int e = 0; e < 8; e++) d[v][e] = st[1] * (d[v][e] - t2 - f[v][e] * t1);
      if (write) store8<VEC>(reinterpret_cast<F*>(a.df) + rc * a.df_row, (gl + v * G * 64) * 8, W, d[v]);
    }
  }
  // the parameters' sums: those of a workgroup's groups added in order, one part of a workgroup to memory
  __shared__ float join[R > 1 ? R * G * 512 : 1];
  float* out = a.parts + (size_t)blockIdx.x * a.n_parts * W;
  auto part = [&](float (*c)[8]) {
    if constexpr (R > 1) {
      __syncthreads();
      float* mine = join + group * G * 512;
#pragma unroll
      for (int v = 0; v < V; v++)
#pragma unroll
        for (int e = 0; e < 8; e++) mine[(gl + v * G * 64) * 8 + e] = c[v][e];
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
          for (int e = 0; e < 8; e++)
#pragma unroll
            for (int g = 1; g < R; g++) c[v][e] += join[g * G * 512 + (gl + v * G * 64) * 8 + e];
      }
    }
    if (group == 0)
#pragma unroll
      for (int v = 0; v < V; v++) store8<VEC>(out, (gl + v * G * 64) * 8, W, c[v]);
    out += W;
  };
  part(cp);
  part(cq);
  if (a.scale) part(cs);
  if (SUMS_B && a.b_post) part(bp);
  if (SUMS_B && a.b_pre) part(bq);
  if (a.gate_kind == 2 && first < a.rows && seq < a.n_seq)
#pragma unroll
    for (int v = 0; v < V; v++) store8<VEC>(gate_parts + (size_t)(unit + seq) * W, (gl + v * G * 64) * 8, W, cg[v]);
}

// the units' parts of the parameters' gradients added in order: 16 values and 64 rows of units to a workgroup
struct SumArgs {
  const float* parts;
  float* out[5];
  int units, n_parts, width;
};
__global__ __launch_bounds__(1024) void gated_norm_sum_kernel(const SumArgs a) {
  __shared__ float sums[1024];
  const int t = threadIdx.x, n = a.n_parts * a.width, c = blockIdx.x * 16 + (t & 15);
  float u = 0.f;
  if (c < n) {
    int i = t >> 4;
    for (; i + 448 < a.units; i += 512) {          // eight loads in flight
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = a.parts[(size_t)(i + 64 * j) * n + c];
#pragma unroll
      for (int j = 0; j < 8; j++) u += v[j];
    }
    for (; i < a.units; i += 64) u += a.parts[(size_t)i * n + c];
  }
  sums[t] = u;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if ((t >> 4) < o) sums[t] += sums[t + 16 * o];
    __syncthreads();
  }
  if (t < 16 && c < n) {
    const int part = c / a.width;
    a.out[part][c - part * a.width] = sums[t];
  }
}
// a sequence's gate: the parts of the units that have rows of it
template <typename F>
__global__ __launch_bounds__(256) void gated_norm_gate_kernel(const NormArgs a) {
  const int nx = (a.width + 255) / 256, b = blockIdx.x / nx, c = (blockIdx.x - b * nx) * 256 + threadIdx.x;
  if (c >= a.width) return;
  const int start = clamp_row(a.cu, b, a.rows), end = clamp_row(a.cu, b + 1, a.rows);
  const float* parts = a.parts + (size_t)a.blocks * a.n_parts * a.width;
  float u = 0.f;
  if (end > start) {
    int i = start / a.per;
    const int last = (end - 1) / a.per;
    for (; i + 7 <= last; i += 8) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = parts[(size_t)(i + j + b) * a.width + c];
#pragma unroll
      for (int j = 0; j < 8; j++) u += v[j];
    }
    for (; i <= last; i++) u += parts[(size_t)(i + b) * a.width + c];
  }
  reinterpret_cast<F*>(a.dgate)[(long long)b * a.dg_row + c] = (F)u;
}

constexpr int kMaxWidth = 8192;
bool aligned(const void* p, long long row, int es) { return !p || ((unsigned long long)p % 16 == 0 && (row * es) % 16 == 0); }

template <typename X, typename F, bool BWD, bool VEC, int G, int V>
int launch_gv(const NormArgs& a, hipStream_t st) {
  const int rows = BWD ? a.units : a.rows;
  const dim3 grid((unsigned)((rows + Block<G>::kRows - 1) / Block<G>::kRows)), block(Block<G>::kThreads);
  if ((unsigned long long)grid.x * block.x >= (1ull << 32)) return AIT_EUNSUPPORTED;      // a launch's work items are counted in 32 bits
  if constexpr (BWD) {
    if (a.b_post || a.b_pre) hipLaunchKernelGGL((gated_norm_bwd_kernel<X, F, G, V, VEC, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((gated_norm_bwd_kernel<X, F, G, V, VEC, false>), grid, block, 0, st, a);
  } else hipLaunchKernelGGL((gated_norm_fwd_kernel<X, F, G, V, VEC>), grid, block, 0, st, a);
  AIT_CHECK_LAUNCH();
  return AIT_OK;
}
template <typename X, typename F, bool BWD>
int launch_xf(const NormArgs& a, bool vec, hipStream_t st) {
  // as many waves as the row fills: one block of eight values a lane up to 6144, two beyond (rows of 5120: backward a
  // sixth faster in ten waves of one block than in eight of two, forward alike; rows of 512: forward 96 us in one wave, 100 in two)
  if (!vec) {
    if (a.width <= 512) return launch_gv<X, F, BWD, false, 1, 1>(a, st);
    if (a.width <= 2048) return launch_gv<X, F, BWD, false, 4, 1>(a, st);
    return a.width <= 4096 ? launch_gv<X, F, BWD, false, 8, 1>(a, st) : launch_gv<X, F, BWD, false, 8, 2>(a, st);
  }
  switch ((a.width + 511) / 512) {
    case 1: return launch_gv<X, F, BWD, true, 1, 1>(a, st);
    case 2: return launch_gv<X, F, BWD, true, 2, 1>(a, st);
    case 3: return launch_gv<X, F, BWD, true, 3, 1>(a, st);
    case 4: return launch_gv<X, F, BWD, true, 4, 1>(a, st);
    case 5: case 6: return launch_gv<X, F, BWD, true, 6, 1>(a, st);
    case 7: case 8: return launch_gv<X, F, BWD, true, 8, 1>(a, st);
    case 9: case 10: return launch_gv<X, F, BWD, true, 10, 1>(a, st);
    case 11: case 12: return launch_gv<X, F, BWD, true, 12, 1>(a, st);
    default: return launch_gv<X, F, BWD, true, 8, 2>(a, st);
  }
}
template <bool BWD>
int launch(const ait_gated_norm& p, const NormArgs& a, bool vec, hipStream_t st) {
  if (p.dtype_x == AIT_DTYPE_BF16) return launch_xf<__bf16, __bf16, BWD>(a, vec, st);
  if (p.dtype_f == AIT_DTYPE_BF16) return launch_xf<float, __bf16, BWD>(a, vec, st);
  return launch_xf<float, float, BWD>(a, vec, st);
}

int check(const ait_gated_norm* p) {
  if (!p || p->rows < 0 || p->width <= 0 || p->n_seq < 0 || !(p->eps >= 0.f)) return AIT_EINVAL;
  if ((p->dtype_x != AIT_DTYPE_F32 && p->dtype_x != AIT_DTYPE_BF16) || (p->dtype_f != AIT_DTYPE_F32 && p->dtype_f != AIT_DTYPE_BF16)) return AIT_EINVAL;
  if (p->width > kMaxWidth || (p->dtype_x == AIT_DTYPE_BF16 && p->dtype_f == AIT_DTYPE_F32)) return AIT_EUNSUPPORTED;
  if ((long long)p->rows + 4096 >= (1ll << 31) || (p->width + 255) / 256 * 256ll * p->n_seq >= (1ll << 32)) return AIT_EUNSUPPORTED;
  if (!p->w_post || !p->w_pre) return AIT_EINVAL;
  if (p->rows > 0 && (!p->x || !p->f)) return AIT_EINVAL;
  if (p->x_row < 0 || p->f_row < 0 || p->gate_row < 0) return AIT_EINVAL;
  if (p->cu_seqlens && !p->gate) return AIT_EINVAL;
  return AIT_OK;
}
NormArgs args_of(const ait_gated_norm& p) {
  NormArgs a{};
  a.x = p.x; a.f = p.f; a.gate = p.gate;
  a.w_post = p.w_post; a.b_post = p.b_post; a.w_pre = p.w_pre; a.b_pre = p.b_pre; a.scale = p.scale;
  a.cu = p.cu_seqlens;
  a.x_row = p.x_row; a.f_row = p.f_row; a.g_row = p.gate_row;
  a.rows = p.rows; a.width = p.width; a.layer = p.layer; a.gate_kind = p.gate ? (p.cu_seqlens ? 2 : 1) : 0; a.n_seq = p.n_seq;
  a.eps = p.eps; a.zero_rest = p.zero_rest;
  return a;
}
bool inputs_aligned(const ait_gated_norm& p) {
  const int xs = p.dtype_x == AIT_DTYPE_F32 ? 4 : 2, fs = p.dtype_f == AIT_DTYPE_F32 ? 4 : 2;
  return p.width % 8 == 0 && aligned(p.x, p.x_row, xs) && aligned(p.f, p.f_row, fs) && aligned(p.gate, p.gate_row, fs) &&
         aligned(p.w_post, 0, 4) && aligned(p.b_post, 0, 4) && aligned(p.w_pre, 0, 4) && aligned(p.b_pre, 0, 4) && aligned(p.scale, 0, 4);
}
// units of the backward: about two workgroups' groups a CU, each with a run of rows
void units_of(const ait_gated_norm& p, int& units, int& per) {
  const int groups = p.width <= 512 ? 2048 : p.width <= 1024 ? 1024 : p.width <= 4096 ? 512 : 256;
  per = p.rows > 0 ? (p.rows + groups - 1) / groups : 1;
  units = (p.rows + per - 1) / per;
}
// rows that a workgroup of the backward has side by side (Block<G>::kRows of the launch)
int groups_of(const ait_gated_norm& p, bool vec) { return p.width <= 512 ? 4 : vec && p.width <= 1024 ? 2 : 1; }
int blocks_of(const ait_gated_norm& p, int units, bool vec) { return (units + groups_of(p, vec) - 1) / groups_of(p, vec); }
int parts_of(const ait_gated_norm& p) { return 2 + (p.scale ? 1 : 0) + (p.b_post ? 1 : 0) + (p.b_pre ? 1 : 0); }
}  // namespace

AIT_API int ait_gated_norm_fwd(const ait_gated_norm* p, void* y, long long y_row, void* h, long long h_row, float* stats, void* stream) {
  AIT_TRY_RC(check(p));
  if (p->rows == 0) return AIT_OK;
  if (!y || !h || y_row < p->width || h_row < p->width || (unsigned long long)stats % 16) return AIT_EINVAL;
  NormArgs a = args_of(*p);
  a.y = y; a.h = h; a.y_row = y_row; a.h_row = h_row; a.stats = stats;
  const bool vec = inputs_aligned(*p) && aligned(y, y_row, p->dtype_x == AIT_DTYPE_F32 ? 4 : 2) && aligned(h, h_row, p->dtype_f == AIT_DTYPE_F32 ? 4 : 2);
  return launch<false>(*p, a, vec, ait_stream(stream));
}

AIT_API size_t ait_gated_norm_bwd_workspace_bytes(const ait_gated_norm* p) {
  if (check(p) != AIT_OK) return 0;
  int units, per;
  units_of(*p, units, per);
  return ((size_t)blocks_of(*p, units, false) * parts_of(*p) + (p->cu_seqlens ? (size_t)units + p->n_seq : 0)) * p->width * sizeof(float);
}

AIT_API int ait_gated_norm_bwd(const ait_gated_norm* p, const float* stats, const void* dy, long long dy_row, const void* dh, long long dh_row,
                               void* dx, long long dx_row, void* df, long long df_row, void* d_gate, long long dg_row, float* d_w_post,
                               float* d_w_pre, float* d_scale, float* d_b_post, float* d_b_pre, void* workspace, size_t workspace_bytes,
                               void* stream) {
  AIT_TRY_RC(check(p));
  if (!d_w_post || !d_w_pre || (p->scale && !d_scale) || (p->b_post && !d_b_post) || (p->b_pre && !d_b_pre)) return AIT_EINVAL;
  if (p->gate && (p->rows > 0 || p->cu_seqlens) && (!d_gate || dg_row < p->width)) return AIT_EINVAL;
  if (p->rows > 0 && (!stats || (unsigned long long)stats % 16 || !dy || !dh || !dx || !df || dx_row < p->width || df_row < p->width || dy_row < 0 || dh_row < 0))
    return AIT_EINVAL;
  const size_t need = ait_gated_norm_bwd_workspace_bytes(p);
  if (need && (!workspace || workspace_bytes < need)) return AIT_EWORKSPACE;
  if ((unsigned long long)workspace % 16) return AIT_EINVAL;
  NormArgs a = args_of(*p);
  a.stats = const_cast<float*>(stats);
  a.dy = dy; a.dh = dh; a.dx = dx; a.df = df; a.dgate = d_gate;
  a.dy_row = dy_row; a.dh_row = dh_row; a.dx_row = dx_row; a.df_row = df_row; a.dg_row = dg_row;
  units_of(*p, a.units, a.per);
  a.n_parts = parts_of(*p);
  a.parts = static_cast<float*>(workspace);
  const hipStream_t st = ait_stream(stream);
  const int xs = p->dtype_x == AIT_DTYPE_F32 ? 4 : 2, fs = p->dtype_f == AIT_DTYPE_F32 ? 4 : 2;
  const bool vec = inputs_aligned(*p) && aligned(dy, dy_row, xs) && aligned(dh, dh_row, fs) && aligned(dx, dx_row, xs) && aligned(df, df_row, fs) &&
                   aligned(d_gate, dg_row, fs);
  a.blocks = blocks_of(*p, a.units, vec);
  if (p->rows > 0) AIT_TRY_RC(launch<true>(*p, a, vec, st));
  SumArgs s{a.parts, {d_w_post, d_w_pre, nullptr, nullptr, nullptr}, a.blocks, a.n_parts, p->width};
  int n = 2;
  if (p->scale) s.out[n++] = d_scale;
  if (p->b_post) s.out[n++] = d_b_post;
  if (p->b_pre) s.out[n++] = d_b_pre;
  hipLaunchKernelGGL(gated_norm_sum_kernel, dim3((unsigned)((a.n_parts * p->width + 15) / 16)), dim3(1024), 0, st, s);
  AIT_CHECK_LAUNCH();
  if (a.gate_kind == 2 && p->n_seq > 0) {
    const dim3 grid((unsigned)((p->width + 255) / 256) * (unsigned)p->n_seq);
    if (p->dtype_f == AIT_DTYPE_F32) hipLaunchKernelGGL(gated_norm_gate_kernel<float>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(gated_norm_gate_kernel<__bf16>, grid, dim3(256), 0, st, a);
    AIT_CHECK_LAUNCH();
  }
  return AIT_OK;
}
