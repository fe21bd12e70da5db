// ait_amd/csrc/packed_attn_bwd.hip -- ait_packed_attn_bwd (layout of the products: packed_attn_impl.h).
//
//   P_ij = exp(s_ij - lse_i),  dP_ij = dO_i . v_j,  dS_ij = P_ij (dP_ij - delta_i),  delta_i = dO_i . O_i
//   (rows whose lse is large: P_ij = w_i exp(s_ij - lse_i), w_i = 1 / sum_j exp(s_ij - lse_i), formed by the first pass)
//   dQ_i = scale sum_j dS_ij k_j,   dK_j = scale sum_i dS_ij q_i,   dV_j = sum_i P_ij dO_i,   d table[bucket] = sum dS_ij
//
// Two passes that each own what they write, so no sum goes through atomics on memory and results repeat bit for bit: the first
// has a block of query rows per workgroup and runs over the keys (three products; it also forms delta and the bias's
// gradient), the second a block of keys and runs over the query rows of every head that shares them (four products).  The two
// score products are computed in both: 14 instead of 10 multiplications per pair and value, against f32 sums of dQ through
// memory.  Of 128-wide bf16 heads dK and dV are formed by workgroups of their own (16 multiplications): with both sets of
// accumulators in one, a wave a SIMD is left or registers spill (734 us against 497).
//
// What bounds it: the matrix unit, the exponentials between its products and the clock the chip holds under both.  3 documents of
// 2500 to 4095, 16 heads on 4 of 128, bf16, causal: 228 us over the query rows, 412 over the keys and 17 to join their two parts;
// 4 of 4096 without a mask: 1036 and 1006 TFLOP/s executed, no bank conflicts, matrix unit 63 and 61 % busy at 1.6 GHz.  12
// documents of 100 to 1800, 8 heads of 64: 48 and 63 us, matrix unit 32 and 25 % busy, bank conflicts in 40 and 22 % of the LDS
// cycles (65 us over the query rows with operand loads in branches, each waited for by itself).  Short sequences (300 of 1 to 49
// in f32 with a bias: 61 and 86 us): the trips to memory in front of a workgroup's one tile.
// (Tried: eight waves a workgroup 291 against 257 and 589 against 515; masked and unmasked blocks as two loops: spills, 1694 us;
// bf16 waves that skip the blocks hidden from them, as 64-wide f32 ones do: 62.6 against 60.5; dK's and dV's workgroups in turn
// instead of dK's first: 459 us against 424.)
#include "packed_attn_impl.h"

namespace {
using namespace ait_packed;

constexpr int NW = 4, NT = NW * 64;      // waves of the pass over keys
// The bias's gradient wants the sums of a 32 x 32 block of dS along its diagonals (63 relative positions).  Each query writes its
// column into a row of its own, shifted so that equal relative positions lie below one another, and a lane adds up one of the
// 64 columns: plain writes and reads of shared memory.  (Added up by f32 atomics in shared memory instead, a block costs about
// ten times as much: 207 us against 60 for the pass over sequences of 17 to 1024 tokens with a distance of 128.)  Where the
// tiles leave no room for it (f32 rows of 128 values) the atomics on kHist sums remain.
constexpr int kHist = 64, kSkew = 32 * 64;
constexpr int kRows = 3 * KB * 4;        // bytes of a stage's rows: lse, delta, weight
template <typename T, int D> constexpr bool kSkewed = D == 64 || sizeof(T) == 2;
template <typename T, int D> constexpr int kSums = kSkewed<T, D> ? kSkew : kHist;      // floats of a wave

struct BwdArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* o;
  const void* d_o;
  const void* rest;   // bf16: what rounding took from o, contiguous; or null
  const float* lse;   // [H][total_q] log2 of the rows' sums
  void* dq;
  void* dk;
  void* dv;
  long long qs, qh, ks, kh, vs, vh, os, oh, dos, doh, dqs, dqh, dks, dkh, dvs, dvh;
  Seqs s;
  Bias bias;
  int H, Hk, d, causal, qnumbers, knumbers, splits, stages, kparts;
  float scale;
  float* delta;       // [H][total_q]
  long long plane;    // floats from delta to the weights [H][total_q]: 1 / a row's sum of 2^(score - lse) where lse is large
                      // (`rounded`), else 0, which stands for 1
  float* part_dq;     // [splits][total_q * H][d], not yet scaled: only where splits > 1
  float* part_kv;     // [kparts][dK, dV][total_k][Hk][d], dK not yet scaled: only where kparts > 1
  float* part_table;  // [splits * qnumbers][H][n_buckets]; null: the table's gradient is not wanted
  void* d_table;
};

template <typename T, int D, bool BIAS, int NW>
__global__ __launch_bounds__(NW * 64, D == 64 || sizeof(T) == 2 ? 2 : 1) void packed_bwd_q_kernel(const BwdArgs a) {
  constexpr int NT = NW * 64, BM = NW * 32, NB = D / 32, NCH = D / 16, kTile = Tile<T, D>::kBytes;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int unit = blockIdx.x % a.H, group = a.H / a.Hk, kvh = unit % a.Hk, head = kvh * group + unit / a.Hk;
  const int number = (int)(blockIdx.x / a.H), nb = a.bias.n_buckets, md = a.bias.max_distance;
  float* part = BIAS && a.part_table ? a.part_table + (((size_t)blockIdx.y * a.qnumbers + number) * a.H + head) * nb : nullptr;
  Place place;
  const bool has = find_place<false>(a.s, 1, BM, number, a.qnumbers, a.causal, place);
  const int seq = place.seq, block = place.block, qstart = place.qstart, qlen = place.qlen;
  if (!has || seq == a.s.n_seq) {
    if constexpr (BIAS)
      if (part)
        for (int b = tid; b < nb; b += NT) part[b] = 0.f;
    if (!has || blockIdx.y) return;
    const int r = block * BM + wave * 32 + (lane & 31);
    if (r < qlen)
      for (int e = 8 * h; e < a.d; e += 16) {
        T* p = reinterpret_cast<T*>(a.dq) + (long long)(qstart + r) * a.dqs + (long long)head * a.dqh + e;
        store4(p, 0.f, 0.f, 0.f, 0.f);
        store4(p + 4, 0.f, 0.f, 0.f, 0.f);
      }
    return;
  }
  const int kstart = place.kstart, klen = place.klen, off = klen - qlen, row0 = block * BM + wave * 32, row = row0 + (lane & 31), pos = min(row, qlen - 1);
  const int kmax = a.causal ? min(klen, pos + off + 1) : klen;
  const int wfirst = min(row0, qlen - 1), wlast = min(row0 + 31, qlen - 1);
  const int wsure = a.causal ? min(klen, wfirst + off + 1) : klen, wend = row0 < qlen ? (a.causal ? min(klen, wlast + off + 1) : klen) : 0;
  const int gend = a.causal ? min(klen, min(block * BM + BM, qlen) + off) : klen;
  const int tiles = gend > 0 ? (gend + KB - 1) / KB : 0, per = (tiles + a.splits - 1) / a.splits;
  const int t0 = blockIdx.y * per, t1 = min(tiles, t0 + per);
  const float sc = a.scale * kLog2e;

  const unsigned kstr = (unsigned)(a.ks * sizeof(T)), vstr = (unsigned)(a.vs * sizeof(T)), dby = a.d * sizeof(T);
  Loader<T, D, NT> lk, lv;
  lk.init(tid, kstr, dby);
  lv.init(tid, vstr, dby);
  const T* kb = reinterpret_cast<const T*>(a.k) + (long long)kstart * a.ks + (long long)kvh * a.kh;
  const T* vb = reinterpret_cast<const T*>(a.v) + (long long)kstart * a.vs + (long long)kvh * a.vh;
  const unsigned lds0 = lds_addr(lds);
  auto fetch = [&](int t, int stage) {
    const long long r = (long long)t * KB;
    lk.load(kb + r * a.ks, klen - r, kstr, dby, lds0 + stage * 2 * kTile, wave);
    lv.load(vb + r * a.vs, klen - r, vstr, dby, lds0 + stage * 2 * kTile + kTile, wave);
  };
  if (t0 < t1) fetch(t0, 0);

  Frag<T> qf[NCH], gf[NCH];
  float delta = 0.f, l2, weight = 0.f;
  bool large;      // a row of this wave's has scores so large that its logarithm does not hold its sum
  {
    const long long at = qstart + pos;
    const T* qr = reinterpret_cast<const T*>(a.q) + at * a.qs + (long long)head * a.qh;
    const T* gr = reinterpret_cast<const T*>(a.d_o) + at * a.dos + (long long)head * a.doh;
    const T* orow = reinterpret_cast<const T*>(a.o) + at * a.os + (long long)head * a.oh;
    Frag<T> of[NCH], rf[NCH];
    const bool there = row < qlen, rest = sizeof(T) == 2 && a.rest;
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      gf[c] = global_frag<T>(gr, 16 * c + 8 * h, a.d, there);
      of[c] = global_frag<T>(orow, 16 * c + 8 * h, a.d, there);
      qf[c] = global_frag<T>(qr, 16 * c + 8 * h, a.d, there);
    }
    l2 = a.lse[(long long)head * a.s.total_q + at];
    if (rest) {
      const T* rr = reinterpret_cast<const T*>(a.rest) + (at * a.H + head) * a.d;
#pragma unroll
      for (int c = 0; c < NCH; c++) rf[c] = global_frag<T>(rr, 16 * c + 8 * h, a.d, there);
    }
#pragma unroll
    for (int c = 0; c < NCH; c++)
#pragma unroll
      for (int e = 0; e < 8; e++) delta = __builtin_fmaf((float)gf[c][e], (float)of[c][e], delta);
    if (rest) {
#pragma unroll
      for (int c = 0; c < NCH; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) delta = __builtin_fmaf((float)gf[c][e], (float)rf[c][e], delta);
    }
    delta = column_sum(delta);
    if (row < qlen && h == 0 && blockIdx.y == 0) a.delta[(long long)head * a.s.total_q + at] = delta;
    large = __any(row < qlen && rounded(l2));
  }
  float* bl = reinterpret_cast<float*>(lds + 2 * a.stages * kTile);      // the head's bias, then per wave: a block's sums by
  float* hist = bl + (BIAS ? bias_row(md) : 0) + wave * (kSums<T, D> + nb);      // relative position, and the sums by bucket
  float* acc_b = hist + kSums<T, D>;
  float far_lo = 0.f, far_hi = 0.f, sum_lo = 0.f, sum_hi = 0.f;
  if constexpr (BIAS) {
    fill_bias<NT>(a.bias, a.H, head, 1, bl, tid);
    if (part) {
      for (int x = lane; x < kSums<T, D> + nb; x += 64) hist[x] = 0.f;
    }
    __syncthreads();
    far_lo = bl[0];
    far_hi = bl[2 * (md + kPad)];
  }
  if (large) {
    // lse = maximum + log2(sum) is one f32, which beyond 2^24 holds nothing of the sum and beyond 2^12 half its digits: the sum over
    // all of the row's keys is formed again, of 2^(score - lse).  (By each wave from memory, without the tiles: hardly a row needs
    // it; where none does, this path costs the passes 0 to 3 %, 64-wide f32 heads over the keys 6.)
    float sum = 0.f;
    for (int k0 = 0; k0 < wend; k0 += 32) {
      f32x16 s;
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = 0.f;
      const bool there = k0 + (lane & 31) < klen;
      const T* kr = kb + (there ? k0 + (lane & 31) : 0) * a.ks;
#pragma unroll
      for (int c = 0; c < NCH; c++) s = mma(global_frag<T>(kr, 16 * c + 8 * h, a.d, there), qf[c], s);
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int j = k0 + 8 * (r >> 2) + 4 * h + (r & 3);
        const float b = BIAS ? bl[min(max(j - pos - off, -md), md) + md + kPad] : 0.f;
        const float e = fast_exp2(__builtin_fmaf(s[r], sc, b) - l2);
        sum += j < kmax ? e : 0.f;
      }
    }
    sum = column_sum(sum);
    if (row < qlen && rounded(l2) && sum > 0.f) weight = 1.f / sum;
  }
  if (row < qlen && h == 0 && blockIdx.y == 0) a.delta[a.plane + (long long)head * a.s.total_q + qstart + pos] = weight;
  if (weight == 0.f) weight = 1.f;
  delta *= weight;
  // (a query that sees one key has no gradient of its scores: exactly zero, not the rounding of dP - delta)
  if (row >= qlen || kmax <= 1) l2 = -kNegInf;

  const int rb = row_base<T, D>(lane), cb = col_base<T, D>(lane);
  f32x16 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int r = 0; r < 16; r++) acc[b][r] = 0.f;

  for (int t = t0; t < t1; t++) {
    const int stage = (t - t0) & (a.stages - 1), k0 = t * KB;
    loads_done_barrier();
    if (a.stages == 2 && t + 1 < t1) fetch(t + 1, stage ^ 1);
    if (k0 < wend) {
    const unsigned char* kt = lds + stage * 2 * kTile;
    const unsigned char* vt = kt + kTile;
    bool near = false, right = false;
    if constexpr (BIAS) {
      right = k0 - (wlast + off) >= md;
      near = !right && k0 + KB - 1 - (wfirst + off) > -md;
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
      if (sizeof(T) == 4 && k0 + 32 * x >= wend) continue;
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        s = mma(row_frag<T, D>(kt, rb, x, c), qf[c], s);
        dp = mma(row_frag<T, D>(vt, rb, x, c), gf[c], dp);
      }
      read_ahead<T, 2 * NCH, 1, 4>();
      const FirstCols<T, D> first(kt, cb, x);
      if (BIAS && (near || large)) {      // (scores rounded as the forward has them; a far block's bias from the outermost values)
        const float* p = bl + (near ? k0 + 32 * x + 4 * h - (pos + off) + md + kPad : right ? bias_row(md) - 32 : 0);
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = __builtin_fmaf(s[r], sc, p[8 * (r >> 2) + (r & 3)]) - l2;
      } else {
        float f = sc;
        if (!BIAS && large) {
#pragma unroll
          for (int r = 0; r < 16; r++) s[r] *= sc;
          f = 1.f;
        }
        const float sub = (BIAS ? (right ? far_hi : far_lo) : 0.f) - l2;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = __builtin_fmaf(s[r], f, sub);
      }
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = fast_exp2(s[r]) * __builtin_fmaf(dp[r], weight, -delta);
      if (k0 + KB > wsure) {
        const int lim = kmax - k0 - 32 * x - 4 * h;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 8 * (r >> 2) + (r & 3) < lim ? s[r] : 0.f;
      }
      if constexpr (BIAS) {
        if (part) {
          if (near) {
            // by key - query + 31 over the block
            float u = 0.f;
            if constexpr (kSkewed<T, D>) {
              float* p = hist + (lane & 31) * 63 + 31 + 4 * h;
#pragma unroll
              for (int r = 0; r < 16; r++) p[8 * (r >> 2) + (r & 3)] = s[r];
              asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // (this wave's own memory, in order: no barrier)
#pragma unroll
              for (int c = 0; c < 32; c++) u += hist[c * 64 + lane];
            } else {
              float* p = hist + 31 - (lane & 31) + 4 * h;
#pragma unroll
              for (int r = 0; r < 16; r++)
                __hip_atomic_fetch_add(p + 8 * (r >> 2) + (r & 3), s[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
              asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
              u = hist[lane];
              hist[lane] = 0.f;
            }
            __hip_atomic_fetch_add(acc_b + bucket(a.bias, k0 + 32 * x - (row0 + 31 + off) + lane), u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          } else {
            float u = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r++) u += s[r];
            sum_lo += right ? 0.f : u;
            sum_hi += right ? u : 0.f;
          }
        }
      }
#pragma unroll
      for (int cc = 0; cc < 2; cc++) {
        const Frag<T> df = acc_frag<T>(s, cc);
#pragma unroll
        for (int b = 0; b < NB; b++) acc[b] = mma(first.get(kt, cb, x, cc, b), df, acc[b]);
      }
      read_ahead<T, 2 * NB, 2, 4, true>();
    }
    }
    if (a.stages == 1 && t + 1 < t1) {
      loads_done_barrier();
      fetch(t + 1, 0);
    }
  }

  if (row < qlen && a.splits > 1) {
    float* p = a.part_dq + (((long long)blockIdx.y * a.s.total_q + qstart + pos) * a.H + head) * a.d;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int dd = 32 * b + 8 * i + 4 * h;
        if (dd < a.d) store4(p + dd, acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]);
      }
  } else if (row < qlen) {
    T* p = reinterpret_cast<T*>(a.dq) + (long long)(qstart + pos) * a.dqs + (long long)head * a.dqh;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int dd = 32 * b + 8 * i + 4 * h;
        if (dd < a.d)
          store4(p + dd, acc[b][4 * i] * a.scale, acc[b][4 * i + 1] * a.scale, acc[b][4 * i + 2] * a.scale, acc[b][4 * i + 3] * a.scale);
      }
  }
  if constexpr (BIAS) {
    if (part) {
      sum_lo = wave_sum(sum_lo);
      sum_hi = wave_sum(sum_hi);
      if (lane == 0) {
        acc_b[bucket(a.bias, -md)] += sum_lo;
        acc_b[bucket(a.bias, md)] += sum_hi;
      }
      __syncthreads();
      const float* w0 = bl + bias_row(md) + kSums<T, D>;
      for (int b = tid; b < nb; b += NT) {
        float u = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) u += w0[w * (kSums<T, D> + nb) + b];
        part[b] = u;
      }
    }
  }
}

// the parts of a row's dQ in their order: one wave per (query row, head)
template <typename T>
__global__ __launch_bounds__(256) void packed_dq_join_kernel(const BwdArgs a) {
  const int dd = (threadIdx.x & 63) * 4;
  const long long n = (long long)a.s.total_q * a.H, id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (id >= n || dd >= a.d) return;
  const int at = (int)(id / a.H), head = (int)(id - (long long)at * a.H);
  if (at < clamped(a.s.cu_q, 0, a.s.total_q) || at >= clamped(a.s.cu_q, a.s.n_seq, a.s.total_q)) return;
  f32x4 u = *reinterpret_cast<const f32x4*>(a.part_dq + id * a.d + dd);
  for (int s = 1; s < a.splits; s++) u += *reinterpret_cast<const f32x4*>(a.part_dq + (s * n + id) * a.d + dd);
  u *= a.scale;
  store4(reinterpret_cast<T*>(a.dq) + (long long)at * a.dqs + (long long)head * a.dqh + dd, u[0], u[1], u[2], u[3]);
}

// d table[b][head]: the workgroups' parts in a fixed order
__global__ __launch_bounds__(256) void packed_table_kernel(const BwdArgs a) {
  __shared__ float sums[256];
  const int head = blockIdx.x, b = blockIdx.y * 16 + (threadIdx.x & 15), nb = a.bias.n_buckets;
  float u = 0.f;
  if (b < nb)
    for (int n = threadIdx.x >> 4; n < a.qnumbers * a.splits; n += 16) u += a.part_table[((size_t)n * a.H + head) * nb + b];
  sums[threadIdx.x] = u;
  __syncthreads();
  if (threadIdx.x < 16 && b < nb) {
    u = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) u += sums[threadIdx.x + 16 * i];
    const size_t at = (size_t)b * a.H + head;
    if (a.bias.bf16) static_cast<__bf16*>(a.d_table)[at] = (__bf16)u;
    else static_cast<float*>(a.d_table)[at] = u;
  }
}

// PARTS: 3 = dK and dV in one pass; 1 / 2: workgroups that form dV alone and workgroups that form dK alone
// XH: 2 = the waves of a pair have the same 32 keys and half of a tile's queries each; 1 = every wave has keys of its own
template <typename T, int D, bool BIAS, int PART, int XH>
__device__ __forceinline__ void bwd_kv(const BwdArgs& a, const int index, unsigned char* lds) {
  constexpr bool DK = PART & 2, DV = PART & 1;
  constexpr int NB = D / 32, NCH = D / 16, kTile = Tile<T, D>::kBytes, BN = NW / XH * 32;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int kvh = index % a.Hk, group = a.H / a.Hk, part = index / a.Hk % a.kparts, number = index / a.Hk / a.kparts, md = a.bias.max_distance;
  Place place;
  if (!find_place<true>(a.s, 1, BN, number, 0, a.causal, place)) return;
  const int block = place.block, kstart = place.kstart, klen = place.klen, kroom = place.kroom;
  // (with a causal mask and more queries than keys the first ones see none: they are left out, whatever they and their dO hold)
  const int blind = a.causal ? max(0, place.qlen - klen) : 0, qstart = place.qstart + blind, qlen = place.qlen - blind;
  const int kc = wave % (NW / XH), xh = wave / (NW / XH), key0 = block * BN + kc * 32, key = key0 + (lane & 31), off = klen - qlen;
  // query rows that see a key j: positions >= j - off with a causal mask
  const int gfirst = a.causal ? max(0, block * BN - off) : 0;
  const int wsure = a.causal ? max(0, min(key0 + 31, klen - 1) - off) : 0;          // from here on every key of the wave is seen
  const int t0 = gfirst / KB, tq = block * BN < klen ? max(0, (qlen + KB - 1) / KB - t0) : 0, all = tq * group;
  // this part's share of the turns, which run over the query tiles of one head after another's
  const int first = (int)((long long)all * part / a.kparts), total = (int)((long long)all * (part + 1) / a.kparts) - first;
  int g = total > 0 ? first / tq : 0, t = t0 + first - g * tq;

  const unsigned qstr = (unsigned)(a.qs * sizeof(T)), gstr = (unsigned)(a.dos * sizeof(T)), dby = a.d * sizeof(T);
  Loader<T, D, NT> lq, lg;
  lq.init(tid, qstr, dby);
  lg.init(tid, gstr, dby);
  const unsigned lds0 = lds_addr(lds), rows0 = lds0 + 4 * kTile;      // behind the tiles: two stages of lse | delta | weight of KB rows
  // the next tile to load: its head, number, rows and rows left (pointers run on: a head's tiles lie one behind another)
  const T *pq = nullptr, *pg = nullptr;
  const float* ps = nullptr;
  int nt = t, nhead = kvh * group + g, left = 0;
  auto to_head = [&]() {
    const long long r = qstart + (long long)nt * KB;
    pq = reinterpret_cast<const T*>(a.q) + r * a.qs + (long long)nhead * a.qh;
    pg = reinterpret_cast<const T*>(a.d_o) + r * a.dos + (long long)nhead * a.doh;
    ps = (wave ? a.delta + (wave == 2 ? a.plane : 0) : a.lse) + (long long)nhead * a.s.total_q + r;
    left = qlen - nt * KB;
  };
  auto fetch = [&](int stage) {
    lq.load(pq, left, qstr, dby, lds0 + stage * 2 * kTile, wave);
    lg.load(pg, left, gstr, dby, lds0 + stage * 2 * kTile + kTile, wave);
    if (wave < 3) {
      const i32x4 rsrc = tile_rsrc(ps, min(KB, left) * 4);
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds"
                   : : "v"(lane * 4), "s"(rsrc), "s"(rows0 + stage * kRows + wave * 256) : "m0", "memory");
    }
    pq += KB * a.qs;
    pg += KB * a.dos;
    ps += KB;
    left -= KB;
    if (++nt == t0 + tq) {
      nt = t0;
      nhead++;
      to_head();
    }
  };
  const float* bl = reinterpret_cast<const float*>(lds + 4 * kTile + 2 * kRows);
  if (total > 0) {
    to_head();
    fetch(0);
  }

  Frag<T> kf[NCH], vf[NCH];
  {
    const bool there = key < klen;
    const long long at = kstart + (there ? key : 0);
    const T* kr = reinterpret_cast<const T*>(a.k) + at * a.ks + (long long)kvh * a.kh;
    const T* vr = reinterpret_cast<const T*>(a.v) + at * a.vs + (long long)kvh * a.vh;
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      kf[c] = global_frag<T>(kr, 16 * c + 8 * h, a.d, there);
      if (DK) vf[c] = global_frag<T>(vr, 16 * c + 8 * h, a.d, there);
    }
  }
  const int rb = row_base<T, D>(lane), cb = col_base<T, D>(lane);
  const float sc = a.scale * kLog2e;
  f32x16 ak[NB], av[NB];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int r = 0; r < 16; r++) ak[b][r] = av[b][r] = 0.f;
  float far_lo = 0.f, far_hi = 0.f;

  for (int it = 0; it < total; it++) {
    const int stage = it & 1, r0 = t * KB;
    if constexpr (BIAS) {
      if (it == 0 || t == t0) {      // another head: its bias
        __syncthreads();
        fill_bias<NT>(a.bias, a.H, kvh * group + g, 1, const_cast<float*>(bl), tid);
        __syncthreads();
        far_lo = bl[0];
        far_hi = bl[2 * (md + kPad)];
      }
    }
    loads_done_barrier();
    if (it + 1 < total) fetch(stage ^ 1);
    if (++t == t0 + tq) { t = t0; g++; }
    // a block that is hidden from this wave (f32: 8192 cycles of the matrix unit; 300 sequences of 1 to 49: 86 us, 89 without)
    if (D == 64 && sizeof(T) == 4 && (key0 >= klen || r0 + 32 * xh >= qlen || (a.causal && r0 + 32 * xh + 31 < key0 - off))) continue;
    const unsigned char* qt = lds + stage * 2 * kTile;
    const unsigned char* gt = qt + kTile;
    const float* rows = reinterpret_cast<const float*>(lds + 4 * kTile + stage * kRows);
    const float weights = rows[128 + lane];
    const int last = min(r0 + KB, qlen) - 1;
    bool near = false, right = false;
    if constexpr (BIAS) {
      right = key0 - (last + off) >= md;
      near = !right && key0 + 31 - (r0 + off) > -md;
    }
#pragma unroll
    for (int xx = 0; xx < 2 / XH; xx++) {
      const int x = XH == 1 ? xx : xh;
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        s = mma(row_frag<T, D>(qt, rb, x, c), kf[c], s);
        if (DK) dp = mma(row_frag<T, D>(gt, rb, x, c), vf[c], dp);
      }
      read_ahead<T, (DK ? 2 : 1) * NCH, 1, 4>();
      const FirstCols<T, D> first(DV ? gt : qt, cb, x);
      const float far = BIAS ? (right ? far_hi : far_lo) : 0.f;
      const float* p = bl + (key - (r0 + 32 * x + 4 * h + off) + md + kPad);
      // (rows of large scores: see the pass over query rows.  With a bias every score is rounded, at the same number of operations)
      const bool large = __any(weights != 0.f);
      float f = sc;
      if (!BIAS && large) {
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] *= sc;
        f = 1.f;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const f32x4 l2 = *reinterpret_cast<const f32x4*>(rows + 32 * x + 8 * i + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          float e;
          if constexpr (BIAS) e = __builtin_fmaf(s[4 * i + j], sc, near ? p[-8 * i - j] : far) - l2[j];
          else e = __builtin_fmaf(s[4 * i + j], f, -l2[j]);
          s[4 * i + j] = fast_exp2(e);
        }
      }
      if constexpr (DK) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const f32x4 dl = *reinterpret_cast<const f32x4*>(rows + 64 + 32 * x + 8 * i + 4 * h);
#pragma unroll
          for (int j = 0; j < 4; j++) dp[4 * i + j] -= dl[j];
        }
      }
      // a row's first positions do not see the wave's last keys; rows behind the sequence and keys behind k_len are zeros in Q,
      // dO, K and V, but their "probabilities" are not; a query that sees one key has no gradient of its scores
      if (large || r0 < wsure || r0 + KB > qlen || key0 + 32 > klen) {
        const int from = a.causal ? key - off : 0, one = klen <= 1 ? qlen : a.causal ? -off : -1;
        if (large) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(rows + 128 + 32 * x + 8 * i + 4 * h);
#pragma unroll
            for (int j = 0; j < 4; j++) s[4 * i + j] *= w[j] == 0.f ? 1.f : w[j];
          }
        }
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int y = r0 + 32 * x + 8 * (r >> 2) + 4 * h + (r & 3);
          const bool seen = y >= from && y < qlen && key < klen;
          if (!seen) s[r] = 0.f;
          if (!seen || y <= one) dp[r] = 0.f;
        }
      }
      if constexpr (DV) {
#pragma unroll
      for (int cc = 0; cc < 2; cc++) {
        const Frag<T> pf = acc_frag<T>(s, cc);
#pragma unroll
        for (int b = 0; b < NB; b++) av[b] = mma(first.get(gt, cb, x, cc, b), pf, av[b]);
      }
      read_ahead<T, 2 * NB, 2, 4, true>();
      }
      if constexpr (DK) {
#pragma unroll
      for (int r = 0; r < 16; r++) s[r] *= dp[r];
#pragma unroll
      for (int cc = 0; cc < 2; cc++) {
        const Frag<T> df = acc_frag<T>(s, cc);
#pragma unroll
        for (int b = 0; b < NB; b++) ak[b] = mma(DV ? col_frag<T, D>(qt, cb, x, cc, b) : first.get(qt, cb, x, cc, b), df, ak[b]);
      }
      read_ahead<T, 2 * NB, 2, 4, !DV>();
      }
    }
  }

  if constexpr (XH == 2) {      // the two waves of a block of keys had half of the query rows each
    float* p = reinterpret_cast<float*>(lds) + kc * NB * 16 * 64 + lane;
#pragma unroll
    for (int g = 0; g < 2; g++) {
      if (!(g ? DV : DK)) continue;
      f32x16* t = g ? av : ak;
      loads_done_barrier();
      if (xh == 1) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int r = 0; r < 16; r++) p[(b * 16 + r) * 64] = t[b][r];
      }
      loads_done_barrier();
      if (xh == 0) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int r = 0; r < 16; r++) t[b][r] += p[(b * 16 + r) * 64];
      }
    }
    if (xh == 1) return;
  }
  if (key >= kroom) return;
  if (a.kparts > 1) {
    float* p = a.part_kv + (((long long)part * 2 * a.s.total_k + kstart + key) * a.Hk + kvh) * a.d;
    const long long dv = (long long)a.s.total_k * a.Hk * a.d;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int dd = 32 * b + 8 * i + 4 * h;
        if (dd < a.d) {
          if (DK) store4(p + dd, ak[b][4 * i], ak[b][4 * i + 1], ak[b][4 * i + 2], ak[b][4 * i + 3]);
          if (DV) store4(p + dv + dd, av[b][4 * i], av[b][4 * i + 1], av[b][4 * i + 2], av[b][4 * i + 3]);
        }
      }
    return;
  }
  T* pk = reinterpret_cast<T*>(a.dk) + (long long)(kstart + key) * a.dks + (long long)kvh * a.dkh;
  T* pv = reinterpret_cast<T*>(a.dv) + (long long)(kstart + key) * a.dvs + (long long)kvh * a.dvh;
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int dd = 32 * b + 8 * i + 4 * h;
      if (dd < a.d) {
        if (DK) store4(pk + dd, ak[b][4 * i] * a.scale, ak[b][4 * i + 1] * a.scale, ak[b][4 * i + 2] * a.scale, ak[b][4 * i + 3] * a.scale);
        if (DV) store4(pv + dd, av[b][4 * i], av[b][4 * i + 1], av[b][4 * i + 2], av[b][4 * i + 3]);
      }
    }
}

// SPLIT: dK and dV by workgroups of their own (the keys' gradients, which have three products to dV's two, first)
template <typename T, int D, bool BIAS, bool SPLIT, int XH>
__global__ __launch_bounds__(NT, D == 128 && sizeof(T) == 4 ? 1 : 2) void packed_bwd_kv_kernel(const BwdArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  if constexpr (SPLIT) {
    const int n = a.knumbers * a.Hk * a.kparts;
    if ((int)blockIdx.x < n) bwd_kv<T, D, BIAS, 2, XH>(a, blockIdx.x, lds);
    else bwd_kv<T, D, BIAS, 1, XH>(a, blockIdx.x - n, lds);
  } else {
    bwd_kv<T, D, BIAS, 3, XH>(a, blockIdx.x, lds);
  }
}

// the parts of dK and dV in their order: a thread has four values of a row and head
template <typename T>
__global__ __launch_bounds__(256) void packed_kv_join_kernel(const BwdArgs a) {
  const int vecs = a.d / 4;
  const long long n = (long long)a.s.total_k * a.Hk * vecs, id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= n) return;
  const long long rh = id / vecs;
  const int dd = (int)(id - rh * vecs) * 4, row = (int)(rh / a.Hk), head = (int)(rh - (long long)row * a.Hk);
  if (row < clamped(a.s.cu_k, 0, a.s.total_k) || (row >= clamped(a.s.cu_k, a.s.n_seq, a.s.total_k) && !a.s.rest)) return;
  f32x4 k = {0.f, 0.f, 0.f, 0.f}, v = k;
  for (int s = 0; s < a.kparts; s++) {
    const float* p = a.part_kv + (2 * s * n + id) * 4;
    k += *reinterpret_cast<const f32x4*>(p);
    v += *reinterpret_cast<const f32x4*>(p + n * 4);
  }
  k *= a.scale;
  store4(reinterpret_cast<T*>(a.dk) + (long long)row * a.dks + (long long)head * a.dkh + dd, k[0], k[1], k[2], k[3]);
  store4(reinterpret_cast<T*>(a.dv) + (long long)row * a.dvs + (long long)head * a.dvh + dd, v[0], v[1], v[2], v[3]);
}
template <typename K>
int set_lds(K kernel, int bytes) {
  if (bytes <= 65536) return AIT_OK;
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess ? AIT_OK : AIT_ELAUNCH;
}
// what the sizes decide for the pass over query rows: waves of a workgroup, parts of the key axis, tiles in flight
struct Shape { int nw, splits, stages, kwide, kparts; };
Shape shape_of(const ait_packed_attn& p) {
  const long long max_q = p.max_q > 0 ? p.max_q : p.total_q, max_k = p.max_k > 0 ? p.max_k : p.total_k;
  Shape r;
  // two waves where a sequence fits them (1 to 49 queries in f32: 61 us, 82 in four), and one tile's memory where there is one
  // (61 us, 121 with room for two)
  r.nw = max_q <= 64 ? 2 : 4;
  r.stages = max_k <= KB ? 1 : 2;
  // (cut as in the forward: 64 queries against 2394 keys take 46 us and 6 to join)
  const long long blocks = p.total_q / (r.nw * 32) > p.n_seq ? p.total_q / (r.nw * 32) : p.n_seq;
  const long long wgs = (blocks > 0 ? blocks : 1) * p.heads, tiles = (max_k + KB - 1) / KB;
  long long s = 512 / wgs;
  if (s > tiles / 2) s = tiles / 2;
  if (s > 64) s = 64;
  r.splits = s < 1 ? 1 : (int)s;
  // Keys: 128 a workgroup for 128-wide bf16 heads, whose products load twice as much for 64 (4 documents of 4096, 16 heads on 4,
  // no mask: 1404 us against 1845; 16 causal ones of 1000: 260 against 284, 64 of 200: 124 against 120); with a bias it would
  // spill, and 64-wide heads gain nothing (documents of 100 to 1800: 61 us against 63; with a bias 70 against 63).
  // Few blocks are cut along the queries, eight tiles at least to a part: of the wide ones, whose longest would outlast the
  // launch under a causal mask, as many parts as make two rounds (3 documents of 2500 to 4095: 409 us in two and 22 to join them,
  // 566 uncut; one of 4096: 201 + 13 in four, 504 uncut), of the others as many as fit at once (one of 2048, 8 heads of 64:
  // 24 + 5 us in two, 31 uncut; two of 512 would lose, 13.5 + 4 against 12.9: eight tiles are all they have)
  const bool split = p.dtype == AIT_DTYPE_BF16 && p.d > 64;
  r.kwide = split && !p.bias_table && max_k >= 512;
  const int bn = r.kwide ? NW * 32 : NW * 16;
  const long long kblocks = p.total_k / bn > p.n_seq ? p.total_k / bn : p.n_seq, turns = (max_q + KB - 1) / KB * (p.heads / p.kv_heads);
  const long long kw = (kblocks > 0 ? kblocks : 1) * p.kv_heads * (split ? 2 : 1);
  s = r.kwide ? (1024 + kw - 1) / kw : 512 / kw;
  if (s > turns / 8) s = turns / 8;
  if (s > 16) s = 16;
  r.kparts = s < 1 ? 1 : (int)s;
  return r;
}

template <typename T, int D, bool BIAS, int XH>
int launch_kv(BwdArgs a, hipStream_t st) {
  const int bytes = 4 * Tile<T, D>::kBytes + 2 * kRows + (BIAS ? bias_row(a.bias.max_distance) * 4 : 0);
  constexpr bool kSplit = D == 128 && sizeof(T) == 2;
  const long long numbers = block_numbers(a.s.total_k, 1, NW / XH * 32, a.s.n_seq, a.s.rest), wgs = numbers * a.Hk * a.kparts * (kSplit ? 2 : 1);
  const long long vecs = (long long)a.s.total_k * a.Hk * (a.d / 4);
  if (!launchable(wgs, NT) || (a.kparts > 1 && !launchable((vecs + 255) / 256, 256))) return AIT_EUNSUPPORTED;
  a.knumbers = (int)numbers;
  AIT_TRY_RC((set_lds(packed_bwd_kv_kernel<T, D, BIAS, kSplit, XH>, bytes)));
  if (a.s.total_k == 0) return AIT_OK;
  hipLaunchKernelGGL((packed_bwd_kv_kernel<T, D, BIAS, kSplit, XH>), dim3((unsigned)wgs), dim3(NT), bytes, st, a);
  AIT_CHECK_LAUNCH();
  if (a.kparts > 1) {
    hipLaunchKernelGGL(packed_kv_join_kernel<T>, dim3((unsigned)((vecs + 255) / 256)), dim3(256), 0, st, a);
    AIT_CHECK_LAUNCH();
  }
  return AIT_OK;
}
template <typename T, int D, bool BIAS, int NWQ>
int launch_q(const BwdArgs& a, hipStream_t st) {
  const int bytes = 2 * a.stages * Tile<T, D>::kBytes + (BIAS ? (bias_row(a.bias.max_distance) + NWQ * (kSums<T, D> + a.bias.n_buckets)) * 4 : 0);
  if (!launchable((long long)a.qnumbers * a.H, NWQ * 64) || (a.splits > 1 && !launchable(((long long)a.s.total_q * a.H + 3) / 4, 256)))
    return AIT_EUNSUPPORTED;
  AIT_TRY_RC((set_lds(packed_bwd_q_kernel<T, D, BIAS, NWQ>, bytes)));
  if (a.s.total_q == 0) return AIT_OK;
  hipLaunchKernelGGL((packed_bwd_q_kernel<T, D, BIAS, NWQ>), dim3((unsigned)(a.qnumbers * a.H), (unsigned)a.splits), dim3(NWQ * 64), bytes, st, a);
  AIT_CHECK_LAUNCH();
  if (a.splits > 1) {
    hipLaunchKernelGGL(packed_dq_join_kernel<T>, dim3((unsigned)(((long long)a.s.total_q * a.H + 3) / 4)), dim3(256), 0, st, a);
    AIT_CHECK_LAUNCH();
  }
  return AIT_OK;
}
template <typename T, int D, bool BIAS>
int launch_b(const BwdArgs& a, const Shape& sh, hipStream_t st) {
  AIT_TRY_RC((sh.nw == 2 ? launch_q<T, D, BIAS, 2>(a, st) : launch_q<T, D, BIAS, 4>(a, st)));
  if constexpr (D == 128 && sizeof(T) == 2 && !BIAS)
    if (sh.kwide) return launch_kv<T, D, BIAS, 1>(a, st);
  return launch_kv<T, D, BIAS, 2>(a, st);
}
template <typename T, int D>
int launch_d(const BwdArgs& a, const Shape& sh, hipStream_t st) {
  return a.bias.table ? launch_b<T, D, true>(a, sh, st) : launch_b<T, D, false>(a, sh, st);
}
template <typename T>
int launch_t(const BwdArgs& a, const Shape& sh, hipStream_t st) {
  return a.d <= 64 ? launch_d<T, 64>(a, sh, st) : launch_d<T, 128>(a, sh, st);
}
long long q_numbers(const ait_packed_attn& p, const Shape& s) { return block_numbers(p.total_q, 1, s.nw * 32, p.n_seq, p.zero_rest ? 1 : 0); }
// floats: delta and weight, the parts of dQ, those of dK and dV, those of the table's gradient
size_t rows_floats(const ait_packed_attn& p) { return ((size_t)p.heads * p.total_q + 3) / 4 * 4; }
size_t dq_floats(const ait_packed_attn& p, const Shape& s) { return s.splits > 1 ? (size_t)s.splits * p.total_q * p.heads * p.d : 0; }
size_t kv_floats(const ait_packed_attn& p, const Shape& s) { return s.kparts > 1 ? (size_t)s.kparts * 2 * p.total_k * p.kv_heads * p.d : 0; }
}  // namespace

AIT_API size_t ait_packed_attn_bwd_workspace_bytes(const ait_packed_attn* p) {
  if (ait_packed::check(p) != AIT_OK) return 0;
  const Shape s = shape_of(*p);
  size_t n = 2 * rows_floats(*p) + dq_floats(*p, s) + kv_floats(*p, s);
  if (p->bias_table) n += (size_t)s.splits * q_numbers(*p, s) * p->heads * p->n_buckets;
  return n * sizeof(float);
}

AIT_API int ait_packed_attn_bwd(const ait_packed_attn* p, const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                                long long k_head, const void* v, long long v_row, long long v_head, const void* o, long long o_row,
                                long long o_head, const void* o_rest, const void* d_o, long long do_row, long long do_head, const float* lse, void* dq,
                                long long dq_row, long long dq_head, void* dk, long long dk_row, long long dk_head, void* dv,
                                long long dv_row, long long dv_head, void* d_table, void* workspace, size_t workspace_bytes, void* stream) {
  AIT_TRY_RC(ait_packed::check(p));
  if (p->n_seq == 0 || (p->total_q == 0 && p->total_k == 0)) return AIT_OK;
  if (!p->cu_q || !p->cu_k) return AIT_EINVAL;
  AIT_TRY_RC(ait_packed::check_strides(p, q, q_row, q_head, p->total_q));
  AIT_TRY_RC(ait_packed::check_strides(p, o, o_row, o_head, p->total_q));
  AIT_TRY_RC(ait_packed::check_strides(p, d_o, do_row, do_head, p->total_q));
  AIT_TRY_RC(ait_packed::check_strides(p, dq, dq_row, dq_head, p->total_q));
  AIT_TRY_RC(ait_packed::check_strides(p, k, k_row, k_head, p->total_k));
  AIT_TRY_RC(ait_packed::check_strides(p, v, v_row, v_head, p->total_k));
  AIT_TRY_RC(ait_packed::check_strides(p, dk, dk_row, dk_head, p->total_k));
  AIT_TRY_RC(ait_packed::check_strides(p, dv, dv_row, dv_head, p->total_k));
  if (p->total_q > 0 && !lse) return AIT_EINVAL;
  if ((unsigned long long)o_rest % 16) return AIT_EUNSUPPORTED;
  const size_t need = ait_packed_attn_bwd_workspace_bytes(p);
  if (!workspace || workspace_bytes < need) return AIT_EWORKSPACE;
  if ((unsigned long long)workspace % 16) return AIT_EINVAL;
  const Shape sh = shape_of(*p);
  BwdArgs a{q, k, v, o, d_o, p->dtype == AIT_DTYPE_BF16 ? o_rest : nullptr, lse, dq, dk, dv, q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head, do_row, do_head,
            dq_row, dq_head, dk_row, dk_head, dv_row, dv_head,
            {p->cu_q, p->cu_k, p->k_len, p->n_seq, p->total_q, p->total_k, p->zero_rest ? 1 : 0, sh.splits == 1 && ait_packed::order_blocks(*p)},
            {p->bias_table, p->bucket_of, p->n_buckets, p->max_distance, p->table_dtype == AIT_DTYPE_BF16},
            p->heads, p->kv_heads, p->d, p->causal, (int)q_numbers(*p, sh), 0, sh.splits, sh.stages, sh.kparts, p->scale,
            static_cast<float*>(workspace), (long long)rows_floats(*p), static_cast<float*>(workspace) + 2 * rows_floats(*p), nullptr, nullptr, d_table};
  a.part_kv = a.part_dq + dq_floats(*p, sh);
  if (p->bias_table && d_table) a.part_table = a.part_kv + kv_floats(*p, sh);
  const hipStream_t st = ait_stream(stream);
  AIT_TRY_RC(p->dtype == AIT_DTYPE_F32 ? launch_t<float>(a, sh, st) : launch_t<__bf16>(a, sh, st));
  if (p->bias_table && d_table) {
    if (p->total_q == 0) a.qnumbers = 0;
    hipLaunchKernelGGL(packed_table_kernel, dim3((unsigned)p->heads, (unsigned)((p->n_buckets + 15) / 16)), dim3(256), 0, st, a);
    AIT_CHECK_LAUNCH();
  }
  return AIT_OK;
}
