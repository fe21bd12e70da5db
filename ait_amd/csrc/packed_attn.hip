// ait_amd/csrc/packed_attn.hip -- ait_packed_attn_fwd: attention over packed sequences, forward (layout of the products:
// packed_attn_impl.h).
//
//   s_ij = scale q_i . k_j + bias[bucket(j - i - (len_k - len_q))],   o_i = sum_j softmax_j(s_ij) v_j
//
// One pass over the keys with the running maximum and sum (kept in units of log2, f32).  A wave has 32 query rows as the columns
// of its score blocks, a workgroup NW waves that share every K / V tile; tiles are double-buffered, the next one's 16-byte loads
// go straight into shared memory while this one is multiplied, one barrier a tile.  The rows of a workgroup are (position,
// head) pairs of one key head: `pack` heads to a position, so that a single new token still fills the block's columns with the
// heads that share its keys.
//
// What bounds it.  Long sequences: the matrix unit and the exponentials beside it, at the clock the chip holds under them: 7
// causal prompts of 33 to 4096 tokens, 16 heads on 4 of 128, bf16: 175 GFLOP in 190 to 196 us a pass, 910 TFLOP/s (a large bf16
// product reaches 1244 here), 223 to 228 for a launch traced by itself.  Of 227 traced, 25 go without the tiles' loads and 13
// without the exponentials; the matrix unit is 48 % busy at 1.7 GHz, no bank conflicts (64-wide heads: a third of the LDS
// cycles, 34 % busy).  (Tried: eight waves a workgroup 247 against 227, two 322 against 231, the next tile's scores under this
// one's exponentials 255 against 227.)  New tokens: memory: 16 caches of 5000 to 8191, 32 heads on 8 of 128: 432 MB in 85 us,
// 5.1 TB/s, and 4.7 us to join the parts.
#include "packed_attn_impl.h"

namespace {
using namespace ait_packed;

struct FwdArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse;          // [H][total_q] log2 of a row's sum (+infinity where a row sees nothing: its probabilities are zero)
  void* rest;          // bf16: what rounding took from o, contiguous
  long long qs, qh, ks, kh, vs, vh, os, oh;      // row and head strides in elements
  Seqs s;
  Bias bias;
  int H, Hk, d, causal, pack, splits, numbers, stages, whole;      // whole: unrounded probabilities (REST)
  float scale;
  float* part_o;      // [splits][total_q * H][d] unnormalised, and
  float* part_ml;     // [splits][total_q * H][2] maximum, sum: only where splits > 1
};

// four values of o; for a backward also what their rounding takes away.  The backward's delta = dO . O is subtracted from
// scores' gradients of like size, so O's rounding to bf16 would be the largest error of dQ and dK.  (Measured against 64 bits: dQ
// off by 0.0025 to 0.0039 of its norm without the rest, 0.0024 with it; bf16 outputs alone are off by 0.0017.)
template <typename T>
__device__ __forceinline__ void store_o(const FwdArgs& a, T* p, long long at, int head, int dd, float v0, float v1, float v2, float v3) {
  store4(p, v0, v1, v2, v3);
  if constexpr (sizeof(T) == 2)
    if (a.rest)
      store4(reinterpret_cast<T*>(a.rest) + (at * a.H + head) * a.d + dd, v0 - (float)(T)v0, v1 - (float)(T)v1, v2 - (float)(T)v2, v3 - (float)(T)v3);
}

// REST (bf16): the probabilities enter the second product as two operands, their bf16 value and what that rounding took, at the
// price of a half more products.  Forwards that a backward follows do it, so that delta belongs to the probabilities and not to
// their rounding: the bias's gradient, a sum over all pairs in which P dP and P delta cancel, is off by 0.0013 to 0.0017 instead
// of 0.0019 to 0.0023, dQ by 0.0024 instead of up to 0.0026.  So do inference calls with few queries a sequence, which wait for
// memory: o is then off by its own rounding (0.0017 of its norm) instead of 0.0023, for 82.8 us instead of 81.4 (16 long caches),
// 7.7 instead of 6.9 (4 short ones), 14.6 instead of 13.5 (300 of up to 49 queries).  Prompts would take 347 us instead of 254
// (7 of 33 to 4096 tokens), sequences of 17 to 1024 with a bias 31.4 instead of 27.0: they round the probabilities once.
template <typename T, int D, int NW, bool BIAS, bool SPLIT, bool REST>
__global__ __launch_bounds__(NW * 64, 2) void packed_fwd_kernel(const FwdArgs a) {
  constexpr int NT = NW * 64, BM = NW * 32, NB = D / 32, NCH = D / 16, kTile = Tile<T, D>::kBytes;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int units = a.H / a.pack, unit = blockIdx.x % units, group = a.H / a.Hk;
  // key heads run fastest (workgroups 8 apart share an L2: they read the same key head where there are 8, 4, 2 or 1 of them)
  const int kvh = unit % a.Hk, head0 = kvh * group + (unit / a.Hk) * a.pack;
  Place place;
  if (!find_place<false>(a.s, a.pack, BM, (int)(blockIdx.x / units), a.numbers, a.causal, place)) return;
  const int seq = place.seq, block = place.block, qstart = place.qstart, qlen = place.qlen;
  if (seq == a.s.n_seq) {          // rows of no sequence
    if constexpr (!SPLIT) {
      const int r = block * BM + wave * 32 + (lane & 31), n = r / a.pack;
      if (n < qlen)
        for (int e = 8 * h; e < a.d; e += 16) {
          T* p = reinterpret_cast<T*>(a.o) + (long long)(qstart + n) * a.os + (long long)(head0 + r - n * a.pack) * a.oh + e;
          store4(p, 0.f, 0.f, 0.f, 0.f);
          store4(p + 4, 0.f, 0.f, 0.f, 0.f);
        }
      if (n < qlen && h == 0 && a.lse) a.lse[(long long)(head0 + r - n * a.pack) * a.s.total_q + qstart + n] = -kNegInf;
    }
    return;
  }
  const int kstart = place.kstart, klen = place.klen, rows = qlen * a.pack, off = klen - qlen;
  const int row0 = block * BM + wave * 32, row = row0 + (lane & 31);
  const int rowc = row < rows ? row : rows - 1, pos = rowc / a.pack, head = head0 + rowc - pos * a.pack;
  const int kmax = a.causal ? min(klen, pos + off + 1) : klen;                           // this lane's query sees keys below it
  const int wfirst = min(row0, rows - 1) / a.pack, wlast = min(row0 + 31, rows - 1) / a.pack;
  const int wsure = a.causal ? min(klen, wfirst + off + 1) : klen, wend = row0 < rows ? (a.causal ? min(klen, wlast + off + 1) : klen) : 0;
  const int gend = a.causal ? min(klen, (min(block * BM + BM, rows) - 1) / a.pack + off + 1) : klen;
  int t0 = 0, t1 = gend > 0 ? (gend + KB - 1) / KB : 0;
  if constexpr (SPLIT) {
    const int per = (t1 + a.splits - 1) / a.splits;
    t0 = blockIdx.y * per;
    t1 = min(t1, t0 + per);
  }

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
  const float* bl = reinterpret_cast<const float*>(lds + 2 * a.stages * kTile);
  float far_lo = 0.f, far_hi = 0.f;
  if (t0 < t1) fetch(t0, 0);
  Frag<T> qf[NCH];
  {
    // (a negative scale: so that the largest product is the largest score)
    const unsigned flip = a.scale < 0.f ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
    const T* qr = reinterpret_cast<const T*>(a.q) + (long long)(qstart + pos) * a.qs + (long long)head * a.qh;
#pragma unroll
    for (int c = 0; c < NCH; c++) {
      qf[c] = global_frag<T>(qr, 16 * c + 8 * h, a.d, row < rows, flip);
    }
  }
  if constexpr (BIAS) {
    const int md = a.bias.max_distance, first = block * BM / a.pack, last = (min(block * BM + BM, rows) - 1) / a.pack;
    const int lowest = bucket(a.bias, -md), highest = bucket(a.bias, md);
    bias_log2(a.bias, (size_t)lowest * a.H + head, (size_t)highest * a.H + head, far_lo, far_hi);
    if (t1 * KB - 1 - (first + off) > -md && t0 * KB - (last + off) < md) {      // (else every key is in the outermost buckets)
      fill_bias<NT>(a.bias, a.H, head0, a.pack, const_cast<float*>(bl), tid);
      __syncthreads();
      bl += (head - head0) * bias_row(md);
    }
  }

  const int rb = row_base<T, D>(lane), cb = col_base<T, D>(lane);
  const float sc = fmaxf(fabsf(a.scale * kLog2e), 1e-30f);      // (0 would make NaN of the hidden scores' -infinity)
  f32x16 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int r = 0; r < 16; r++) acc[b][r] = 0.f;
  float m = kNegInf, l = 0.f;

  for (int t = t0; t < t1; t++) {
    const int stage = (t - t0) & (a.stages - 1), k0 = t * KB;
    loads_done_barrier();
    if (a.stages == 2 && t + 1 < t1) fetch(t + 1, stage ^ 1);
    if (k0 < wend) {
    const unsigned char* kt = lds + stage * 2 * kTile;
    const unsigned char* vt = kt + kTile;
    f32x16 s[2];
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int r = 0; r < 16; r++) s[x][r] = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; c++)
#pragma unroll
      for (int x = 0; x < 2; x++)
        if (sizeof(T) == 2 || x == 0 || k0 + 32 < wend) s[x] = mma(row_frag<T, D>(kt, rb, x, c), qf[c], s[x]);      // (f32: 512 cycles saved)
    read_ahead<T, 2 * NCH, 1, 4>();
    const FirstCols<T, D> first(vt, cb, 0);
    // the block's scores are f * s + add: scaled already where a bias is added value by value
    float f = sc, add = 0.f;
    if constexpr (BIAS) {
      const int md = a.bias.max_distance;
      if (k0 - (wlast + off) >= md) {
        add = far_hi;
      } else if (k0 + KB - 1 - (wfirst + off) <= -md) {
        add = far_lo;
      } else {
        const float* p = bl + (k0 + 4 * h - (pos + off) + md + kPad);
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int r = 0; r < 16; r++) s[x][r] = __builtin_fmaf(s[x][r], sc, p[32 * x + 8 * (r >> 2) + (r & 3)]);
        f = 1.f;
      }
    }
    if (k0 + KB > wsure) {
      const int lim = kmax - k0 - 4 * h;
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int r = 0; r < 16; r++) s[x][r] = 32 * x + 8 * (r >> 2) + (r & 3) < lim ? s[x][r] : kNegInf;
    }
    float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int r = 1; r < 16; r++) top = fmaxf(fmaxf(top, s[0][r]), s[1][r]);
    top = __builtin_fmaf(column_max(top), f, add);
    // The maximum is only followed where it rises by more than 2^8 (a published idea: T. Dao, Hot Chips 2025): what is summed
    // stays below 2^8 and the same bits are significant, and nearly every block is spared the rescaling of the accumulators
    if (__any(top > m + 8.f)) {
      const float mn = fmaxf(m, top), alpha = fast_exp2(m - (mn == kNegInf ? 0.f : mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[b][r] *= alpha;
    }
    if (__any(rounded(m))) {
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int r = 0; r < 16; r++) s[x][r] = __builtin_fmaf(s[x][r], f, add);
      f = 1.f;
      add = 0.f;
    }
    const float sub = add - (m == kNegInf ? 0.f : m);
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        s[x][r] = fast_exp2(__builtin_fmaf(s[x][r], f, sub));
        l += s[x][r];
      }
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int cc = 0; cc < 2; cc++) {
        if (sizeof(T) == 4 && k0 + 32 * x + 16 * cc >= wend) continue;
        const Frag<T> pf = acc_frag<T>(s[x], cc);
#pragma unroll
        for (int b = 0; b < NB; b++) {
          const Frag<T> vf = x == 0 ? first.get(vt, cb, x, cc, b) : col_frag<T, D>(vt, cb, x, cc, b);
          acc[b] = mma(vf, pf, acc[b]);
          if constexpr (REST) acc[b] = mma(vf, acc_rest<T>(s[x], cc, pf), acc[b]);
        }
      }
    read_ahead<T, 4 * NB, 2, 4, true, REST ? 2 : 1>();
    }
    if (a.stages == 1 && t + 1 < t1) {
      loads_done_barrier();
      fetch(t + 1, 0);
    }
  }

  if (row >= rows) return;
  l = column_sum(l);
  const long long at = (long long)(qstart + pos);
  if constexpr (SPLIT) {
    const long long id = (long long)blockIdx.y * a.s.total_q * a.H + at * a.H + head;
    if (h == 0) {
      a.part_ml[2 * id] = m;
      a.part_ml[2 * id + 1] = l;
    }
    float* p = a.part_o + id * a.d;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int dd = 32 * b + 8 * i + 4 * h;
        if (dd < a.d) store4(p + dd, acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]);
      }
  } else {
    const bool none = l == 0.f;        // a row that sees nothing: zeros, whatever the keys beside it hold
    const float inv = 1.f / l;
    if (a.lse && h == 0) a.lse[(long long)head * a.s.total_q + at] = none ? -kNegInf : m + __builtin_amdgcn_logf(l);
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[b][r] = none ? 0.f : acc[b][r] * inv;
    T* p = reinterpret_cast<T*>(a.o) + at * a.os + (long long)head * a.oh;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int dd = 32 * b + 8 * i + 4 * h;
        if (dd < a.d) store_o<T>(a, p + dd, at, head, dd, acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]);
      }
  }
}

// The parts of a row joined: one wave per (query row, head).  A lane has one part's maximum and sum (there are at most 64); then
// LD lanes take four values each and 64 / LD parts go at a time, added up in a fixed order.
constexpr int kMaxSplits = 64;
template <typename T, int LD>
__global__ __launch_bounds__(256) void packed_join_kernel(const FwdArgs a) {
  const int lane = threadIdx.x & 63;
  const long long n = (long long)a.s.total_q * a.H, id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (id >= n) return;
  const int at = (int)(id / a.H);
  const bool in = at >= clamped(a.s.cu_q, 0, a.s.total_q) && at < clamped(a.s.cu_q, a.s.n_seq, a.s.total_q);
  if (!in && !a.s.rest) return;                          // no sequence's row: left as it is, or set to zero
  const int head = (int)(id - (long long)at * a.H), dd = (lane % LD) * 4, splits = in ? a.splits : 0;
  float m = kNegInf, l = 0.f;
  if (lane < splits) {
    m = a.part_ml[2 * (lane * n + id)];
    l = a.part_ml[2 * (lane * n + id) + 1];
  }
  const float top = wave_max(m), w = fast_exp2(m - (top == kNegInf ? 0.f : top));      // (NaN scores leave m alone and make l NaN)
  l = wave_sum(lane < splits ? l * w : 0.f);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < splits; s0 += 64 / LD) {
    const int s = s0 + lane / LD;
    const float ws = __shfl(w, s & 63, 64);
    if (s < splits && dd < a.d && ws != 0.f) o += *reinterpret_cast<const f32x4*>(a.part_o + (s * n + id) * a.d + dd) * ws;
  }
#pragma unroll
  for (int x = LD; x < 64; x *= 2)
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] += __shfl_xor(o[e], x, 64);
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (a.lse && lane == 0) a.lse[(long long)head * a.s.total_q + at] = l == 0.f ? -kNegInf : top + __builtin_amdgcn_logf(l);
  if (lane < LD && dd < a.d)
    store_o<T>(a, reinterpret_cast<T*>(a.o) + (long long)at * a.os + (long long)head * a.oh + dd, at, head, dd, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
}

template <typename T, int D, int NW, bool BIAS, bool SPLIT, bool REST>
int launch(const FwdArgs& a, int bias_bytes, hipStream_t st) {
  const int bytes = 2 * a.stages * Tile<T, D>::kBytes + bias_bytes;
  if (!launchable((long long)a.numbers * (a.H / a.pack), NW * 64) || (SPLIT && !launchable(((long long)a.s.total_q * a.H + 3) / 4, 256)))
    return AIT_EUNSUPPORTED;
  if (bytes > 65536 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(packed_fwd_kernel<T, D, NW, BIAS, SPLIT, REST>), hipFuncAttributeMaxDynamicSharedMemorySize,
                          bytes) != hipSuccess)
    return AIT_ELAUNCH;
  hipLaunchKernelGGL((packed_fwd_kernel<T, D, NW, BIAS, SPLIT, REST>), dim3((unsigned)(a.numbers * (a.H / a.pack)), (unsigned)a.splits), dim3(NW * 64),
                     bytes, st, a);
  AIT_CHECK_LAUNCH();
  if constexpr (SPLIT) {
    hipLaunchKernelGGL((packed_join_kernel<T, D / 4>), dim3((unsigned)(((long long)a.s.total_q * a.H + 3) / 4)), dim3(256), 0, st, a);
    AIT_CHECK_LAUNCH();
  }
  return AIT_OK;
}
template <typename T, int D, int NW, bool BIAS, bool SPLIT>
int launch_rest(const FwdArgs& a, int bias_bytes, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (a.whole) return launch<T, D, NW, BIAS, SPLIT, true>(a, bias_bytes, st);
  return launch<T, D, NW, BIAS, SPLIT, false>(a, bias_bytes, st);
}
template <typename T, int D, int NW>
int launch_nw(const FwdArgs& a, int bias_bytes, hipStream_t st) {
  if (a.bias.table) return a.splits > 1 ? launch_rest<T, D, NW, true, true>(a, bias_bytes, st) : launch_rest<T, D, NW, true, false>(a, bias_bytes, st);
  return a.splits > 1 ? launch_rest<T, D, NW, false, true>(a, 0, st) : launch_rest<T, D, NW, false, false>(a, 0, st);
}
template <typename T, int D>
int launch_d(const FwdArgs& a, int nw, int bias_bytes, hipStream_t st) {
  return nw == 2 ? launch_nw<T, D, 2>(a, bias_bytes, st) : launch_nw<T, D, 4>(a, bias_bytes, st);
}
template <typename T>
int launch_t(const FwdArgs& a, int nw, int bias_bytes, hipStream_t st) {
  return a.d <= 64 ? launch_d<T, 64>(a, nw, bias_bytes, st) : launch_d<T, 128>(a, nw, bias_bytes, st);
}

// what the sizes decide: heads packed to a position, waves of a workgroup, parts of the key axis, tiles in flight
struct Shape { int pack, nw, splits, stages; bool few; };
Shape shape_of(const ait_packed_attn& p) {
  Shape r;
  const int group = p.heads / p.kv_heads;
  const long long max_q = p.max_q > 0 ? p.max_q : p.total_q, max_k = p.max_k > 0 ? p.max_k : p.total_k;
  // a few new tokens: the heads of a key head share a workgroup's columns, and its keys are read once (16 long caches, 4 heads to
  // a key head: 86 us, 185 with a workgroup to a head; with a bias, whose heads each want a row in shared memory, 13.3 and 20.9)
  r.few = max_q * group <= 128;
  r.pack = r.few && (!p.bias_table || (long long)group * bias_row(p.max_distance) * 4 <= 32768) ? group : 1;
  // up to 64 rows in two waves, in four what is longer (sequences of 1 to 49 in f32: 36.3 us against 43.5 in four; prompts: 322 us
  // in two, 231 in four); for single tokens two measure as four and better than one (with bias 11.3, 11.7, 13.3 us)
  r.nw = max_q * r.pack <= 64 ? 2 : 4;
  // sequences of one tile have no second one to load ahead: half the memory, twice the workgroups beside one another (sequences
  // of 1 to 49 in f32: 36.3 us, 55.1 with room for two)
  r.stages = max_k <= KB ? 1 : 2;
  // Few rows leave most of the chip idle: the key axis is cut, two tiles at least to a part.  As many parts as fit the chip at
  // once with two workgroups a CU: a round more costs as much as all of them (64 queries against 2394 keys in f32: 37 us in 19
  // parts, 608 workgroups, 33.6 in 16; forward and backward 465 us uncut, 172 cut); twice as many gain new tokens nothing (84.2 us against 84.0)
  const long long rows = (long long)p.total_q * r.pack, blocks = rows / (r.nw * 32) > p.n_seq ? rows / (r.nw * 32) : p.n_seq;
  const long long wgs = (blocks > 0 ? blocks : 1) * (p.heads / r.pack), tiles = (max_k + KB - 1) / KB;
  long long s = 512 / wgs;
  if (s > tiles / 2) s = tiles / 2;
  if (s > kMaxSplits) s = kMaxSplits;
  r.splits = s < 1 ? 1 : (int)s;
  return r;
}
size_t workspace(const ait_packed_attn& p, const Shape& s) {
  return s.splits > 1 ? (size_t)s.splits * p.total_q * p.heads * (p.d + 2) * sizeof(float) : 0;
}
}  // namespace

namespace ait_packed {
int check(const ait_packed_attn* p) {
  if (!p || p->n_seq < 0 || p->total_q < 0 || p->total_k < 0 || p->heads <= 0 || p->kv_heads <= 0 || p->heads % p->kv_heads || p->d <= 0)
    return AIT_EINVAL;
  if (p->dtype != AIT_DTYPE_F32 && p->dtype != AIT_DTYPE_BF16) return AIT_EINVAL;
  if (p->max_q < 0 || p->max_k < 0 || !(p->scale == p->scale)) return AIT_EINVAL;
  if (p->d > 128 || p->d % 8) return AIT_EUNSUPPORTED;
  if (p->bias_table) {
    if (!p->bucket_of || p->n_buckets <= 0 || p->max_distance < 0) return AIT_EINVAL;
    if (p->table_dtype != AIT_DTYPE_F32 && p->table_dtype != AIT_DTYPE_BF16) return AIT_EINVAL;
    if (p->n_buckets > AIT_MAX_BUCKETS || p->max_distance > AIT_MAX_BIAS_DISTANCE) return AIT_EUNSUPPORTED;
  }
  if ((p->n_seq > 0 && p->total_q > 0) && (!p->cu_q || !p->cu_k)) return AIT_EINVAL;
  // 32-bit counters: block numbers times heads, and rows times heads
  if ((long long)p->total_q * p->heads + (long long)(p->n_seq + 1LL) * p->heads >= (1LL << 31)) return AIT_EUNSUPPORTED;
  if ((long long)p->total_k * p->heads + (long long)(p->n_seq + 1LL) * p->heads >= (1LL << 40)) return AIT_EUNSUPPORTED;
  return AIT_OK;
}
int check_strides(const ait_packed_attn* p, const void* base, long long row, long long head, long long rows) {
  const int es = p->dtype == AIT_DTYPE_F32 ? 4 : 2;
  if (rows > 0 && !base) return AIT_EINVAL;
  if ((unsigned long long)base % 16 || (row * es) % 16 || (head * es) % 16 || row < 0 || head < 0) return AIT_EUNSUPPORTED;
  if (row * es * KB >= (1LL << 31)) return AIT_EUNSUPPORTED;      // a tile's 32-bit offsets
  return AIT_OK;
}
}  // namespace ait_packed

AIT_API size_t ait_packed_attn_fwd_workspace_bytes(const ait_packed_attn* p) {
  if (ait_packed::check(p) != AIT_OK) return 0;
  return workspace(*p, shape_of(*p));
}

AIT_API int ait_packed_attn_fwd(const ait_packed_attn* p, const void* q, long long q_row, long long q_head, const void* k, long long k_row,
                                long long k_head, const void* v, long long v_row, long long v_head, void* o, long long o_row,
                                long long o_head, float* lse, void* o_rest, void* workspace_ptr, size_t workspace_bytes, void* stream) {
  AIT_TRY_RC(ait_packed::check(p));
  if (p->n_seq == 0 || p->total_q == 0) return AIT_OK;
  AIT_TRY_RC(ait_packed::check_strides(p, q, q_row, q_head, p->total_q));
  AIT_TRY_RC(ait_packed::check_strides(p, o, o_row, o_head, p->total_q));
  AIT_TRY_RC(ait_packed::check_strides(p, k, k_row, k_head, p->total_k));
  AIT_TRY_RC(ait_packed::check_strides(p, v, v_row, v_head, p->total_k));
  if ((unsigned long long)o_rest % 16) return AIT_EUNSUPPORTED;
  const Shape sh = shape_of(*p);
  const size_t need = workspace(*p, sh);
  if (need && (!workspace_ptr || workspace_bytes < need)) return AIT_EWORKSPACE;
  if ((unsigned long long)workspace_ptr % 16) return AIT_EINVAL;
  FwdArgs a{q, k, v, o, lse, p->dtype == AIT_DTYPE_BF16 ? o_rest : nullptr, q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head,
            {p->cu_q, p->cu_k, p->k_len, p->n_seq, p->total_q, p->total_k, p->zero_rest ? 1 : 0, sh.splits == 1 && ait_packed::order_blocks(*p)},
            {p->bias_table, p->bucket_of, p->n_buckets, p->max_distance, p->table_dtype == AIT_DTYPE_BF16},
            p->heads, p->kv_heads, p->d, p->causal, sh.pack, sh.splits,
            (int)ait_packed::block_numbers(p->total_q, sh.pack, sh.nw * 32, p->n_seq, p->zero_rest ? 1 : 0), sh.stages, o_rest || sh.few, p->scale, nullptr, nullptr};
  if (need) {
    a.part_o = static_cast<float*>(workspace_ptr);
    a.part_ml = a.part_o + (size_t)sh.splits * p->total_q * p->heads * p->d;
  }
  const int bias_bytes = p->bias_table ? sh.pack * bias_row(p->max_distance) * 4 : 0;
  return p->dtype == AIT_DTYPE_F32 ? launch_t<float>(a, sh.nw, bias_bytes, ait_stream(stream)) : launch_t<__bf16>(a, sh.nw, bias_bytes, ait_stream(stream));
}
