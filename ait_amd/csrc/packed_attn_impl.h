// ait_amd/csrc/packed_attn_impl.h -- shared by packed_attn.hip (forward) and packed_attn_bwd.hip.
//
// Attention over sequences that lie one behind another in memory.  Every product runs on 32 x 32 matrix blocks in the
// TRANSPOSED form: the scores as S^T = K Q^T, so that an accumulator column -- one lane and its partner 32 lanes away -- is
// one query.  The softmax's running maximum, its sum and the rescaling are then values of a lane, the probabilities leave the
// accumulators in the operand order of the second product (O^T = V^T P^T), and nothing passes through shared memory between
// the two.  V^T comes out of the row-major tile by gfx950's transposing LDS read.
//
// One operand block ("Frag") is eight values a lane: of row / column lane & 31, reduction indices 8 (lane >> 5) + 0..7 of a
// chunk of 16.  bf16: one v_mfma_f32_32x32x16_bf16 per chunk; f32: eight v_mfma_f32_32x32x2_f32, instruction e taking element e
// of both halves -- the same chunk, so the kernels are one source for both types (f32 products are exact f32 products).
#pragma once
#include "common.h"

namespace ait_packed {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) unsigned char lds_u8;

constexpr int KB = 64;              // keys (or, in the gradient of keys and values, queries) of a tile in shared memory
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kNegInf = -__builtin_inff(), kMaxFinite = 3.402823466e38f;
// A score scale q.k + bias is an f32 value.  Up to kRounded in size (in units of log2, where a step of f32 is 2^-16) products,
// bias and what is subtracted from them go through one multiply-add, which keeps more than that.  Beyond it the score is rounded
// first, everywhere alike, so that a row whose every score is far from zero (a mask's value in the bias, or products of that
// size) has one softmax, whichever block a key lies in, and the same one in the backward.
constexpr float kRounded = 256.f;
__device__ __forceinline__ bool rounded(float t) { return fabsf(t) > kRounded && fabsf(t) <= kMaxFinite; }

template <typename T> struct FragOf;
template <> struct FragOf<__bf16> { using type = bf16x8; };
template <> struct FragOf<float> { using type = f32x8; };
template <typename T> using Frag = typename FragOf<T>::type;

__device__ __forceinline__ f32x16 mma(const bf16x8& a, const bf16x8& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const f32x8& a, const f32x8& b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// eight accumulator values (registers 8 cc .. 8 cc + 7) as an operand: reduction index 16 cc + 8 (e / 4) + 4 (lane >> 5) + e % 4
// of the 32 the block has.  bf16: rounded to nearest even here -- the one rounding of the probabilities (and of dS in the
// backward), to the type of the tensor they are multiplied with, as the matrix unit asks; sums stay in f32.  Against 64 bits it
// leaves o off by 0.0021 and the gradients by 0.0024 of their norm, where the outputs' own rounding to bf16 makes 0.0017; a
// second operand with what it took (acc_rest) would cost every product that has one of them as much again.
template <typename T>
__device__ __forceinline__ Frag<T> acc_frag(const f32x16& c, int cc) {
  Frag<T> f;
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = (T)c[8 * cc + e];
  return f;
}

// what that rounding took, as a second operand
template <typename T>
__device__ __forceinline__ Frag<T> acc_rest(const f32x16& c, int cc, const Frag<T>& f) {
  Frag<T> r;
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = (T)(c[8 * cc + e] - (float)f[e]);
  return r;
}

// The order of a chain of N products whose left operands come from shared memory by R reads each: AHEAD operands are read before
// the first product, then one more behind every product.  Left alone, the compiler reads an operand, waits for it and multiplies:
// a trip to shared memory (over 100 cycles) in front of every 32-cycle product.  (f32: an operand feeds 8 products of 64 cycles.)
// READ: the first AHEAD operands are there already.  M: products that share a left operand.
template <typename T, int N, int R, int AHEAD, bool READ = false, int M = 1>
__device__ __forceinline__ void read_ahead() {
  if constexpr (sizeof(T) == 2) {
    if constexpr (!READ) __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * R, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; i++) {
      __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * M, 0);
  }
}

// ---- tiles in shared memory: KB rows of D values, 16-byte chunk c of row r at position c ^ swz(r) -------------------------
// Row operands (16 bytes of 32 consecutive rows) and transposed reads (32 bytes of four consecutive rows) both spread over
// all 64 banks.  Chunk positions differ from chunks in the low bits only, so every offset below is one base XOR a constant.
template <typename T, int D>
struct Tile {
  static constexpr int kRow = D * (int)sizeof(T);
  static constexpr int kChunks = kRow / 16;
  static constexpr int kBytes = KB * kRow;
  __device__ static __forceinline__ int swz(int r) {
    return kChunks >= 16 ? (4 * (r & 3) | ((r >> 2) & 3)) : (2 * (r & 3) | ((r >> 2) & 1));
  }
};

// operand block of tile rows 32 rt .. + 31, values 16 c .. + 15 of each.  `base` = row_base<T, D>(lane)
template <typename T, int D>
__device__ __forceinline__ int row_base(int lane) {
  const int r = lane & 31, h = lane >> 5;
  return r * Tile<T, D>::kRow + (((sizeof(T) == 4 ? 2 * h : h) ^ Tile<T, D>::swz(r)) * 16);
}
template <typename T, int D>
__device__ __forceinline__ Frag<T> row_frag(const unsigned char* tile, int base, int rt, int c) {
  const unsigned char* p = tile + rt * 32 * Tile<T, D>::kRow;
  if constexpr (sizeof(T) == 2) {
    return *reinterpret_cast<const bf16x8*>(p + (base ^ (c * 32)));
  } else {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p + (base ^ (c * 64)));
    const f32x4 hi = *reinterpret_cast<const f32x4*>(p + (base ^ (c * 64) ^ 16));
    f32x8 f;
#pragma unroll
    for (int e = 0; e < 4; e++) { f[e] = lo[e]; f[4 + e] = hi[e]; }
    return f;
  }
}

// operand block of the tile TRANSPOSED: row = value 32 db + (lane & 31), reduction = tile rows 32 rt + 16 cc + the order of
// acc_frag.  `base` = col_base<T, D>(lane)
template <typename T, int D>
__device__ __forceinline__ int col_base(int lane) {
  const int h = lane >> 5;
  if constexpr (sizeof(T) == 2) {      // the address a lane gives to the transposing read: four rows, 16 values, per 16 lanes
    const int i = lane & 15, r = 4 * h + (i >> 2), chunk = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    return r * Tile<T, D>::kRow + (chunk ^ Tile<T, D>::swz(r)) * 16 + (i & 1) * 8;
  } else {
    const int d = lane & 31;
    return 4 * h * Tile<T, D>::kRow + ((d >> 2) ^ Tile<T, D>::swz(4 * h)) * 16 + (d & 3) * 4;
  }
}
template <typename T, int D>
__device__ __forceinline__ Frag<T> col_frag(const unsigned char* tile, int base, int rt, int cc, int db) {
  constexpr int R = Tile<T, D>::kRow;
  const unsigned char* p = tile + (rt * 32 + cc * 16) * R;
  if constexpr (sizeof(T) == 2) {
    constexpr int kUp = Tile<T, D>::kChunks >= 16 ? 32 : 0;      // what eight rows further down change in the swizzle
    const int b = base ^ (db * 64);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + b));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + (b ^ kUp) + 8 * R));
    s16x8 v;
#pragma unroll
    for (int e = 0; e < 4; e++) { v[e] = lo[e]; v[4 + e] = hi[e]; }
    return __builtin_bit_cast(bf16x8, v);
  } else {
    const int b = base ^ (db * 128);
    f32x8 f;
#pragma unroll
    for (int e = 0; e < 8; e++)
      f[e] = *reinterpret_cast<const float*>(p + (b ^ ((4 * (e & 3) | 2 * (e >> 2)) * 16)) + (8 * (e >> 2) + (e & 3)) * R);
    return f;
  }
}

// The first four transposed operands of a product, read before what comes between it and the product in front (exponentials,
// selects, branches: the compiler moves no read across them).  f32 operands are eight reads each and feed 512 cycles: not kept.
template <typename T, int D>
struct FirstCols {
  static constexpr int NB = D / 32;
  Frag<T> f[sizeof(T) == 2 ? 4 : 1];
  __device__ __forceinline__ FirstCols(const unsigned char* tile, int base, int rt) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = col_frag<T, D>(tile, base, rt, i / NB, i % NB);
      __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
    }
  }
  __device__ __forceinline__ Frag<T> get(const unsigned char* tile, int base, int rt, int cc, int b) const {
    if constexpr (sizeof(T) == 2) {
      if (cc * NB + b < 4) return f[(cc * NB + b) & 3];
    }
    return col_frag<T, D>(tile, base, rt, cc, b);
  }
};

// ---- global -> shared memory -----------------------------------------------------------------------------------------------
// 16 bytes a lane straight into shared memory.  The buffer descriptor ends behind the sequence's last row (tile by tile: a
// 64-bit base and at most KB rows of 32-bit offsets, so long caches need no wider offsets), and what lies outside arrives as
// zeros: rows of the next sequence, the cache's unwritten tail and the padding of d to D never reach a product.
__device__ __forceinline__ i32x4 tile_rsrc(const void* base, unsigned bytes) {
  const unsigned long long p = (unsigned long long)base;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)p);
  r[1] = __builtin_amdgcn_readfirstlane((int)((unsigned)(p >> 32) & 0xffffu));
  r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
  r[3] = 0x00027000;
  // a vector instruction's scalar result (readfirstlane) must be five wait states old where a memory instruction reads it; the
  // compiler keeps to that for its own instructions but does not look into the asm of the loads below
  asm volatile("s_nop 4" : "+s"(r));
  return r;
}
__device__ __forceinline__ void load_lds16(unsigned voff, const i32x4& rsrc, unsigned dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(voff), "s"(rsrc), "s"(dst) : "m0", "memory");
}
// all of this wave's memory operations are done, and every wave of the workgroup says the same
__device__ __forceinline__ void loads_done_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T, int D, int NT>
struct Loader {
  static constexpr int kN = Tile<T, D>::kBytes / (NT * 16);          // instructions of a wave per tile
  unsigned voff[kN];
  // stride: bytes from row to row; d_bytes: bytes of a row that exist (a multiple of 16)
  __device__ __forceinline__ void init(int tid, unsigned stride, unsigned d_bytes) {
#pragma unroll
    for (int j = 0; j < kN; j++) {
      const int p = (tid >> 6) * kN * 64 + j * 64 + (tid & 63);
      const int r = p / Tile<T, D>::kChunks, c = (p % Tile<T, D>::kChunks) ^ Tile<T, D>::swz(r);
      voff[j] = (unsigned)(c * 16) < d_bytes ? (unsigned)r * stride + c * 16 : 0x80000000u;
    }
  }
  // rows: how many of the tile's rows exist (any number; 0 or less: all zeros)
  __device__ __forceinline__ void load(const void* base, long long rows, unsigned stride, unsigned d_bytes, unsigned lds, int wave) const {
    const unsigned n = rows <= 0 ? 0u : (unsigned)(rows < KB ? rows : KB);
    const i32x4 rsrc = tile_rsrc(base, n ? (n - 1) * stride + d_bytes : 0u);
#pragma unroll
    for (int j = 0; j < kN; j++) load_lds16(voff[j], rsrc, (unsigned)__builtin_amdgcn_readfirstlane((int)(lds + (wave * kN + j) * 1024)));
  }
};

__device__ __forceinline__ unsigned lds_addr(const void* p) { return (unsigned)(size_t)(const lds_u8*)p; }

// Eight values of a row in memory as an operand; values >= d, and rows that are not there (`row` is then any row that is): zero.
// No branch around the load, so that a row's loads are in flight together.  flip: the sign bits to turn over, as bits (negated
// as a vector of bf16 behind the select, one value in two came out of the compiler with the wrong sign)
template <typename T>
__device__ __forceinline__ Frag<T> global_frag(const T* row, int at, int d, bool there, unsigned flip = 0) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  struct Words { u32x4 w[sizeof(T) / 2]; };
  const T* p = row + min(at, d - 8);
  const bool in = there && at < d;
  Words f;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; i++) {
    const u32x4 v = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
    for (int e = 0; e < 4; e++) f.w[i][e] = (in ? v[e] : 0u) ^ flip;
  }
  return __builtin_bit_cast(Frag<T>, f);
}

// four consecutive values of a row
template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 2) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    bf16x4 v;
    v[0] = (__bf16)a; v[1] = (__bf16)b; v[2] = (__bf16)c; v[3] = (__bf16)d;
    *reinterpret_cast<bf16x4*>(p) = v;
  } else {
    f32x4 v;
    v[0] = a; v[1] = b; v[2] = c; v[3] = d;
    *reinterpret_cast<f32x4*>(p) = v;
  }
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// the two lanes of an accumulator column (32 apart): both get both values, in the same order
__device__ __forceinline__ void column_pair(float v, float& lo, float& hi) {
  lo = hi = v;      // the upper half of one register swaps places with the lower half of the other (as attn_impl.h swap16)
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(lo), "+v"(hi));
}
__device__ __forceinline__ float column_max(float v) {
  float a, b;
  column_pair(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float column_sum(float v) {
  float a, b;
  column_pair(v, a, b);
  return a + b;
}

// ---- which rows a workgroup has ---------------------------------------------------------------------------------------------
// Row blocks of BM are numbered so that no host knows the lengths: block j of sequence b has number start(b) * mul / BM + b + j.
// A sequence of n rows needs at most n / BM + 1 of the n / BM + 1 numbers up to its successor's first, so numbers never clash;
// the few unused ones are workgroups that end at once.  Lengths and starts come from device memory and are clamped to the
// tensors they index, so that a bad table gives wrong rows, never a wrong address.
__device__ __forceinline__ int clamped(const int* cu, int i, int total) {
  const int v = cu[i];
  return v < 0 ? 0 : v > total ? total : v;
}
// With `rest` the rows behind the last sequence count as one more, number n_seq: the blocks that set them to zero.
__device__ __forceinline__ bool find_block(const int* cu, int n_seq, int rest, int total, int mul, int bm, int number, int& seq, int& block,
                                           int& start, int& len) {
  // 64 candidates at a time, one per lane: up to 64 sequences cost one trip to memory
  const int lane = threadIdx.x & 63;
  int lo = 0, count = n_seq + rest, begin = 0, end = 0;
  while (true) {
    const int step = (count + 63) / 64, b = lo + lane * step;
    const bool there = lane * step < count;
    const int c = clamped(cu, min(b, n_seq), total), next = clamped(cu, min(b + 1, n_seq), total), e = b < n_seq ? next : total;
    // (the first candidate counts in any case; what follows a later one is later, in a table that ascends)
    const unsigned long long ok = __ballot(there && (lane == 0 || (int)((long long)c * mul / bm) + b <= number));
    const int t = 63 - __builtin_clzll(ok);
    lo += t * step;
    count = min(step, count - t * step);
    begin = __builtin_amdgcn_readlane(c, t);
    end = __builtin_amdgcn_readlane(e, t);
    if (step == 1) break;
  }
  seq = lo;
  start = begin;
  len = end - begin;
  block = number - (int)((long long)start * mul / bm) - lo;
  return block >= 0 && (long long)block * bm < (long long)len * mul;
}
// inclusive sum over the lanes
__device__ __forceinline__ int lane_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);      // row_shr 1, 2, 4, 8: inside 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);      // the last lane of rows 0 and 2 to rows 1 and 3,
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);      // of the first half to the second
  return v;
}
// The same blocks in another order: those with the most turns first, whatever their sequence, so that a launch does not end on
// the long ones (7 prompts of 33 to 4096 tokens: 217 us against 227, sequences of 17 to 1024 with a bias 61 against 73 in the pass
// over query rows).  At most 64 sequences, `rest` among them.
// A block of rows j (of ROWS rows) of a sequence takes turns(j) = ceil(min(all, (j + 1) rows_per + off) / KB) turns if it
// ascends, ceil((all - max(0, j rows_per - off)) / KB) if not -- the key tiles of a query block, the query tiles of a key block;
// `flat`: every block takes ceil(all / KB).  The blocks with more than L turns are counted in closed form and L is found by
// bisection; among those with L + 1 turns the order is by sequence.
struct Turns { int blocks, all, off, rows_per; bool flat, ascends; };
__device__ __forceinline__ int blocks_over(const Turns& s, int L) {      // blocks with more than L >= 0 turns
  const int need = L * KB;
  if (s.all <= need) return 0;
  if (s.flat) return s.blocks;
  if (s.ascends) {      // (j + 1) rows_per + off > need
    const int first = need - s.off;
    return s.blocks - min(s.blocks, first > 0 ? first / s.rows_per : 0);
  }
  const int room = s.all - need - 1 + s.off;      // all - max(0, j rows_per - off) > need: j rows_per <= room
  return room < 0 ? 0 : min(s.blocks, room / s.rows_per + 1);
}
__device__ __forceinline__ bool heaviest_first(const Turns& s, int number, int most, int& seq, int& block) {
  if (__builtin_amdgcn_readlane(lane_scan(s.blocks), 63) <= number) return false;
  int lo = -1, hi = most;      // over(lo) > number >= over(hi); over(-1): all blocks
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__builtin_amdgcn_readlane(lane_scan(blocks_over(s, mid)), 63) > number) lo = mid;
    else hi = mid;
  }
  const int more = blocks_over(s, lo + 1), here = (lo < 0 ? s.blocks : blocks_over(s, lo)) - more;      // this lane's with lo + 1 turns
  const int skip = number - __builtin_amdgcn_readlane(lane_scan(more), 63), upto = lane_scan(here);
  seq = __builtin_ctzll(__ballot(upto > skip));
  const int k = skip - __builtin_amdgcn_readlane(upto - here, seq);
  // the k-th of them: in an ascending sequence the blocks with more turns are the last ones, else the first
  const int m = __builtin_amdgcn_readlane(more, seq), n = __builtin_amdgcn_readlane(here, seq), b = __builtin_amdgcn_readlane(s.blocks, seq);
  block = __builtin_amdgcn_readlane((int)(s.ascends && !s.flat), seq) ? b - m - n + k : m + k;
  return true;
}
static inline long long block_numbers(long long total, int mul, int bm, int n_seq, int rest) {
  return total * mul / bm + n_seq + rest;
}

struct Seqs {
  const int* cu_q;
  const int* cu_k;
  const int* k_len;        // may be null: the keys of a sequence end where the next one's begin
  int n_seq, total_q, total_k, rest;
  int ordered;             // blocks in the order of heaviest_first
};
__device__ __forceinline__ void keys_of(const Seqs& s, int seq, int& start, int& len) {
  const int from = s.cu_k[seq], to = s.cu_k[seq + 1];
  int l = s.total_k;
  if (s.k_len) l = s.k_len[seq];
  start = min(max(from, 0), s.total_k);
  len = max(0, min(min(max(to, 0), s.total_k) - start, l));
}

// A workgroup's place: block `number` of the query rows (mul rows to a position, bm to a block) or, KEYS, of the key rows (bm to a
// block, counted over the rows that the sequences occupy: keys behind k_len get zeros), and its sequence's queries and keys.
struct Place { int seq, block, qstart, qlen, kstart, klen, kroom; };
template <bool KEYS>
__device__ __forceinline__ bool find_place(const Seqs& s, int mul, int bm, int number, int numbers, bool causal, Place& p) {
  if (s.ordered) {
    const int lane = threadIdx.x & 63, n = s.n_seq + s.rest, b = lane < n ? lane : n - 1;
    const bool seq = b < s.n_seq;
    // (the loads together, then what is done with them)
    const int to = min(b + 1, s.n_seq), q0 = s.cu_q[b], q1 = s.cu_q[to], k0 = s.cu_k[b], k1 = s.cu_k[to];
    int l = s.total_k;
    if (s.k_len) l = s.k_len[min(b, s.n_seq - 1)];
    const int qs = min(max(q0, 0), s.total_q), qe = seq ? min(max(q1, 0), s.total_q) : s.total_q;
    const int ks = min(max(k0, 0), s.total_k), ke = seq ? min(max(k1, 0), s.total_k) : s.total_k;
    const int len = max(0, qe - qs), room = max(0, ke - ks), kl = seq ? max(0, min(room, l)) : 0;
    const int off = kl - len, rows = KEYS ? room : len * mul, per = KEYS || mul == 1 ? bm : max(1, bm / mul);
    const Turns t{lane < n && rows > 0 ? (rows - 1) / bm + 1 : 0, KEYS ? (kl > 0 ? len : 0) : kl, off, per, !causal, !KEYS};
    if (!heaviest_first(t, number, (KEYS ? s.total_q : s.total_k) / KB + 1, p.seq, p.block)) return false;
    p.qstart = __builtin_amdgcn_readlane(qs, p.seq);
    p.qlen = __builtin_amdgcn_readlane(len, p.seq);
    p.kstart = __builtin_amdgcn_readlane(ks, p.seq);
    p.klen = __builtin_amdgcn_readlane(kl, p.seq);
    p.kroom = __builtin_amdgcn_readlane(room, p.seq);
    return true;
  }
  if constexpr (KEYS) {
    if (!find_block(s.cu_k, s.n_seq, s.rest, s.total_k, 1, bm, number, p.seq, p.block, p.kstart, p.kroom)) return false;
    p.qstart = p.qlen = p.klen = 0;
    if (p.seq < s.n_seq) {
      int ks;
      keys_of(s, p.seq, ks, p.klen);
      p.qstart = clamped(s.cu_q, p.seq, s.total_q);
      p.qlen = max(0, clamped(s.cu_q, p.seq + 1, s.total_q) - p.qstart);
    }
  } else {      // a sequence's last rows first: with a causal mask they have the most to do
    if (!find_block(s.cu_q, s.n_seq, s.rest, s.total_q, mul, bm, numbers - 1 - number, p.seq, p.block, p.qstart, p.qlen)) return false;
    if (p.seq < s.n_seq) keys_of(s, p.seq, p.kstart, p.klen);
  }
  return true;
}
static inline int order_blocks(const ait_packed_attn& p) {
  const long long max_k = p.max_k > 0 ? p.max_k : p.total_k;
  return p.n_seq < 64 && max_k > 4 * KB && p.total_q < (1 << 24) && p.total_k < (1 << 24);
}

// ---- the bias: one value per relative position and head, constant beyond max_distance on either side --------------------------
// A workgroup keeps the values of its heads in shared memory, kPad of the outermost ones on either side: a 64 x 32 block that
// touches the inner range reads them at one address per lane plus constants; a block that does not adds one constant.
struct Bias {
  const void* table;       // [n_buckets, H], f32 or bf16; null: no bias
  const int* bucket_of;    // [2 max_distance + 1], by key - query + max_distance
  int n_buckets, max_distance, bf16;
};
constexpr int kPad = 96;
__host__ __device__ static inline int bias_row(int max_distance) { return 2 * (max_distance + kPad) + 1; }
__device__ __forceinline__ int bucket(const Bias& b, int rel) {
  const int m = b.max_distance, i = (rel < -m ? -m : rel > m ? m : rel) + m, v = b.bucket_of[i];
  return v < 0 ? 0 : v >= b.n_buckets ? b.n_buckets - 1 : v;
}
// in units of the exponent to base 2.  Finite values stay finite (those beyond 2.358e38 count as that): a row that sees only a
// mask's lowest value still has its softmax
__device__ __forceinline__ float to_log2(float t) {
  const float v = t * kLog2e;
  return fabsf(t) <= kMaxFinite ? fminf(fmaxf(v, -kMaxFinite), kMaxFinite) : v;
}
// two values at once (a trip to memory each, if one waited for the other)
__device__ __forceinline__ void bias_log2(const Bias& b, size_t at0, size_t at1, float& v0, float& v1) {
  float t0, t1;
  if (b.bf16) {
    const __bf16 *p = static_cast<const __bf16*>(b.table), u0 = p[at0], u1 = p[at1];
    t0 = (float)u0;
    t1 = (float)u1;
  } else {
    t0 = static_cast<const float*>(b.table)[at0];
    t1 = static_cast<const float*>(b.table)[at1];
  }
  v0 = to_log2(t0);
  v1 = to_log2(t1);
}

template <int NT>
__device__ __forceinline__ void fill_bias(const Bias& b, int H, int head0, int heads, float* lds, int tid) {
  const int w = bias_row(b.max_distance);
  for (int x = tid; x < w; x += 2 * NT) {
    const int y = min(x + NT, w - 1);      // (the last value may be written twice)
    const int bx = bucket(b, x - b.max_distance - kPad), by = bucket(b, y - b.max_distance - kPad);
    for (int g = 0; g < heads; g++) {
      float u, v;
      bias_log2(b, (size_t)bx * H + head0 + g, (size_t)by * H + head0 + g, u, v);
      lds[g * w + x] = u;
      lds[g * w + y] = v;
    }
  }
}

int check(const ait_packed_attn* p);
// a launch's work items are counted in 32 bits
static inline bool launchable(long long workgroups, int threads) { return workgroups * threads < (1LL << 32) && workgroups < (1LL << 31); }
int check_strides(const ait_packed_attn* p, const void* base, long long row, long long head, long long rows);

}  // namespace ait_packed
