// Attention over packed sequences, forward and backward (gfx950).
//
//   row p of sequence i (sq queries, sk keys) sees keys [0, hi(p)):
//     hi(p) = sk, or causal min(sk, p + 1 + sk - sq), none if that is <= 0
//   S = scale Q K^T, P = softmax(S), O = P V (0 where no key is seen)
//   lse = log2 sum 2^(S log2 e), kept for the backward
//   D = sum_d dO O, dV = P^T dO, dS = P (dO V^T - D)
//   (with O as it was before its rounding: the forward of a training step
//   leaves what the rounding took off; without it D's error is the largest of
//   the gradients of Q and K, 2.8e-3 against 2.4e-3 of them in bf16)
//   dQ = scale dS K, dK = scale dS^T Q, both sums over the group's heads
//
// Rounded to 16 bits are P before its products with V and dO, and dS before its
// own, because the matrix unit takes nothing wider at this rate; all sums stay
// in 32 bits.  Against a form that rounds only at the end the output's error is
// 1.1 times as large and the gradients' 1.45 times (1.8e-3 for 1.6e-3 and 2.4e-3
// for 1.7e-3 in bf16); two parts of 16 bits each would take it back for three
// products more of the backward's seven, and one of the forward's two.
//
// Times of single kernels below are the shortest of 20 under the profiler, some
// 5% above what they take in passes without it.
//
// The stream's sequences are given on the device, so the grid has as many
// tiles as could be needed and a block finds its own (sequence, tile) by
// adding up the sequences' tile counts.  No tile holds rows of two
// sequences: nothing of one request reaches another's sums, NaN included.
// The places before the first and behind the last sequence are taken as
// sequences without keys, so they come out as zeros.

#include "attn_tiles.h"

#include <algorithm>

namespace {

constexpr int BM = 128;     // rows of a block: four waves of 32
constexpr int BN = 64;      // rows of a tile in LDS
constexpr int BLOCK = 256;
constexpr float LOG2E = 1.4426950408889634f;

struct Strides {
  long t, b, h;             // elements; the head's elements are adjacent
};

struct Packing {
  const int* cu_q;          // [n + 1]
  const int* cu_k;
  int n, tq, tk;            // sequences, places of the two streams
};

struct Span {
  int q0, sq, k0, sk;       // the sequence's places and lengths
  int tile;                 // the block's tile of it
};

__device__ __forceinline__ int bounded(const int* cu, int i, int lo, int hi) {
  return max(lo, min(cu[i], hi));
}

// sequence i - 1 of the stream; 0 and n + 1 are what lies before and behind
__device__ __forceinline__ void span_of(const int* cu, int n, int total, int i,
                                        int& from, int& len) {
  from = i == 0 ? 0 : bounded(cu, i - 1, 0, total);
  const int to = i > n ? total : bounded(cu, i, from, total);
  len = max(to - from, 0);
}

// The wave's sum, as a scalar.  Moves within the vector unit: through LDS the
// dozen sums of find_span() took longer than a tile's products.
__device__ __forceinline__ int wave_sum(int v) {
#define ADD(CTRL, ROWS) \
  v += __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false)
  ADD(0x111, 0xf);      // row_shr 1, 2, 4, 8: sums of 16 in their last lane
  ADD(0x112, 0xf);
  ADD(0x114, 0xf);
  ADD(0x118, 0xf);
  ADD(0x142, 0xa);      // row_bcast 15 into rows 1 and 3, 31 into 2 and 3
  ADD(0x143, 0xc);
#undef ADD
  return __builtin_amdgcn_readlane(v, WAVE - 1);
}

// The `slot`-th tile of BM rows of the query (or key) stream.
//
// Under a causal mask a tile of queries has the more keys the further back it
// lies, one of keys the more queries the further in front.  Where the
// sequences fit a wave's lanes, tiles are handed out by that: level L holds
// the L-th tile (from the other end for keys) of every sequence that has one,
// and the highest level goes first, so that the last blocks to start are the
// shortest.  8 documents of 45 to 2048 tokens, 16 heads of 128, forward: 94 us
// in stream order, 82 so, with the CUs busy 76% of the time.
template <bool KEYS>
__device__ __forceinline__ bool find_span(const Packing& pk, int slot,
                                          int lane, Span& s) {
  const int* cu = KEYS ? pk.cu_k : pk.cu_q;
  const int total = KEYS ? pk.tk : pk.tq;
  for (int base = 0; base < pk.n + 2; base += WAVE) {
    const int i = base + lane;
    int from = 0, len = 0;
    if (i < pk.n + 2) span_of(cu, pk.n, total, i, from, len);
    const int tiles = (len + BM - 1) / BM;
    int w;                    // the lane whose sequence it is
    if (pk.n + 2 <= WAVE) {
      if (slot >= wave_sum(tiles)) return false;
      // the highest level at or above which there are more tiles than `slot`
      int lo = 0, hi = total / BM + 1;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (wave_sum(max(0, tiles - mid)) > slot) lo = mid; else hi = mid;
      }
      slot -= wave_sum(max(0, tiles - lo - 1));
      const unsigned long long in = __ballot(tiles > lo);
      const int rank = __popcll(in & ((1ull << lane) - 1));
      w = __ffsll((unsigned long long)__ballot(tiles > lo && rank == slot)) -
          1;
      s.tile = KEYS ? __builtin_amdgcn_readlane(tiles, w) - 1 - lo : lo;
    } else {
      int upto = tiles;
#pragma unroll
      for (int off = 1; off < WAVE; off <<= 1) {
        const int x = __shfl_up(upto, off, WAVE);
        if (lane >= off) upto += x;
      }
      const unsigned long long hit = __ballot(upto > slot);
      if (!hit) {
        slot -= __builtin_amdgcn_readlane(upto, WAVE - 1);
        continue;
      }
      w = __ffsll((unsigned long long)hit) - 1;
      s.tile = slot - (__builtin_amdgcn_readlane(upto, w) -
                       __builtin_amdgcn_readlane(tiles, w));
    }
    const int seq = base + w;
    const int f = __builtin_amdgcn_readlane(from, w);
    const int l = __builtin_amdgcn_readlane(len, w);
    int of = 0, ol = 0;       // of the other stream
    if (seq > 0 && seq <= pk.n) {
      if (pk.cu_q == pk.cu_k && pk.tq == pk.tk) of = f, ol = l;
      else if (KEYS) span_of(pk.cu_q, pk.n, pk.tq, seq, of, ol);
      else span_of(pk.cu_k, pk.n, pk.tk, seq, of, ol);
    }
    s.q0 = KEYS ? of : f;
    s.sq = KEYS ? ol : l;
    s.k0 = KEYS ? f : of;
    s.sk = KEYS ? l : ol;
    return true;
  }
  return false;
}

// keys that row p of the sequence sees
template <bool CAUSAL>
__device__ __forceinline__ int keys_of(const Span& s, int p) {
  return CAUSAL ? max(0, min(s.sk, p + 1 + s.sk - s.sq)) : s.sk;
}

__device__ __forceinline__ f32x16 zeros16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// head h of the block: heads of one group follow each other in steps of ng,
// so that they run on one XCD (blocks go round the eight) and share its L2
__device__ __forceinline__ int head_of(int x, int ng, int rep) {
  return (x % ng) * rep + x / ng;
}

// ------------------------------------------------------------------ forward
// A wave holds 32 rows of Q as the right operand of S^T = K Q^T, and P^T, which
// that leaves in its registers, is the right operand of O^T = V^T P^T; the four
// waves share the tiles of K and V, of which the next one comes into the other
// of two images while one is used.  Two blocks of 187 registers at D = 128 and
// four of 122 at 64 run on a CU, each at another place of its loop, so that one
// does its exponentials beside the other's products.
//
// At D = 64 the vector unit bounds it (active 69% of the time, the matrix unit
// busy 31%): an element takes some six of its instructions and two products; 15
// documents of 1 to 2048 tokens, 32 heads, take 161 us, 630 TFLOP/s.  At 128
// both are near (51% and 48%): 8192 + 5003 + 3001 + 188 tokens, 32 heads, fp16
// take 890 us without the profiler, 930 TFLOP/s, and under it the clock falls
// to 1.6 GHz, where shorter work runs at 2.1: that is the power's doing.  Where
// sequences are few and uneven, the longest tiles are more than a CU's share
// of the work: ten prompts of 0 to 2048 tokens, 32 heads, 89 us (680; CUs busy
// 81% of the time), eight documents of 45 to 2048, 16 heads, 82 us (640).
//
// Taken back: 64 rows a wave at D = 64 (half the reads of K and V: equal, for
// short prompts 9.0 us against 7.5), the next tile's scores beside this one's
// exponentials (equal at 128, where nothing spills, and 155 us -> 165 at 64), a
// higher priority for the products (equal), images of K and V apart (equal).
template <class T, int D, bool CAUSAL, int HALVES>
__global__ __launch_bounds__(BLOCK * HALVES, 2) void packed_fwd_kernel(
    const unsigned short* __restrict__ q, const unsigned short* __restrict__ k,
    const unsigned short* __restrict__ v, unsigned short* __restrict__ o,
    unsigned short* __restrict__ low, float* __restrict__ lse, Packing pk,
    int b, int nh, int ng, float c, Strides qs, Strides ks, Strides vs) {
  constexpr int IMG = 2 * BN * D;
  __shared__ __attribute__((aligned(16))) unsigned short kv0_lds[HALVES * IMG];
  __shared__ __attribute__((aligned(16))) unsigned short kv1_lds[HALVES * IMG];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
  const int half = HALVES == 1 ? 0
                               : __builtin_amdgcn_readfirstlane(tid >> 8);
  const int h = lane >> 5, n = lane & 31;
  const Places<D> at_lane(lane);
  Span s;
  const unsigned x = blockIdx.x % (b * nh), slot = blockIdx.x / (b * nh);
  if (!find_span<false>(pk, slot, lane, s)) return;
  const int bi = x / nh, head = head_of(x % nh, ng, nh / ng);
  const int hk = head / (nh / ng);

  const int p0 = s.tile * BM + wave * 32;       // the wave's first row
  const int p = p0 + n;                         // the lane's row
  const bool mine = p < s.sq;
  const long row = s.q0 + min(p, s.sq - 1);
  constexpr int NF = D / 16, ND = D / 32;
  typename T::x8 qf[NF];
  {
    const unsigned short* src = q + row * qs.t + bi * qs.b + head * qs.h;
#pragma unroll
    for (int f = 0; f < NF; ++f)
      qf[f] = *(const typename T::x8*)(src + 16 * f + 8 * h);
  }
  const int most = keys_of<CAUSAL>(s, min(s.tile * BM + BM, s.sq) - 1);
  const int wave_most = keys_of<CAUSAL>(s, min(p0 + 31, s.sq - 1));
  const int wave_least = keys_of<CAUSAL>(s, min(p0, s.sq - 1));
  const int lane_most = keys_of<CAUSAL>(s, min(p, s.sq - 1));
  const int tiles = (most + BN - 1) / BN;
  const unsigned short* kp = k + s.k0 * ks.t + bi * ks.b + hk * ks.h;
  const unsigned short* vp = v + s.k0 * vs.t + bi * vs.b + hk * vs.h;

  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = zeros16();
  float m = -INFINITY, ms = 0.f, l = 0.f;
  auto fetch = [&](int t, unsigned short* img) {
    if (HALVES > 1 && t >= tiles) return;
    const int last = s.sk - 1 - t * BN;
    load_tile<D, BN, 4>(img, kp + (long)t * BN * ks.t, ks.t, last, wave, lane);
    load_tile<D, BN, 4>(img + BN * D, vp + (long)t * BN * vs.t, vs.t, last,
                        wave, lane);
  };
  auto step = [&](int t, const unsigned short* img) {
    const int at = t * BN;
    if (p0 >= s.sq || at >= wave_most) return;
    f32x16 st[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      st[u] = zeros16();
#pragma unroll
      for (int f = 0; f < NF; ++f)
        st[u] = T::mfma32(read_rows<T, D>(img, 32 * u, f, at_lane), qf[f],
                            st[u]);
    }
    reads_ahead<2 * NF, 1>();
    if (at + BN > wave_least) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (at + 32 * u + 16 * (r >> 3) + 8 * h + (r & 7) >= lane_most)
            st[u][r] = -INFINITY;
    }
    float mt = st[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) mt = fmaxf(mt, st[u][r]);
    mt = half_max(mt) * c;
    // The maximum moves whenever it can: the largest weight is then one, with
    // nothing to round.  Let lag behind by up to 2^8 it would move seldom, for
    // 5% of the forward's time, and the output's error be 1.30 of its last
    // rounding's rather than 1.13 (2048 tokens, D = 64).  With and without
    // gradients alike: a recomputed forward gives the same bits.
    if (__any(mt > m)) {
      const float mn = fmaxf(m, mt);
      const float a = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      ms = mn == -INFINITY ? 0.f : mn;
      l *= a;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= a;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        st[u][r] = __builtin_amdgcn_exp2f(fmaf(st[u][r], c, -ms));
        l += st[u][r];
      }
    const unsigned short* vi = img + BN * D;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const typename T::x8 pf = pack8<T>(st[u], 8 * x);
#pragma unroll
        for (int i = 0; i < ND; ++i)
          acc[i] = T::mfma32(read_cols<T, D>(vi, 32 * u + 16 * x, i, at_lane),
                             pf, acc[i]);
      }
    reads_ahead<4 * ND, 2>();
  };
  // one tile is used while the next one comes in; each half of the waves has
  // every other tile
  unsigned short* const img0 = kv0_lds + half * IMG;
  unsigned short* const img1 = kv1_lds + half * IMG;
  auto turn = [&](int t, unsigned short* img, unsigned short* next) {
    __builtin_amdgcn_s_waitcnt(0x0f70);         // vmcnt(0)
    __syncthreads();
    if (t + HALVES < tiles) fetch(t + HALVES + half, next);
    step(t + half, img);
  };
  if (tiles > 0) fetch(half, img0);
  for (int t = 0; t < tiles; t += 2 * HALVES) {
    turn(t, img0, img1);
    if (t + HALVES < tiles) turn(t + HALVES, img1, img0);
  }
  if constexpr (HALVES == 2) {
    // the second half's sums, handed over through the images
    static_assert(sizeof(kv0_lds) >= 2 * (16 * ND + 2) * WAVE * 4,
                  "room for them");
    constexpr int EACH = (16 * ND + 2) * WAVE;
    float* to = (float*)(wave < 2 ? kv0_lds : kv1_lds) + (wave & 1) * EACH +
                lane;
    __syncthreads();
    if (half) {
      to[0] = m;
      to[WAVE] = l;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) to[(2 + i * 16 + r) * WAVE] = acc[i][r];
    }
    __syncthreads();
    if (half) return;
    const float other = to[0], top = fmaxf(m, other);
    const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    const float e = other == -INFINITY ? 0.f
                                       : __builtin_amdgcn_exp2f(other - top);
    m = top;
    l = l * a + to[WAVE] * e;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[i][r] = acc[i][r] * a + to[(2 + i * 16 + r) * WAVE] * e;
  }
  if (!mine) return;
  l = half_sum(l);
  const float by = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (h == 0 && lse)
    lse[((long)bi * nh + head) * pk.tq + s.q0 + p] =
        l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
  const long at = ((row * b + bi) * nh + head) * D;
  if (low) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
      store_cols<T, true>(o + at + 32 * i, acc[i], by, h, low + at + 32 * i);
  } else {
#pragma unroll
    for (int i = 0; i < ND; ++i)
      store_cols<T>(o + at + 32 * i, acc[i], by, h);
  }
}

// ----------------------------------------------------------------- backward
// dQ: rows of queries, over their keys, as in the forward.  S and dP are found
// again; the other kernel's blocks could add dQ up, but only by atomics, whose
// order changes results.  Each row's D is found on the way, and left for the
// other kernel (a kernel of its own: backward 247 us, so 235).
//
// Eight documents of 45 to 2048 tokens, 16 heads of 128: 110 us, 710 TFLOP/s;
// fifteen of 1 to 2048, 32 heads of 64: 215 us, 710.  The matrix unit is busy
// 33% and 38% of the time, the vector unit active 26% and 51%, and the waves
// wait 28% and 34% of theirs; two waves on a SIMD do not cover more of each
// other's waits.  Eight waves on a tile there keep all of a CU's waves in step:
// the backward takes 280 us for 244, and 587 for 466.
template <class T, int D, bool CAUSAL, int HALVES>
__global__ __launch_bounds__(BLOCK * HALVES, 2) void packed_bwd_dq_kernel(
    const unsigned short* __restrict__ q, const unsigned short* __restrict__ k,
    const unsigned short* __restrict__ v,
    const unsigned short* __restrict__ dout,
    const unsigned short* __restrict__ o,
    const unsigned short* __restrict__ low, const float* __restrict__ lse,
    float* __restrict__ dot, unsigned short* __restrict__ dq, Packing pk,
    int b, int nh, int ng, float scale, Strides qs, Strides ks, Strides vs,
    Strides os) {
  constexpr int IMG = 2 * BN * D;
  __shared__ __attribute__((aligned(16))) unsigned short kv0_lds[HALVES * IMG];
  __shared__ __attribute__((aligned(16))) unsigned short kv1_lds[HALVES * IMG];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
  const int half = HALVES == 1 ? 0
                               : __builtin_amdgcn_readfirstlane(tid >> 8);
  const int h = lane >> 5, n = lane & 31;
  const Places<D> at_lane(lane);
  Span s;
  const unsigned x = blockIdx.x % (b * nh), slot = blockIdx.x / (b * nh);
  if (!find_span<false>(pk, slot, lane, s)) return;
  const int bi = x / nh, head = head_of(x % nh, ng, nh / ng);
  const int hk = head / (nh / ng);
  const float c = scale * LOG2E;

  const int p0 = s.tile * BM + wave * 32;
  const int p = p0 + n;
  const long row = s.q0 + min(p, s.sq - 1);
  constexpr int NF = D / 16, ND = D / 32;
  typename T::x8 qf[NF], df[NF];
  {
    const unsigned short* src = q + row * qs.t + bi * qs.b + head * qs.h;
    const unsigned short* dsrc = dout + row * os.t + bi * os.b + head * os.h;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      qf[f] = *(const typename T::x8*)(src + 16 * f + 8 * h);
      df[f] = *(const typename T::x8*)(dsrc + 16 * f + 8 * h);
    }
  }
  const long stat = ((long)bi * nh + head) * pk.tq + row;
  const float rl = lse[stat];
  float rd = 0.f;
  {
    const long at = ((row * b + bi) * nh + head) * D + 8 * h;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const typename T::x8 e = *(const typename T::x8*)(o + at + 16 * f);
      const typename T::x8 r = *(const typename T::x8*)(low + at + 16 * f);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        rd += ((float)e[i] + (float)r[i]) * (float)df[f][i];
    }
    rd = half_sum(rd);
    if (h == 0 && half == 0 && p < s.sq) dot[stat] = rd;
  }
  const int most = keys_of<CAUSAL>(s, min(s.tile * BM + BM, s.sq) - 1);
  const int wave_most = keys_of<CAUSAL>(s, min(p0 + 31, s.sq - 1));
  const int wave_least = keys_of<CAUSAL>(s, min(p0, s.sq - 1));
  const int lane_most = keys_of<CAUSAL>(s, min(p, s.sq - 1));
  const int tiles = (most + BN - 1) / BN;
  const unsigned short* kp = k + s.k0 * ks.t + bi * ks.b + hk * ks.h;
  const unsigned short* vp = v + s.k0 * vs.t + bi * vs.b + hk * vs.h;

  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = zeros16();

  auto fetch = [&](int t, unsigned short* img) {
    if (HALVES > 1 && t >= tiles) return;
    const int last = s.sk - 1 - t * BN;
    load_tile<D, BN, 4>(img, kp + (long)t * BN * ks.t, ks.t, last, wave, lane);
    load_tile<D, BN, 4>(img + BN * D, vp + (long)t * BN * vs.t, vs.t, last,
                        wave, lane);
  };
  auto step = [&](int t, const unsigned short* img) {
    const int at = t * BN;
    if (p0 >= s.sq || at >= wave_most) return;
    const bool edge = at + BN > wave_least;
    const unsigned short* vi = img + BN * D;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x16 st = zeros16(), dp = zeros16();
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        st = T::mfma32(read_rows<T, D>(img, 32 * u, f, at_lane), qf[f], st);
        dp = T::mfma32(read_rows<T, D>(vi, 32 * u, f, at_lane), df[f], dp);
      }
      reads_ahead<2 * NF, 1>();
#pragma unroll
      for (int r = 0; r < 16; ++r)
        dp[r] = __builtin_amdgcn_exp2f(fmaf(st[r], c, -rl)) * (dp[r] - rd);
      if (edge) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (at + 32 * u + 16 * (r >> 3) + 8 * h + (r & 7) >= lane_most)
            dp[r] = 0.f;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const typename T::x8 sf = pack8<T>(dp, 8 * x);
#pragma unroll
        for (int i = 0; i < ND; ++i)
          acc[i] = T::mfma32(
              read_cols<T, D>(img, 32 * u + 16 * x, i, at_lane), sf, acc[i]);
      }
      reads_ahead<2 * ND, 2>();
    }
  };
  // one tile is used while the next one comes in; each half of the waves has
  // every other tile
  unsigned short* const img0 = kv0_lds + half * IMG;
  unsigned short* const img1 = kv1_lds + half * IMG;
  auto turn = [&](int t, unsigned short* img, unsigned short* next) {
    __builtin_amdgcn_s_waitcnt(0x0f70);         // vmcnt(0)
    __syncthreads();
    if (t + HALVES < tiles) fetch(t + HALVES + half, next);
    step(t + half, img);
  };
  if (tiles > 0) fetch(half, img0);
  for (int t = 0; t < tiles; t += 2 * HALVES) {
    turn(t, img0, img1);
    if (t + HALVES < tiles) turn(t + HALVES, img1, img0);
  }
  if constexpr (HALVES == 2) {
    static_assert(sizeof(kv0_lds) >= 2 * 16 * ND * WAVE * 4, "room for them");
    float* to = (float*)(wave < 2 ? kv0_lds : kv1_lds) +
                (wave & 1) * 16 * ND * WAVE + lane;
    __syncthreads();
    if (half) {
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) to[(i * 16 + r) * WAVE] = acc[i][r];
    }
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] += to[(i * 16 + r) * WAVE];
  }
  if (p >= s.sq) return;
  unsigned short* dst = dq + ((row * b + bi) * nh + head) * D;
#pragma unroll
  for (int i = 0; i < ND; ++i) store_cols<T>(dst + 32 * i, acc[i], scale, h);
}

// dK and dV: rows of keys, over the queries that see them, for each head of
// the group in turn (one block sums them all, so no atomics).
//
// At D = 128 a wave's two sums alone take 128 registers.  So that two waves
// still fit a SIMD, K's and V's fragments stay in LDS, and eight waves work on
// the 128 keys: four on the first 32 queries of a tile, four on the others,
// whose sums are added at the end (one wave a SIMD: 228 us for 165 then, and
// 546 for 361 at D = 64).
//
// The same documents as for dQ: 153 us, 680 TFLOP/s, and 274 us, 740.  The
// matrix unit is busy 31% and 37% of the time, the vector unit active 25% and
// 39%, and the waves wait 40% and 31% of theirs.  Each 32 x 32 tile reads Q and
// dO along both axes, and at 128 K and V too, from LDS, without conflicts.
//
// Eight waves keep in step, which costs time; at D = 64, where K and V are in
// registers, two blocks of four waves fit a CU instead, and are taken (MANY)
// where tiles are many.
// Three such blocks, K in LDS for that: eight sequences of 1024 tokens 101 ->
// 96 us, the fifteen documents 444 -> 468, 8192 + 5003 + 3001 + 188 1620 ->
// 1740; not kept.
template <int D, bool MANY>
struct Dkv {
  static constexpr int HALVES = MANY ? 1 : 2;
  static constexpr int BQ = D == 128 ? 64 : 64 * HALVES;   // queries of a tile
  static constexpr int WAVES = 4 * HALVES;
};

template <int D>
constexpr long SHARE = BM * D / 4;    // of four numbers: one tile's dK (or dV)

template <class T, int D, bool CAUSAL, bool MANY>
__global__ __launch_bounds__((Dkv<D, MANY>::WAVES * 64), 2)
void packed_bwd_dkv_kernel(
    const unsigned short* __restrict__ q, const unsigned short* __restrict__ k,
    const unsigned short* __restrict__ v,
    const unsigned short* __restrict__ dout, const float* __restrict__ lse,
    const float* __restrict__ dot, unsigned short* __restrict__ dk,
    unsigned short* __restrict__ dv, float* __restrict__ sums, int shares,
    Packing pk, int b, int nh, int ng, float scale, Strides qs, Strides ks,
    Strides vs, Strides os) {
  constexpr int HALVES = Dkv<D, MANY>::HALVES;
  constexpr int WAVES = Dkv<D, MANY>::WAVES, BQ = Dkv<D, MANY>::BQ;
  constexpr bool KV_LDS = D == 128;
  // Q, dO, then the rows' lse and D
  constexpr int IMG = 2 * BQ * D + 4 * BQ;
  __shared__ __attribute__((aligned(16))) unsigned short qd0_lds[IMG];
  __shared__ __attribute__((aligned(16))) unsigned short qd1_lds[IMG];
  __shared__ __attribute__((aligned(16)))
  unsigned short kv_lds[KV_LDS ? 2 * BM * D : 8];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = wave & 3, half = wave >> 2;
  const int h = lane >> 5, n = lane & 31;
  const Places<D> at_lane(lane);
  Span s;
  const unsigned x = blockIdx.x % (b * ng * shares);
  if (!find_span<true>(pk, blockIdx.x / (b * ng * shares), lane, s)) return;
  const int hk = x % ng, bi = x / ng % b, share = x / ng / b, rep = nh / ng;
  const float c = scale * LOG2E;

  const int j0 = s.tile * BM + part * 32;       // the wave's first key
  const int j = j0 + n;                         // the lane's key
  const long row = s.k0 + min(j, s.sk - 1);
  constexpr int NF = D / 16, ND = D / 32;
  typename T::x8 kf[KV_LDS ? 1 : NF], vf[KV_LDS ? 1 : NF];
  if constexpr (KV_LDS) {
    const long from = s.k0 + s.tile * BM;
    const int last = s.sk - 1 - s.tile * BM;
    load_tile<D, BM, WAVES>(kv_lds, k + from * ks.t + bi * ks.b + hk * ks.h,
                            ks.t, last, wave, lane);
    load_tile<D, BM, WAVES>(kv_lds + BM * D,
                            v + from * vs.t + bi * vs.b + hk * vs.h, vs.t,
                            last, wave, lane);
  } else {
    const unsigned short* ksrc = k + row * ks.t + bi * ks.b + hk * ks.h;
    const unsigned short* vsrc = v + row * vs.t + bi * vs.b + hk * vs.h;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      kf[f] = *(const typename T::x8*)(ksrc + 16 * f + 8 * h);
      vf[f] = *(const typename T::x8*)(vsrc + 16 * f + 8 * h);
    }
  }
  const Places<D> kv_lane(lane, false);
  auto k_frag = [&](int f) __attribute__((always_inline)) {
    if constexpr (KV_LDS) return read_rows<T, D>(kv_lds, 32 * part, f, kv_lane);
    else return kf[f];
  };
  auto v_frag = [&](int f) __attribute__((always_inline)) {
    if constexpr (KV_LDS)
      return read_rows<T, D>(kv_lds + BM * D, 32 * part, f, kv_lane);
    else return vf[f];
  };
  // the first query that sees the block's first key
  const int ahead = CAUSAL ? s.sk - s.sq : 0;
  const int first = CAUSAL ? max(0, s.tile * BM - ahead) / BQ : 0;
  const int per = max(0, (s.sq + BQ - 1) / BQ - first);
  // the block's share of the heads' tiles
  const int begin = rep * per * share / shares;
  int left = rep * per * (share + 1) / shares - begin;

  f32x16 ak[ND], av[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) ak[i] = av[i] = zeros16();

  // tile `at` of head hk * rep + r
  auto fetch = [&](int r, int at, unsigned short* img) {
    const int head = hk * rep + r, last = s.sq - 1 - at;
    const unsigned short* qp =
        q + (s.q0 + at) * qs.t + bi * qs.b + head * qs.h;
    const unsigned short* dp =
        dout + (s.q0 + at) * os.t + bi * os.b + head * os.h;
    load_tile<D, BQ, WAVES>(img, qp, qs.t, last, wave, lane);
    load_tile<D, BQ, WAVES>(img + BQ * D, dp, os.t, last, wave, lane);
    // four bytes a lane: the rows' statistics, by one wave each
    constexpr int EACH = BQ / WAVE;
    if (wave < 2 * EACH) {
      const float* src = (wave / EACH ? dot : lse) +
                         ((long)bi * nh + head) * pk.tq + s.q0 + at +
                         min(wave % EACH * WAVE + lane, last);
      __builtin_amdgcn_global_load_lds(
          (global_char*)src,
          (lds_char*)(img + 2 * BQ * D + 2 * WAVE * wave), 4, 0, 0);
    }
  };
  auto part_step = [&](int at, int u, const unsigned short* img)
                       __attribute__((always_inline)) {
    const int a0 = at + 32 * u;
    // no key of the wave is seen by these rows
    if (a0 >= s.sq || (CAUSAL && j0 > a0 + 31 + ahead)) return;
    const unsigned short* di = img + BQ * D;
    const float* sl = (const float*)(img + 2 * BQ * D) + 32 * u + 8 * h;
    const float* sd = sl + BQ;
    f32x16 st = zeros16(), dp = zeros16();
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      st = T::mfma32(read_rows<T, D>(img, 32 * u, f, at_lane), k_frag(f), st);
      dp = T::mfma32(read_rows<T, D>(di, 32 * u, f, at_lane), v_frag(f), dp);
    }
    reads_ahead<2 * NF, KV_LDS ? 2 : 1>();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int y = 16 * (r >> 3) + (r & 7);
      st[r] = __builtin_amdgcn_exp2f(fmaf(st[r], c, -sl[y]));
      dp[r] = st[r] * (dp[r] - sd[y]);
    }
    if (a0 + 32 > s.sq || (CAUSAL && j0 + 31 > a0 + ahead)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int y = a0 + 16 * (r >> 3) + 8 * h + (r & 7);
        if (y >= s.sq || (CAUSAL && j > y + ahead)) st[r] = dp[r] = 0.f;
      }
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const typename T::x8 pf = pack8<T>(st, 8 * y);
      const typename T::x8 sf = pack8<T>(dp, 8 * y);
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        av[i] = T::mfma32(read_cols<T, D>(di, 32 * u + 16 * y, i, at_lane),
                          pf, av[i]);
        ak[i] = T::mfma32(read_cols<T, D>(img, 32 * u + 16 * y, i, at_lane),
                          sf, ak[i]);
      }
    }
    reads_ahead<4 * ND, 2>();
  };
  // one tile is used while the next one comes in
  int r1 = left ? begin / per : 0;    // the next tile's head and number
  int t1 = left ? begin % per : 0;
  auto turn = [&](int at, unsigned short* img, unsigned short* next)
                  __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0f70);         // vmcnt(0)
    __syncthreads();
    if (++t1 == per) {
      t1 = 0;
      ++r1;
    }
    if (--left) fetch(r1, (first + t1) * BQ, next);
    if (j0 >= s.sk) return;
#pragma unroll
    for (int u = 0; u < BQ / 32 / HALVES; ++u)
      part_step(at, HALVES * u + half, img);
  };
  if (left) fetch(r1, (first + t1) * BQ, qd0_lds);
  while (left) {
    turn((first + t1) * BQ, qd0_lds, qd1_lds);
    if (left) turn((first + t1) * BQ, qd1_lds, qd0_lds);
  }
  if constexpr (HALVES == 2) {
    // the second half's sums, handed over through the images
    static_assert(sizeof(qd0_lds) >= 2 * 16 * ND * WAVE * 4, "room for them");
    float* to = (float*)(part < 2 ? qd0_lds : qd1_lds) +
                (part & 1) * 16 * ND * WAVE + lane;
    auto hand_over = [&](f32x16(&acc)[ND]) __attribute__((always_inline)) {
      __syncthreads();
      if (half) {
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) to[(i * 16 + r) * WAVE] = acc[i][r];
      }
      __syncthreads();
      if (!half) {
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] += to[(i * 16 + r) * WAVE];
      }
    };
    hand_over(ak);
    hand_over(av);
    if (half) return;
  }
  if (shares > 1) {           // left as the registers hold them
    const long unit = (long)(blockIdx.x / (b * ng * shares)) * (b * ng) + bi *
                      ng + hk;
    f32x4* to = (f32x4*)sums + (unit * shares + share) * 2 * SHARE<D> +
                part * 4 * ND * WAVE + lane;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const f32x4 a = {ak[i][4 * y], ak[i][4 * y + 1], ak[i][4 * y + 2],
                         ak[i][4 * y + 3]};
        const f32x4 v = {av[i][4 * y], av[i][4 * y + 1], av[i][4 * y + 2],
                         av[i][4 * y + 3]};
        to[(4 * i + y) * WAVE] = a;
        to[SHARE<D> + (4 * i + y) * WAVE] = v;
      }
    return;
  }
  if (j >= s.sk) return;
  const long at = ((row * b + bi) * ng + hk) * D;
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    store_cols<T>(dk + at + 32 * i, ak[i], scale, h);
    store_cols<T>(dv + at + 32 * i, av[i], 1.f, h);
  }
}

// The shares' sums of a tile's dK and dV, added up in order: a wave for 32 keys
// and 32 columns of one of them.
template <class T, int D>
__global__ __launch_bounds__(BLOCK) void packed_bwd_add_kernel(
    const float* __restrict__ sums, unsigned short* __restrict__ dk,
    unsigned short* __restrict__ dv, int shares, Packing pk, int b, int ng,
    float scale) {
  constexpr int ND = D / 32;
  const int lane = threadIdx.x & 63;
  const int part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = blockIdx.y % ND, second = blockIdx.y / ND;
  const f32x4* from = (const f32x4*)sums +
                      ((long)blockIdx.x * shares * 2 + second) * SHARE<D> +
                      (part * ND + i) * 4 * WAVE + lane;
  Span s;
  const unsigned x = blockIdx.x % (b * ng);
  if (!find_span<true>(pk, blockIdx.x / (b * ng), lane, s)) return;
  f32x16 acc = zeros16();
#pragma unroll 4
  for (int k = 0; k < shares; ++k)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const f32x4 z = from[k * 2 * SHARE<D> + y * WAVE];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[4 * y + e] += z[e];
    }
  const int j = s.tile * BM + part * 32 + (lane & 31);
  if (j >= s.sk) return;
  store_cols<T>((second ? dv : dk) +
                    ((long)(s.k0 + j) * b * ng + x) * D + 32 * i,
                acc, second ? 1.f : scale, lane >> 5);
}

// each sequence may end in a part of a tile
dim3 grid_for(long heads, int total, int n) {
  const long blocks = heads * ((long)total / BM + n + 2);
  if (blocks * 512 >= 1l << 32)
    throw std::runtime_error("packed attention: too many tiles for one launch");
  return dim3((unsigned)blocks);
}

}  // namespace

#define PACKED_MASK(RUN, T, D)                       \
  do {                                               \
    if (causal) RUN(T, D, true); else RUN(T, D, false); \
  } while (0)
#define PACKED_DISPATCH(RUN)                         \
  do {                                               \
    if (fp16) {                                      \
      if (d == 128) PACKED_MASK(RUN, Fp16, 128);     \
      else PACKED_MASK(RUN, Fp16, 64);               \
    } else {                                         \
      if (d == 128) PACKED_MASK(RUN, Bf16, 128);     \
      else PACKED_MASK(RUN, Bf16, 64);               \
    }                                                \
  } while (0)

// Tiles of a stream, where every other sequence ends in a part of one.
static long tiles_of(int n, int total, long heads) {
  return heads * (total / BM + (n + 1) / 2);
}

// Whether a tile of queries has eight waves, four for every other tile of keys,
// so that its block is done in half the time: where there are hardly more than
// two blocks for each of 256 CUs, and sequences are not short.  Forward and
// dQ, us, with four waves and with eight: 2048 tokens, 16 heads of 128, 272
// blocks, 46 + 46 and 39 + 40; 4096 tokens, 8 heads, 264, 82 + 81 and 67 + 66,
// 16 heads, 528, 98 + 95 and 85 + 78; two of 2048, 16 heads, 528, 53 + 52 and
// 51 + 49; 1500 + 900 tokens, 32 heads of 64, 608, 29 + 36 and 32 + 39; five
// of 310 tokens in all 7.0 and 7.7.  At D = 64 a prompt: 2048 tokens, 16 heads,
// 34 and 28, 4096 tokens, 8 heads, 59 and 48, 16 heads 65 and 55, two of 2048
// 35 and 33, 1500 + 900 tokens 26 and 21, and a whole pass with gradients 116
// and 101, 196 and 162, 242 and 219, 137 and 130, 95 and 82; 600 + 600 tokens
// 13 and 11.5, with gradients 81 in both.
static bool in_halves(int n, int tq, int tk, int b, int nh) {
  return tiles_of(n, tq, (long)b * nh) <= 576 && tk / std::max(n, 1) >= 512;
}

void launch_packed_attn_fwd(const void* q, const void* k, const void* v,
                            void* o, void* low, float* lse, const int* cu_q,
                            const int* cu_k, int n, int tq, int tk, int b,
                            int nh, int ng, int d, float scale, bool causal,
                            bool fp16, const long* qs, const long* ks,
                            const long* vs, hipStream_t stream) {
  const Packing pk = {cu_q, cu_k, n, tq, tk};
  const dim3 grid = grid_for((long)b * nh, tq, n);
#define LAUNCH(T, DD, CC, HALVES)                                           \
  hipLaunchKernelGGL((packed_fwd_kernel<T, DD, CC, HALVES>), grid,          \
                     dim3(BLOCK * HALVES), 0, stream,                       \
                     (const unsigned short*)q, (const unsigned short*)k,    \
                     (const unsigned short*)v, (unsigned short*)o,          \
                     (unsigned short*)low, lse, pk, b, nh, ng,              \
                     scale * LOG2E, Strides{qs[0], qs[1], qs[2]},           \
                     Strides{ks[0], ks[1], ks[2]},                          \
                     Strides{vs[0], vs[1], vs[2]})
#define RUN(T, DD, CC)                                                      \
  do {                                                                      \
    if (halves) LAUNCH(T, DD, CC, 2); else LAUNCH(T, DD, CC, 1);            \
  } while (0)
  const bool halves = in_halves(n, tq, tk, b, nh);
  PACKED_DISPATCH(RUN);
#undef RUN
#undef LAUNCH
  HIP_CHECK_LAUNCH();
}


// From so many blocks on, three for each of 256 CUs, four waves do at D = 64.
// Backward with eight and four waves, us, 16 heads: 4096 tokens in two
// sequences, 528 blocks, 99 and 108, 6144 in three, 800 blocks, 132 and 121;
// 1024 in each of eight, 1088, 110 and 100; 32 heads, 300 in each of twelve,
// 1088, 75 and 60; the fifteen documents, 1120, 467 and 444.  The rule does not
// look at lengths, for which few long sequences pay: 32/8 heads, 8192 + 5003
// tokens, 832 blocks, 1435 and 1508.
static constexpr long FOUR_WAVES = 768;

// Into how many shares a tile's work for dK and dV is cut, so that there are
// two blocks for each of 256 CUs (of a causal mask's tiles the first has twice
// the average to do), but none of fewer than two tiles of queries; where every
// CU has a block already, only long sequences are.  Sequences are taken to be
// of one length.  The shares' sums are written and read once more, in 32 bits,
// in at most ROOM floats (134 MB).
//
// Backward in one share and so, us: 4096 tokens, 32/8 heads of 128 655 and 502
// (four shares: 522), of 64 370 and 283; 16384 tokens, 8/2 heads of 128 2540
// and 1850; 1024 tokens, 32/8 heads of 128 151 and 84; 8192 tokens, 8/1 heads
// of 128 1950 and 590; 4096 tokens, 8 heads of 128 233 and 212.  In two shares
// all the same: 2048 tokens, 16 heads of 128 126 and 130, five sequences of
// 6921 tokens, 32/8 heads of 64 228 and 256; these two set the bound on tiles
// where every CU has a block.
int packed_attn_shares(int n, int tq, int tk, int b, int nh, int ng, int d,
                       long* floats) {
  constexpr long FILL = 512, LEAST = 2, ROOM = 1l << 25;
  const long blocks = tiles_of(n, tk, (long)b * ng);
  const int bq = d == 128 ? Dkv<128, false>::BQ : Dkv<64, false>::BQ;
  const long tiles = (long)(nh / ng) * (tq / std::max(n, 1)) / (2 * bq);
  long fill = (FILL + blocks / 2) / std::max(blocks, 1l);
  if (blocks >= FILL / 2 && tiles < d * 3 / 16) fill = 1;
  const long each = (long)b * ng * ((long)tk / BM + n + 2) * 2 * BM * d;
  const long shares = std::max(
      1l, std::min(std::min(std::min(fill, tiles / LEAST), 8l), ROOM / each));
  *floats = shares > 1 ? each * shares : 0;
  return (int)shares;
}

void launch_packed_attn_bwd(const void* dout, const void* q, const void* k,
                            const void* v, const void* o, const void* low,
                            const float* lse, float* dot, void* dq, void* dk,
                            void* dv, float* sums, int shares, const int* cu_q,
                            const int* cu_k, int n, int tq, int tk, int b,
                            int nh, int ng, int d, float scale, bool causal,
                            bool fp16, const long* os, const long* qs,
                            const long* ks, const long* vs,
                            hipStream_t stream) {
  const Packing pk = {cu_q, cu_k, n, tq, tk};
  const Strides so = {os[0], os[1], os[2]}, sq = {qs[0], qs[1], qs[2]},
                sk = {ks[0], ks[1], ks[2]}, sv = {vs[0], vs[1], vs[2]};
  if (tq > 0) {
    const dim3 grid = grid_for((long)b * nh, tq, n);
#define LAUNCH(T, DD, CC, HALVES)                                            \
  hipLaunchKernelGGL((packed_bwd_dq_kernel<T, DD, CC, HALVES>), grid,        \
                     dim3(BLOCK * HALVES), 0, stream,                        \
                     (const unsigned short*)q, (const unsigned short*)k,     \
                     (const unsigned short*)v, (const unsigned short*)dout,  \
                     (const unsigned short*)o, (const unsigned short*)low,   \
                     lse, dot, (unsigned short*)dq, pk, b, nh, ng, scale,    \
                     sq, sk, sv, so)
#define RUN(T, DD, CC)                                                       \
  do {                                                                       \
    if (halves) LAUNCH(T, DD, CC, 2); else LAUNCH(T, DD, CC, 1);             \
  } while (0)
    const bool halves = in_halves(n, tq, tk, b, nh);
    PACKED_DISPATCH(RUN);
#undef RUN
#undef LAUNCH
    HIP_CHECK_LAUNCH();
  }
  if (tk > 0) {
    const dim3 grid = grid_for((long)b * ng * shares, tk, n);
#define LAUNCH(T, DD, CC, FOUR)                                              \
  hipLaunchKernelGGL((packed_bwd_dkv_kernel<T, DD, CC, FOUR>),               \
                     grid, dim3(Dkv<DD, FOUR>::WAVES * 64), 0, stream,       \
                     (const unsigned short*)q, (const unsigned short*)k,     \
                     (const unsigned short*)v, (const unsigned short*)dout,  \
                     lse, dot, (unsigned short*)dk, (unsigned short*)dv,     \
                     sums, shares, pk, b, nh, ng, scale, sq, sk, sv, so)
#define RUN(T, DD, CC)                                                       \
  do {                                                                       \
    if (DD == 64 && many) LAUNCH(T, 64, CC, true);                           \
    else LAUNCH(T, DD, CC, false);                                           \
  } while (0)
    const bool many = tiles_of(n, tk, (long)b * ng) >= FOUR_WAVES;
    PACKED_DISPATCH(RUN);
#undef RUN
#undef LAUNCH
    HIP_CHECK_LAUNCH();
    if (shares > 1) {
      const dim3 tiles(grid_for((long)b * ng, tk, n).x, d / 16);
#define ADD(T, DD)                                                           \
  hipLaunchKernelGGL((packed_bwd_add_kernel<T, DD>), tiles, dim3(BLOCK), 0,  \
                     stream, sums, (unsigned short*)dk, (unsigned short*)dv, \
                     shares, pk, b, ng, scale)
      if (fp16) { if (d == 128) ADD(Fp16, 128); else ADD(Fp16, 64); }
      else { if (d == 128) ADD(Bf16, 128); else ADD(Bf16, 64); }
#undef ADD
      HIP_CHECK_LAUNCH();
    }
  }
}
