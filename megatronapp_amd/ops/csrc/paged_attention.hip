// Attention of single tokens over a paged cache (gfx950).
//
//   row i sees the first lengths[slot] tokens of its table's pages
//   o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s = scale log2(e) q k
//
// The row's keys are cut into pieces so that few rows fill the card too; each
// piece leaves its own o and log2 of its sum, and a second launch joins them:
//   o = sum_i 2^(L_i - M) o_i / sum_i 2^(L_i - M),  M = max L_i
// A row without tokens gives zeros.  A page number out of the pool leaves its
// tokens out.

#include "attn_tiles.h"

#include <algorithm>

namespace {

constexpr int BLOCK = 256;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int KEYS = 32;      // of one step of a wave
constexpr int HEADS = 16;     // query heads of a block, of one key head

struct Cache {
  const unsigned short* k;
  const unsigned short* v;
  const int* tables;          // [slots, width]
  const int* lengths;         // [slots]
  const int* slots;           // [b], or the rows themselves
  long kp, kh, kt, vp, vh, vt;  // strides of pages, heads, tokens
  int pages, page, width, count;  // pages, tokens of one, table, its rows
};

struct Out {
  unsigned short* o;          // [b, nh, D], where there is one piece
  float* part;                // [b, nh, pieces, D]
  float* lse;                 // [b, nh, pieces]
  int pieces;
};

__device__ __forceinline__ int slot_at(const Cache& c, int row) {
  return c.slots ? c.slots[row] : row;
}

__device__ __forceinline__ int length_at(const Cache& c, int slot) {
  if (slot < 0 || slot >= c.count) return 0;
  return (int)min((long)max(c.lengths[slot], 0), (long)c.width * c.page);
}

// An image of [KEYS][D] that only the transposing reads use: 32 lanes read
// 32 bytes of 8 rows, so the pairs of 16-byte slots are what is permuted.
template <int D>
__device__ __forceinline__ int pair_slot(int row, int slot) {
  return D == 128 ? slot ^ ((row & 7) << 1) : slot ^ (((row >> 1) & 3) << 1);
}

template <class T, int D>
__global__ __launch_bounds__(BLOCK, 2) void paged_rows_kernel(
    const unsigned short* __restrict__ q, long qb, long qh, Cache c, Out out,
    int nh, int ng, float scale) {
  constexpr int NF = D / 32, ND = D / 16;
  constexpr int SLOTS = D / 8, PER = WAVE / SLOTS, NV = KEYS / PER;
  // each wave's V rows; at the end the waves' sums
  __shared__ __attribute__((aligned(16))) unsigned short v_lds[4 * KEYS * D];
  __shared__ float m_lds[4][HEADS], l_lds[4][HEADS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int rep = nh / ng, tiles = (rep + HEADS - 1) / HEADS;
  const int hk = blockIdx.x % ng, ht = blockIdx.x / ng % tiles;
  const int piece = blockIdx.x / ng / tiles % out.pieces;
  const int row = blockIdx.x / ng / tiles / out.pieces;
  const int heads = min(HEADS, rep - ht * HEADS);
  const int head = hk * rep + ht * HEADS + min(n, heads - 1);

  const int slot = slot_at(c, row);
  const int len = length_at(c, slot);
  // this piece's keys; pieces begin at pages' sixteenths
  const int per = ((len + out.pieces - 1) / out.pieces + KEYS - 1) / KEYS * KEYS;
  const int from = min(piece * per, len), to = min(from + per, len);
  const int* table = c.tables + (long)max(0, min(slot, c.count - 1)) * c.width;

  typename T::x8 qf[NF];
  const unsigned short* src = q + row * qb + head * qh + 8 * g;
#pragma unroll
  for (int f = 0; f < NF; ++f) qf[f] = *(const typename T::x8*)(src + 32 * f);

  f32x4 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, ms = 0.f, l = 0.f;
  unsigned short* img = v_lds + wave * KEYS * D;

  typename T::x8 kn[2][NF];
  s16x8 vn[NV];
  bool okn[2];
  // keys behind the piece are read as its last one, and masked
  auto fetch = [&](int at) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int first = min(at + 16 * i, (to - 1) & ~15);
      int page = __builtin_amdgcn_readfirstlane(table[first / c.page]);
      okn[i] = page >= 0 && page < c.pages;
      page = okn[i] ? page : 0;
      const int in = first % c.page, last = to - 1 - first;
      const unsigned short* kp = c.k + page * c.kp + hk * c.kh +
                                 (long)(in + min(n, last)) * c.kt + 8 * g;
#pragma unroll
      for (int f = 0; f < NF; ++f)
        kn[i][f] = *(const typename T::x8*)(kp + 32 * f);
      const unsigned short* vp = c.v + page * c.vp + hk * c.vh;
#pragma unroll
      for (int x = 0; x < NV / 2; ++x) {
        const int r = x * PER + lane / SLOTS;
        vn[i * NV / 2 + x] = *(const s16x8*)(
            vp + (long)(in + min(r, last)) * c.vt + 8 * (lane % SLOTS));
      }
    }
  };
  const int step = 4 * KEYS;
  int at = from + wave * KEYS;
  if (at < to) fetch(at);
  for (; at < to; at += step) {
    typename T::x8 kc[2][NF];
    bool ok[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ok[i] = okn[i];
#pragma unroll
      for (int f = 0; f < NF; ++f) kc[i][f] = kn[i][f];
#pragma unroll
      for (int x = 0; x < NV / 2; ++x) {
        const int r = 16 * i + x * PER + lane / SLOTS;
        // a page out of the pool may hold anything
        *(s16x8*)(img + r * D + 8 * pair_slot<D>(r, lane % SLOTS)) =
            ok[i] ? vn[i * NV / 2 + x] : s16x8{0, 0, 0, 0, 0, 0, 0, 0};
      }
    }
    if (at + step < to) fetch(at + step);

    // S^T: keys 4g + r of each sixteen, head n
    f32x4 st[2];
    float mt = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      st[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < NF; ++f) st[i] = T::mfma16(kc[i][f], qf[f], st[i]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (!ok[i] || at + 16 * i + 4 * g + r >= to) st[i][r] = -INFINITY;
        mt = fmaxf(mt, st[i][r]);
      }
    }
    mt = fmaxf(mt, __shfl_xor(mt, 16, WAVE));
    mt = fmaxf(mt, __shfl_xor(mt, 32, WAVE)) * scale;
    if (__any(mt > m + 8.f)) {
      const float mn = fmaxf(m, mt);
      const float a = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      ms = mn == -INFINITY ? 0.f : mn;
      l *= a;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] *= a;
    }
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        st[i][r] = __builtin_amdgcn_exp2f(fmaf(st[i][r], scale, -ms));
        l += st[i][r];
      }
      w[2 * i] = pack2<T>(st[i][0], st[i][1]);
      w[2 * i + 1] = pack2<T>(st[i][2], st[i][3]);
    }
    // lane g holds keys 4g + j and 16 + 4g + j, as V^T's reads do
    const typename T::x8 pf = __builtin_bit_cast(typename T::x8, w);
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      s16x8 vf;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int r = 16 * y + 4 * g + ((lane >> 2) & 3);
        const int sl = 2 * i + ((lane >> 1) & 1);
        s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4*)(img + r * D + 8 * pair_slot<D>(r, sl) +
                         4 * (lane & 1)));
#pragma unroll
        for (int j = 0; j < 4; ++j) vf[4 * y + j] = x[j];
      }
      acc[i] = T::mfma16(__builtin_bit_cast(typename T::x8, vf), pf, acc[i]);
    }
  }

  // the waves' sums, joined
  l += __shfl_xor(l, 16, WAVE);
  l += __shfl_xor(l, 32, WAVE);
  if (g == 0) {
    m_lds[wave][n] = m;
    l_lds[wave][n] = l;
  }
  __syncthreads();             // the V rows are done with, too
  float mx = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) mx = fmaxf(mx, m_lds[w][n]);
  const float a =
      m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
  // two waves at a time: [2][HEADS][D + 4] floats fit
  float* sums = (float*)v_lds;
  constexpr int ROW = D;
#pragma unroll
  for (int turn = 0; turn < 4; ++turn) {
    if (wave == turn) {
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        f32x4* p = (f32x4*)(sums + n * ROW + ((i * 16 + 4 * g) ^ ((n & 7) << 2)));
        f32x4 x = acc[i];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] *= a;
        if (turn) {
          const f32x4 y = *p;
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] += y[r];
        }
        *p = x;
      }
    }
    __syncthreads();
  }
  for (int x = tid; x < heads * D / 4; x += BLOCK) {
    const int hh = x / (D / 4), d = x % (D / 4) * 4;
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, m_lds[w][hh]);
#pragma unroll
    for (int w = 0; w < 4; ++w)
      ll += m_lds[w][hh] == -INFINITY
                ? 0.f
                : l_lds[w][hh] * __builtin_amdgcn_exp2f(m_lds[w][hh] - mm);
    const float by = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);
    f32x4 y = *(f32x4*)(sums + hh * ROW + (d ^ ((hh & 7) << 2)));
    const long r = (long)row * nh + hk * rep + ht * HEADS + hh;
    if (out.part) {
      f32x4 z = {y[0] * by, y[1] * by, y[2] * by, y[3] * by};
      *(f32x4*)(out.part + (r * out.pieces + piece) * D + d) = z;
      if (d == 0)
        out.lse[r * out.pieces + piece] =
            ll == 0.f ? -INFINITY : mm + __builtin_amdgcn_logf(ll);
    } else {
      u32x2 z = {pack2<T>(y[0] * by, y[1] * by), pack2<T>(y[2] * by, y[3] * by)};
      *(u32x2*)(out.o + r * D + d) = z;
    }
  }
}

// a wave joins the pieces of two (D = 64: four) heads of a row
template <class T, int D>
__global__ __launch_bounds__(BLOCK) void paged_join_kernel(Out out,
                                                           long heads) {
  constexpr int LANES = D / 4;
  const long r = ((long)blockIdx.x * BLOCK + threadIdx.x) / LANES;
  const int d = threadIdx.x % LANES * 4;
  if (r >= heads) return;
  const float* lse = out.lse + r * out.pieces;
  const float* part = out.part + r * out.pieces * D + d;
  float mx = -INFINITY, l = 0.f;
  for (int i = 0; i < out.pieces; ++i) mx = fmaxf(mx, lse[i]);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < out.pieces; ++i) {
    const float x = lse[i];
    if (x == -INFINITY) continue;
    const float w = __builtin_amdgcn_exp2f(x - mx);
    const f32x4 y = *(const f32x4*)(part + (long)i * D);
    l += w;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += w * y[j];
  }
  const float by = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  u32x2 z = {pack2<T>(o[0] * by, o[1] * by), pack2<T>(o[2] * by, o[3] * by)};
  *(u32x2*)(out.o + r * D + d) = z;
}

}  // namespace

// pieces of a row, so that its blocks and the other rows' fill the card
int paged_attn_pieces(int b, int nh, int ng, int max_length) {
  const long blocks = (long)b * ng * ((nh / ng + HEADS - 1) / HEADS);
  const long fill = (1024 + blocks - 1) / blocks;
  const long most = (max_length + 4 * KEYS - 1) / (4 * KEYS);
  return (int)std::max(1l, std::min(std::min(fill, most), 64l));
}

void launch_paged_attn(const void* q, long qb, long qh, const void* k,
                       const void* v, const long* ks, const long* vs,
                       const int* tables, const int* lengths, const int* slots,
                       int b, int nh, int ng, int d, int pages, int page,
                       int width, int count, int pieces, void* o, float* part,
                       float* lse, float scale, bool fp16,
                       hipStream_t stream) {
  const Cache c = {(const unsigned short*)k, (const unsigned short*)v, tables,
                   lengths, slots, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                   pages, page, width, count};
  const Out out = {(unsigned short*)o, part, lse, pieces};
  const long blocks =
      (long)b * pieces * ng * ((nh / ng + HEADS - 1) / HEADS);
  const long lanes = (long)b * nh * (d / 4);
  if (blocks * BLOCK >= 1l << 32 || lanes >= 1l << 32)
    throw std::runtime_error("paged attention: too many rows for one launch");
#define RUN(T, DD)                                                          \
  do {                                                                      \
    hipLaunchKernelGGL((paged_rows_kernel<T, DD>), dim3((unsigned)blocks),  \
                       dim3(BLOCK), 0, stream, (const unsigned short*)q,    \
                       qb, qh, c, out, nh, ng, scale * LOG2E);              \
    HIP_CHECK_LAUNCH();                                                     \
    if (part) {                                                             \
      hipLaunchKernelGGL((paged_join_kernel<T, DD>),                        \
                         dim3((unsigned)((lanes + BLOCK - 1) / BLOCK)),     \
                         dim3(BLOCK), 0, stream, out, (long)b * nh);        \
      HIP_CHECK_LAUNCH();                                                   \
    }                                                                       \
  } while (0)
  if (fp16) { if (d == 128) RUN(Fp16, 128); else RUN(Fp16, 64); }
  else { if (d == 128) RUN(Bf16, 128); else RUN(Bf16, 64); }
#undef RUN
}
