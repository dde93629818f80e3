// Attention of single tokens over a paged cache (gfx950).
//
//   row i sees the first lengths[slot] tokens of its table's pages
//   o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s = scale log2(e) q k
//
// The row's keys are cut into pieces so that few rows fill the card too; each
// piece leaves its own o and log2 of its sum, and a second launch joins them:
//   o = sum_i 2^(L_i - M) o_i / sum_i 2^(L_i - M),  M = max L_i
// A row without tokens gives zeros.  A page number out of the pool leaves its
// tokens out.  The weights are rounded to 16 bits before their product with V,
// which the matrix unit takes nothing wider for at this rate (the output's
// error is 1.1 times what its last rounding alone leaves); scores, sums and
// what is joined of pieces stay in 32 bits.
//
// Rows of a group begin with the same pages.  Their queries, for all heads of
// a key head, are the rows of a matrix product over these pages, done once
// for the group; what each row has of its own follows as above, and the
// pieces of both are joined.  Both kinds of blocks are one launch: the
// group's products are bound by the matrix units, the rows' own pages by
// memory, and each fills what the other leaves.

#include "attn_tiles.h"

#include <algorithm>

namespace {

constexpr int BLOCK = 256;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int KEYS = 32;      // of one step of a wave
constexpr int HEADS = 16;     // query heads of a block, of one key head

constexpr int BM = 128;       // queries of a group's block, 32 a wave
constexpr int BN = 64;        // keys of its step

struct Cache {
  const unsigned short* k;
  const unsigned short* v;
  const int* tables;          // [slots, width]
  const int* lengths;         // [slots]
  const int* slots;           // [b], or the rows themselves
  long kp, kh, kt, vp, vh, vt;  // strides of pages, heads, tokens
  int pages, page, width, count;  // pages, tokens of one, table, its rows
  unsigned long magic;        // 2^shift / (page / 16), rounded up
  int shift;
};

// Groups of rows that share their first pages; none: groups == 0.
struct Groups {
  const int* rows;            // [groups + 1]
  const int* lengths;         // [groups]
  int groups, b;
  int tiles, pieces, blocks;  // blocks of BM queries, cuts of the prefix
};

struct Out {
  unsigned short* o;          // [b, nh, D], of rows in one piece
  float* part;                // [b, nh, pieces, D]
  float* lse;                 // [b, nh, pieces]
  int pieces;                 // of a row at most, the groups' ones first
  int evenly;                 // into which a row is cut if it has the keys
  int extra;                  // blocks for the pieces beyond that
};

// The pieces of a row's own keys: `evenly` for the sake of the card, but none
// of fewer than LEAST keys, and more where they would have more than MOST.
constexpr int LEAST = 256, MOST = 1024;

__host__ __device__ constexpr int cuts(int keys, int evenly, int most) {
  const int fill = std::min((keys + LEAST - 1) / LEAST, evenly);
  const int n = std::max(fill, (keys + MOST - 1) / MOST);
  return std::max(1, std::min(n, most));
}

// the page and the place in it of a token, at a multiple of 16
//
// With p = page / 16 and shift = 37 + floor(log2 p), magic is at most 2^37 and
// off by less than one.  x = token / 16 is below 2^27, so the product fits 64
// bits and is off by less than 2^27, where 2^shift / p, one part in p of a
// page, is above 2^36: the quotient is exact for any multiple of 16.
__device__ __forceinline__ int page_of(const Cache& c, int token, int& in) {
  const int i = (int)(((unsigned long)(token >> 4) * c.magic) >> c.shift);
  in = token - i * c.page;
  return i;
}

__device__ __forceinline__ int slot_at(const Cache& c, int row) {
  return c.slots ? c.slots[row] : row;
}

__device__ __forceinline__ int length_at(const Cache& c, int slot) {
  if (slot < 0 || slot >= c.count) return 0;
  return (int)min((long)max(c.lengths[slot], 0), (long)c.width * c.page);
}

// tokens that a group's rows share: whole pages
__device__ __forceinline__ int shared_of(const Cache& c, const Groups& gr,
                                         int g) {
  const int n = max(0, min(gr.lengths[g], c.width * c.page));
  return n / c.page * c.page;
}

__device__ __forceinline__ int group_row(const Groups& gr, int g) {
  return max(0, min(gr.rows[g], gr.b));
}

// tokens of the row that its group's blocks do: the last group that begins
// at or before it, if it reaches so far
__device__ __forceinline__ int shared_at(const Cache& c, const Groups& gr,
                                         int row) {
  if (gr.groups == 0) return 0;
  int lo = 0, hi = gr.groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (gr.rows[mid] <= row) lo = mid; else hi = mid;
  }
  return row >= gr.rows[lo] && row < gr.rows[lo + 1] ? shared_of(c, gr, lo)
                                                      : 0;
}

// The row of a group whose table is read for all: the first that holds all of
// what they share, or the longest.  Rows that hold less have nothing in their
// tables behind that.
__device__ __forceinline__ int lead_row(const Cache& c, int from, int to,
                                        int shared, int lane) {
  int most = -1, at = from;      // the lane's longest
  for (int base = from; base < to; base += WAVE) {
    const int row = base + lane;
    const int len = row < to ? length_at(c, slot_at(c, row)) : -1;
    const unsigned long long whole = __ballot(len >= shared);
    if (whole) return base + __builtin_ctzll(whole);
    if (len > most) most = len, at = row;
  }
#pragma unroll
  for (int off = 1; off < WAVE; off <<= 1) {
    const int len = __shfl_xor(most, off, WAVE);
    const int row = __shfl_xor(at, off, WAVE);
    if (len > most || (len == most && row < at)) most = len, at = row;
  }
  return __builtin_amdgcn_readfirstlane(at);
}

// A lane's worth of a table: 64 page numbers from `base` on, read ahead so
// that no step waits for its page's number.
struct Pages {
  int id, base;
};

__device__ __forceinline__ int page_at(const Cache& c, const int* table,
                                       int i, int lane, Pages& p, bool& ok) {
  if (i < p.base || i >= p.base + WAVE) {
    p.base = i;
    p.id = table[min(i + lane, c.width - 1)];
  }
  const int page = __builtin_amdgcn_readlane(p.id, i - p.base);
  ok = page >= 0 && page < c.pages;
  return ok ? page : 0;
}

// An image of [KEYS][D] that only the transposing reads use: 32 lanes read
// 32 bytes of 8 rows, so the pairs of 16-byte slots are what is permuted.
template <int D>
__device__ __forceinline__ int pair_slot(int row, int slot) {
  return D == 128 ? slot ^ ((row & 7) << 1) : slot ^ (((row >> 1) & 3) << 1);
}

// --------------------------------------------------------- a row's own keys
// the pieces of a row that no block of its own stands for
__device__ __forceinline__ int extra_of(const Cache& c, const Groups& gr,
                                        const Out& out, int row) {
  const int len = length_at(c, slot_at(c, row));
  return max(cuts(len - min(shared_at(c, gr, row), len), out.evenly,
                  out.pieces - gr.pieces) - out.evenly, 0);
}

// The row and the piece of the index-th of these, or false behind the last.
__device__ __forceinline__ bool find_extra(const Cache& c, const Groups& gr,
                                           const Out& out, int index, int lane,
                                           int& row, int& piece) {
  for (int base = 0; base < gr.b; base += WAVE) {
    const int own = base + lane < gr.b ? extra_of(c, gr, out, base + lane) : 0;
    int sum = own;
#pragma unroll
    for (int off = 1; off < WAVE; off <<= 1) {
      const int x = __shfl_up(sum, off, WAVE);
      if (lane >= off) sum += x;
    }
    const int total = __builtin_amdgcn_readlane(sum, WAVE - 1);
    if (index < total) {
      const int at = __builtin_ctzll(__ballot(index < sum));
      row = base + at;
      piece = out.evenly + index - __builtin_amdgcn_readlane(sum - own, at);
      return true;
    }
    index -= total;
  }
  return false;
}

// Four waves take every fourth step of 32 keys, for up to 16 query heads of
// one key head (S^T = K Q^T by 16 x 16 products, so grouped heads read K and V
// once).  K goes straight into registers, V by registers into the wave's own
// LDS, out of which it is read transposed; the next step's loads are under way
// while one is used, and page numbers come 64 at a time.  Memory bounds it: 32
// rows of 2048 tokens, 8 key heads of 128, take 52 us, 5.1 TB/s; one row of
// 8192 takes 17 us, mostly latencies of its pieces' 8 steps and of the join.
// Steps of 64 keys at D = 64 lose 15%.

// What a block's waves tell each other at the end.
struct WaveSums {
  float m[4][HEADS], l[4][HEADS];
};

// `image`: each wave's V rows, [4][KEYS][D]; at the end the waves' sums
template <class T, int D>
__device__ __forceinline__ void own_keys(const unsigned short* q, long qb,
                                         long qh, const Cache& c,
                                         const Groups& gr, const Out& out,
                                         int nh, int ng, float scale, int hk,
                                         int ht, int row, int piece,
                                         unsigned short* image,
                                         WaveSums& lds) {
  constexpr int NF = D / 32, ND = D / 16;
  constexpr int SLOTS = D / 8, PER = WAVE / SLOTS, NV = KEYS / PER;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int rep = nh / ng;
  const int heads = min(HEADS, rep - ht * HEADS);
  const int head = hk * rep + ht * HEADS + min(n, heads - 1);

  // under way before the lengths are known: Q, and the first page numbers
  typename T::x8 qf[NF];
  const unsigned short* src = q + row * qb + head * qh + 8 * g;
#pragma unroll
  for (int f = 0; f < NF; ++f) qf[f] = *(const typename T::x8*)(src + 32 * f);
  const int slot = slot_at(c, row);
  const int* table = c.tables + (long)max(0, min(slot, c.count - 1)) * c.width;
  Pages ids = {0, -WAVE};
  if (c.count > 0 && c.width > 0) ids = {table[min(lane, c.width - 1)], 0};
  const int len = length_at(c, slot);
  // this piece's keys
  const int shared = shared_at(c, gr, row);
  const int begin = min(shared, len), own = len - begin;
  const int pieces = cuts(own, out.evenly, out.pieces - gr.pieces);
  if (piece >= pieces) return;
  const int per = ((own + pieces - 1) / pieces + KEYS - 1) / KEYS * KEYS;
  const int from = begin + min(piece * per, own);
  const int to = min(from + per, len);

  f32x4 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, ms = 0.f, l = 0.f;
  unsigned short* img = image + wave * KEYS * D;

  typename T::x8 kn[2][NF];
  s16x8 vn[NV];
  bool okn[2];
  // keys behind the piece are read as its last one, and masked
  auto fetch = [&](int at) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int first = min(at + 16 * i, (to - 1) & ~15);
      int in;
      const int index = page_of(c, first, in);
      const long page = page_at(c, table, index, lane, ids, okn[i]);
      const int last = to - 1 - first;
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
    if (__any(mt > m)) {
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
    lds.m[wave][n] = m;
    lds.l[wave][n] = l;
  }
  __syncthreads();             // the V rows are done with, too
  float mx = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) mx = fmaxf(mx, lds.m[w][n]);
  const float a =
      m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
  // [HEADS][D] floats, the waves' added one after the other
  float* sums = (float*)image;
  constexpr int ROW = D;
#pragma unroll
  for (int turn = 0; turn < 4; ++turn) {
    if (wave == turn) {
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        f32x4* p =
            (f32x4*)(sums + n * ROW + ((i * 16 + 4 * g) ^ ((n & 7) << 2)));
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
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, lds.m[w][hh]);
    // a wave without a maximum has a sum of zero, or saw nothing but NaN
#pragma unroll
    for (int w = 0; w < 4; ++w)
      ll += lds.l[w][hh] *
            (lds.m[w][hh] == -INFINITY
                 ? 1.f
                 : __builtin_amdgcn_exp2f(lds.m[w][hh] - mm));
    const float by = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);
    f32x4 y = *(f32x4*)(sums + hh * ROW + (d ^ ((hh & 7) << 2)));
    const long r = (long)row * nh + hk * rep + ht * HEADS + hh;
    if (shared || pieces > 1) {
      f32x4 z = {y[0] * by, y[1] * by, y[2] * by, y[3] * by};
      const long at = r * out.pieces + gr.pieces + piece;
      *(f32x4*)(out.part + at * D + d) = z;
      if (d == 0)
        out.lse[at] =
            ll == 0.f ? -INFINITY : mm + __builtin_amdgcn_logf(ll);
    } else {
      u32x2 z = {pack2<T>(y[0] * by, y[1] * by),
                 pack2<T>(y[2] * by, y[3] * by)};
      *(u32x2*)(out.o + r * D + d) = z;
    }
  }
}

// The first blocks take the extra pieces, which are of the longest rows.  A
// launch without any has a kernel of its own, with fewer registers (at D = 64
// 104 and four blocks on a CU, not 130 and three: 256 rows on 0..300 tokens
// 17 us against 19).
template <class T, int D, bool EXTRA>
__device__ __forceinline__ void rows_block(const unsigned short* q, long qb,
                                           long qh, const Cache& c,
                                           const Groups& gr, const Out& out,
                                           int nh, int ng, float scale,
                                           unsigned block,
                                           unsigned short* image,
                                           WaveSums& sums) {
  const int tiles = (nh / ng + HEADS - 1) / HEADS;
  if (!EXTRA || block >= (unsigned)out.extra) {
    const unsigned unit = EXTRA ? block - out.extra : block;
    const int index = unit / ng / tiles;
    own_keys<T, D>(q, qb, qh, c, gr, out, nh, ng, scale, unit % ng,
                   unit / ng % tiles, index / out.evenly, index % out.evenly,
                   image, sums);
    return;
  }
  int row, piece;
  for (unsigned unit = block;
       find_extra(c, gr, out, unit / ng / tiles, threadIdx.x & 63, row, piece);
       unit += out.extra) {
    own_keys<T, D>(q, qb, qh, c, gr, out, nh, ng, scale, unit % ng,
                   unit / ng % tiles, row, piece, image, sums);
    __syncthreads();          // the sums are read, and their place is free
  }
}

// ------------------------------------------------------ a group's first keys
// A forward of packed sequences, but for where its rows and its keys lie: 32
// queries a wave (rows times the heads of a key head), tiles of 64 keys in two
// images.  Its products are bound by the matrix and vector units, so that the
// rows' own keys, read beside them, cost little: 64 rows on 4096 + 33..700
// tokens, 32/8 heads of 128, take 34 us (113 MB, 4.7 GFLOP) and the join 5;
// 256 rows on 16384 + 1..1024 171 (611 MB, 71 GFLOP) and 8; in fp16 the same.
// Each row for itself, joined: 97 and 1190.
template <class T, int D>
__device__ __forceinline__ void shared_keys(
    const unsigned short* q, long qb, long qh, const Cache& c,
    const Groups& gr, const Out& out, int nh, int ng, float scale,
    unsigned block, unsigned short* img0, unsigned short* img1) {
  constexpr int NF = D / 16, ND = D / 32;
  constexpr int PER = WAVE / (D / 8);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, n = lane & 31, rep = nh / ng;
  const Places<D> at_lane(lane);
  const int hk = block % ng, piece = block / ng % gr.pieces;
  const int g = block / ng / gr.pieces % gr.groups;
  const int first_row = group_row(gr, g), end_row = group_row(gr, g + 1);
  const int queries = (end_row - first_row) * rep;
  const int shared = shared_of(c, gr, g);
  if (queries <= 0 || shared == 0) return;
  const int per = ((shared + gr.pieces - 1) / gr.pieces + BN - 1) / BN * BN;
  const int from = min(piece * per, shared), to = min(from + per, shared);
  const int lead = lead_row(c, first_row, end_row, shared, lane);
  const int slot = max(0, min(slot_at(c, lead), c.count - 1));
  const int* table = c.tables + (long)slot * c.width;
  const int turns = (to - from + BN - 1) / BN;
  // no tile lies in two pages: one number is enough
  const bool whole = c.page % BN == 0;
  const unsigned short* kb = c.k + hk * c.kh + wave * PER * c.kt;
  const unsigned short* vb = c.v + hk * c.vh + wave * PER * c.vt;
  const long k_step = 4 * PER * c.kt, v_step = 4 * PER * c.vt;
  const unsigned k_off = lane_offset<D>(c.kt, wave, lane);
  const unsigned v_off = lane_offset<D>(c.vt, wave, lane);
  Pages ids = {0, -WAVE};

  // as many blocks go round the group's queries as the host expects to need
  for (int tile = block / ng / gr.pieces / gr.groups; tile * BM < queries;
       tile += gr.tiles) {
    const int x0 = tile * BM + wave * 32;
    const int x = min(x0 + n, queries - 1);
    const int row = first_row + x / rep, head = hk * rep + x % rep;
    const int sees = min(length_at(c, slot_at(c, row)), to);
    typename T::x8 qf[NF];
    const unsigned short* src = q + row * qb + head * qh;
#pragma unroll
    for (int f = 0; f < NF; ++f)
      qf[f] = *(const typename T::x8*)(src + 16 * f + 8 * h);
    f32x16 acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    float m = -INFINITY, ms = 0.f, l = 0.f;
    // rows of a group as a rule see all of it
    const bool all = __all(sees >= to);

    int fine = 0, fine_next = 0;    // which sixteenths' pages are in the pool
    auto fetch = [&](int t, unsigned short* img) {
      bool ok;
      if (whole) {
        int in;
        const int index = page_of(c, from + t * BN, in);
        const long page = page_at(c, table, index, lane, ids, ok);
        fine_next = ok ? 15 : 0;
        const unsigned short* kr = kb + page * c.kp + in * c.kt;
        const unsigned short* vr = vb + page * c.vp + in * c.vt;
#pragma unroll
        for (int i = 0; i < BN / PER / 4; ++i) {
          const int r0 = (i * 4 + wave) * PER;
          load_lds16(img + r0 * D, kr, k_off);
          load_lds16(img + (BN + r0) * D, vr, v_off);
          kr += k_step;
          vr += v_step;
        }
        return;
      }
      int pg[4], in[4];
      fine_next = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // keys behind the piece are read as its last sixteen, and masked
        const int index =
            page_of(c, min(from + t * BN + 16 * i, (to - 1) & ~15), in[i]);
        pg[i] = page_at(c, table, index, lane, ids, ok);
        fine_next |= (int)ok << i;
      }
#pragma unroll
      for (int i = 0; i < BN / PER / 4; ++i) {
        const int r0 = (i * 4 + wave) * PER, x = r0 >> 4;
        const long page = x < 2 ? (x == 0 ? pg[0] : pg[1])
                                : (x == 2 ? pg[2] : pg[3]);
        const int base = x < 2 ? (x == 0 ? in[0] : in[1])
                               : (x == 2 ? in[2] : in[3]);
        // kb and vb begin at the wave's rows of the first sixteenth
        const long at = base - (r0 & ~15) + i * 4 * PER;
        load_lds16(img + r0 * D, kb + page * c.kp + at * c.kt, k_off);
        load_lds16(img + (BN + r0) * D, vb + page * c.vp + at * c.vt, v_off);
      }
    };
    auto step = [&](int t, const unsigned short* img) {
      const int at = from + t * BN;
      if (x0 >= queries) return;
      f32x16 st[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) st[u][r] = 0.f;
#pragma unroll
        for (int f = 0; f < NF; ++f)
          st[u] = T::mfma32(read_rows<T, D>(img, 32 * u, f, at_lane), qf[f],
                             st[u]);
      }
      reads_ahead<2 * NF, 1>();
      if (!all || at + BN > to || fine != 15) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (at + 32 * u + 16 * (r >> 3) + 8 * h + (r & 7) >= sees ||
                !(fine >> (2 * u + (r >> 3)) & 1))
              st[u][r] = -INFINITY;
      }
      float mt = st[0][0];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, st[u][r]);
      mt = half_max(mt) * scale;
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
          st[u][r] = __builtin_amdgcn_exp2f(fmaf(st[u][r], scale, -ms));
          l += st[u][r];
        }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const typename T::x8 pf = pack8<T>(st[u], 8 * y);
#pragma unroll
          for (int i = 0; i < ND; ++i)
            acc[i] = T::mfma32(
                read_cols<T, D>(img + BN * D, 32 * u + 16 * y, i, at_lane), pf,
                acc[i]);
        }
    };
    auto turn = [&](int t, unsigned short* img, unsigned short* next) {
      __builtin_amdgcn_s_waitcnt(0x0f70);         // vmcnt(0)
      __syncthreads();
      fine = fine_next;
      if (t + 1 < turns) fetch(t + 1, next);
      if (fine != 15) {       // what stands for a page out of the pool
        for (int i = 0; i < 4; ++i)
          if (!(fine >> i & 1))
            for (int x = tid; x < 2 * D; x += BLOCK)
              *(s16x8*)(img + (BN + 16 * i) * D + 8 * x) =
                  s16x8{0, 0, 0, 0, 0, 0, 0, 0};
        __syncthreads();
      }
      step(t, img);
    };
    __syncthreads();          // the images of the tile before are done with
    if (turns > 0) fetch(0, img0);
    for (int t = 0; t < turns; t += 2) {
      turn(t, img0, img1);
      if (t + 1 < turns) turn(t + 1, img1, img0);
    }
    if (x0 + n < queries) {
      l = half_sum(l);
      const float by = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      const long r = ((long)row * nh + head) * out.pieces + piece;
      if (h == 0)
        out.lse[r] = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
      float* dst = out.part + r * D + 4 * h;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          f32x4 z = {acc[i][4 * y] * by, acc[i][4 * y + 1] * by,
                     acc[i][4 * y + 2] * by, acc[i][4 * y + 3] * by};
          *(f32x4*)(dst + 32 * i + 8 * y) = z;
        }
    }
  }
}

template <class T, int D, bool EXTRA>
__global__ __launch_bounds__(BLOCK, 2) void paged_rows_kernel(
    const unsigned short* __restrict__ q, long qb, long qh, Cache c, Groups gr,
    Out out, int nh, int ng, float scale) {
  __shared__ __attribute__((aligned(16))) unsigned short image[4 * KEYS * D];
  __shared__ WaveSums sums;
  rows_block<T, D, EXTRA>(q, qb, qh, c, gr, out, nh, ng, scale, blockIdx.x,
                          image, sums);
}

template <class T, int D>
__global__ __launch_bounds__(BLOCK, 2) void paged_groups_kernel(
    const unsigned short* __restrict__ q, long qb, long qh, Cache c, Groups gr,
    Out out, int nh, int ng, float scale) {
  // two arrays, so that reads of one do not wait for what comes into the other
  __shared__ __attribute__((aligned(16))) unsigned short img0[2 * BN * D];
  __shared__ __attribute__((aligned(16))) unsigned short img1[2 * BN * D];
  __shared__ WaveSums sums;
  static_assert(2 * BN >= 4 * KEYS, "room for the rows' image");
  if (blockIdx.x < gr.blocks)
    shared_keys<T, D>(q, qb, qh, c, gr, out, nh, ng, scale, blockIdx.x, img0,
                      img1);
  else
    rows_block<T, D, true>(q, qb, qh, c, gr, out, nh, ng, scale,
                           blockIdx.x - gr.blocks, img0, sums);
}

// -------------------------------------------------------------------- joining
// A wave for each head of a row.  The pieces' log-sums come in at once, a lane
// each, and each half-wave adds up every other piece (at D = 64 each quarter
// every fourth).
template <class T, int D>
__global__ __launch_bounds__(BLOCK) void paged_join_kernel(Cache c, Groups gr,
                                                           Out out, int nh,
                                                           long heads) {
  constexpr int LANES = D / 4, PARTS = WAVE / LANES;
  const int lane = threadIdx.x & 63, d = lane % LANES * 4;
  const long r = (long)blockIdx.x * (BLOCK / WAVE) +
                 __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= heads) return;
  // under way before it is known which of them there are: all the log-sums,
  // and the first of the outputs
  const float* lse = out.lse + r * out.pieces;
  const float* part = out.part + r * out.pieces * D + d;
  float x0 = lane < out.pieces ? lse[lane] : 0.f;
  float x1 = lane + WAVE < out.pieces ? lse[lane + WAVE] : 0.f;
  constexpr int AHEAD = 4;
  f32x4 y[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    y[k] = *(const f32x4*)(
        part + (long)min(k * PARTS + lane / LANES, out.pieces - 1) * D);
  // a row that shares nothing has no pieces of a group
  const int row = (int)(r / nh), len = length_at(c, slot_at(c, row));
  const int shared = shared_at(c, gr, row), first = shared ? 0 : gr.pieces;
  const int own = cuts(len - min(shared, len), out.evenly,
                       out.pieces - gr.pieces);
  if (!shared && own == 1) return;      // its block wrote o
  const int last = gr.pieces + own;
  if (lane < first || lane >= last) x0 = -INFINITY;
  if (lane + WAVE < first || lane + WAVE >= last) x1 = -INFINITY;
  float mx = fmaxf(x0, x1);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    mx = fmaxf(mx, __shfl_xor(mx, off, WAVE));
  const float w0 = x0 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x0 - mx);
  const float w1 = x1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x1 - mx);
  float l = w0 + w1;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off, WAVE);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  // all lanes stay in: a lane that left would not hand over its weights
  auto add = [&](int i, const f32x4& z) __attribute__((always_inline)) {
    const float a = __shfl(w0, i & 63, WAVE), b = __shfl(w1, i & 63, WAVE);
    const float w = i < WAVE ? a : b;
    // a piece of no keys adds nothing, nor does one that is not there
    if (i < last && w != 0.f) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += w * z[j];
    }
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) add(k * PARTS + lane / LANES, y[k]);
#pragma unroll 4
  for (int base = AHEAD * PARTS; base < last; base += PARTS) {
    const int i = base + lane / LANES;
    add(i, *(const f32x4*)(part + (long)min(i, last - 1) * D));
  }
#pragma unroll
  for (int off = LANES; off < WAVE; off <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], off, WAVE);
  const float by = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (lane < LANES) {
    u32x2 z = {pack2<T>(o[0] * by, o[1] * by), pack2<T>(o[2] * by, o[3] * by)};
    *(u32x2*)(out.o + r * D + d) = z;
  }
}

}  // namespace

// How the work is cut: pieces of a row's own keys, at most and in general, and
// of its group's (none: every row reads its shared pages for itself).
//
// A group's blocks run beside the rows' ones, one of each on a CU where there
// are enough; both should end together.  A step of 64 keys of a group's block
// takes the time in which the card reads some 9 MB of rows' own keys at D = 128
// (half of that at 64), and rows are taken to have half of the longest one's
// own keys; four steps are worth a piece.  256 rows on 16384 + 1..1024 tokens:
// 257, 185, 171, 186, 206 us in 2, 3, 4, 6, 8 pieces; 64 rows on 4096 +
// 33..700: 58, 48, 39, 40, 46 us in 3, 4, 6, 8, 16.  Rows that read little
// more than SHARE bytes of shared keys in all, mostly out of L2, are done
// sooner each for itself (24 rows in four groups, 51 MB: 13 us against 16; 16
// rows, 134 MB: 24 us against 17).
//
// Rows in general are cut until there are two blocks for each of 256 CUs: at
// 8 key heads 16 rows on 4096 tokens take 96, 59, 53, 57 us in 1, 2, 4, 8
// pieces, 64 rows on 1024 at D = 64 27, 32, 39 us in 1, 2, 4.  Keys fewer than
// LEAST are worth no piece: one row on 500 takes 8 us in one and 11 in two and
// joined, 8 rows on 1024 14.5 us in pieces of 256, 15.8 in ones of 512.  Above
// MOST keys a row is cut again, which only its own length decides: 64 rows on
// 0, 100 .. 6300 tokens take 244, 158, 160, 164 us at MOST = 4096, 2048, 1024,
// 512, 63 rows on 100 beside one on 8100 39, 27, 27 us at 2048, 1024, 512.
// These pieces have no blocks of their own, which would mostly find nothing to
// do: 512 blocks share them out.  With a block for every piece that a row may
// have, 128 rows on 200 tokens beside one on 60000 take 114 us, and 86 so.
// Unless all rows are of the one group, a row may have `max_length` keys of its
// own, whatever the others share: one of 20000 beside two that share as many,
// 32/8 heads of 128, take 49 us, and 303 if the row may have no more keys of
// its own than those.  Half as many blocks stand by for such rows: four groups
// of 16 rows, each on 4096 tokens, take 48 us without any, 49 and, with all, 51.
// ROOM bounds the memory that a row's own pieces take, and four times as much
// that of all: every row of the batch has room for its group's pieces, in a
// group or not.  One piece of each is always there.
void paged_attn_pieces(int b, int nh, int ng, int d, int max_length,
                       int groups, int max_rows, long max_prefix, int* own,
                       int* shared, int* evenly, int* extra) {
  constexpr long SHARE = 96l << 20, FILL = 512, ROOM = 64l << 20;
  const long part = ROOM / ((long)b * nh * (d + 1) * 4);   // in pieces
  const long blocks = (long)b * ng * ((nh / ng + HEADS - 1) / HEADS);
  *shared = 0;
  long most = max_length, longest = most;     // own keys, of these and of all
  const long rows = std::min((long)b, (long)groups * max_rows);
  if (rows * max_prefix * ng * d * 4 > SHARE) {
    max_prefix = std::min(max_prefix, most);
    most = std::max(1l, most - max_prefix);
    if (groups == 1 && max_rows >= b) longest = most;
    const long units =
        (long)groups * ng * (((long)max_rows * (nh / ng) + BM - 1) / BM);
    const long steps = (max_prefix + BN - 1) / BN;
    const long beside = (long)b * most * ng / 34000;   // in steps
    // little beside them: two of a group's blocks on a CU
    const long room = beside * 4 < steps * units / 256 ? 512 : 256;
    const long per = std::max(4l, beside);
    *shared = (int)std::max(
        1l, std::min(std::min(std::min((steps + per - 1) / per, room / units),
                              64l), 3 * part));
  }
  *evenly = 1;
  while (*evenly < 64 && blocks * *evenly < FILL) *evenly *= 2;
  const int cap = (int)std::max((long)*evenly, std::min(part, 64l));
  *evenly = std::min(*evenly, cuts((int)most, *evenly, cap));
  *own = cuts((int)longest, *evenly, cap);
  // rows in general may need none of them
  const bool few = cuts((int)most, *evenly, cap) == *evenly;
  *extra = (int)std::min(blocks * (*own - *evenly), few ? FILL / 2 : FILL);
}

void launch_paged_attn(const void* q, long qb, long qh, const void* k,
                       const void* v, const long* ks, const long* vs,
                       const int* tables, const int* lengths, const int* slots,
                       const int* group_rows, const int* group_lengths,
                       int groups, int max_rows, int b, int nh, int ng, int d,
                       int pages, int page, int width, int count, int own,
                       int shared, int evenly, int extra, void* o, float* part,
                       float* lse,
                       float scale, bool fp16, hipStream_t stream) {
  const unsigned long p16 = page / 16;
  const int shift = 37 + 63 - __builtin_clzl(p16);
  const Cache c = {(const unsigned short*)k, (const unsigned short*)v, tables,
                   lengths, slots, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                   pages, page, width, count, ((1ul << shift) + p16 - 1) / p16,
                   shift};
  const long units = (long)b * ng * ((nh / ng + HEADS - 1) / HEADS);
  const Out out = {(unsigned short*)o, part, lse, own + shared, evenly, extra};
  const int tiles =
      (int)std::max(1l, ((long)max_rows * (nh / ng) + BM - 1) / BM);
  const long first = shared ? (long)groups * tiles * ng * shared : 0;
  const long blocks = first + extra + units * evenly;
  const long heads = (long)b * nh, each = BLOCK / WAVE;
  if (blocks * BLOCK >= 1l << 32 || heads * WAVE >= 1l << 32)
    throw std::runtime_error("paged attention: too many rows for one launch");
  const Groups gr = {group_rows, group_lengths, shared ? groups : 0, b, tiles,
                     shared, (int)first};
#define RUN(T, DD)                                                          \
  do {                                                                      \
    if (shared)                                                             \
      hipLaunchKernelGGL((paged_groups_kernel<T, DD>),                      \
                         dim3((unsigned)blocks), dim3(BLOCK), 0, stream,    \
                         (const unsigned short*)q, qb, qh, c, gr, out, nh,  \
                         ng, scale * LOG2E);                                \
    else if (extra)                                                         \
      hipLaunchKernelGGL((paged_rows_kernel<T, DD, true>),                  \
                         dim3((unsigned)blocks), dim3(BLOCK), 0, stream,    \
                         (const unsigned short*)q, qb, qh, c, gr, out, nh,  \
                         ng, scale * LOG2E);                                \
    else                                                                    \
      hipLaunchKernelGGL((paged_rows_kernel<T, DD, false>),                 \
                         dim3((unsigned)blocks), dim3(BLOCK), 0, stream,    \
                         (const unsigned short*)q, qb, qh, c, gr, out, nh,  \
                         ng, scale * LOG2E);                                \
    HIP_CHECK_LAUNCH();                                                     \
    if (part) {                                                             \
      hipLaunchKernelGGL((paged_join_kernel<T, DD>),                        \
                         dim3((unsigned)((heads + each - 1) / each)),       \
                         dim3(BLOCK), 0, stream, c, gr, out, nh, heads);    \
      HIP_CHECK_LAUNCH();                                                   \
    }                                                                       \
  } while (0)
  if (fp16) { if (d == 128) RUN(Fp16, 128); else RUN(Fp16, 64); }
  else { if (d == 128) RUN(Bf16, 128); else RUN(Bf16, 64); }
#undef RUN
}
