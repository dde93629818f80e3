// Pieces shared by the packed and the paged attention kernels: element
// traits, the LDS image of a [rows][D] tile, its asynchronous loader and the
// fragment readers.
//
// Lane maps of the matrix instructions (l = lane, h = l >> 5, n = l & 31):
//   32x32x16  A[m = n][k = 8h + j], B[k = 8h + j][n], j = 0..7
//             C[m = (r & 3) + 8 (r >> 2) + 4h][n], r = 0..15
//   16x16x32  A[m = l & 15][k = 8 (l >> 4) + j], B likewise
//             C[m = 4 (l >> 4) + r][n = l & 15], r = 0..3
//   transposing LDS read of 4 x 16 bit, per 16 lanes: lane l gets element
//             (l & 3) of what lanes 4j + ((l >> 2) & 3), j = 0..3, address
//
// A C tile becomes the B (or A) operand of the next product without moving
// data between lanes: the product's rows m may be fed in any order, and with
// tile_row(m) as the row that A's lane m reads, lane h holds rows
// 16 (r >> 3) + 8h + (r & 7), which is just what an operand's lane holds.
#pragma once

#include "common.h"

#include <stdexcept>
#include <string>

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;

struct Bf16 {
  typedef __attribute__((ext_vector_type(8))) __bf16 x8;
  typedef __attribute__((ext_vector_type(2))) __bf16 x2;
  static __device__ __forceinline__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_float(unsigned short u) {
    return bf2f(u);
  }
};

struct Fp16 {
  typedef __attribute__((ext_vector_type(8))) _Float16 x8;
  typedef __attribute__((ext_vector_type(2))) _Float16 x2;
  static __device__ __forceinline__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_float(unsigned short u) {
    return (float)__builtin_bit_cast(_Float16, u);
  }
};

// two floats to 16 bits each, to nearest even
template <class T>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  f32x2 f = {a, b};
  return __builtin_bit_cast(unsigned,
                            __builtin_convertvector(f, typename T::x2));
}

// eight floats of a C tile as half of a product's operand
template <class T>
__device__ __forceinline__ typename T::x8 pack8(const f32x16& c, int at) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2<T>(c[at + 2 * i], c[at + 2 * i + 1]);
  return __builtin_bit_cast(typename T::x8, w);
}

__device__ __forceinline__ int tile_row(int m) {
  return 16 * (m >> 4) + 8 * ((m >> 2) & 1) + (m & 3) + 4 * ((m >> 3) & 1);
}

// ---------------------------------------------------------------- LDS image
// Row r of a tile lies at r * D * 2 bytes, its 16-byte slots in another
// order for each row, so that both readers below meet every bank once: 16
// lanes that read one slot of 16 rows, and 32 lanes that read 4 slots of 4
// rows (a 256-byte row of banks holds one row at D = 128, two at D = 64).
template <int D>
__device__ __forceinline__ int slot_of(int row, int slot) {
  if (D == 128) return slot ^ (((row & 3) << 2) | ((row >> 2) & 3));
  return slot ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
}

typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef const __attribute__((address_space(1))) char global_char;

// 16 bytes a lane from `base` + `off` straight to LDS: base is the wave's, off
// the lane's, so the address takes no vector instruction.
__device__ __forceinline__ void load_lds16(unsigned short* dst,
                                           const unsigned short* base,
                                           unsigned off) {
  __builtin_amdgcn_global_load_lds((global_char*)((const char*)base + off),
                                   (lds_char*)dst, 16, 0, 0);
}

// The lane's place in what one instruction of `wave` loads of an image: rows
// of `stride` elements apart (less than 2^27).
template <int D>
__device__ __forceinline__ unsigned lane_offset(long stride, int wave,
                                                int lane) {
  constexpr int SLOTS = D / 8, PER = WAVE / SLOTS;
  const int row = wave * PER + lane / SLOTS;   // only its low bits count
  return (unsigned)(lane / SLOTS) * (unsigned)stride * 2 +
         16 * slot_of<D>(row, lane % SLOTS);
}

// ROWS rows of D elements from `src` into the image at `dst`, by WAVES waves
// (a multiple of four); rows behind `last` (>= 0) are read as row `last`.
// The caller waits for them.
template <int D, int ROWS, int WAVES>
__device__ __forceinline__ void load_tile(unsigned short* dst,
                                          const unsigned short* src,
                                          long stride, int last, int wave,
                                          int lane) {
  constexpr int SLOTS = D / 8;             // of a row
  constexpr int PER = WAVE / SLOTS;        // rows of one instruction
  if (last >= ROWS - 1) {
    const unsigned off = lane_offset<D>(stride, wave, lane);
#pragma unroll
    for (int i = 0; i < ROWS / PER / WAVES; ++i) {
      const int first = (i * WAVES + wave) * PER;
      load_lds16(dst + first * D, src + (long)first * stride, off);
    }
    return;
  }
#pragma unroll 1
  for (int i = 0; i < ROWS / PER / WAVES; ++i) {
    const int first = (i * WAVES + wave) * PER;
    const int row = first + lane / SLOTS;
    const unsigned short* p = src + (long)min(row, last) * stride +
                              8 * slot_of<D>(row, lane % SLOTS);
    __builtin_amdgcn_global_load_lds(
        (global_char*)p, (lds_char*)(dst + first * D), 16, 0, 0);
  }
}

// Where a lane reads in an image, in bytes: `rows` for its row n (or
// tile_row(n)) as an operand of 32x32x16, `cols` for what the transposing reads
// address.  All other places of a tile are these with some of the slot's bits
// flipped and multiples of 16 rows added, which cost an instruction and
// nothing.
template <int D>
struct Places {
  unsigned rows, cols;
  __device__ __forceinline__ Places(int lane, bool permuted = true) {
    const int h = lane >> 5, n = lane & 31, r = permuted ? tile_row(n) : n;
    rows = r * 2 * D + 16 * slot_of<D>(r, h);
    const int c = 8 * h + ((lane >> 2) & 3);
    cols = c * 2 * D +
           16 * slot_of<D>(c, 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) +
           8 * (lane & 1);
  }
};

// operand of 32x32x16: the lane's row of those from row0 on, elements
// 16f + 8h ..
template <class T, int D>
__device__ __forceinline__ typename T::x8 read_rows(const unsigned short* img,
                                                    int row0, int f,
                                                    const Places<D>& p) {
  return *(const typename T::x8*)((const char*)img + row0 * 2 * D +
                                  (p.rows ^ 32 * f));
}

// operand of 32x32x16 whose k are the image's rows row0 .. row0 + 15 and
// whose m (or n) are its columns 32 c ..
template <class T, int D>
__device__ __forceinline__ typename T::x8 read_cols(const unsigned short* img,
                                                    int row0, int c,
                                                    const Places<D>& p) {
  s16x8 v;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)((const char*)img + (row0 + 4 * i) * 2 * D +
                     (p.cols ^ (64 * c + 16 * i))));
#pragma unroll
    for (int j = 0; j < 4; ++j) v[4 * i + j] = x[j];
  }
  return __builtin_bit_cast(typename T::x8, v);
}

// For the scheduler: N products whose operands take READS reads of LDS each,
// with those of four products ahead all along (it waits for each read just
// before the product else; forward of 10 prompts 90 -> 87 us).
template <int N, int READS>
__device__ __forceinline__ void reads_ahead() {
  constexpr int MFMA = 0x008, DS_READ = 0x100;
  __builtin_amdgcn_sched_group_barrier(DS_READ, 4 * READS, 0);
#pragma unroll
  for (int i = 0; i < N - 4; ++i) {
    __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
    __builtin_amdgcn_sched_group_barrier(DS_READ, READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(MFMA, 4, 0);
}

// this lane's and the other half-wave's value (a bit cast of a vector's
// element takes its first one, so the elements are copied out before)
__device__ __forceinline__ void half_pair(float v, float& a, float& b) {
  const unsigned x = __builtin_bit_cast(unsigned, v);
  auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  const unsigned lo = s[0], hi = s[1];
  a = __builtin_bit_cast(float, lo);
  b = __builtin_bit_cast(float, hi);
}

__device__ __forceinline__ float half_max(float v) {
  float a, b;
  half_pair(v, a, b);
  return fmaxf(a, b);
}

__device__ __forceinline__ float half_sum(float v) {
  float a, b;
  half_pair(v, a, b);
  return a + b;
}

// A 32x32 C tile (rows d, columns n) as 16-byte pieces of row n: the two
// half-waves exchange so that h = 0 gets elements 0..7 and h = 1 8..15 of
// each sixteen.  `p` points at element 0 of row n, aligned to 16 bytes; `low`,
// where there is one, gets what the rounding left out.
template <class T, bool LOW = false>
__device__ __forceinline__ void store_cols(unsigned short* p, const f32x16& c,
                                           float by, int h,
                                           unsigned short* low = nullptr) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    unsigned a[2], b[2], la[2], lb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x[4] = {c[8 * k + 2 * i] * by, c[8 * k + 2 * i + 1] * by,
                          c[8 * k + 4 + 2 * i] * by,
                          c[8 * k + 5 + 2 * i] * by};
      a[i] = pack2<T>(x[0], x[1]);
      b[i] = pack2<T>(x[2], x[3]);
      if (LOW) {
        la[i] = pack2<T>(x[0] - T::to_float(a[i] & 0xffff),
                         x[1] - T::to_float(a[i] >> 16));
        lb[i] = pack2<T>(x[2] - T::to_float(b[i] & 0xffff),
                         x[3] - T::to_float(b[i] >> 16));
      }
    }
    auto s0 = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
    auto s1 = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
    u32x4 w = {s0[0], s1[0], s0[1], s1[1]};
    *(u32x4*)(p + 16 * k + 8 * h) = w;
    if (LOW) {
      s0 = __builtin_amdgcn_permlane32_swap(la[0], lb[0], false, false);
      s1 = __builtin_amdgcn_permlane32_swap(la[1], lb[1], false, false);
      u32x4 y = {s0[0], s1[0], s0[1], s1[1]};
      *(u32x4*)(low + 16 * k + 8 * h) = y;
    }
  }
}
