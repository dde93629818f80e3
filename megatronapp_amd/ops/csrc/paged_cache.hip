// The pages of a key/value cache: fork, free, compact, extend, write, copy.
//
//   pages   [planes, P, groups, page, d]  planes = layers x (key, value)
//   refs    [P]      sequences that hold the page, 0: free
//   tables  [slots, W]  a sequence's pages in order, -1 behind them
//   lengths [slots]  its tokens; ceil(length / page) entries are in use
//
// A part-filled page belongs to one sequence; full pages may be shared, and
// are never written again.  All bookkeeping stays on the device and does not
// go by the order of atomics: pages are handed out lowest first by scans, and
// counts are only added to.  A call that cannot be carried out (a slot or a
// page out of range, a target named twice, no free page) changes nothing and
// leaves a bit in `status`.
//
// The content moves at the speed of a copy; the tables are small.  A plan is
// one block's work (scans over refs), what it decides is applied by a second
// launch that fills the card.

#include "common.h"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace {

constexpr int PLAN = 1024;    // threads of a planning block
constexpr int WAVES = PLAN / WAVE;
constexpr int BLOCK = 256;

enum Status {
  BAD_SLOT = 1, NO_PAGE = 2, BAD_PAGE = 4, TOO_LONG = 8, SHARED = 16
};

struct Pool {
  int* refs;
  int* tables;
  int* lengths;
  int* status;
  int pages, slots, width, page;   // page: tokens of one
};

// inclusive sum over the block; `total` is everybody's
template <class N>
__device__ __forceinline__ N block_scan(N v, N* lds, N& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < WAVE; off <<= 1) {
    const N x = __shfl_up(v, off, WAVE);
    if (lane >= off) v += x;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = v;
  __syncthreads();
  N before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const N x = lds[w];
    before += w < wave ? x : 0;
    total += x;
  }
  return v + before;
}

__device__ __forceinline__ int pages_for(int tokens, int page) {
  return (int)(((long)tokens + page - 1) / page);
}

// A thread's four of the counts from `base` on; -1 behind the last.
__device__ __forceinline__ void four_refs(const Pool& p, int base, int* f) {
  const int at = base + 4 * threadIdx.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = at + i < p.pages ? p.refs[at + i] : -1;
}

// The lowest `need` free pages, in order, to `out`; false if there are fewer.
// `f`: the first counts, which the caller read before it knew `need`.
__device__ bool lowest_free(const Pool& p, int need, int* out, int* lds,
                            int* f) {
  int found = 0;
  for (int base = 0; base < p.pages && found < need; base += 4 * PLAN) {
    if (base) four_refs(p, base, f);
    int free = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) free += f[i] == 0;
    int total;
    int k = found + block_scan(free, lds, total) - free;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f[i] == 0) {
        if (k < need) out[k] = base + 4 * threadIdx.x + i;
        ++k;
      }
    found += total;
  }
  return found >= need;
}

// ---------------------------------------------------------------------- fork
// plan[0]: whether to go on; then for each pair the parent's length, its
// part-filled page and the page that takes its tokens (-1: none)
//
// Four beams of 201 tokens, 24 layers: 9.5 us, the latency of two launches that
// wait for each other (one cannot do: a page may only be written once the whole
// call is known to be sound).  63 samples of 8237 tokens, 32 layers: 121 us;
// 743 MB would take 148 at a copy's 5.0 TB/s, but all read the same page.
struct Pair {
  int length, from, to, pad;
};

__global__ __launch_bounds__(PLAN) void fork_plan_kernel(
    Pool p, const int* src, const int* dst, int n, int* go, Pair* plan,
    int* rows, int* fresh) {
  if (blockIdx.x > 0) {       // the parents' rows, before any is replaced
    const int i = blockIdx.x - 1;
    const int s = src[i];
    if (s < 0 || s >= p.slots) return;
    for (int j = threadIdx.x; j < p.width; j += PLAN)
      rows[(long)i * p.width + j] = p.tables[(long)s * p.width + j];
    return;
  }
  __shared__ int lds[WAVES];
  __shared__ int bad;
  extern __shared__ unsigned named[];   // a bit for each slot
  int refs[4];
  four_refs(p, 0, refs);
  if (threadIdx.x == 0) bad = 0;
  for (int i = threadIdx.x; i < (p.slots + 31) / 32; i += PLAN) named[i] = 0;
  __syncthreads();
  int copies = 0;
  Pair mine = {0, -1, -1, 0};
  for (int base = 0; base < n; base += PLAN) {
    const int i = base + threadIdx.x;
    Pair pr = {0, -1, -1, 0};
    bool copy = false;
    if (i < n) {
      const int s = src[i], t = dst[i];
      if (s < 0 || s >= p.slots || t < 0 || t >= p.slots) {
        atomicOr(&bad, BAD_SLOT);
      } else {
        if (atomicOr(&named[t >> 5], 1u << (t & 31)) & (1u << (t & 31)))
          atomicOr(&bad, BAD_SLOT);
        pr.length = p.lengths[s];
        if (pr.length < 0 || pages_for(pr.length, p.page) > p.width) {
          atomicOr(&bad, TOO_LONG);
          pr.length = 0;
        }
        if (s != t && pr.length % p.page) {
          pr.from = p.tables[(long)s * p.width + pr.length / p.page];
          if (pr.from < 0 || pr.from >= p.pages) atomicOr(&bad, BAD_PAGE);
          copy = true;
        }
      }
    }
    int total;
    const int k = copies + block_scan((int)copy, lds, total) - copy;
    if (copy) pr.to = k;      // the k-th free page, below
    mine = pr;
    if (i < n && n > PLAN) plan[i] = pr;
    copies += total;
  }
  __shared__ int few[PLAN];   // the pages, where they are not many
  int* out = copies <= PLAN ? few : fresh;
  const bool enough = lowest_free(p, copies, out, lds, refs);
  __threadfence_block();
  __syncthreads();
  if (n <= PLAN) {            // a pair a thread, still in its registers
    if ((int)threadIdx.x < n) {
      if (mine.to >= 0) mine.to = enough ? out[mine.to] : -1;
      plan[threadIdx.x] = mine;
    }
  } else {
    for (int i = threadIdx.x; i < n; i += PLAN)
      if (plan[i].to >= 0) plan[i].to = enough ? out[plan[i].to] : -1;
  }
  if (threadIdx.x == 0) {
    const int code = bad | (enough ? 0 : NO_PAGE);
    if (code) atomicOr(p.status, code);
    *go = code == 0;
  }
}

__global__ __launch_bounds__(BLOCK) void fork_apply_kernel(
    Pool p, const int* src, const int* dst, const int* go, const Pair* plan,
    const int* rows, char* pages, int planes, int groups, int token) {
  const int i = blockIdx.x;
  const Pair pr = plan[i];      // read at once with whether it holds
  const int from = src[i], into = dst[i];
  if (!*go) return;
  if (blockIdx.y == 0) {
    if (from == into) return;
    int* row = p.tables + (long)into * p.width;
    const int full = pr.length / p.page;
    for (int j = threadIdx.x; j < p.width; j += BLOCK) {
      const int old = row[j];
      if (old >= 0 && old < p.pages) atomicSub(p.refs + old, 1);
      int page = -1;
      if (j < full) page = rows[(long)i * p.width + j];
      else if (j == full) page = pr.to;
      if (page >= 0 && page < p.pages) atomicAdd(p.refs + page, 1);
      row[j] = page;
    }
    if (threadIdx.x == 0) p.lengths[into] = pr.length;
    return;
  }
  if (pr.to < 0) return;
  // the part-filled page's tokens, `token` bytes of each head of a plane
  const long head = (long)p.page * token, page = head * groups;
  char* plane = pages + (long)(blockIdx.y - 1) * p.pages * page;
  const char* a = plane + pr.from * page;
  char* b = plane + pr.to * page;
  const int part = pr.length % p.page * token / 16;   // 16-byte pieces
  for (int x = threadIdx.x; x < part * groups; x += BLOCK) {
    const long at = x / part * head + x % part * 16;
    *(float4*)(b + at) = *(const float4*)(a + at);
  }
}

// ---------------------------------------------------------------------- free
__global__ __launch_bounds__(BLOCK) void free_kernel(Pool p,
                                                     const int* slots) {
  const int s = slots[blockIdx.x];
  if (s < 0 || s >= p.slots) {
    if (threadIdx.x == 0) atomicOr(p.status, BAD_SLOT);
    return;
  }
  // exchanged, so that a slot named twice gives its pages back once
  for (int j = threadIdx.x; j < p.width; j += BLOCK) {
    const int page = atomicExch(p.tables + (long)s * p.width + j, -1);
    if (page >= 0 && page < p.pages) atomicSub(p.refs + page, 1);
  }
  if (threadIdx.x == 0) p.lengths[s] = 0;
}

// ------------------------------------------------------------------- compact
// Live pages behind the first `live` places go to the holes among these, in
// order.  moves[0]: how many; then (from, to) each; map: every page's place.
//
// 43 sequences of up to 2386 tokens in 1500 pages, 22 more retired, 16 layers:
// 320 us, of which the plan 6; 1.52 GB at 4.8 TB/s, near a copy's 5.0.
__global__ __launch_bounds__(PLAN) void compact_plan_kernel(Pool p, int* map,
                                                            int* moves,
                                                            int* movers) {
  __shared__ int lds[WAVES];
  int total, live = 0;
  for (int i = threadIdx.x; i < p.pages; i += PLAN) live += p.refs[i] > 0;
  block_scan(live, lds, total);
  live = total;
  int before = 0, holes = 0;
  for (int base = 0; base < p.pages; base += 4 * PLAN) {
    const int at = base + 4 * threadIdx.x;
    int n = 0;
    bool f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = at + i < p.pages && p.refs[at + i] > 0;
      n += f[i];
    }
    int k = before + block_scan(n, lds, total) - n;
    int h = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = at + i;
      if (x < p.pages) {
        map[x] = x;
        if (f[i]) {
          if (x >= live) movers[k] = x;      // the k-th live page
          ++k;
        } else if (x < live) {
          moves[2 + 2 * (x - k)] = x;        // the (x - k)-th hole
          ++h;
        }
      }
    }
    before += total;
    block_scan(h, lds, total);
    holes += total;
  }
  __threadfence_block();
  __syncthreads();
  for (int i = threadIdx.x; i < holes; i += PLAN) {
    const int to = moves[2 + 2 * i], from = movers[live - holes + i];
    moves[3 + 2 * i] = from;
    map[from] = to;
    p.refs[to] = p.refs[from];
    p.refs[from] = 0;
  }
  if (threadIdx.x == 0) {
    moves[0] = holes;
    moves[1] = live;
  }
}

// source and target never overlap, so several loads may be in flight
__device__ __forceinline__ void copy_page(char* pages, long bytes, int count,
                                          int plane, int from, int to) {
  const char* __restrict__ a = pages + ((long)plane * count + from) * bytes;
  char* __restrict__ b = pages + ((long)plane * count + to) * bytes;
#pragma unroll 4
  for (long x = (long)threadIdx.x * 16; x < bytes; x += BLOCK * 16)
    *(float4*)(b + x) = *(const float4*)(a + x);
}

__global__ __launch_bounds__(BLOCK) void compact_apply_kernel(
    Pool p, const int* map, const int* moves, char* pages, int planes,
    long bytes) {
  const long entries = (long)p.slots * p.width;
  for (long i = (long)blockIdx.x * BLOCK + threadIdx.x; i < entries;
       i += (long)gridDim.x * BLOCK) {
    const int page = p.tables[i];
    if (page >= 0 && page < p.pages) p.tables[i] = map[page];
  }
  const long items = (long)moves[0] * planes;
  for (long i = blockIdx.x; i < items; i += gridDim.x) {
    const int k = (int)(i / planes);
    copy_page(pages, bytes, p.pages, (int)(i % planes), moves[3 + 2 * k],
              moves[2 + 2 * k]);
  }
}

// ---------------------------------------------------------------------- copy
// 500 pages, 16 layers, 8 heads of 64: 415 us, 2.1 GB at 5.05 TB/s.
__global__ __launch_bounds__(BLOCK) void copy_kernel(const int* src,
                                                     const int* dst, int n,
                                                     char* pages, int planes,
                                                     int count, long bytes,
                                                     int* status) {
  const long items = (long)n * planes;
  for (long i = blockIdx.x; i < items; i += gridDim.x) {
    const int k = (int)(i / planes);
    const int a = src[k], b = dst[k];
    if (a < 0 || a >= count || b < 0 || b >= count) {
      if (threadIdx.x == 0) atomicOr(status, BAD_PAGE);
    } else if (a != b) {
      copy_page(pages, bytes, count, (int)(i % planes), a, b);
    }
  }
}

// -------------------------------------------------------------------- extend
// Room for counts[i] (or `each`) more tokens of each slot; lengths grow.  One
// block, for its scans: 256 rows by a token, 12000 pages, take 15 us.
__global__ __launch_bounds__(PLAN) void extend_kernel(Pool p, const int* slots,
                                                      const int* counts,
                                                      int each, int n,
                                                      int* offsets,
                                                      int* fresh) {
  __shared__ int lds[WAVES];
  __shared__ long wide[WAVES];   // all that is asked for may pass 32 bits
  __shared__ int bad;
  extern __shared__ unsigned named[];
  int refs[4];
  four_refs(p, 0, refs);
  if (threadIdx.x == 0) bad = 0;
  for (int i = threadIdx.x; i < (p.slots + 31) / 32; i += PLAN) named[i] = 0;
  __syncthreads();
  long need = 0;
  for (int base = 0; base < n; base += PLAN) {
    const int i = base + threadIdx.x;
    long more = 0;
    if (i < n) {
      const int s = slots[i], c = counts ? counts[i] : each;
      if (s < 0 || s >= p.slots || c < 0) {
        atomicOr(&bad, BAD_SLOT);
      } else {
        if (atomicOr(&named[s >> 5], 1u << (s & 31)) & (1u << (s & 31)))
          atomicOr(&bad, BAD_SLOT);
        const int len = p.lengths[s];
        if (len < 0 || (long)len + c > (long)p.width * p.page)
          atomicOr(&bad, TOO_LONG);
        else
          more = pages_for(len + c, p.page) - pages_for(len, p.page);
      }
    }
    long total;
    const long k = need + block_scan(more, wide, total) - more;
    if (i < n) offsets[i] = (int)k;   // used where all of it fits
    need += total;
  }
  __syncthreads();
  bool ok = bad == 0;
  // `fresh` holds as many as there are pages
  ok = ok && need <= p.pages && lowest_free(p, (int)need, fresh, lds, refs);
  __threadfence_block();
  __syncthreads();
  if (!ok) {
    if (threadIdx.x == 0) atomicOr(p.status, bad ? bad : NO_PAGE);
    return;
  }
  for (int i = threadIdx.x >> 6; i < n; i += WAVES) {   // a wave each
    const int s = slots[i], c = counts ? counts[i] : each;
    const int have = pages_for(p.lengths[s], p.page);
    const int more = pages_for(p.lengths[s] + c, p.page) - have;
    for (int j = threadIdx.x & 63; j < more; j += WAVE) {
      const int page = fresh[offsets[i] + j];
      p.tables[(long)s * p.width + have + j] = page;
      p.refs[page] = 1;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += PLAN)
    p.lengths[slots[i]] += counts ? counts[i] : each;
}

// --------------------------------------------------------------------- write
// Token t of the stream is token t - cu[i] of the last cu[i + 1] - cu[i] of
// slot i's sequence (one each without cu).  Sixteen lanes for each token and
// head.  256 rows' tokens, 8 heads of 128: 6.5 us, one launch's latency; prompts
// of 5883 tokens 9.4 us, 48 MB at 5.1 TB/s.
__global__ __launch_bounds__(BLOCK) void write_kernel(
    Pool p, const int* slots, const int* cu, int n, int tokens, char* keys,
    char* values, const char* k, const char* v, int groups, int token, long kt,
    long kh, long vt, long vh) {
  const long item = (long)blockIdx.x * (BLOCK / 16) + threadIdx.x / 16;
  const long t = item / groups;
  const int g = (int)(item % groups), x = threadIdx.x % 16;
  if (t >= tokens) return;
  int i = (int)t, back = 1;          // tokens from the sequence's end
  if (cu) {
    int lo = 0, hi = n;              // the last i with cu[i] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (cu[mid] <= t) lo = mid; else hi = mid;
    }
    i = lo;
    if (n == 0 || t < cu[i] || t >= cu[i + 1]) return;
    back = cu[i + 1] - (int)t;
  }
  const int s = slots[i];
  if (s < 0 || s >= p.slots) {
    atomicOr(p.status, BAD_SLOT);
    return;
  }
  const int at = p.lengths[s] - back;
  if (at < 0 || at / p.page >= p.width) {
    atomicOr(p.status, TOO_LONG);
    return;
  }
  const int page = p.tables[(long)s * p.width + at / p.page];
  if (page < 0 || page >= p.pages) {
    atomicOr(p.status, BAD_PAGE);
    return;
  }
  // where an extension found no page, the last place is in an older one
  if (p.refs[page] > 1) {
    atomicOr(p.status, SHARED);
    return;
  }
  const long to =
      (((long)page * groups + g) * p.page + at % p.page) * token;
  for (int b = x * 16; b < token; b += 256) {
    *(float4*)(keys + to + b) = *(const float4*)(k + t * kt + g * kh + b);
    *(float4*)(values + to + b) = *(const float4*)(v + t * vt + g * vh + b);
  }
}

Pool pool_of(int* refs, int* tables, int* lengths, int* status, int pages,
             int slots, int width, int page) {
  return {refs, tables, lengths, status, pages, slots, width, page};
}

}  // namespace

void launch_cache_fork(int* refs, int* tables, int* lengths, int* status,
                       int pages, int slots, int width, int page, void* data,
                       int planes, int groups, int token, const int* src,
                       const int* dst, int n, int* scratch,
                       hipStream_t stream) {
  const Pool p =
      pool_of(refs, tables, lengths, status, pages, slots, width, page);
  int* go = scratch;                        // [4]
  Pair* plan = (Pair*)(scratch + 4);        // [n] of 4
  int* fresh = scratch + 4 + 4l * n;        // [n]
  int* rows = fresh + n;                    // [n, W]
  hipLaunchKernelGGL(fork_plan_kernel, dim3(n + 1), dim3(PLAN),
                     (slots + 31) / 32 * 4, stream, p, src, dst, n, go, plan,
                     rows, fresh);
  HIP_CHECK_LAUNCH();
  hipLaunchKernelGGL(fork_apply_kernel, dim3(n, planes + 1), dim3(BLOCK), 0,
                     stream, p, src, dst, go, plan, rows, (char*)data, planes,
                     groups, token);
  HIP_CHECK_LAUNCH();
}

void launch_cache_free(int* refs, int* tables, int* lengths, int* status,
                       int pages, int slots, int width, int page,
                       const int* list, int n, hipStream_t stream) {
  const Pool p =
      pool_of(refs, tables, lengths, status, pages, slots, width, page);
  hipLaunchKernelGGL(free_kernel, dim3(n), dim3(BLOCK), 0, stream, p, list);
  HIP_CHECK_LAUNCH();
}

void launch_cache_compact(int* refs, int* tables, int* lengths, int* status,
                          int pages, int slots, int width, int page,
                          void* data, int planes, long bytes, int* scratch,
                          hipStream_t stream) {
  const Pool p =
      pool_of(refs, tables, lengths, status, pages, slots, width, page);
  int* moves = scratch;                     // [2 + 2 P]
  int* map = scratch + 2 + 2l * pages;      // [P]
  int* movers = map + pages;                // [P]
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(PLAN), 0, stream, p,
                     map, moves, movers);
  HIP_CHECK_LAUNCH();
  // at most half the pages move
  const long items = std::max<long>(
      (long)pages / 2 * planes, ((long)slots * width + BLOCK - 1) / BLOCK);
  hipLaunchKernelGGL(compact_apply_kernel,
                     dim3((unsigned)std::min<long>(std::max<long>(items, 1),
                                                   4096)),
                     dim3(BLOCK), 0, stream, p, map, moves, (char*)data,
                     planes, bytes);
  HIP_CHECK_LAUNCH();
}

void launch_cache_copy(const int* src, const int* dst, int n, void* data,
                       int planes, int pages, long bytes, int* status,
                       hipStream_t stream) {
  hipLaunchKernelGGL(copy_kernel,
                     dim3((unsigned)std::min<long>((long)n * planes, 4096)),
                     dim3(BLOCK), 0, stream, src, dst, n, (char*)data, planes,
                     pages, bytes, status);
  HIP_CHECK_LAUNCH();
}

void launch_cache_extend(int* refs, int* tables, int* lengths, int* status,
                         int pages, int slots, int width, int page,
                         const int* list, const int* counts, int each, int n,
                         int* scratch, hipStream_t stream) {
  const Pool p =
      pool_of(refs, tables, lengths, status, pages, slots, width, page);
  hipLaunchKernelGGL(extend_kernel, dim3(1), dim3(PLAN), (slots + 31) / 32 * 4,
                     stream, p, list, counts, each, n, scratch, scratch + n);
  HIP_CHECK_LAUNCH();
}

void launch_cache_write(int* refs, int* tables, int* lengths, int* status,
                        int pages, int slots, int width, int page,
                        const int* list, const int* cu, int n, int tokens,
                        void* keys, void* values, const void* k, const void* v,
                        int groups, int token, long kt, long kh, long vt,
                        long vh, hipStream_t stream) {
  const Pool p =
      pool_of(refs, tables, lengths, status, pages, slots, width, page);
  const long items = (long)tokens * groups;
  hipLaunchKernelGGL(write_kernel,
                     dim3((unsigned)((items + BLOCK / 16 - 1) / (BLOCK / 16))),
                     dim3(BLOCK), 0, stream, p, list, cu, n, tokens,
                     (char*)keys, (char*)values, (const char*)k,
                     (const char*)v, groups, token, kt, kh, vt, vh);
  HIP_CHECK_LAUNCH();
}
