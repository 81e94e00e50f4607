// Routes sorted by expert, the tokens' rows in that order, and the way back with weights; their gradients.
//
//   key(r) = ids[r], or E outside [0, E);  place(r) = number of routes q with (key(q), q) < (key(r), r)
//   sort:    rows[place(t, j)] = x[t]                      its gradient: dx[t] = sum_j drows[place(t, j)]
//   unsort:  out[t] = sum_j w[t, j] rows[place(t, j)]      its gradients: drows[place(t, j)] = w[t, j] dout[t],
//                                                          dw[t, j] = <dout[t], rows[place(t, j)]>
// Routes without an expert have no place outside this file; the rows behind the last expert's hold zeros.  Nothing depends on
// the order of atomics: they only count.
#include <algorithm>
#include <cmath>

#include "awq_launch.h"
#include "awq_mx_common.h"

namespace awq {

typedef u32x4 u32x4_any __attribute__((aligned(2)));  // 16 bytes at any address of a 16-bit element

// ------------------------------------------------------------------ rows in pieces of 16 bytes
// Piece p of a row of n elements of ES bytes.  The last one ends with the row and overlaps the one before it, so no row
// needs a remainder; rows shorter than a piece go by elements.
template <int ES>
struct Pieces {
  static constexpr int VEC = 16 / ES;
  static __device__ __forceinline__ int start(int p, int n) { return min(p * VEC, n - VEC); }
  // PAST the caches: for more rows than those hold
  template <bool PAST = false>
  static __device__ __forceinline__ u32x4 load(const void* row, int p, int n) {
    if (n >= VEC) {
      const u32x4_any* const at = (const u32x4_any*)((const char*)row + (int64_t)start(p, n) * ES);
      if constexpr (PAST) return __builtin_nontemporal_load(at);
      else return *at;
    }
    u32x4 v = {0, 0, 0, 0};
    for (int i = 0; i < n; ++i) {
      if constexpr (ES == 4) v[i] = ((const uint32_t*)row)[i];
      else v[i >> 1] |= (uint32_t)((const uint16_t*)row)[i] << (16 * (i & 1));
    }
    return v;
  }
  template <bool PAST = false>
  static __device__ __forceinline__ void store(void* row, int p, int n, const u32x4& v) {
    if (n >= VEC) {
      u32x4_any* const at = (u32x4_any*)((char*)row + (int64_t)start(p, n) * ES);
      if constexpr (PAST) __builtin_nontemporal_store(v, at);
      else *at = v;
      return;
    }
    for (int i = 0; i < n; ++i) {
      if constexpr (ES == 4) ((uint32_t*)row)[i] = v[i];
      else ((uint16_t*)row)[i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
    }
  }
};

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);
template <typename T>
__device__ __forceinline__ void unpack(const u32x4& p, float* v) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(f32x4, p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = from_bits<T>((uint16_t)(p[i] & 0xFFFF)), v[2 * i + 1] = from_bits<T>((uint16_t)(p[i] >> 16));
  }
}
template <typename T>
__device__ __forceinline__ u32x4 packed(const float* v) {
  u32x4 p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) p[i] = __builtin_bit_cast(uint32_t, v[i]);
    else p[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
  }
  return p;
}

// Which token and piece a thread has: rows of at most half a block's pieces share blocks, longer ones take one or several.
struct RowGrid {
  int pieces, per_block;  // tokens of a block, two at least; 1 where a row has blocks of its own
};
struct TokenPiece {
  int64_t token;
  int piece;
};
__device__ __forceinline__ TokenPiece token_piece(const RowGrid& g) {
  if (g.per_block == 1) return {(int64_t)blockIdx.x, (int)(blockIdx.y * blockDim.x + threadIdx.x)};
  const int mine = (int)threadIdx.x / g.pieces;
  // threads behind the block's last token have no piece
  return {(int64_t)blockIdx.x * g.per_block + mine, mine < g.per_block ? (int)threadIdx.x - mine * g.pieces : g.pieces};
}

// ------------------------------------------------------------------ sort
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64;

struct SortArgs {
  const void *x, *ids;
  int64_t ldx;
  void* rows;
  int *offsets, *experts, *places;
  int64_t T;
  int H, E, topk, id64, R;
  int own;       // tokens of a block
  int segments;  // 0: every block counts all routes
  int per;       // routes of a segment
  int* counts;   // [segments][E + 1], the last for routes without an expert
};
__device__ __forceinline__ int sort_key(const SortArgs& a, int64_t r) {
  const int64_t e = mx_route_id(a.ids, a.id64, r);
  return e >= 0 && e < a.E ? (int)e : a.E;
}

// Sum of the threads' c before this one's, on top of carry, which grows by all of them.
__device__ __forceinline__ int block_scan(int c, int* carry, int* tot) {
  const int t = threadIdx.x, wave = t >> 6, incl = wave_incl_scan_i32(c);
  if ((t & 63) == 63) tot[wave] = incl;
  __syncthreads();
  int first = incl - c + *carry, all = 0;
  for (int w = 0; w < kSortWaves; ++w) {
    if (w < wave) first += tot[w];
    all += tot[w];
  }
  *carry += all;
  __syncthreads();
  return first;
}

// A block counts a segment: 16384 routes 2.8 us, 131072 4.8, its launch and one round of loads and LDS adds.
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs a) {
  __shared__ int count[1025];
  for (int e = threadIdx.x; e <= a.E; e += kSortThreads) count[e] = 0;
  __syncthreads();
  const int64_t start = (int64_t)blockIdx.x * a.per, end = min(start + a.per, (int64_t)a.R);
#pragma unroll 4
  for (int64_t r = start + threadIdx.x; r < end; r += kSortThreads) atomicAdd(&count[sort_key(a, r)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= a.E; e += kSortThreads) a.counts[(int64_t)blockIdx.x * (a.E + 1) + e] = count[e];
}

// A block places the routes of its tokens and copies their rows.  Bound by its chain (ids, counts, scan, places, rows): 4 tokens 4.3
// us, 2048 tokens, top 8, H = 2048 with the counts' launch 19.5, where a copy of the same bytes takes 15.  To place its routes it
// counts those in front of its own and all of them, by expert: in LDS where they are few, else those in front of it in its segment
// and the rest from the segments' counts.  Its own, at most kMostOwn, are placed by one wave, 64 at a time in their order; lanes
// of the same expert find each other by its bits.
constexpr int kMostOwn = 1024;
template <int ES>  // 0: no rows
__global__ void __launch_bounds__(kSortThreads) sort_kernel(SortArgs a) {
  __shared__ int before[1025], rest[1025], tot[kSortWaves], all[kSortThreads], front[kSortThreads], place[kMostOwn];
  const int t = threadIdx.x;
  const int64_t token0 = (int64_t)blockIdx.x * a.own;
  const int first = (int)token0 * a.topk, mine = min(a.own * a.topk, a.R - first), segment = a.segments ? first / a.per : 0;
  for (int e = t; e <= a.E; e += kSortThreads) before[e] = rest[e] = 0;
  __syncthreads();
  const int last = a.segments ? first : a.R;
#pragma unroll 4
  for (int r = segment * a.per + t; r < last; r += kSortThreads) atomicAdd((r < first ? before : rest) + sort_key(a, r), 1);
  __syncthreads();
  int carry = 0;
  // routes without an expert come last; they are placed to say which rows to clear
  for (int e0 = 0; e0 <= a.E; e0 += kSortThreads) {
    const int e = e0 + t;
    int count = 0, ahead = 0;
    if (a.segments) {  // the threads of an expert share the segments
      const int wide = min(a.E + 1 - e0, kSortThreads), shares = min(kSortThreads / wide, 16), share = t / wide;
      if (share < shares) {
#pragma unroll 8
        for (int s = share; s < a.segments; s += shares) {
          const int c = a.counts[(int64_t)s * (a.E + 1) + e0 + t - share * wide];
          count += c;
          ahead += s < segment ? c : 0;
        }
      }
      all[t] = count, front[t] = ahead;
      __syncthreads();
      if (e <= a.E)
        for (int i = 1; i < shares; ++i) count += all[i * wide + t], ahead += front[i * wide + t];
    } else if (e <= a.E) {
      count = before[e] + rest[e];
    }
    const int at = block_scan(e <= a.E ? count : 0, &carry, tot);
    if (e > a.E) continue;
    if (blockIdx.x == 0) a.offsets[e] = at;  // offsets[E]: the first place of a route without an expert
    before[e] += at + ahead;
  }
  __syncthreads();
  if (t < 64) {
    for (int r0 = 0; r0 < mine; r0 += 64) {
      const bool has = r0 + t < mine;
      const int e = has ? sort_key(a, first + r0 + t) : a.E;
      uint64_t same = __ballot(has);
      for (int bit = 1; bit <= a.E; bit <<= 1) {
        const uint64_t set = __ballot(e & bit);
        same &= e & bit ? set : ~set;
      }
      const int rank = __popcll(same & ((1ull << t) - 1)), at = before[e];
      if (has) {
        place[r0 + t] = e < a.E ? at + rank : ~(at + rank);
        a.places[first + r0 + t] = e < a.E ? at + rank : -1;
        a.experts[at + rank] = e < a.E ? e : -1;
      }
      __builtin_amdgcn_wave_barrier();
      if (has && rank == 0) before[e] = at + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
  if constexpr (ES > 0) {
    __syncthreads();
    const int pieces = (a.H + 16 / ES - 1) / (16 / ES), tokens = mine / a.topk;
    for (int64_t i = t; i < (int64_t)tokens * pieces; i += kSortThreads) {
      const int token = (int)(i / pieces), p = (int)(i - (int64_t)token * pieces);
      const u32x4 v = Pieces<ES>::load((const char*)a.x + (token0 + token) * a.ldx * ES, p, a.H);
      for (int j = 0; j < a.topk; ++j) {
        const int at = place[token * a.topk + j];
        Pieces<ES>::store((char*)a.rows + (int64_t)(at < 0 ? ~at : at) * a.H * ES, p, a.H, at < 0 ? u32x4{0, 0, 0, 0} : v);
      }
    }
  }
}

// Many rows, by blocks of their own: more of them, which the memory's queues stay full with.  16384 tokens, top 8, H = 2048: 101 us,
// 604 MB read and written, 6.0 TB/s.
template <int ES, bool PAST>
__global__ void __launch_bounds__(256) sort_rows_kernel(SortArgs a, RowGrid g) {
  const TokenPiece tp = token_piece(g);
  if (tp.token >= a.T || tp.piece >= g.pieces) return;
  const u32x4 v = Pieces<ES>::load((const char*)a.x + tp.token * a.ldx * ES, tp.piece, a.H);
  const int* const places = a.places + tp.token * a.topk;
  for (int j = 0; j < a.topk; ++j) {
    const int p = places[j];
    if (p >= 0) {
      Pieces<ES>::template store<PAST>((char*)a.rows + (int64_t)p * a.H * ES, tp.piece, a.H, v);
    }
  }
  // as many rows as the token has routes, behind the last expert's
  const int64_t first = a.offsets[a.E] + tp.token * a.topk;
  for (int64_t p = first; p < min(first + a.topk, (int64_t)a.R); ++p)
    Pieces<ES>::store((char*)a.rows + p * a.H * ES, tp.piece, a.H, u32x4{0, 0, 0, 0});
}

// ------------------------------------------------------------------ unsort
struct UnsortArgs {
  const void *rows, *weights, *upstream;
  const int *places, *total;
  int64_t T, ldu;
  int H, topk, w_dtype, R;
  void *out, *grad_rows, *grad_weights;
  int64_t ldo;
};

// A thread has a piece of a token's row, the loads of eight of its routes at once in flight.  HBM-bound: 1000 tokens, top 8, H = 4096
// 14.6 us, 5.0 TB/s; 16384, H = 2048 111 us, 5.4 TB/s, the gradient of sort, without weights, 101 us.
template <typename T, bool WEIGHTED, bool PAST>
__global__ void __launch_bounds__(256) unsort_kernel(UnsortArgs a, RowGrid g) {
  constexpr int ES = (int)sizeof(T), VEC = kVec<T>, AT_ONCE = 8;
  const TokenPiece tp = token_piece(g);
  if (tp.token >= a.T || tp.piece >= g.pieces) return;
  float s[VEC] = {};
  for (int j0 = 0; j0 < a.topk; j0 += AT_ONCE) {
    int place[AT_ONCE];
    float w[AT_ONCE];
    u32x4 v[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int64_t r = tp.token * a.topk + j0 + j;
      place[j] = j0 + j < a.topk ? a.places[r] : -1;
      if ((unsigned)place[j] >= (unsigned)a.R) place[j] = -1;
      if constexpr (WEIGHTED) w[j] = place[j] >= 0 ? mx_route_weight(a.weights, a.w_dtype, r) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (place[j] >= 0) v[j] = Pieces<ES>::template load<PAST>((const char*)a.rows + (int64_t)place[j] * a.H * ES, tp.piece, a.H);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (place[j] >= 0) {
        float f[VEC];
        unpack<T>(v[j], f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] = WEIGHTED ? fmaf(f[i], w[j], s[i]) : s[i] + f[i];
      }
  }
  Pieces<ES>::store((char*)a.out + tp.token * a.ldo * ES, tp.piece, a.H, packed<T>(s));
}

// A block has a token: its upstream row is read once and goes out k times, weighted, while it meets the experts' rows.  HBM-bound:
// 16384 tokens, top 8, H = 2048 204 us, 1.14 GB read and written, 5.6 TB/s.
template <typename T, bool ROWS, bool WEIGHTS, int PAST>  // stores past the caches, 2: loads as well
__global__ void __launch_bounds__(256) unsort_grad_kernel(UnsortArgs a) {
  constexpr int ES = (int)sizeof(T), VEC = kVec<T>, AT_ONCE = 8;
  __shared__ float part[4][AT_ONCE];
  const int t = threadIdx.x, pieces = (a.H + VEC - 1) / VEC;
  const int64_t token = blockIdx.x;
  for (int j0 = 0; j0 < a.topk; j0 += AT_ONCE) {
    int place[AT_ONCE];
    float w[AT_ONCE], dot[AT_ONCE] = {};
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int64_t r = token * a.topk + j0 + j;
      place[j] = j0 + j < a.topk ? a.places[r] : -1;
      if ((unsigned)place[j] >= (unsigned)a.R) place[j] = -1;
      if constexpr (ROWS) w[j] = place[j] < 0 ? 0.f : a.weights ? mx_route_weight(a.weights, a.w_dtype, r) : 1.f;
    }
    for (int p = t; p < pieces; p += 256) {
      float u[VEC];
      unpack<T>(Pieces<ES>::load((const char*)a.upstream + token * a.ldu * ES, p, a.H), u);
      if constexpr (WEIGHTS) {
        u32x4 v[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
          if (place[j] >= 0) v[j] = Pieces<ES>::template load<(PAST > 1)>((const char*)a.rows + (int64_t)place[j] * a.H * ES, p, a.H);
        // elements that the piece before has too
        const int twice = a.H >= VEC ? p * VEC - Pieces<ES>::start(p, a.H) : 0;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
          if (place[j] >= 0) {
            float f[VEC];
            unpack<T>(v[j], f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) dot[j] = i >= twice ? fmaf(f[i], u[i], dot[j]) : dot[j];
          }
      }
      if constexpr (ROWS) {
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
          if (place[j] >= 0) {
            float f[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = w[j] * u[i];
            Pieces<ES>::template store<(PAST > 0)>((char*)a.grad_rows + (int64_t)place[j] * a.H * ES, p, a.H, packed<T>(f));
          }
      }
    }
    if constexpr (WEIGHTS) {
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        for (int d = 32; d; d >>= 1) dot[j] += __shfl_xor(dot[j], d);
        if ((t & 63) == 0) part[t >> 6][j] = dot[j];
      }
      __syncthreads();
      if (t < AT_ONCE && j0 + t < a.topk) {
        const float s = (part[0][t] + part[1][t]) + (part[2][t] + part[3][t]);
        const int64_t r = token * a.topk + j0 + t;
        if (a.w_dtype == AWQ_DTYPE_F32) ((float*)a.grad_weights)[r] = s;
        else ((uint16_t*)a.grad_weights)[r] = a.w_dtype == AWQ_DTYPE_F16 ? f2h_bits(s) : f2bf_bits(s);
      }
      __syncthreads();
    }
  }
  if constexpr (ROWS) {
    const int64_t first = max(a.total[0], 0) + token * a.topk;
    for (int64_t r = first; r < min(first + a.topk, (int64_t)a.R); ++r)
      for (int p = t; p < pieces; p += 256) Pieces<ES>::store((char*)a.grad_rows + r * a.H * ES, p, a.H, u32x4{0, 0, 0, 0});
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

// Segments that the routes are counted in, 0 where every block counts all of them and no other launch does (64 experts, top 8,
// H = 2048: 576 tokens 9.2 us, with segments 11.1, 896 11.9 and 12.0, 1000 13.1 and 12.8, 2048 24.3 and 19.5; 8000 tokens, top 1,
// H = 512 8.6 and 9.7).  A block reads every segment's counts and, on average, half a segment's ids, of which each costs it about
// eight counts.
static int sort_segments(int64_t R, int E) {
  if (R <= 8192) return 0;
  const int64_t per = std::max<int64_t>(512, (int64_t)std::sqrt((double)R * E / 2));
  return (int)std::min<int64_t>(cdiv(R, per), 1024);
}
// Whether rows go past the caches, of which the last holds 256 MB: where they do not fit there anyway.  16384 tokens, top 8,
// H = 2048 (537 MB): moe_sort 130 -> 117 us, moe_unsort 121 -> 115, without weights 119 -> 104, its gradients 221 -> 206; half as
// many tokens 61 -> 63, 53 -> 60 and 46 -> 53, but the gradients, which hold the rows twice, 116 -> 98 with their stores alone.
static bool past_caches(int64_t R, int64_t row_bytes, int64_t mib) { return R * row_bytes > mib << 20; }

size_t moe_sort_workspace_bytes(int64_t T, int E, int topk) { return (size_t)sort_segments(T * topk, E) * (size_t)(E + 1) * 4; }

// Threads and blocks of a launch over tokens and pieces of their rows.
struct RowLaunch {
  RowGrid g;
  dim3 grid, block;
};
static RowLaunch row_launch(int64_t T, int64_t H, int vec) {
  const int pieces = (int)cdiv(H, vec), ny = (int)cdiv(pieces, 256);
  if (pieces <= 128) {
    const int per = 256 / pieces;
    return {{pieces, per}, dim3((unsigned)cdiv(T, per)), dim3(256)};
  }
  return {{pieces, 1}, dim3((unsigned)T, (unsigned)ny), dim3((unsigned)(cdiv(cdiv(pieces, ny), 64) * 64))};
}

int launch_moe_sort(const MoeSortCall& c, hipStream_t st) {
  SortArgs a{};
  a.x = c.x, a.ids = c.ids, a.ldx = c.ldx, a.rows = c.rows, a.offsets = c.offsets, a.experts = c.experts, a.places = c.places;
  a.T = c.T, a.H = (int)c.H, a.E = c.E, a.topk = c.topk, a.id64 = c.id64, a.R = (int)(c.T * c.topk);
  a.counts = (int*)c.workspace;
  a.segments = sort_segments(a.R, c.E);
  if (a.segments) {
    a.per = (int)cdiv(a.R, a.segments);
    a.segments = (int)cdiv(a.R, a.per);
    sort_count_kernel<<<(unsigned)a.segments, kSortThreads, 0, st>>>(a);
    if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  }
  // blocks that wait for counts do not keep HBM busy, a launch more costs 3 us: 134 MB of rows 30.7 us, apart 33.1, 268 MB (4096
  // tokens, top 8, H = 4096) 69.3 and 59.2
  const bool apart = past_caches(a.R, c.H * c.elem_bytes, 192);
  a.own = (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(c.T, 512), kMostOwn / c.topk));
  const dim3 grid((unsigned)std::max<int64_t>(1, cdiv(c.T, a.own)));
  if (apart) sort_kernel<0><<<grid, kSortThreads, 0, st>>>(a);
  else if (c.elem_bytes == 2) sort_kernel<2><<<grid, kSortThreads, 0, st>>>(a);
  else sort_kernel<4><<<grid, kSortThreads, 0, st>>>(a);
  if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  if (!apart) return AWQ_OK;
  const RowLaunch l = row_launch(c.T, c.H, 16 / c.elem_bytes);
  const bool past = past_caches(a.R, c.H * c.elem_bytes, 384);
  if (c.elem_bytes == 2 && past) sort_rows_kernel<2, true><<<l.grid, l.block, 0, st>>>(a, l.g);
  else if (c.elem_bytes == 2) sort_rows_kernel<2, false><<<l.grid, l.block, 0, st>>>(a, l.g);
  else if (past) sort_rows_kernel<4, true><<<l.grid, l.block, 0, st>>>(a, l.g);
  else sort_rows_kernel<4, false><<<l.grid, l.block, 0, st>>>(a, l.g);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

static UnsortArgs unsort_args(const MoeUnsortCall& c) {
  UnsortArgs a{};
  a.rows = c.rows, a.weights = c.weights, a.upstream = c.upstream, a.places = c.places, a.total = c.total;
  a.T = c.T, a.ldu = c.ldu, a.H = (int)c.H, a.topk = c.topk, a.w_dtype = c.w_dtype, a.R = (int)(c.T * c.topk);
  a.out = c.out, a.grad_rows = c.grad_rows, a.grad_weights = c.grad_weights, a.ldo = c.ldo;
  return a;
}

template <typename T>
static void unsort_typed(const UnsortArgs& a, hipStream_t st) {
  const RowLaunch l = row_launch(a.T, a.H, kVec<T>);
  const bool past = past_caches(a.R, a.H * (int64_t)sizeof(T), 384);
  if (a.weights && past) unsort_kernel<T, true, true><<<l.grid, l.block, 0, st>>>(a, l.g);
  else if (a.weights) unsort_kernel<T, true, false><<<l.grid, l.block, 0, st>>>(a, l.g);
  else if (past) unsort_kernel<T, false, true><<<l.grid, l.block, 0, st>>>(a, l.g);
  else unsort_kernel<T, false, false><<<l.grid, l.block, 0, st>>>(a, l.g);
}
int launch_moe_unsort(const MoeUnsortCall& c, hipStream_t st) {
  const UnsortArgs a = unsort_args(c);
  if (c.dtype == AWQ_DTYPE_F16) unsort_typed<f16>(a, st);
  else if (c.dtype == AWQ_DTYPE_BF16) unsort_typed<bf16>(a, st);
  else unsort_typed<float>(a, st);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

template <typename T>
static void unsort_grad_typed(const UnsortArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.T);
  const int64_t row = a.H * (int64_t)sizeof(T);
  const bool out = past_caches(a.R, row, 192), in = past_caches(a.R, row, 384);
  if (a.grad_rows && a.grad_weights) {
    if (in) unsort_grad_kernel<T, true, true, 2><<<grid, 256, 0, st>>>(a);
    else if (out) unsort_grad_kernel<T, true, true, 1><<<grid, 256, 0, st>>>(a);
    else unsort_grad_kernel<T, true, true, 0><<<grid, 256, 0, st>>>(a);
  } else if (a.grad_rows) {
    if (in) unsort_grad_kernel<T, true, false, 1><<<grid, 256, 0, st>>>(a);
    else unsort_grad_kernel<T, true, false, 0><<<grid, 256, 0, st>>>(a);
  } else {
    if (in) unsort_grad_kernel<T, false, true, 2><<<grid, 256, 0, st>>>(a);
    else unsort_grad_kernel<T, false, true, 0><<<grid, 256, 0, st>>>(a);
  }
}
int launch_moe_unsort_grad(const MoeUnsortCall& c, hipStream_t st) {
  const UnsortArgs a = unsort_args(c);
  if (c.dtype == AWQ_DTYPE_F16) unsort_grad_typed<f16>(a, st);
  else if (c.dtype == AWQ_DTYPE_BF16) unsort_grad_typed<bf16>(a, st);
  else unsort_grad_typed<float>(a, st);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

}  // namespace awq_host
