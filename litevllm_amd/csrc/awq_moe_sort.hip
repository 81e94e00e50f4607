// Routes sorted by expert, the tokens' rows in that order, and the way back with weights; their gradients.
//
//   key(r) = ids[r], or E outside [0, E);  place(r) = number of routes q with (key(q), q) < (key(r), r)
//   sort:    rows[place(t, j)] = x[t]                      its gradient: dx[t] = sum_j drows[place(t, j)]
//   unsort:  out[t] = sum_j w[t, j] rows[place(t, j)]      its gradients: drows[place(t, j)] = w[t, j] dout[t],
//                                                          dw[t, j] = <dout[t], rows[place(t, j)]>
// Routes without an expert have no place outside this file; the rows behind the last expert's hold zeros.  Nothing depends on
// the order of atomics: they only count.
#include <algorithm>

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
  static __device__ __forceinline__ u32x4 load(const void* row, int p, int n) {
    if (n >= VEC) return *(const u32x4_any*)((const char*)row + (int64_t)start(p, n) * ES);
    u32x4 v = {0, 0, 0, 0};
    for (int i = 0; i < n; ++i) {
      if constexpr (ES == 4) v[i] = ((const uint32_t*)row)[i];
      else v[i >> 1] |= (uint32_t)((const uint16_t*)row)[i] << (16 * (i & 1));
    }
    return v;
  }
  static __device__ __forceinline__ void store(void* row, int p, int n, const u32x4& v) {
    if (n >= VEC) {
      *(u32x4_any*)((char*)row + (int64_t)start(p, n) * ES) = v;
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
  int pieces, per_block;  // tokens of a block; 1 where a row has blocks of its own
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
  // many routes
  int* hist;  // [blocks][E]
  int blocks;
  int64_t per;  // routes of a block, a multiple of kSortThreads
};
__device__ __forceinline__ int sort_key(const SortArgs& a, int64_t r) {
  const int64_t e = mx_route_id(a.ids, a.id64, r);
  return e >= 0 && e < a.E ? (int)e : a.E;
}

// offsets[e] for the experts 512 c + t from their counts, with the offset before them; returns it.
__device__ __forceinline__ int scan_experts(int c, int* carry, int* tot) {
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

// Up to kCountRoutes routes in one launch: the blocks of a token count the places of its routes themselves, one comparison a
// route and place with the route's number in the low bits; one more block has the offsets.
constexpr int kCountRoutes = 4096, kCountBits = 12;
template <int ES>
__global__ void __launch_bounds__(kSortThreads) sort_few_kernel(SortArgs a) {
  constexpr int AT_ONCE = 8;
  const int t = threadIdx.x, wave = t >> 6;
  if ((int64_t)blockIdx.x == a.T) {
    __shared__ int hist[1025], tot[kSortWaves];
    if (blockIdx.y > 0) return;
    for (int e = t; e <= a.E; e += kSortThreads) hist[e] = 0;
    __syncthreads();
    for (int r = t; r < a.R; r += kSortThreads) atomicAdd(&hist[sort_key(a, r)], 1);
    __syncthreads();
    int carry = 0;
    for (int e0 = 0; e0 < a.E; e0 += kSortThreads) {
      const int e = e0 + t, first = scan_experts(e < a.E ? hist[e] : 0, &carry, tot);
      if (e < a.E) a.offsets[e] = first;
    }
    if (t == 0) a.offsets[a.E] = carry;
    return;
  }
  __shared__ int part[kSortWaves][AT_ONCE];
  const int64_t token = blockIdx.x;
  const int pieces = (a.H + 16 / ES - 1) / (16 / ES);
  for (int j0 = 0; j0 < a.topk; j0 += AT_ONCE) {
    int mine[AT_ONCE], count[AT_ONCE] = {};
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int r = (int)token * a.topk + min(j0 + j, a.topk - 1);
      mine[j] = sort_key(a, r) << kCountBits | r;
    }
    for (int r0 = 0; r0 < a.R; r0 += kSortThreads) {
      const int r = r0 + t, key = r < a.R ? sort_key(a, r) << kCountBits | r : 0x7FFFFFFF;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) count[j] += __popcll(__ballot(key < mine[j]));
    }
    if ((t & 63) == 0) {
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) part[wave][j] = count[j];
    }
    __syncthreads();
    int place[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      place[j] = 0;
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) place[j] += part[w][j];
    }
    if (blockIdx.y == 0) {
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        if (t != j || j0 + j >= a.topk) continue;
        const int e = mine[j] >> kCountBits;
        a.places[token * a.topk + j0 + j] = e < a.E ? place[j] : -1;
        a.experts[place[j]] = e < a.E ? e : -1;
      }
    }
    for (int p = blockIdx.y * kSortThreads + t; p < pieces; p += gridDim.y * kSortThreads) {
      const u32x4 v = Pieces<ES>::load((const char*)a.x + token * a.ldx * ES, p, a.H);
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j)
        if (j0 + j < a.topk)
          Pieces<ES>::store((char*)a.rows + (int64_t)place[j] * a.H * ES, p, a.H, mine[j] >> kCountBits < a.E ? v : u32x4{0, 0, 0, 0});
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs a) {
  __shared__ int hist[1025];
  for (int e = threadIdx.x; e <= a.E; e += kSortThreads) hist[e] = 0;
  __syncthreads();
  const int64_t start = (int64_t)blockIdx.x * a.per, end = min(start + a.per, (int64_t)a.R);
  for (int64_t r = start + threadIdx.x; r < end; r += kSortThreads) atomicAdd(&hist[sort_key(a, r)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += kSortThreads) a.hist[(int64_t)blockIdx.x * a.E + e] = hist[e];
}

// Block b places its routes: behind the experts before, the same expert's routes of the blocks before and of the waves
// before.  A wave has consecutive routes, 64 at a time in order; lanes of the same expert find each other by its bits.
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortArgs a) {
  extern __shared__ int next[];  // [kSortWaves][E + 1]: next place of a wave's routes to an expert
  __shared__ int tot[kSortWaves];
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63, ld = a.E + 1;
  for (int i = t; i < kSortWaves * ld; i += kSortThreads) next[i] = 0;
  __syncthreads();
  const int64_t start = (int64_t)blockIdx.x * a.per + wave * (a.per / kSortWaves);
  const int64_t end = min(start + a.per / kSortWaves, (int64_t)a.R);
  int* const mine = next + wave * ld;
  for (int64_t r = start + lane; r < end; r += 64) atomicAdd(&mine[sort_key(a, r)], 1);
  __syncthreads();
  int carry = 0;
  for (int e0 = 0; e0 < a.E; e0 += kSortThreads) {
    const int e = e0 + t;
    int total = 0, before = 0;
    if (e < a.E) {
#pragma unroll 8
      for (int b = 0; b < a.blocks; ++b) {
        const int c = a.hist[(int64_t)b * a.E + e];
        total += c;
        before += b < (int)blockIdx.x ? c : 0;
      }
    }
    const int first = scan_experts(total, &carry, tot);
    if (e < a.E) {
      if (blockIdx.x == 0) a.offsets[e] = first;
      int at = first + before;
      for (int w = 0; w < kSortWaves; ++w) {
        const int c = next[w * ld + e];
        next[w * ld + e] = at;
        at += c;
      }
    }
  }
  if (blockIdx.x == 0 && t == 0) a.offsets[a.E] = carry;
  for (int64_t p = carry + (int64_t)blockIdx.x * kSortThreads + t; p < a.R; p += (int64_t)gridDim.x * kSortThreads) a.experts[p] = -1;
  __syncthreads();
  for (int64_t r0 = start; r0 < end; r0 += 64) {
    const int64_t r = r0 + lane;
    const int e = r < end ? sort_key(a, r) : a.E;
    uint64_t same = __ballot(r < end);
    for (int bit = 1; bit <= a.E; bit <<= 1) {
      const uint64_t set = __ballot(e & bit);
      same &= e & bit ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1)), at = mine[e];
    if (r < end) {
      a.places[r] = e < a.E ? at + rank : -1;
      if (e < a.E) a.experts[at + rank] = e;
    }
    __builtin_amdgcn_wave_barrier();
    if (r < end && rank == 0) mine[e] = at + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

template <int ES>
__global__ void __launch_bounds__(256) sort_rows_kernel(SortArgs a, RowGrid g) {
  const TokenPiece tp = token_piece(g);
  if (tp.token >= a.T || tp.piece >= g.pieces) return;
  const u32x4 v = Pieces<ES>::load((const char*)a.x + tp.token * a.ldx * ES, tp.piece, a.H);
  const int* const places = a.places + tp.token * a.topk;
  for (int j = 0; j < a.topk; ++j) {
    const int p = places[j];
    if (p >= 0) Pieces<ES>::store((char*)a.rows + (int64_t)p * a.H * ES, tp.piece, a.H, v);
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

template <typename T, bool WEIGHTED>
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
      if (place[j] >= 0) v[j] = Pieces<ES>::load((const char*)a.rows + (int64_t)place[j] * a.H * ES, tp.piece, a.H);
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

// A block has a token: its upstream row is read once and goes out k times, weighted, while it meets the experts' rows.
template <typename T, bool ROWS, bool WEIGHTS>
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
          if (place[j] >= 0) v[j] = Pieces<ES>::load((const char*)a.rows + (int64_t)place[j] * a.H * ES, p, a.H);
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
            Pieces<ES>::store((char*)a.grad_rows + (int64_t)place[j] * a.H * ES, p, a.H, packed<T>(f));
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

static int64_t sort_per(int64_t R) { return cdiv(cdiv(R, 256), kSortThreads) * kSortThreads; }

size_t moe_sort_workspace_bytes(int64_t T, int E, int topk) {
  const int64_t R = T * topk;
  return R <= kCountRoutes ? 0 : (size_t)cdiv(R, sort_per(R)) * E * 4;
}

// Threads and blocks of a launch over tokens and pieces of their rows.
struct RowLaunch {
  RowGrid g;
  dim3 grid, block;
};
static RowLaunch row_launch(int64_t T, int64_t H, int vec) {
  const int pieces = (int)cdiv(H, vec), ny = (int)cdiv(pieces, 256);
  if (pieces <= 128) {
    const int per = 256 / pieces;
    return {{pieces, per == 1 ? 2 : per}, dim3((unsigned)cdiv(T, per)), dim3(256)};
  }
  return {{pieces, 1}, dim3((unsigned)T, (unsigned)ny), dim3((unsigned)(cdiv(cdiv(pieces, ny), 64) * 64))};
}

int launch_moe_sort(const MoeSortCall& c, hipStream_t st) {
  SortArgs a{};
  a.x = c.x, a.ids = c.ids, a.ldx = c.ldx, a.rows = c.rows, a.offsets = c.offsets, a.experts = c.experts, a.places = c.places;
  a.T = c.T, a.H = (int)c.H, a.E = c.E, a.topk = c.topk, a.id64 = c.id64, a.R = (int)(c.T * c.topk);
  const int vec = 16 / c.elem_bytes;
  if (a.R <= kCountRoutes) {
    const dim3 grid((unsigned)(c.T + 1), (unsigned)std::max<int64_t>(1, cdiv(cdiv(c.H, vec), kSortThreads)));
    if (c.elem_bytes == 2) sort_few_kernel<2><<<grid, kSortThreads, 0, st>>>(a);
    else sort_few_kernel<4><<<grid, kSortThreads, 0, st>>>(a);
    return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
  }
  a.hist = (int*)c.workspace;
  a.per = sort_per(a.R);
  a.blocks = (int)cdiv(a.R, a.per);
  sort_count_kernel<<<(unsigned)a.blocks, kSortThreads, 0, st>>>(a);
  if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  sort_place_kernel<<<(unsigned)a.blocks, kSortThreads, (size_t)kSortWaves * (c.E + 1) * 4, st>>>(a);
  if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  if (c.H == 0) return AWQ_OK;
  const RowLaunch l = row_launch(c.T, c.H, vec);
  if (c.elem_bytes == 2) sort_rows_kernel<2><<<l.grid, l.block, 0, st>>>(a, l.g);
  else sort_rows_kernel<4><<<l.grid, l.block, 0, st>>>(a, l.g);
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
  if (a.weights) unsort_kernel<T, true><<<l.grid, l.block, 0, st>>>(a, l.g);
  else unsort_kernel<T, false><<<l.grid, l.block, 0, st>>>(a, l.g);
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
  if (a.grad_rows && a.grad_weights) unsort_grad_kernel<T, true, true><<<grid, 256, 0, st>>>(a);
  else if (a.grad_rows) unsort_grad_kernel<T, true, false><<<grid, 256, 0, st>>>(a);
  else unsort_grad_kernel<T, false, true><<<grid, 256, 0, st>>>(a);
}
int launch_moe_unsort_grad(const MoeUnsortCall& c, hipStream_t st) {
  const UnsortArgs a = unsort_args(c);
  if (c.dtype == AWQ_DTYPE_F16) unsort_grad_typed<f16>(a, st);
  else if (c.dtype == AWQ_DTYPE_BF16) unsort_grad_typed<bf16>(a, st);
  else unsort_grad_typed<float>(a, st);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

}  // namespace awq_host
