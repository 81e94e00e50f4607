// Products of microscaled fp4 matrices with few rows: operands straight from memory to registers (format,
// modes and operand order: awq_mx_common.h).
//
// What bounds them is the read of the weights, once: a block has 16 columns (gate_up: 32 gate rows and the 32 up
// rows of the same outputs), its waves share K, each asks for all that it will use before the first product, and
// the waves' sums meet in LDS, in wave order.
#include "awq_launch.h"
#include "awq_mx_common.h"

namespace awq {

// The fragments of a pair of steps (256 along K, one line of a row): a load of a wave takes half a line of each of
// its 16 rows.  (Quarters of the wave with 32 neighbouring bytes each, whose scales are neighbours too: 12.6 us for
// the reads of K = 4096, N = 24576 where these take 10.1; non-temporal loads 11.2, as weights in use stay in the MALL.)
struct MxPair {
  u32x4 c[2];
  uint32_t s[2];
};
// A whole pair; its scales still as they lie in memory, all of a half's four in every lane: nothing here waits for a
// load.
__device__ __forceinline__ MxPair mx_load_pair(const uint8_t* codes, const uint8_t* scales, int pair, int q) {
  MxPair f;
  const u32x4* at = (const u32x4*)(codes + (int64_t)pair * 128) + q;
  f.c[0] = at[0];
  f.c[1] = at[4];
  __builtin_memcpy(f.s, scales + 8 * pair, 8);
  return f;
}
// The pair that K ends in, in the same form: behind the end codes 0 and the scale 2^-127.
__device__ __forceinline__ MxPair mx_load_last(const uint8_t* codes, const uint8_t* scales, int pair, int q, int KB) {
  MxPair f{{u32x4{0u, 0u, 0u, 0u}, u32x4{0u, 0u, 0u, 0u}}, {0u, 0u}};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int block = 8 * pair + 4 * h + q;
    if (block < KB) {
      f.c[h] = *(const u32x4*)(codes + (int64_t)block * 16);
      f.s[h] = (uint32_t)scales[block] << (8 * q);
    }
  }
  return f;
}
// c += a . b^T over the pair
__device__ __forceinline__ f32x4 mx_mfma_pair(const MxPair& a, const MxPair& b, f32x4 c, int q) {
  c = mx_mfma(a.c[0], b.c[0], c, a.s[0] >> (8 * q), b.s[0] >> (8 * q));
  return mx_mfma(a.c[1], b.c[1], c, a.s[1] >> (8 * q), b.s[1] >> (8 * q));
}

// The at most kMxScanRoutes routes in a wave's lanes: a lane holds the expert of the route with its number, or -1.
__device__ __forceinline__ int mx_scan_ids(const MxArgs& p, int lane) {
  const int64_t e = lane < p.routes ? mx_route_id(p.ids, p.id64, lane) : -1;
  return e >= 0 && e < p.experts ? (int)e : -1;
}
// The routes that share a route's expert, as a mask; first: the lowest of them, -1 if the route has no expert.
struct MxScan {
  uint64_t its;
  int expert, first;
};
__device__ __forceinline__ MxScan mx_scan(int mine, int route) {
  const int e = __builtin_amdgcn_readlane(mine, route);
  const uint64_t its = __ballot(mine == e);
  return {its, e, e < 0 ? -1 : __ffsll((unsigned long long)its) - 1};
}
__device__ __forceinline__ void mx_scan_list(const MxScan& f, int lane, int* list) {
  if (f.its >> lane & 1) list[__popcll(f.its & ((1ull << lane) - 1))] = lane;
}
static_assert(kMxScanRoutes <= 64, "a lane each");

// Grid x: column blocks, y: row tiles of 16 (with SCAN: routes).
// X16: a is 16-bit and quantised by every block for itself, into LDS, while its weights are on their way: one
// launch less where the rows are few and short.
// SCAN (gate_up): no table of tiles; block y takes up to 16 routes of route y's expert from y on, which it finds in
// the ids itself, if 16, 32, .. or none of the expert's lie in front of y.  A route's place is its own number.
template <int MODE, int NT, int WAVES, bool X16, bool SCAN>
__global__ void __launch_bounds__(WAVES * 64) mx_rows_kernel(MxArgs p) {
  constexpr int THREADS = WAVES * 64;
  __shared__ float red[WAVES][NT][256];
  __shared__ int list[SCAN ? kMxScanRoutes : 1];
  extern __shared__ __align__(16) uint8_t xq[];  // X16: codes [xrows][K/2 + 16], scales [xrows][K/32]
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, q = lane >> 4;
  MxRows t;
  if constexpr (SCAN) {
    // every wave looks for itself, so that its weights are asked for at once
    MxScan f = mx_scan(mx_scan_ids(p, lane), blockIdx.y);
    const uint64_t before = (1ull << blockIdx.y) - 1;
    if (f.first < 0 || (__popcll(f.its & before) & 15) != 0) return;
    f.its &= ~before;
    if (wave == 0) mx_scan_list(f, lane, list);
    t = {f.expert, 0, min((int)__popcll(f.its), 16)};
  } else {
    if (MODE != kMxDense && (int)blockIdx.y >= p.tile_count[0]) return;
    t = mx_rows<MODE, 16>(p, blockIdx.y);
  }
  constexpr int COLS = MODE == kMxGateUp ? 8 * NT : 16 * NT;
  const int n0 = (int)blockIdx.x * COLS, KB = p.K / 32, pairs = KB / 8;  // whole ones

  const uint8_t *wc[NT], *wsc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    int64_t row;
    if constexpr (MODE == kMxGateUp) row = (j < NT / 2 ? n0 + 16 * j : p.N + n0 + 16 * (j - NT / 2)) + r;
    else row = min(n0 + 16 * j + r, p.N - 1);
    row += (int64_t)t.expert * p.wrows;
    wc[j] = p.w + row * (p.K / 2);
    wsc[j] = p.ws + row * KB;
  }
  const int ld = p.K / 2 + 16;
  const uint8_t *ac, *asc;
  if constexpr (SCAN && !X16) __syncthreads();  // the list
  if constexpr (!X16) {
    const int64_t row = SCAN ? list[min(r, t.rows - 1)] / p.topk : mx_a_row<MODE>(p, t, r);
    ac = p.a + row * (p.K / 2);
    asc = p.as + row * p.as_ld;
  }
  f32x4 acc[NT];
  MxPair b[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (wave < pairs) {
#pragma unroll
    for (int j = 0; j < NT; ++j) b[j] = mx_load_pair(wc[j], wsc[j], wave, q);
  }
  if constexpr (X16) {
    if constexpr (SCAN) __syncthreads();  // the list
    const int pieces = p.K / 8;
    for (int m = 0; m < t.rows; ++m) {
      const int64_t row = SCAN ? list[m] / p.topk : t.first + m;
      const uint16_t* x = p.x + row * p.ldx;
      uint8_t *codes = xq + m * ld, *scales = xq + p.xrows * ld + m * KB;
      for (int i = tid; i < pieces; i += THREADS) {
        if (p.out_bf16) mx_quantize8<bf16>(x, codes, scales, i);
        else mx_quantize8<f16>(x, codes, scales, i);
      }
    }
    __syncthreads();
    const int m = min(r, t.rows - 1);
    ac = xq + m * ld;
    asc = xq + p.xrows * ld + m * KB;
  }
  // a pair at a time: two or four under way in a wave measured the same, other waves fill in (unrolled: 3 tokens through
  // 64 experts, H = 7168, I = 2048 127 us against 115, H = 2048, I = 1024 22.7 against 23.2)
#pragma unroll 1
  for (int pair = wave; pair < pairs; pair += WAVES) {
    if (pair != wave) {
#pragma unroll
      for (int j = 0; j < NT; ++j) b[j] = mx_load_pair(wc[j], wsc[j], pair, q);
    }
    const MxPair a = mx_load_pair(ac, asc, pair, q);
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = mx_mfma_pair(a, b[j], acc[j], q);
  }
  if ((KB & 7) != 0 && wave == pairs % WAVES) {
    const MxPair a = mx_load_last(ac, asc, pairs, q, KB);
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = mx_mfma_pair(a, mx_load_last(wc[j], wsc[j], pairs, q, KB), acc[j], q);
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int u = 0; u < 4; ++u) red[wave][j][(4 * q + u) * 16 + r] = acc[j][u];
  __syncthreads();

  auto sum = [&](int j, int at) {
    float v = red[0][j][at];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += red[w][j][at];
    return v;
  };
  if constexpr (MODE == kMxGateUp) {
    // 32 lanes hold a row's 32 columns: their largest magnitude, then the codes, two to a byte
    static_assert(NT == 4, "32 gate and 32 up rows");
    const int n = tid & 31;
    for (int m = tid >> 5; m < t.rows; m += THREADS / 32) {
      const int at = m * 16 + (n & 15);
      const float v = mx_gated(sum(n >> 4, at), sum((n >> 4) + 2, at), p.act);
      uint32_t top = mx_abs_bits(v);
#pragma unroll
      for (int d = 1; d < 32; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
      const uint32_t byte = mx_scale_byte(top);
      const float other = __shfl_xor(v, 1);
      const int64_t place = SCAN ? list[m] : t.first + m;
      if ((n & 1) == 0) {
        const uint32_t code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, v, other, mx_scale_value(byte == 255u ? 0u : byte), 0);
        p.h[place * (p.N / 2) + (n0 + n) / 2] = byte == 255u ? (uint8_t)0 : (uint8_t)code;
      }
      if (n == 0) p.hs[place * (p.N / 32) + n0 / 32] = (uint8_t)byte;
    }
  } else {
    for (int i = tid; i < NT * 256; i += THREADS) {
      const int j = i >> 8, at = i & 255, m = at >> 4, n = n0 + j * 16 + (at & 15);
      if (m >= t.rows || n >= p.N) continue;
      float v = sum(j, at);
      if constexpr (MODE == kMxDense) {
        v += load_bias(p.bias, p.bias_dtype, n);
        p.c[(int64_t)(t.first + m) * p.ldc + n] = p.out_bf16 ? f2bf_bits(v) : f2h_bits(v);
      } else {
        p.y[(int64_t)p.order[t.first + m] * p.N + n] = v;
      }
    }
  }
}

// The down product of at most kMxScanRoutes routes with the weighted sum over each token's slots, in one launch: a
// block has COLS columns of all experts, its waves an expert at a time, and the routes' sums meet in LDS.  A route's
// place is its own number.
// COLS = 8: rows 8 .. 15 of both operands of an MFMA are rows 0 .. 7 again, half of K on, so that a wave still loads 16 half
// lines at once; two of the four quadrants of the product count, and are added up.
constexpr int kDownWaves = 16;

template <typename T, int COLS>
__global__ void __launch_bounds__(kDownWaves * 64) mx_down_combine_kernel(MxArgs p, const void* weights, int w_dtype,
                                                                          uint16_t* out, int64_t ldo) {
  constexpr int THREADS = kDownWaves * 64, U = 2 /* pairs under way; four do not fit the registers */, PARTS = 16 / COLS;
  __shared__ float y[kMxScanRoutes][COLS];
  __shared__ int slot[kDownWaves][kMxScanRoutes], has[kMxScanRoutes];
  __shared__ float weight[kMxScanRoutes];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane % COLS, q = lane >> 4;
  if (tid < p.routes) {
    const int64_t e = mx_route_id(p.ids, p.id64, tid);
    has[tid] = e >= 0 && e < p.experts;
    weight[tid] = mx_route_weight(weights, w_dtype, tid);
  }
  // a lane's part of K: pairs `from` .. `from` + share - 1; what is left behind the parts is part 0's
  const int n0 = (int)blockIdx.x * COLS, KB = p.K / 32, share = KB / 8 / PARTS, part = (lane & 15) / COLS, from = part * share;
  const int expert = mx_scan_ids(p, lane);
  for (int k = wave; k < p.routes; k += kDownWaves) {
    const MxScan f = mx_scan(expert, k);
    if (f.first != k) continue;  // another wave's, or nobody's
    mx_scan_list(f, lane, slot[wave]);
    __builtin_amdgcn_wave_barrier();
    const int64_t row = (int64_t)f.expert * p.wrows + min(n0 + r, p.N - 1);
    const uint8_t *wc = p.w + row * (p.K / 2) + from * 128, *wsc = p.ws + row * KB + from * 8;
    const int n = (int)__popcll(f.its);
    for (int at = 0; at < n; at += COLS) {
      const int mine = slot[wave][min(at + r, n - 1)];
      const uint8_t *ac = p.a + (int64_t)mine * (p.K / 2) + from * 128, *asc = p.as + (int64_t)mine * p.as_ld + from * 8;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      // the operands swapped: a lane holds four columns of the route in lane r
      for (int first = 0; first < share; first += U) {
        MxPair a[U], b[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (first + u < share) b[u] = mx_load_pair(wc, wsc, first + u, q);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (first + u < share) a[u] = mx_load_pair(ac, asc, first + u, q);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (first + u < share) acc = mx_mfma_pair(b[u], a[u], acc, q);
      }
      for (int pair = PARTS * share; 8 * pair < KB; ++pair) {
        const int end = part == 0 ? KB : 0;
        acc = mx_mfma_pair(mx_load_last(wc, wsc, pair, q, end), mx_load_last(ac, asc, pair, q, end), acc, q);
      }
      if constexpr (PARTS == 2) {
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[u] += __shfl(acc[u], (lane + 40) & 63);
      }
      if (lane < COLS * 4 && part == 0 && at + r < n) *(f32x4*)&y[mine][4 * q] = acc;
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  const int tokens = p.routes / p.topk;
  for (int i = tid; i < tokens * COLS; i += THREADS) {
    const int t = i / COLS, n = i % COLS;
    if (n0 + n >= p.N) continue;
    float s = 0.f;
    for (int j = 0; j < p.topk; ++j) {
      const int route = t * p.topk + j;
      if (has[route]) s = fmaf(y[route][n], weight[route], s);
    }
    out[(int64_t)t * ldo + n0 + n] = to_bits<T>(s);
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

template <int MODE, int NT, int WAVES, bool X16, bool SCAN>
static int launch_rows(const MxArgs& p, int64_t row_tiles, hipStream_t st) {
  constexpr int COLS = MODE == kMxGateUp ? 8 * NT : 16 * NT;
  auto kernel = mx_rows_kernel<MODE, NT, WAVES, X16, SCAN>;
  const size_t lds = X16 ? (size_t)p.xrows * (p.K / 2 + 16 + p.K / 32) : 0;
  kernel<<<dim3((unsigned)cdiv(p.N, COLS), (unsigned)row_tiles), dim3(WAVES * 64), lds, st>>>(p);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

// Up to 16 rows, and more, in row tiles that each read the weights, while these give a block per CU at most, or two for
// short K (us with these kernels and with tiles: M = 20, N = 512, K = 2048 3.3, 5.2; M = 32, N = 2048, K = 4096 5.0, 7.1;
// M = 64, N = 1024, K = 4096 4.9, 7.2; two: M = 64, N = 2048, K = 2048 4.5, 5.4, K = 4096 7.5, 7.2; M = 32, N = 4096, K = 2048
// 4.5, 5.3, K = 4096 7.6, 7.2; more: M = 64, N = 4096, K = 2048 7.0, 5.4).
bool mx_takes_rows(int64_t M, int64_t N, int64_t K) { return M <= 16 || cdiv(M, 16) * cdiv(N, 16) <= (K <= 2048 ? 512 : 256); }

// Up to here every block quantises a's rows for itself (M = 8, K = 4096, N = 24576: 17.2 us against 13.4 and 1.6 for a
// launch of its own; M = 2 12.4 against 12.0 and 1.6).
bool mx_quantizes_itself(int64_t M, int64_t K) { return M <= 16 && M * K <= 16384; }

// 16 columns a block where that gives a block per CU at most, else 32 (K = 4096, us, 16 and 32 columns: N = 4096, M = 1
// 4.0, 5.2, M = 16 4.8, 6.4; N = 6144 5.7, 5.3 and 7.9, 6.5; N = 24576 12.0, 11.9 and 18.4, 14.9); 16 waves where a CU has
// one block (K = 12288, N = 4096: 4 waves 10.1, 8 8.1, 16 7.7).
template <bool X16>
static int launch_rows_dense(const MxArgs& p, hipStream_t st) {
  const int64_t tiles = cdiv(p.M, 16);
  if (p.N <= 16 * 256) return launch_rows<kMxDense, 1, 16, X16, false>(p, tiles, st);
  if (p.N <= 32 * 256) return launch_rows<kMxDense, 2, 16, X16, false>(p, tiles, st);
  return launch_rows<kMxDense, 2, 8, X16, false>(p, tiles, st);
}
int launch_mx_rows_gemm(const MxArgs& p, hipStream_t st) {
  return p.x ? launch_rows_dense<true>(p, st) : launch_rows_dense<false>(p, st);
}

int launch_mx_grouped(const MxArgs& p, bool gate_up, int rows, int64_t row_tiles, hipStream_t st) {
  if (rows > 16) return launch_mx_tile_grouped(p, gate_up, rows, row_tiles, st);
  if (gate_up) return launch_rows<kMxGateUp, 4, 4, false, false>(p, row_tiles, st);
  return launch_rows<kMxDown, 2, 4, false, false>(p, row_tiles, st);
}

int launch_mx_scan_gate_up(const MxArgs& p, hipStream_t st) {
  if (p.x) return launch_rows<kMxGateUp, 4, 4, true, true>(p, p.routes, st);
  return launch_rows<kMxGateUp, 4, 4, false, true>(p, p.routes, st);
}

int launch_mx_down_combine(const MxArgs& p, const void* weights, int w_dtype, void* out, int64_t ldo, hipStream_t st) {
  auto go = [&](auto kernel, int cols) {
    kernel<<<dim3((unsigned)cdiv(p.N, cols)), dim3(kDownWaves * 64), 0, st>>>(p, weights, w_dtype, (uint16_t*)out, ldo);
  };
  // 8 columns where that gives a block per CU at most (N = 2048: the whole call 23.1 us against 26.9 for 4 tokens through 64
  // experts, I = 1024; N = 2880 41.0 against 38.1)
  const bool narrow = p.N <= 8 * 256;
  if (p.out_bf16) narrow ? go(mx_down_combine_kernel<bf16, 8>, 8) : go(mx_down_combine_kernel<bf16, 16>, 16);
  else narrow ? go(mx_down_combine_kernel<f16, 8>, 8) : go(mx_down_combine_kernel<f16, 16>, 16);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

}  // namespace awq_host
