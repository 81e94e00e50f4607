// Mixture of experts over microscaled fp4 stacks: the places of the routes, the grouped products
// (awq_mx_gemm.hip) and the weighted sum.
#include <algorithm>

#include "awq_launch.h"
#include "awq_mx_common.h"

namespace awq {

constexpr int kOrderThreads = 1024, kOneBlockRoutes = 6144;

// The places of the routes, sorted by expert: order[place] = route, and the table of row tiles, at most `rows` places of
// one expert each.  The order inside an expert is that of atomics; no result depends on it, since every place's row is
// computed by itself and summed by its route.  Routes without an expert get no place.
//
// Up to kOneBlockRoutes routes block 0 does it alone.  More: its LDS atomics, on few addresses, would take longer than
// the rest (16384 routes to 64 experts: 19 us), so at most 256 blocks of kOrderThreads routes, or of several times as many,
// count and rank theirs, and a second
// launch adds up the counts (6 us for both; the whole call with one block and with several: 4096 routes 70 and 78 us, 5600
// 89 and 91, 8192 126 and 123).
struct MxOrder {
  const void* ids;
  int id64, R, E, rows;
  int *order, *tiles, *tile_count;
  int blocks;         // of routes; 1: block 0 does everything
  int64_t per;        // routes of a block, a multiple of kOrderThreads
  int *rank, *hist;   // rank[route] in its block and expert; hist[blocks][E]
};

// First place and first tile of every expert (thread e has expert e's) from its count, and its rows of the table if
// `write`.
__device__ __forceinline__ int mx_first_place(const MxOrder& o, int c, bool write) {
  __shared__ int tot[2][kOrderThreads / 64];
  const int t = threadIdx.x, wave = t >> 6, nt = (c + o.rows - 1) / o.rows;
  const int ic = wave_incl_scan_i32(c), it = wave_incl_scan_i32(nt);
  if ((t & 63) == 63) tot[0][wave] = ic, tot[1][wave] = it;
  __syncthreads();
  int first = ic - c, ft = it - nt;
  for (int w = 0; w < wave; ++w) first += tot[0][w], ft += tot[1][w];
  if (write) {
    for (int i = 0; i < nt; ++i) {
      int* row = o.tiles + 3 * (ft + i);
      row[0] = t;
      row[1] = first + i * o.rows;
      row[2] = min(o.rows, c - i * o.rows);
    }
    if (t == kOrderThreads - 1) o.tile_count[0] = ft + nt;
  }
  return first;
}

// Blocks of routes first, then blocks that quantise the tokens.
template <typename T>
__global__ void __launch_bounds__(kOrderThreads) mx_prepare_kernel(MxOrder o, const uint16_t* __restrict__ x, int64_t ldx, int64_t pieces,
                                                                   int per_row, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                   int lds) {
  __shared__ int count[kOrderThreads];
  const int t = threadIdx.x;
  if ((int)blockIdx.x >= o.blocks) {
    const int64_t i = (int64_t)((int)blockIdx.x - o.blocks) * kOrderThreads + t;
    if (i >= pieces) return;  // whole blocks of 32: pieces % 4 == 0
    const int64_t row = i / per_row;
    const int piece = (int)(i - row * per_row);
    mx_quantize8<T>(x + row * ldx, codes + row * per_row * 4, scales + row * lds, piece);
    return;
  }
  count[t] = 0;
  __syncthreads();
  if (o.blocks > 1) {
    const int64_t start = (int64_t)blockIdx.x * o.per, end = min(start + o.per, (int64_t)o.R);
    for (int64_t r = start + t; r < end; r += kOrderThreads) {
      const int64_t e = mx_route_id(o.ids, o.id64, r);
      if (e >= 0 && e < o.E) o.rank[r] = atomicAdd(&count[e], 1);
    }
    __syncthreads();
    if (t < o.E) o.hist[(int64_t)blockIdx.x * o.E + t] = count[t];
    return;
  }
  constexpr int MOST = kOneBlockRoutes / kOrderThreads;
  int64_t e[MOST];
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const int r = t + j * kOrderThreads;
    e[j] = r < o.R ? mx_route_id(o.ids, o.id64, r) : -1;
    if (e[j] >= o.E) e[j] = -1;
  }
#pragma unroll
  for (int j = 0; j < MOST; ++j)
    if (e[j] >= 0) atomicAdd(&count[e[j]], 1);
  __syncthreads();
  // E <= kOrderThreads: one expert per thread
  const int first = mx_first_place(o, count[t], true);
  count[t] = first;  // from here on the expert's next place
  __syncthreads();
#pragma unroll
  for (int j = 0; j < MOST; ++j)
    if (e[j] >= 0) o.order[atomicAdd(&count[e[j]], 1)] = t + j * kOrderThreads;
}

// The second launch of many routes: block b places the routes of block b.
__global__ void __launch_bounds__(kOrderThreads) mx_place_kernel(MxOrder o) {
  __shared__ int base[kOrderThreads];
  const int t = threadIdx.x;
  int total = 0, before = 0;
  if (t < o.E) {
#pragma unroll 8
    for (int b = 0; b < o.blocks; ++b) {
      const int c = o.hist[(int64_t)b * o.E + t];
      total += c;
      before += b < (int)blockIdx.x ? c : 0;
    }
  }
  base[t] = mx_first_place(o, total, blockIdx.x == 0) + before;
  __syncthreads();
  const int64_t start = (int64_t)blockIdx.x * o.per, end = min(start + o.per, (int64_t)o.R);
  for (int64_t r = start + t; r < end; r += kOrderThreads) {
    const int64_t e = mx_route_id(o.ids, o.id64, r);
    if (e >= 0 && e < o.E) o.order[base[e] + o.rank[r]] = (int)r;
  }
}

// out[t] = the sum over a token's slots, in slot order, of weight * y: fp32, one rounding.  A slot
// without an expert adds nothing (its row of y was never written).  Bound by the read of y (2048 tokens, top 8, H = 2048:
// 134 MB in 26 us, 5.4 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) mx_combine_kernel(const float* __restrict__ y, const void* __restrict__ ids, int id64,
                                                         const void* __restrict__ w, int w_dtype, int E, int64_t T_, int H, int topk,
                                                         uint16_t* __restrict__ out, int64_t ldo) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = i / (H / 4);
  if (t >= T_) return;
  const int c = (int)(i - t * (H / 4)) * 4;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  constexpr int AT_ONCE = 8;  // slots under way
  for (int j = 0; j < topk; j += AT_ONCE) {
    bool has[AT_ONCE];
    float g[AT_ONCE];
    f32x4 v[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const int64_t r = t * topk + j + k, e = j + k < topk ? mx_route_id(ids, id64, r) : -1;
      has[k] = e >= 0 && e < E;
      if (has[k]) g[k] = mx_route_weight(w, w_dtype, r);
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k)
      if (has[k]) v[k] = *(const f32x4*)(y + (t * topk + j + k) * H + c);
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k)
      if (has[k])
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] = fmaf(v[k][u], g[k], s[u]);
  }
  u32x2 o = {pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3])};
  uint16_t* at = out + t * ldo + c;
  if (((uintptr_t)at & 7) == 0) {
    *(u32x2*)at = o;
  } else {
#pragma unroll
    for (int u = 0; u < 4; ++u) at[u] = (uint16_t)(o[u >> 1] >> (16 * (u & 1)));
  }
}

}  // namespace awq

namespace awq_host {
using namespace awq;

// Rows of a row tile by what an expert gets on average, so that its weights are read about once.  64 experts, H = 2048,
// I = 1024, us: 2 routes an expert 42.9 with 16 rows, 42.7 with 64, 3 46.7 and 44.2, 4 47.8 and 45.2 (128 experts, H = 4096,
// I = 1536: 1 156 and 162); 32 52.8 with 64 rows, 54.2 with 128, 37 54.6 and 55.4, 44 60.8 and 57.8, 62 74 and 63 (32 experts,
// H = 4096, I = 1536: 32 88.6 and 89.0, 45 92.8 and 91.5, 62 124 and 102).
static int mx_moe_rows(int64_t R, int E) { return R <= (int64_t)2 * E ? 16 : (R <= (int64_t)40 * E ? 64 : 128); }

// Bytes between rows of the tokens' scales: whole words, which the gathering kernel counts on.
static int64_t scale_stride(int64_t K) { return cdiv(K / 32, 4) * 4; }

MxMoeWorkspace mx_moe_workspace(int64_t T, int64_t H, int64_t I, int E, int topk) {
  MxMoeWorkspace w{};
  const int64_t R = T * topk;
  auto al = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  w.max_tiles = R / mx_moe_rows(R, E) + std::min<int64_t>(R, E);
  w.order = 256;  // the tile count sits in front
  w.tiles = al(w.order + R * 4);
  w.order_per = cdiv(R, (int64_t)256 * kOrderThreads) * kOrderThreads;
  w.order_blocks = R <= kOneBlockRoutes ? 1 : cdiv(R, w.order_per);
  w.rank = al(w.tiles + w.max_tiles * 12);
  w.hist = al(w.rank + (w.order_blocks > 1 ? R * 4 : 0));
  w.x = al(w.hist + (w.order_blocks > 1 ? w.order_blocks * E * 4 : 0));
  w.xs = al(w.x + T * (H / 2));
  w.h = al(w.xs + T * scale_stride(H));
  w.hs = al(w.h + R * (I / 2));
  w.y = al(w.hs + R * (I / 32));
  w.total = al(w.y + R * H * 4);
  return w;
}

// Few routes take two launches, which find their experts in the ids, instead of four with a table: 5 to 7 us less, against
// slower streams (every block quantises its tokens, a wave of down has an expert to itself).  So it is for few routes an
// expert and, if each route had an expert of its own, up to 320 MiB of weights.  us with two launches and with four, R routes to
// E experts, H, I: R = 8, E = 64, 2048, 1024 11.3, 17.6; 32 23.0, 30.1; 64 32.3, 34.4; R = 16, E = 16, 2048, 5632 36.6, 43.0, 32
// 59.1, 57.4; R = 16, E = 32, 2880, 2880 37.9, 40.7, 32 64.5, 59.5; R = 32, E = 32, 4096, 1536 54.4, 56.3, 64 70.4, 68.8;
// R = 32, E = 256, 7168, 2048 149, 141; R = 16, E = 8, 4096, 1536 28.6, 29.8, 24 31.5, 29.8.
static bool mx_scans(int64_t R, int64_t H, int64_t I, int E) {
  return R <= kMxScanRoutes && R <= 2 * (int64_t)E && R * (3 * H * I / 32 * 17) <= (int64_t)320 << 20;
}

int launch_mx_moe(const MxMoeCall& c, hipStream_t st) {
  const int64_t R = c.T * c.topk;
  if (R > 0x7FFFFFFFLL) return AWQ_ERR_UNSUPPORTED;
  const MxMoeWorkspace w = mx_moe_workspace(c.T, c.H, c.I, c.E, c.topk);
  char* ws = (char*)c.workspace;
  if (mx_scans(R, c.H, c.I, c.E)) {
    // two launches: gate_up, which finds its routes and quantises its tokens itself, and down with the weighted sum
    MxArgs g{};
    if (c.H <= 4096) {
      g.x = (const uint16_t*)c.x, g.ldx = c.ldx, g.xrows = 16;
    } else {
      const int rc = launch_mx_quantize(c.x, c.ldx, (uint8_t*)(ws + w.x), (uint8_t*)(ws + w.xs), c.H / 32, c.T, c.H, c.act_dtype, st);
      if (rc != AWQ_OK) return rc;
      g.a = (const uint8_t*)(ws + w.x), g.as = (const uint8_t*)(ws + w.xs);
    }
    g.w = c.gate_up, g.ws = c.gate_up_scales;
    g.K = (int)c.H, g.N = (int)c.I, g.wrows = 2 * c.I, g.a_rows = c.T, g.as_ld = (int)(c.H / 32);
    g.ids = c.ids, g.id64 = c.id64, g.routes = (int)R, g.experts = c.E, g.topk = c.topk;
    g.act = c.act_kind, g.out_bf16 = c.act_dtype == AWQ_DTYPE_BF16;
    g.h = (uint8_t*)(ws + w.h), g.hs = (uint8_t*)(ws + w.hs);
    const int rc = launch_mx_scan_gate_up(g, st);
    if (rc != AWQ_OK) return rc;
    MxArgs d = g;
    d.x = nullptr, d.a = g.h, d.as = g.hs;
    d.w = c.down, d.ws = c.down_scales;
    d.K = (int)c.I, d.N = (int)c.H, d.wrows = c.H, d.a_rows = R, d.as_ld = (int)(c.I / 32);
    return launch_mx_down_combine(d, c.weights, c.weights_dtype, c.out, c.ldo, st);
  }
  int* order = (int*)(ws + w.order);
  int* tiles = (int*)(ws + w.tiles);
  const int rows = mx_moe_rows(R, c.E);
  const int64_t pieces = c.T * (c.H / 8);
  if (cdiv(pieces, kOrderThreads) + w.order_blocks > 0x7FFFFFFFLL) return AWQ_ERR_UNSUPPORTED;
  MxOrder o{c.ids, c.id64, (int)R, c.E, rows, order, tiles, (int*)ws, (int)w.order_blocks, w.order_per, (int*)(ws + w.rank), (int*)(ws + w.hist)};
  auto prepare = [&](auto kernel) {
    kernel<<<dim3((unsigned)(w.order_blocks + cdiv(pieces, kOrderThreads))), dim3(kOrderThreads), 0, st>>>(
        o, (const uint16_t*)c.x, c.T > 1 ? c.ldx : c.H, pieces, (int)(c.H / 8), (uint8_t*)(ws + w.x), (uint8_t*)(ws + w.xs),
        (int)scale_stride(c.H));
  };
  c.act_dtype == AWQ_DTYPE_BF16 ? prepare(mx_prepare_kernel<bf16>) : prepare(mx_prepare_kernel<f16>);
  if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  if (w.order_blocks > 1) {
    mx_place_kernel<<<dim3((unsigned)w.order_blocks), dim3(kOrderThreads), 0, st>>>(o);
    if (hipGetLastError() != hipSuccess) return AWQ_ERR_LAUNCH;
  }

  MxArgs g{};
  g.a = (const uint8_t*)(ws + w.x), g.as = (const uint8_t*)(ws + w.xs);
  g.w = c.gate_up, g.ws = c.gate_up_scales;
  g.K = (int)c.H, g.N = (int)c.I, g.wrows = 2 * c.I, g.a_rows = c.T, g.as_ld = (int)scale_stride(c.H);
  g.tiles = tiles, g.tile_count = (const int*)ws, g.order = order;
  g.topk = c.topk, g.act = c.act_kind;
  g.h = (uint8_t*)(ws + w.h), g.hs = (uint8_t*)(ws + w.hs);
  int rc = launch_mx_grouped(g, true, rows, w.max_tiles, st);
  if (rc != AWQ_OK) return rc;

  MxArgs d = g;
  d.a = g.h, d.as = g.hs;
  d.w = c.down, d.ws = c.down_scales;
  d.K = (int)c.I, d.N = (int)c.H, d.wrows = c.H, d.a_rows = R, d.as_ld = (int)(c.I / 32);
  d.y = (float*)(ws + w.y);
  rc = launch_mx_grouped(d, false, rows, w.max_tiles, st);
  if (rc != AWQ_OK) return rc;

  const dim3 grid((unsigned)cdiv(c.T * (c.H / 4), 256));
  if (c.act_dtype == AWQ_DTYPE_BF16)
    mx_combine_kernel<bf16><<<grid, 256, 0, st>>>(d.y, c.ids, c.id64, c.weights, c.weights_dtype, c.E, c.T, (int)c.H, c.topk,
                                                 (uint16_t*)c.out, c.ldo);
  else
    mx_combine_kernel<f16><<<grid, 256, 0, st>>>(d.y, c.ids, c.id64, c.weights, c.weights_dtype, c.E, c.T, (int)c.H, c.topk,
                                                (uint16_t*)c.out, c.ldo);
  return hipGetLastError() == hipSuccess ? AWQ_OK : AWQ_ERR_LAUNCH;
}

}  // namespace awq_host
