// Group norm + activation (+ stochastic depth, + skip), NHWC, gfx950.
//
//   mean, var over the hw * (c / groups) values of a group of one image
//   h = (x - mean) * rsqrt(var + eps);  z = h * weight + bias
//   y = act(z) * drop[image] + residual
//
// and with g = dy * drop * act'(z), A = sum_group weight g,
// B = sum_group weight g h, m = hw * c / groups:
//
//   dbias = sum g;  dweight = sum g h;  dx = rstd (weight g - (A + h B) / m)
//
// What a block can hold of an image is normed by one block in one launch
// (group_norm_slab.hip); this file streams the rest: statistics, then their
// use.
//
// An image is a row-major [hw, c] matrix. A thread owns VEC neighbouring
// channels, keeps their coefficients in registers and streams rows; a block
// takes cpb such channel slots times 256 / cpb rows at a time (DfdPlan). All
// statistics are held in fp32; sums over a long axis are made by thread,
// block and chunk, joined in a fixed order, without atomics, so a result is
// the same every time.

#include "group_norm_device.h"

namespace {

constexpr int kBlock = 256, kGroupBlock = 1024;  // most threads of gn_bwd_group
constexpr int kTileRows = 4;  // rows of a tile that one thread takes

struct GnPlan {
  // Where 16 bytes do not divide the channels, `fold` rows are taken as one of
  // c = fold * channels: a whole number of vectors. Channel i of such a row is
  // channel i % channels of the image. Without it 23x274x152x151 bf16 (vectors
  // of 4 bytes) takes 702 us forward and backward, and so 513.
  int vec, fold, c;
  long long hw;
  int cpb, ctiles, chunks;
  int span;  // groups that a tile of channels can reach into
};

GnPlan gn_plan(const GnArgs& a) {
  GnPlan g = {};
  for (g.vec = 16 / gn_elem(a.type); g.vec > 1; g.vec /= 2) {
    g.fold = g.vec / gcd_of(a.c, g.vec);
    if (a.hw % g.fold == 0 && gn_aligned(a, g.vec)) break;
  }
  if (g.vec == 1) g.fold = 1;
  g.c = a.c * g.fold;
  g.hw = a.hw / g.fold;
  // A thread takes 16 rows at least, for a block's sums have a price: 32x336
  // x38x38 bf16 takes 32 us forward and 48 backward with 16, 37 and 53 with 4.
  // Where that leaves CUs without work it takes fewer: 1x480x75x75 fp16 26 and
  // 27 with 4, 21 and 34 with 16.
  DfdPlan p = {};
  for (int rows = 16; rows >= 4; rows /= 2) {
    p = dfd_plan(g.c / g.vec, g.hw, a.n, rows);
    if (a.n * p.chunks * p.ctiles >= 256) break;
  }
  const long long tile = kTileRows * (kBlock / p.cpb);
  const long long tiles = (g.hw + tile - 1) / tile;
  long long chunks = p.chunks;
  if (chunks < g.hw >> 20) chunks = g.hw >> 20;  // a block's rows are in div_small's range
  if (chunks > tiles) chunks = tiles;
  const int cpg = a.c / a.groups;
  g.cpb = p.cpb;
  g.ctiles = p.ctiles;
  g.chunks = (int)chunks;
  g.span = (p.cpb * g.vec + cpg - 2) / cpg + 1;
  return g;
}

// Which rows and channels a thread of the streaming kernels takes. Blocks run
// over channel tiles first, then chunks of rows, then images; the kernels that
// use the statistics run from the last to the first (forward and backward of
// 26x256x300x300 bf16 take 1582 us so and 1590 from the first; 26x480x75x75 238
// and 236: next to nothing of what was read last is still cached).
//
// What matters for the memory is that the blocks which run together read
// neighbouring rows, and that loads and stores pass by the caches: 2000 blocks
// each at a place of its own copy 1.2 GB in 489 us, the same blocks taking
// turns in 459, 73000 short ones in 417, and these past the caches in 384. So
// the kernels that sum take every chunks-th tile of rows, and those that do not
// are short. 26x256x300x300 bf16 (1.2 GB a tensor), us, before and so: stats
// 228 and 182, apply 519 and 400, backward sums 444 and 386, dx 728 and 608: 6
// TB/s, as that copy. All eight reads and writes are then at the memory's rate,
// and what the caches could save of them is little (the reads of both passes
// at 32 images' distance or at one: the same time).
//
// Past the caches is right for tensors larger than they are, and the kernels
// have this form alone. With plain loads and stores 26x256x300x300 takes 1738 us
// for 1582 and 64x144x150x150 (415 MB) 625 for 584, but 26x480x75x75 (140 MB) 234
// for 238, 16x144x150x150 (104 MB) 170 for 180, and forward 32x336x38x38 28.9 for
// 31.1.
struct Place {
  long long image;
  int c0, rg, nrg;
  // tiles of rows from first on, every step-th row, before end
  long long first, step, end;
  bool in;
};

template <int VEC>
DFD_DEV Place gn_place(int b, long long hw, int c, int cpb, int ctiles, int chunks, int turns) {
  Place p;
  const int ct = b % ctiles;
  const int ch = (b / ctiles) % chunks;
  p.image = b / (ctiles * chunks);
  const int slot = threadIdx.x % cpb;
  p.rg = threadIdx.x / cpb;
  p.nrg = kBlock / cpb;
  const int v = ct * cpb + slot;
  p.in = p.rg < p.nrg && v * VEC < c;
  p.c0 = v * VEC;
  const long long tile = kTileRows * p.nrg;
  if (turns) {  // a few tiles in a row
    p.first = ch * turns * tile;
    p.step = tile;
    p.end = p.first + turns * tile < hw ? p.first + turns * tile : hw;
  } else {  // every chunks-th of the image's
    p.first = ch * tile;
    p.step = chunks * tile;
    p.end = hw;
  }
  return p;
}

// Blocks go to the 8 XCDs in turn. Those that take the same rows, other
// channels, are given the same XCD, one after another: where a tile's part of a
// row does not end with a cache line, they share it in one L2. 20x1032x84x83
// fp16 takes 182 us forward and 302 backward so, 212 and 332 otherwise; 26x960
// x75x75 bf16, whose tiles do end with lines, 155 and 268, and 159 and 275.
DFD_DEV int gn_near(int b, int ctiles) {
  const int set = 8 * ctiles;
  if (ctiles == 1 || b >= (int)gridDim.x / set * set) return b;
  const int r = b % set;
  return b - r + r % 8 * ctiles + r / 8;
}

// Per-channel coefficients of a block's channels, made once in LDS and read
// from there into registers: coef(channel, k) for the k-th of K.
template <int K, int VEC, typename F>
DFD_DEV void gn_coefs(float* lds, const Place& p, int c, int cpb, int ctiles, int b, F coef,
                      float (&out)[K][VEC]) {
  const int first = b % ctiles * cpb * VEC;
  const int width = c - first < cpb * VEC ? c - first : cpb * VEC;
  for (int i = threadIdx.x; i < width; i += kBlock) {
    float v[K];
    coef(first + i, v);
#pragma unroll
    for (int k = 0; k < K; ++k) lds[k * cpb * VEC + i] = v[k];
  }
  __syncthreads();
  if (p.in) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[k][i] = lds[k * cpb * VEC + p.c0 - first + i];
  }
}

// f(row, vectors..) for the thread's rows, U at a time; rows beyond the last
// load that one again and are dropped, so that the loads of a turn are all in
// flight together.
template <int U, typename T, int VEC, typename F>
DFD_DEV void gn_rows(const Place& at, const T* __restrict__ p, const T* __restrict__ q,
                     long long hw, int c, F f) {
  for (long long tile = at.first; tile < at.end; tile += at.step) {
#pragma unroll
    for (int s = 0; s < kTileRows; s += U) {
      const long long r = tile + s * at.nrg + at.rg;
      DfdVec<T, VEC> v[U], w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long row = r + u * at.nrg < hw ? r + u * at.nrg : hw - 1;
        v[u] = dfd_vload_once<T, VEC>(p + row * c);
        if (q) w[u] = dfd_vload_once<T, VEC>(q + row * c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + u * at.nrg < hw) f(r + u * at.nrg, v[u], w[u]);
    }
  }
}

template <int L>
DFD_DEV void gn_store_groups(const Columns& sum, Moments* part, int g0, int g1, int cpg,
                             int first, int width, int each) {
  for (int g = g0 + threadIdx.x / L; g <= g1; g += kBlock / L) {
    const int from = g * cpg > first ? (g * cpg - first) / each : 0;
    const int to = (g + 1) * cpg < first + width ? ((g + 1) * cpg - first) / each : sum.cols;
    const Moments m = sum.join_columns<L>(from, to - from);
    if (threadIdx.x % L == 0) part[g - g0] = m;
  }
}

// part[image][chunk][tile][span] = the moments that the chunk's rows and the
// tile's channels have of each group the tile reaches into (at most span).
template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void gn_stats_kernel(
    const T* __restrict__ x, Moments* __restrict__ part, long long hw, int c, int cpg, int cpb,
    int ctiles, int chunks, int span) {
  extern __shared__ float lds[];
  const int b = gn_near(blockIdx.x, ctiles);
  const Place p = gn_place<VEC>(b, hw, c, cpb, ctiles, chunks, 0);
  const int first = b % ctiles * cpb * VEC;  // the tile's channels
  const int width = c - first < cpb * VEC ? c - first : cpb * VEC;
  // a vector within one group is one column
  const bool whole = cpg % VEC == 0;
  const int each = whole ? VEC : 1;
  Columns sum(lds, width / each, p.nrg, whole ? cpg / VEC : cpg);
  // the block's rows: its tiles, less what the image's last one lacks
  const long long tile = kTileRows * p.nrg, last = (hw - 1) / tile * tile;
  const long long turns = (last - p.first) / p.step;
  int here = (int)((turns + 1) * tile);
  if (p.first + turns * p.step == last) here -= (int)(last + tile - hw);
  if (p.in) {
    float s1[VEC] = {}, s2[VEC] = {}, pivot[VEC] = {};
    const T* base = x + p.image * hw * c + p.c0;
    if (p.first + p.rg < hw) {
      // about the thread's own first row: its values are of the set's own size
      const DfdVec<T, VEC> one = dfd_vload<T, VEC>(base + (p.first + p.rg) * c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) pivot[i] = DfdCvt<T>::to_f32(one.v[i]);
    }
    gn_rows<4, T, VEC>(p, base, nullptr, hw, c,
                       [&](long long, const DfdVec<T, VEC>& v, const DfdVec<T, VEC>&) {
#pragma unroll
                         for (int i = 0; i < VEC; ++i) {
                           const float d = DfdCvt<T>::to_f32(v.v[i]) - pivot[i];
                           s1[i] += d;
                           s2[i] += d * d;
                         }
                       });
    sum.put<VEC>(p.rg, threadIdx.x % cpb, whole, sum.row_count(p.rg, here, 1), pivot, s1, s2);
  }
  sum.join_rows(here, each);
  const int g0 = first / cpg, g1 = (first + width - 1) / cpg;
  if (sum.small_groups(g1 - g0 + 1))
    gn_store_groups<16>(sum, part + (long long)b * span, g0, g1, cpg, first, width, each);
  else
    gn_store_groups<kWave>(sum, part + (long long)b * span, g0, g1, cpg, first, width, each);
}

// A group's WAVES waves join the moments of the chunks, of the tiles that reach
// into the group, and of the group's places in a folded row.
template <int WAVES>
constexpr int final_block() {
  return WAVES > 1 ? WAVES * kWave : kBlock;
}

template <int WAVES>
__global__ __launch_bounds__(final_block<WAVES>()) void gn_finalize_kernel(
    const Moments* __restrict__ part, float* __restrict__ mean, float* __restrict__ rstd,
    long long total, int cpg, int groups, int fold, int tile, int ctiles, int chunks, int span,
    float eps) {
  __shared__ Moments joined[WAVES];
  const int lanes = WAVES * kWave;
  const long long id = (long long)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes;
  if (id >= total) return;  // the whole block, where a group has more than one wave
  const long long image = id / groups;
  const int g = (int)(id - image * groups);
  const int most = (cpg + tile - 2) / tile + 1;  // tiles that can reach into a group
  const float inv_most = 1.f / (float)most, inv_chunks = 1.f / (float)chunks;
  const int wave = threadIdx.x % lanes / kWave;
  const int all = fold * chunks * most, each = (all + WAVES - 1) / WAVES;
  const int begin = wave * each, count = all - begin < each ? all - begin : each;
  Moments m = gather<kWave>(count, [&](int i) {
    const int e = begin + i;
    const int f = div_small(e, inv_most), place = div_small(f, inv_chunks);
    const int ch = f - place * chunks;
    const int from = (place * groups + g) * cpg;  // the group's first channel in the row
    const int t = from / tile + (e - f * most);
    if (t * tile >= from + cpg) return Moments{0.f, 0.f, 0.f};
    return part[((image * chunks + ch) * ctiles + t) * span + (from / cpg - t * tile / cpg)];
  });
  if (WAVES > 1) {
    if (threadIdx.x % kWave == 0) joined[wave] = m;
    __syncthreads();
    m = gather<16>(WAVES, [&](int e) { return joined[e]; });
  }
  if (threadIdx.x % lanes == 0) {
    mean[id] = m.mean;
    rstd[id] = rsqrtf(m.m2 * __builtin_amdgcn_rcpf(m.n) + eps);
  }
}

template <typename T, int VEC, Act ACT>
__global__ __launch_bounds__(kBlock) void gn_apply_kernel(
    const T* __restrict__ x, Params weight, Params bias,
    const T* __restrict__ residual, const float* __restrict__ drop, T* __restrict__ y,
    const float* __restrict__ mean, const float* __restrict__ rstd, long long hw, int c,
    int groups, int cpg, int cpb, int ctiles, int chunks, int turns) {
  extern __shared__ float lds[];
  const int b = gn_near(gridDim.x - 1 - blockIdx.x, ctiles);
  const Place p = gn_place<VEC>(b, hw, c, cpb, ctiles, chunks, turns);
  const float inv_cpg = 1.f / (float)cpg, inv_channels = 1.f / (float)(cpg * groups);
  float k[3][VEC];  // mean, factor, bias
  gn_coefs<3, VEC>(lds, p, c, cpb, ctiles, b, [&](int i, float (&v)[3]) {
    const int ch = i - div_small(i, inv_channels) * cpg * groups;
    const long long s = p.image * groups + div_small(ch, inv_cpg);
    v[0] = mean[s];
    v[1] = rstd[s] * weight.at(ch, 1.f);
    v[2] = bias.at(ch, 0.f);
  }, k);
  if (!p.in) return;
  const float keep = drop ? drop[p.image] : 1.f;
  const long long off = p.image * hw * c + p.c0;
  gn_rows<4, T, VEC>(
      p, x + off, residual ? residual + off : nullptr, hw, c,
      [&](long long r, const DfdVec<T, VEC>& v, const DfdVec<T, VEC>& res) {
        DfdVec<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float z = gn_act((DfdCvt<T>::to_f32(v.v[i]) - k[0][i]) * k[1][i] + k[2][i], ACT) * keep;
          if (residual) z += DfdCvt<T>::to_f32(res.v[i]);
          o.v[i] = DfdCvt<T>::from_f32(z);
        }
        dfd_vstore_once<T, VEC>(y + off + r * c, o);
      });
}

// part[image][chunk][2][c] = sum g, sum g (x - mean) over the chunk's rows.
template <typename T, int VEC, Act ACT>
__global__ __launch_bounds__(kBlock) void gn_bwd_sums_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, Params weight,
    Params bias, const float* __restrict__ drop,
    const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ part,
    long long hw, int c, int groups, int cpg, int cpb, int ctiles, int chunks) {
  __shared__ float l1[kBlock * VEC], l2[kBlock * VEC];
  extern __shared__ float lds[];
  const int b = gn_near(blockIdx.x, ctiles);
  const Place p = gn_place<VEC>(b, hw, c, cpb, ctiles, chunks, 0);
  const float inv_cpg = 1.f / (float)cpg, inv_channels = 1.f / (float)(cpg * groups);
  float k[3][VEC];  // mean, factor, bias
  gn_coefs<3, VEC>(lds, p, c, cpb, ctiles, b, [&](int i, float (&v)[3]) {
    const int ch = i - div_small(i, inv_channels) * cpg * groups;
    const long long s = p.image * groups + div_small(ch, inv_cpg);
    v[0] = mean[s];
    v[1] = rstd[s] * weight.at(ch, 1.f);
    v[2] = bias.at(ch, 0.f);
  }, k);
  float s1[VEC] = {}, s2[VEC] = {};
  if (p.in) {
    const long long off = p.image * hw * c + p.c0;
    gn_rows<2, T, VEC>(p, x + off, dy + off, hw, c,
                              [&](long long, const DfdVec<T, VEC>& v, const DfdVec<T, VEC>& u) {
#pragma unroll
                                for (int i = 0; i < VEC; ++i) {
                                  const float d = DfdCvt<T>::to_f32(v.v[i]) - k[0][i];
                                  const float g = DfdCvt<T>::to_f32(u.v[i]) *
                                                  gn_act_slope(d * k[1][i] + k[2][i], ACT);
                                  s1[i] += g;
                                  s2[i] += g * d;
                                }
                              });
    const float keep = drop ? drop[p.image] : 1.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      s1[i] *= keep;
      s2[i] *= keep;
    }
  }
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    l1[t * VEC + i] = s1[i];
    l2[t * VEC + i] = s2[i];
  }
  __syncthreads();
  for (int s = p.nrg; s > 1;) {
    const int h = (s + 1) / 2;
    if (p.rg + h < s) {
      const int o = t + h * cpb;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        l1[t * VEC + i] += l1[o * VEC + i];
        l2[t * VEC + i] += l2[o * VEC + i];
      }
    }
    __syncthreads();
    s = h;
  }
  if (p.in && p.rg == 0) {
    const long long chunk = b / ctiles;
    float* out = part + chunk * 2 * c + p.c0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      out[i] = l1[t * VEC + i];
      out[c + i] = l2[t * VEC + i];
    }
  }
}

// A block takes some whole groups of an image, `width` channels: their sums
// over the chunks and the places in a folded row,
//   k[image][group] = (A / m, B rstd / m), so that
//     dx = rstd (weight g - k.x - (x - mean) k.y)
//   sums[image][2][c] = sum g, sum g h, if the parameters want them
__global__ __launch_bounds__(kGroupBlock) void gn_bwd_group_kernel(
    const float* __restrict__ part, Params weight, const float* __restrict__ rstd,
    float2* __restrict__ k, float* __restrict__ sums, long long hw, int c, int groups,
    int fold, int chunks, int width, int tiles) {
  extern __shared__ float lds[];  // [2][parts * cols], [2][cols]
  const long long image = blockIdx.x / tiles;
  const int c0 = (int)(blockIdx.x % tiles) * width;
  const int cols = c - c0 < width ? c - c0 : width;
  const int cpg = c / groups;
  const int threads = blockDim.x;
  const int parts = cols < threads ? threads / cols : 1;
  // part[image][chunk][2][fold][c]
  const float* src = part + image * chunks * 2 * fold * c + c0;
  const float inv_fold = 1.f / (float)fold;
  for (int i = threadIdx.x; i < parts * cols; i += threads) {
    const int p = i / cols, col = i - p * cols;
    float a = 0.f, b = 0.f;
#pragma unroll 8
    for (int e = p; e < chunks * fold; e += parts) {
      const int ch = div_small(e, inv_fold);
      const float* at = src + ((long long)ch * 2 * fold + (e - ch * fold)) * c + col;
      a += at[0];
      b += at[(long long)fold * c];
    }
    lds[i] = a;
    lds[parts * cols + i] = b;
  }
  __syncthreads();
  // the columns' sums, 16 lanes each, in place where a column is one part
  float* col_a = parts > 1 ? lds + 2 * parts * cols : lds;
  float* col_b = col_a + cols;
  for (int col = threadIdx.x / 16; col < cols; col += threads / 16) {
    float a = 0.f, b = 0.f;
    for (int p = threadIdx.x % 16; p < parts; p += 16) {
      a += lds[p * cols + col];
      b += lds[(parts + p) * cols + col];
    }
    a = lanes_sum<16>(a);
    b = lanes_sum<16>(b);
    if (threadIdx.x % 16 == 0) {
      col_a[col] = a;
      col_b[col] = b;
      if (sums) {
        float* out = sums + image * 2 * c + c0 + col;
        out[0] = a;
        out[c] = b * rstd[image * groups + (c0 + col) / cpg];
      }
    }
  }
  __syncthreads();
  const int lane = threadIdx.x % kWave;
  for (int g = threadIdx.x / kWave; g < cols / cpg; g += threads / kWave) {
    float a = 0.f, b = 0.f;
    for (int e = lane; e < cpg; e += kWave) {
      const float w = weight.at(c0 + g * cpg + e, 1.f);
      a += w * col_a[g * cpg + e];
      b += w * col_b[g * cpg + e];
    }
    a = lanes_sum<kWave>(a);
    b = lanes_sum<kWave>(b);
    if (lane == 0) {
      const long long id = image * groups + c0 / cpg + g;
      const float m = (float)hw * (float)cpg;
      const float r = rstd[id];
      k[id] = make_float2(a / m, b * r * r / m);
    }
  }
}

// dbias[c], dweight[c] from the images' sums: 32 channels a block, 32 threads
// for each of them. Slice blockIdx.y takes `per` images; its result is 2 c
// after the one before.
__global__ __launch_bounds__(1024) void gn_bwd_params_kernel(
    const float* __restrict__ sums, float* __restrict__ dweight, float* __restrict__ dbias,
    long long n, int c, int per) {
  __shared__ float l1[1024], l2[1024];
  const int t = threadIdx.x;
  const int ch = blockIdx.x * 32 + t % 32;
  const long long first = (long long)blockIdx.y * per;
  const long long end = first + per < n ? first + per : n;
  float s1 = 0.f, s2 = 0.f;
  if (ch < c) {
#pragma unroll 4
    for (long long i = first + t / 32; i < end; i += 32) {
      s1 += sums[i * 2 * c + ch];
      s2 += sums[i * 2 * c + c + ch];
    }
  }
  l1[t] = s1;
  l2[t] = s2;
  for (int h = 512; h >= 32; h /= 2) {
    __syncthreads();
    if (t < h) {
      l1[t] += l1[t + h];
      l2[t] += l2[t + h];
    }
  }
  if (t < 32 && ch < c) {
    if (dbias) dbias[blockIdx.y * 2ll * c + ch] = l1[t];
    if (dweight) dweight[blockIdx.y * 2ll * c + ch] = l2[t];
  }
}

template <typename T, int VEC, Act ACT>
__global__ __launch_bounds__(kBlock) void gn_bwd_dx_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, Params weight,
    Params bias, const float* __restrict__ drop,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    const float2* __restrict__ k, T* __restrict__ dx, long long hw, int c, int groups, int cpg,
    int cpb, int ctiles, int chunks, int turns) {
  extern __shared__ float lds[];
  const int b = gn_near(gridDim.x - 1 - blockIdx.x, ctiles);
  const Place p = gn_place<VEC>(b, hw, c, cpb, ctiles, chunks, turns);
  const float inv_cpg = 1.f / (float)cpg, inv_channels = 1.f / (float)(cpg * groups);
  float q[5][VEC];  // mean, factor, bias, and what is taken off
  gn_coefs<5, VEC>(lds, p, c, cpb, ctiles, b, [&](int i, float (&v)[5]) {
    const int ch = i - div_small(i, inv_channels) * cpg * groups;
    const long long s = p.image * groups + div_small(ch, inv_cpg);
    const float r = rstd[s];
    const float2 kk = k[s];
    v[0] = mean[s];
    v[1] = r * weight.at(ch, 1.f);
    v[2] = bias.at(ch, 0.f);
    v[3] = r * kk.x;
    v[4] = r * kk.y;
  }, q);
  if (!p.in) return;
  const float keep = drop ? drop[p.image] : 1.f;
  const long long off = p.image * hw * c + p.c0;
  gn_rows<4, T, VEC>(p, x + off, dy + off, hw, c,
                  [&](long long r, const DfdVec<T, VEC>& v, const DfdVec<T, VEC>& u) {
                    DfdVec<T, VEC> o;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                      const float d = DfdCvt<T>::to_f32(v.v[i]) - q[0][i];
                      const float g = DfdCvt<T>::to_f32(u.v[i]) * keep *
                                      gn_act_slope(d * q[1][i] + q[2][i], ACT);
                      o.v[i] = DfdCvt<T>::from_f32(g * q[1][i] - q[3][i] - d * q[4][i]);
                    }
                    dfd_vstore_once<T, VEC>(dx + off + r * c, o);
                  });
}

}  // namespace

long long gn_fwd_ws(const GnArgs& a) {
  if (gn_slab_fits(a, false)) return 0;
  const GnPlan p = gn_plan(a);
  return a.n * p.chunks * p.ctiles * p.span * (long long)(sizeof(Moments) / sizeof(float));
}

// Images that one block of the parameters' kernel adds up; where there are
// more, the slices' results are added in a second launch: backward of 16384x256
// x1x1 bf16 49 us so and 105 by one launch, 4096x448x3x3 61 and 68.
static int gn_slice(const GnArgs& a) {
  const long long per = a.n <= 512 ? a.n : a.n <= 64 * 256 ? 256 : (a.n + 63) / 64;
  return (int)per;
}
static int gn_slices(const GnArgs& a) { return (int)((a.n + gn_slice(a) - 1) / gn_slice(a)); }

// The images' sums for the parameters, and the slices'; streaming, the chunks'
// and groups' too.
long long gn_bwd_ws(const GnArgs& a) {
  const long long sums = (a.n + gn_slices(a)) * 2 * a.c;
  if (gn_slab_fits(a, true)) return sums;
  const GnPlan p = gn_plan(a);
  return sums + a.n * p.chunks * p.c * 2 + a.n * a.groups * 2;
}

// Tiles of a block of the kernels that make no sums: 26x256x300x300 bf16 takes
// 407 us forward with two, 449 with one and 411 with four, for a block's
// coefficients have a price; 4x144x150x150 14.4 with one and 16.5 with two.
static int gn_turns(const GnArgs& a, const GnPlan& p) {
  const long long tile = kTileRows * (kBlock / p.cpb);
  const long long tiles = (p.hw + tile - 1) / tile;
  return a.n * p.ctiles * tiles >= 4096 ? 2 : 1;
}
static int gn_short_chunks(const GnArgs& a, const GnPlan& p) {
  const long long rows = (long long)gn_turns(a, p) * kTileRows * (kBlock / p.cpb);
  return (int)((p.hw + rows - 1) / rows);
}

hipError_t gn_fwd(const GnArgs& a, hipStream_t stream) {
  if (gn_slab_fits(a, false)) return gn_slab_fwd(a, stream);
  const GnPlan p = gn_plan(a);
  const int chunks = gn_short_chunks(a, p);
  if (gn_too_many(a.n * chunks * p.ctiles, kBlock) ||
      gn_too_many(a.n * a.groups, kWave))
    return hipErrorInvalidConfiguration;
  const dim3 fine((unsigned)(a.n * chunks * p.ctiles));
  const int coef = 3 * (int)sizeof(float) * p.cpb * p.vec;
  const Params weight = {a.weight, a.ptype}, bias = {a.bias, a.ptype};
  const dim3 grid((unsigned)(a.n * p.chunks * p.ctiles));
  const long long groups = a.n * a.groups;
  // Few groups of many chunks have 16 waves each: forward of 1x256x300x300 fp16
  // takes 38 us so and 54 by one wave; where there are many, 42x800x42x43 bf16
  // takes 82 us by one and 91 by 16.
  const bool alone = groups <= 512 && p.fold * p.chunks > 128;
  const int each = kBlock / kWave;  // groups a block, where they have one wave
  const dim3 finals((unsigned)(alone ? groups : (groups + each - 1) / each));
  const int cpg = a.c / a.groups;
  const int cols = p.cpb * (cpg % p.vec == 0 ? 1 : p.vec);
  const int lds = columns_lds(kBlock, kBlock / p.cpb, cols);
  GN_TYPE(a.type, GN_VEC(p.vec, {
            const T* x = static_cast<const T*>(a.x);
            gn_stats_kernel<T, V><<<grid, kBlock, lds, stream>>>(
                x, reinterpret_cast<Moments*>(a.ws), p.hw, p.c, cpg, p.cpb, p.ctiles,
                p.chunks, p.span);
            const auto finalize = alone ? gn_finalize_kernel<16> : gn_finalize_kernel<1>;
            finalize<<<finals, alone ? final_block<16>() : kBlock, 0, stream>>>(
                reinterpret_cast<const Moments*>(a.ws), a.mean, a.rstd, groups, cpg, a.groups,
                p.fold, p.cpb * p.vec, p.ctiles, p.chunks, p.span, a.eps);
            GN_ACT(a.act, gn_apply_kernel<T, V, A><<<fine, kBlock, coef, stream>>>(
                              x, weight, bias, static_cast<const T*>(a.residual), a.drop,
                              static_cast<T*>(a.y), a.mean, a.rstd, p.hw, p.c, a.groups, cpg,
                              p.cpb, p.ctiles, chunks, gn_turns(a, p)));
          }));
  return hipGetLastError();
}

hipError_t gn_bwd(const GnArgs& a, hipStream_t stream) {
  float* sums = a.dweight || a.dbias ? a.ws : nullptr;
  if (gn_slab_fits(a, true)) {
    const hipError_t e = gn_slab_bwd(a, sums, stream);
    if (e != hipSuccess) return e;
  } else {
    const GnPlan p = gn_plan(a);
    const Params weight = {a.weight, a.ptype}, bias = {a.bias, a.ptype};
    const dim3 grid((unsigned)(a.n * p.chunks * p.ctiles));
    const int chunks = gn_short_chunks(a, p);
    const dim3 fine((unsigned)(a.n * chunks * p.ctiles));
    const int coef = (int)sizeof(float) * p.cpb * p.vec;  // LDS of one coefficient
    float2* k = reinterpret_cast<float2*>(a.ws + (a.n + gn_slices(a)) * 2 * a.c);
    float* part = reinterpret_cast<float*>(k + a.n * a.groups);
    // Whole groups of about 32 channels: many blocks, and many threads a
    // channel, since the chunks are read one after another. More of both
    // where there are few: backward of 1x288x150x150 fp16 34.0 us and 35.6
    // without, 1x32x296x293 bf16 21.8 and 24.2.
    const int cpg = a.c / a.groups;
    const bool few = a.n * a.c < 32 * 128;
    const int some = few ? 8 : 32, threads = few ? kGroupBlock : kGroupBlock / 2;
    const int width = cpg >= some ? cpg : some / cpg * cpg;
    const int tiles = (a.c + width - 1) / width;
    const int lds = 2 * (int)sizeof(float) * (width > 2 * threads ? width : 2 * threads);
    if (gn_too_many(a.n * chunks * p.ctiles, kBlock) || gn_too_many(a.n * tiles, kGroupBlock))
      return hipErrorInvalidConfiguration;
    GN_TYPE(a.type, GN_VEC(p.vec, GN_ACT(a.act, {
              const T* x = static_cast<const T*>(a.x);
              const T* dy = static_cast<const T*>(a.dy);
              gn_bwd_sums_kernel<T, V, A><<<grid, kBlock, 3 * coef, stream>>>(
                  dy, x, weight, bias, a.drop, a.mean, a.rstd, part, p.hw, p.c, a.groups,
                  cpg, p.cpb, p.ctiles, p.chunks);
              gn_bwd_group_kernel<<<dim3((unsigned)(a.n * tiles)), threads, lds, stream>>>(
                  part, weight, a.rstd, k, sums, a.hw, a.c, a.groups, p.fold, p.chunks, width,
                  tiles);
              if (a.dx)
                gn_bwd_dx_kernel<T, V, A><<<fine, kBlock, 5 * coef, stream>>>(
                    dy, x, weight, bias, a.drop, a.mean, a.rstd, k, static_cast<T*>(a.dx),
                    p.hw, p.c, a.groups, cpg, p.cpb, p.ctiles, chunks, gn_turns(a, p));
            })));
  }
  if (sums) {
    const unsigned blocks = (a.c + 31) / 32;
    const int slices = gn_slices(a);
    long long n = a.n;
    if (slices > 1) {
      float* parts = a.ws + a.n * 2 * a.c;
      gn_bwd_params_kernel<<<dim3(blocks, slices), 1024, 0, stream>>>(
          sums, parts + a.c, parts, n, a.c, gn_slice(a));
      sums = parts;
      n = slices;
    }
    gn_bwd_params_kernel<<<dim3(blocks), 1024, 0, stream>>>(sums, a.dweight, a.dbias, n, a.c,
                                                            (int)n);
  }
  return hipGetLastError();
}
