// Group norm + activation of one slab by one block: the rows of an image by
// some whole groups of channels, held in LDS between the statistics and their
// use, so that x (and dy) are read from memory once and a pass is one launch.
// group_norm.hip has the formulas, and takes what is too large here.
//
// A thread takes rows rg, rg + nrg, .. of its slot of VEC channels, and reads
// back from LDS only what it wrote. Its sums, about its own first row, are
// joined over columns of LDS (a channel, or a vector's channels together) and
// then over each group's columns, always in the same order.
//
// These are small shapes, where a launch's fixed costs count: the loops stay
// rolled, since code that runs once costs more to fetch than to run. Forward,
// 64x160x19x19 bf16 takes 12.0 us (two passes over rows in registers, all
// unrolled: 17.4; streaming: 17.9 in three launches), 32x256x19x19 fp16 9.0 (its
// 12 MB at the rate of a large copy: 1.9; streaming 16.7), 1x1632x10x10 fp16 7.3
// (streaming 13.8); backward 15.9 and 12.8 (streaming 25.8 and 24.6). What is left
// is a block's chain: by a clock in the kernel 2.3 to 3.7 us until the rows are
// there, 2.3 for the sums, 1.0 to 2.6 for the activation and its stores.

#include "group_norm_device.h"

namespace {

constexpr int kMaxThreads = 1024;
constexpr int kLds = 160 * 1024;

struct SlabPlan {
  int vec, threads;        // threads 0: no block can hold a slab
  int width, nslots, nrg;  // channels of a block, its vectors, rows at a time
  int slices;              // blocks an image
  int lds;
};

bool slab_try(const GnArgs& a, int tensors, int vec, int width, int threads, SlabPlan* p) {
  const int cpg = a.c / a.groups;
  p->vec = vec;
  p->threads = threads;
  p->width = width < a.c ? width : a.c;
  p->nslots = p->width / vec;
  p->slices = (a.c + p->width - 1) / p->width;
  if (p->nslots > threads) return false;
  p->nrg = threads / p->nslots;
  const int cols = tensors == 1 && cpg % vec == 0 ? p->nslots : p->width;
  const long long data = (long long)a.hw * p->width * gn_elem(a.type) * tensors;
  const long long lds = (data + 15) / 16 * 16 + columns_lds(threads, p->nrg, cols);
  p->lds = (int)lds;
  return lds <= kLds;
}

// How the image is cut.
SlabPlan slab_plan(const GnArgs& a, int tensors) {
  SlabPlan best = {}, p = {};
  const int cpg = a.c / a.groups;
  const int es = gn_elem(a.type);
  // div_small's range, and offsets in an int
  if (a.hw >= (1 << 16) || a.c >= (1 << 14)) return best;
  const int widest = gn_vec(a);
  for (int vec = widest; vec >= 1; vec >>= 1) {
    const int unit = cpg / gcd_of(cpg, vec) * vec;
    // A row's part of a slab is 64 bytes or more: backward of 64x256x38x38 bf16
    // in parts of 32 bytes takes 90 us, streaming 61; less only for a few blocks.
    // Of many images of few rows a slab is 2 KB or more: a block has its own price.
    int m = 1;
    while (m * unit < a.c &&
           (m * unit * es < 64 ||
            (m * unit * es * a.hw < 2048 && a.n * a.c / (m * unit) > 4096)))
      ++m;
    for (; m >= 1; m /= 2) {
      const int width = m * unit < a.c ? m * unit : a.c;
      const long long blocks = a.n * ((a.c + width - 1) / width);
      const bool few = blocks < 128;
      if (width * es < 64 && width < a.c && !few) break;
      // 512 slabs of 13 KB: 12.7 us by 256 threads, 13.6 by 512; 256 of 29 KB:
      // 14.5 us by 512, 15.9 by 1024; 28 of 80 KB: 13.9 us by 1024; 8192 of
      // 3 KB (1024x256x7x7 bf16): 20.8 us by 64, 24.6 by 128, 36.8 by 256;
      // 16384x256x1x1 bf16: 31 us by 64 in slabs of 512 bytes, 435 by 256 in
      // slabs of 64.
      const long long bytes = a.hw * width * es;
      const int threads = blocks <= 64 ? 1024 : bytes <= 4096 ? 64 : bytes <= 16384 ? 256 : 512;
      if (!slab_try(a, tensors, vec, width, threads, &p)) continue;
      // Narrow loads cost what wide ones do: of more than 16 a thread, streaming
      // is faster. us by a slab and streaming, forward and backward: fp16
      // 1x1632x10x10 (5 rows a thread) 7.4 and 14.2, 8.8 and 19.4; 1x960x38x38
      // (21) 16.7 and 16.6, 25.4 and 22.0; 4x336x38x38 (30) 21.3 and 16.2;
      // backward of 1x192x75x75 (17) 31.5 and 21.4; fp32 46x96x41x43 (31) 39.2
      // and 27.4.
      if (vec * es < 16 && a.hw > 16 * p.nrg) continue;
      // One block alone on a CU does not hide its chain. us by a slab and
      // streaming, bf16: forward of 64x1020x25x25 in 960 blocks 80 and 58,
      // backward of 128x256x24x24 in 1024 60 and 53, of 32x512x28x28 in 512 36
      // and 46, of 128x1632x10x10 in 1024 63 and 70.
      if (2 * p.lds > kLds && blocks > 512) continue;
      // With less than a block for every other CU, narrower vectors make more
      // and smaller slabs.
      if (best.threads == 0 || (a.n * best.slices < 128 && p.slices > best.slices)) best = p;
      break;
    }
    if (best.threads != 0 && a.n * best.slices >= 128) break;
  }
  return best;
}

// A thread's part of the slab.
template <int VEC>
struct Slab {
  long long image;
  int c0, width;  // the block's channels
  int slot, rg;
  bool in;
  int group[VEC];  // its channels' groups within the slab

  DFD_DEV Slab(int c, int cpg, int width_, int nslots, int nrg, int slices) {
    image = blockIdx.x / slices;
    c0 = (int)(blockIdx.x - image * slices) * width_;
    width = c - c0 < width_ ? c - c0 : width_;
    rg = div_small(threadIdx.x, 1.f / (float)nslots);
    slot = threadIdx.x - rg * nslots;
    in = rg < nrg && slot * VEC < width;
    int g = div_small(slot * VEC, 1.f / (float)cpg);
    int left = (g + 1) * cpg - slot * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      group[i] = g;
      if (--left == 0) {
        ++g;
        left = cpg;
      }
    }
  }
};

template <typename T, int VEC, Act ACT>
__global__ __launch_bounds__(kMaxThreads) void gn_slab_fwd_kernel(
    const T* __restrict__ x, Params weight, Params bias, const T* __restrict__ residual,
    const float* __restrict__ drop, T* __restrict__ y, float* __restrict__ mean,
    float* __restrict__ rstd, int hw, int c, int groups, int width, int nslots, int nrg,
    int slices, int data_bytes, float eps) {
  extern __shared__ __align__(16) unsigned char lds[];
  DfdVec<T, VEC>* data = reinterpret_cast<DfdVec<T, VEC>*>(lds);
  float* scratch = reinterpret_cast<float*>(lds + data_bytes);
  const int cpg = c / groups;
  const Slab<VEC> s(c, cpg, width, nslots, nrg, slices);
  const long long base = s.image * hw * c + s.c0 + s.slot * VEC;
  float ka[VEC], kb[VEC], mu[VEC];
  // a vector within one group is one column
  const bool whole = cpg % VEC == 0;
  Columns sum(scratch, whole ? s.width / VEC : s.width, nrg, whole ? cpg / VEC : cpg);
  if (s.in) {
    weight.load<VEC>(s.c0 + s.slot * VEC, 1.f, ka);
    bias.load<VEC>(s.c0 + s.slot * VEC, 0.f, kb);
    float pivot[VEC] = {}, a[VEC] = {}, b[VEC] = {};
    constexpr int U = 4;  // loads in flight; those beyond the rows are dropped
    for (int row = s.rg; row < hw; row += U * nrg) {
      DfdVec<T, VEC> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = row + u * nrg < hw ? row + u * nrg : row;
        v[u] = dfd_vload<T, VEC>(x + base + (long long)r * c);
      }
      if (row == s.rg) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) pivot[i] = DfdCvt<T>::to_f32(v[0].v[i]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row + u * nrg >= hw) continue;
        data[(row + u * nrg) * nslots + s.slot] = v[u];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = DfdCvt<T>::to_f32(v[u].v[i]) - pivot[i];
          a[i] += d;
          b[i] += d * d;
        }
      }
    }
    sum.put<VEC>(s.rg, s.slot, whole, sum.row_count(s.rg, hw, 1), pivot, a, b);
  }
  sum.join_rows(hw, whole ? VEC : 1);
  sum.join_groups(eps);
  if (!s.in) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    mu[i] = sum.sums[s.group[i]];
    const float rs = sum.sums[sum.groups + s.group[i]];
    ka[i] *= rs;
    if (s.rg == 0 && (i == 0 || s.group[i] != s.group[i - 1])) {
      // by each vector that reaches into the group: they all have the same
      const long long g = s.image * groups + s.c0 / cpg + s.group[i];
      mean[g] = mu[i];
      rstd[g] = rs;
    }
  }
  const float keep = drop ? drop[s.image] : 1.f;
#pragma unroll 2
  for (int row = s.rg; row < hw; row += nrg) {
    const DfdVec<T, VEC> v = data[row * nslots + s.slot];
    DfdVec<T, VEC> res, o;
    if (residual) res = dfd_vload<T, VEC>(residual + base + (long long)row * c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float z = gn_act((DfdCvt<T>::to_f32(v.v[i]) - mu[i]) * ka[i] + kb[i], ACT) * keep;
      if (residual) z += DfdCvt<T>::to_f32(res.v[i]);
      o.v[i] = DfdCvt<T>::from_f32(z);
    }
    dfd_vstore<T, VEC>(y + base + (long long)row * c, o);
  }
}

// sums[image][2][c] = sum g, rstd * sum g (x - mean), for the parameters.
template <typename T, int VEC, Act ACT>
__global__ __launch_bounds__(kMaxThreads) void gn_slab_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, Params weight, Params bias,
    const float* __restrict__ drop, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* __restrict__ dx, float* __restrict__ sums, int hw,
    int c, int groups, int width, int nslots, int nrg, int slices, int data_bytes) {
  extern __shared__ __align__(16) unsigned char lds[];
  DfdVec<T, VEC>* xs = reinterpret_cast<DfdVec<T, VEC>*>(lds);
  DfdVec<T, VEC>* dys = xs + hw * nslots;
  float* scratch = reinterpret_cast<float*>(lds + data_bytes);
  const int cpg = c / groups;
  const Slab<VEC> s(c, cpg, width, nslots, nrg, slices);
  const long long base = s.image * hw * c + s.c0 + s.slot * VEC;
  const long long g0 = s.image * groups + s.c0 / cpg;
  const float keep = drop ? drop[s.image] : 1.f;
  float mu[VEC], rs[VEC], ka[VEC], kb[VEC], a[VEC] = {}, b[VEC] = {};
  auto slope = [&](const DfdVec<T, VEC>& v, const DfdVec<T, VEC>& u, int i, float& d) {
    d = DfdCvt<T>::to_f32(v.v[i]) - mu[i];
    return DfdCvt<T>::to_f32(u.v[i]) * keep * gn_act_slope(d * ka[i] + kb[i], ACT);
  };
  if (s.in) {
    weight.load<VEC>(s.c0 + s.slot * VEC, 1.f, ka);
    bias.load<VEC>(s.c0 + s.slot * VEC, 0.f, kb);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      mu[i] = mean[g0 + s.group[i]];
      rs[i] = rstd[g0 + s.group[i]];
      ka[i] *= rs[i];
    }
#pragma unroll 2
    for (int row = s.rg; row < hw; row += nrg) {
      const DfdVec<T, VEC> v = dfd_vload<T, VEC>(x + base + (long long)row * c);
      const DfdVec<T, VEC> u = dfd_vload<T, VEC>(dy + base + (long long)row * c);
      xs[row * nslots + s.slot] = v;
      dys[row * nslots + s.slot] = u;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float d;
        const float g = slope(v, u, i, d);
        a[i] += g;
        b[i] += g * d;
      }
    }
  }
  Columns sum(scratch, s.width, nrg, cpg);
  if (s.in) {
    float* ra = sum.raw + s.rg * s.width + s.slot * VEC;
    float* rb = ra + nrg * s.width;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      ra[i] = a[i];
      rb[i] = b[i];
    }
  }
  sum.over_rows();
  if (sums)
    for (int ch = threadIdx.x; ch < s.width; ch += blockDim.x) {
      float sa = 0.f, sb = 0.f;
      for (int p = 0; p < sum.parts; ++p) {
        sa += sum.part[p * s.width + ch];
        sb += sum.part[(sum.parts + p) * s.width + ch];
      }
      float* out = sums + s.image * 2 * c + s.c0 + ch;
      out[0] = sa;
      out[c] = sb * rstd[g0 + div_small(ch, sum.inv_cpg)];
    }
  if (!dx) return;
  sum.over_groups([&](int ch) { return weight.at(s.c0 + ch, 1.f); });
  if (!s.in) return;
  const float inv_m = 1.f / ((float)hw * (float)cpg);
  float k0[VEC], k1[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    k0[i] = sum.sums[s.group[i]] * inv_m * rs[i];
    k1[i] = sum.sums[sum.groups + s.group[i]] * inv_m * rs[i] * rs[i] * rs[i];
  }
  for (int row = s.rg; row < hw; row += nrg) {
    const DfdVec<T, VEC> v = xs[row * nslots + s.slot];
    const DfdVec<T, VEC> u = dys[row * nslots + s.slot];
    DfdVec<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float d;
      const float g = slope(v, u, i, d);
      o.v[i] = DfdCvt<T>::from_f32(g * ka[i] - k0[i] - d * k1[i]);
    }
    dfd_vstore<T, VEC>(dx + base + (long long)row * c, o);
  }
}

int slab_data(const GnArgs& a, const SlabPlan& p, int tensors) {
  return (int)((a.hw * p.width * gn_elem(a.type) * tensors + 15) / 16 * 16);
}

}  // namespace

bool gn_slab_fits(const GnArgs& a, bool backward) {
  return slab_plan(a, backward ? 2 : 1).threads != 0;
}

hipError_t gn_slab_fwd(const GnArgs& a, hipStream_t stream) {
  const SlabPlan p = slab_plan(a, 1);
  if (gn_too_many(a.n * p.slices, p.threads)) return hipErrorInvalidConfiguration;
  const Params weight = {a.weight, a.ptype}, bias = {a.bias, a.ptype};
  const dim3 grid((unsigned)(a.n * p.slices));
  GN_TYPE(a.type, GN_VEC(p.vec, GN_ACT(a.act, {
            gn_slab_fwd_kernel<T, V, A><<<grid, p.threads, p.lds, stream>>>(
                static_cast<const T*>(a.x), weight, bias, static_cast<const T*>(a.residual),
                a.drop, static_cast<T*>(a.y), a.mean, a.rstd, (int)a.hw, a.c, a.groups,
                p.width, p.nslots, p.nrg, p.slices, slab_data(a, p, 1), a.eps);
          })));
  return hipGetLastError();
}

hipError_t gn_slab_bwd(const GnArgs& a, float* sums, hipStream_t stream) {
  const SlabPlan p = slab_plan(a, 2);
  if (gn_too_many(a.n * p.slices, p.threads)) return hipErrorInvalidConfiguration;
  const Params weight = {a.weight, a.ptype}, bias = {a.bias, a.ptype};
  const dim3 grid((unsigned)(a.n * p.slices));
  GN_TYPE(a.type, GN_VEC(p.vec, GN_ACT(a.act, {
            gn_slab_bwd_kernel<T, V, A><<<grid, p.threads, p.lds, stream>>>(
                static_cast<const T*>(a.dy), static_cast<const T*>(a.x), weight, bias, a.drop,
                a.mean, a.rstd, static_cast<T*>(a.dx), sums, (int)a.hw, a.c, a.groups,
                p.width, p.nslots, p.nrg, p.slices, slab_data(a, p, 2));
          })));
  return hipGetLastError();
}
