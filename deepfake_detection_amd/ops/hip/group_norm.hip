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
// An image is a row-major [hw, c] matrix. A thread owns VEC neighbouring
// channels, keeps their coefficients in registers and streams rows; a block
// takes cpb such channel slots times 256 / cpb rows at a time (DfdPlan). All
// statistics are held in fp32; sums over a long axis are made by thread,
// block and chunk, joined in a fixed order, without atomics, so a result is
// the same every time.

#include "common.h"
#include "group_norm.h"

namespace {

constexpr int kBlock = 256;

struct GnPlan {
  int vec, cpb, ctiles, chunks, rows_per_chunk;
};

bool gn_aligned(const void* p, int bytes) {
  return (reinterpret_cast<unsigned long long>(p) % bytes) == 0;
}

int gn_elem(GnType t) { return t == GnType::kF32 ? 4 : 2; }

GnPlan gn_plan(const GnArgs& a) {
  const int es = gn_elem(a.type);
  int vec = dfd_pick_vec(a.c, es);
  const void* ptrs[] = {a.x, a.y, a.residual, a.dy, a.dx};
  for (const void* p : ptrs)
    while (vec > 1 && !gn_aligned(p, vec * es)) vec >>= 1;
  const DfdPlan p = dfd_plan(a.c / vec, a.hw, a.n);
  // rounding up the rows of a chunk can leave the last chunks without any
  const int chunks = (int)((a.hw + p.rows_per_chunk - 1) / p.rows_per_chunk);
  return {vec, p.cpb, p.ctiles, chunks, p.rows_per_chunk};
}

// (count, mean, sum of squares about the mean) of a set of values; joining
// two such sets loses nothing to a large common offset, which a plain sum of
// squares would.
struct Moments {
  float n, mean, m2;
};

DFD_DEV Moments join(const Moments& a, const Moments& b) {
  const float n = a.n + b.n;
  if (n == 0.f) return a;
  const float d = b.mean - a.mean;
  const float w = b.n / n;
  return {n, a.mean + d * w, a.m2 + b.m2 + d * d * a.n * w};
}

// The norm's weight or bias, in fp32 or in a halved model's own type.
struct Params {
  const void* p;
  GnType type;
  DFD_DEV float at(int i, float otherwise) const {
    if (p == nullptr) return otherwise;
    switch (type) {
      case GnType::kBf16:
        return DfdCvt<__hip_bfloat16>::to_f32(static_cast<const __hip_bfloat16*>(p)[i]);
      case GnType::kF16:
        return DfdCvt<__half>::to_f32(static_cast<const __half*>(p)[i]);
      default:
        return static_cast<const float*>(p)[i];
    }
  }
};

struct Place {
  long long image;
  int c0, rg, nrg;
  long long r0, r1;
  bool in;
};

// Which rows and channels a thread of the streaming kernels takes. Blocks run
// over channel tiles first, then chunks of rows, then images.
template <int VEC>
DFD_DEV Place gn_place(long long hw, int c, int cpb, int ctiles, int chunks, int rows) {
  Place p;
  const int b = blockIdx.x;
  const int ct = b % ctiles;
  const int ch = (b / ctiles) % chunks;
  p.image = b / (ctiles * chunks);
  const int slot = threadIdx.x % cpb;
  p.rg = threadIdx.x / cpb;
  p.nrg = kBlock / cpb;
  const int v = ct * cpb + slot;
  p.in = p.rg < p.nrg && v * VEC < c;
  p.c0 = v * VEC;
  p.r0 = (long long)ch * rows;
  p.r1 = p.r0 + rows < hw ? p.r0 + rows : hw;
  return p;
}

// part[image][chunk][c] = (mean, m2) of the chunk's rows.
template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void gn_stats_kernel(
    const T* __restrict__ x, float2* __restrict__ part, long long hw, int c, int cpb,
    int ctiles, int chunks, int rows) {
  __shared__ float lm[kBlock * VEC], lv[kBlock * VEC], ln[kBlock];
  const Place p = gn_place<VEC>(hw, c, cpb, ctiles, chunks, rows);
  float s1[VEC] = {}, s2[VEC] = {}, pivot[VEC] = {};
  float cnt = 0.f;
  if (p.in && p.r0 + p.rg < p.r1) {
    const T* base = x + p.image * hw * c + p.c0;
    // about the thread's own first row: its values are of the set's own size
    DfdVec<T, VEC> first = dfd_vload<T, VEC>(base + (p.r0 + p.rg) * c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) pivot[i] = DfdCvt<T>::to_f32(first.v[i]);
    cnt = 1.f;
    for (long long r = p.r0 + p.rg + p.nrg; r < p.r1; r += p.nrg) {
      const DfdVec<T, VEC> v = dfd_vload<T, VEC>(base + r * c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = DfdCvt<T>::to_f32(v.v[i]) - pivot[i];
        s1[i] += d;
        s2[i] += d * d;
      }
      cnt += 1.f;
    }
  }
  const int t = threadIdx.x;
  const float inv = cnt > 0.f ? 1.f / cnt : 0.f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    lm[t * VEC + i] = pivot[i] + s1[i] * inv;
    const float m2 = s2[i] - s1[i] * s1[i] * inv;
    lv[t * VEC + i] = m2 < 0.f ? 0.f : m2;  // a NaN stays one
  }
  ln[t] = cnt;
  __syncthreads();
  for (int s = p.nrg; s > 1;) {
    const int h = (s + 1) / 2;
    if (p.rg + h < s) {
      const int o = t + h * cpb;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const Moments m = join({ln[t], lm[t * VEC + i], lv[t * VEC + i]},
                               {ln[o], lm[o * VEC + i], lv[o * VEC + i]});
        lm[t * VEC + i] = m.mean;
        lv[t * VEC + i] = m.m2;
      }
      ln[t] += ln[o];
    }
    __syncthreads();
    s = h;
  }
  if (p.in && p.rg == 0) {
    const long long chunk = blockIdx.x / ctiles;  // image * chunks + chunk
    float2* out = part + chunk * c + p.c0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = make_float2(lm[t * VEC + i], lv[t * VEC + i]);
  }
}

// One wave a group: joins the chunks' and channels' moments.
__global__ __launch_bounds__(kBlock) void gn_finalize_kernel(
    const float2* __restrict__ part, float* __restrict__ mean, float* __restrict__ rstd,
    long long total, long long hw, int c, int groups, int chunks, int rows, float eps) {
  const long long id = (long long)blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
  if (id >= total) return;
  const int lane = threadIdx.x % kWave;
  const int cpg = c / groups;
  const long long image = id / groups;
  const int g = (int)(id - image * groups);
  const float2* src = part + image * chunks * c + (long long)g * cpg;
  Moments m = {0.f, 0.f, 0.f};
  for (int e = lane; e < chunks * cpg; e += kWave) {
    const int ch = e / cpg;
    const float2 v = src[(long long)ch * c + (e - ch * cpg)];
    const long long left = hw - (long long)ch * rows;
    m = join(m, {(float)(left < rows ? left : rows), v.x, v.y});
  }
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) {
    const Moments o = {__shfl_xor(m.n, off), __shfl_xor(m.mean, off), __shfl_xor(m.m2, off)};
    m = lane & off ? join(o, m) : join(m, o);
  }
  if (lane == 0) {
    mean[id] = m.mean;
    rstd[id] = 1.f / sqrtf(m.m2 / m.n + eps);
  }
}

template <typename T, int VEC, Act ACT>
__global__ __launch_bounds__(kBlock) void gn_apply_kernel(
    const T* __restrict__ x, Params weight, Params bias,
    const T* __restrict__ residual, const float* __restrict__ drop, T* __restrict__ y,
    const float* __restrict__ mean, const float* __restrict__ rstd, long long hw, int c,
    int groups, int cpb, int ctiles, int chunks, int rows) {
  const Place p = gn_place<VEC>(hw, c, cpb, ctiles, chunks, rows);
  if (!p.in) return;
  float mu[VEC], a[VEC], b[VEC];
  const int cpg = c / groups;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const long long s = p.image * groups + (p.c0 + i) / cpg;
    mu[i] = mean[s];
    a[i] = rstd[s] * weight.at(p.c0 + i, 1.f);
    b[i] = bias.at(p.c0 + i, 0.f);
  }
  const float keep = drop ? drop[p.image] : 1.f;
  const long long off = p.image * hw * c + p.c0;
  for (long long r = p.r0 + p.rg; r < p.r1; r += p.nrg) {
    const DfdVec<T, VEC> v = dfd_vload<T, VEC>(x + off + r * c);
    DfdVec<T, VEC> res, o;
    if (residual) res = dfd_vload<T, VEC>(residual + off + r * c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float z = act_fwd((DfdCvt<T>::to_f32(v.v[i]) - mu[i]) * a[i] + b[i], ACT) * keep;
      if (residual) z += DfdCvt<T>::to_f32(res.v[i]);
      o.v[i] = DfdCvt<T>::from_f32(z);
    }
    dfd_vstore<T, VEC>(y + off + r * c, o);
  }
}

// part[image][chunk][2][c] = sum g, sum g (x - mean) over the chunk's rows.
template <typename T, int VEC, Act ACT>
__global__ __launch_bounds__(kBlock) void gn_bwd_sums_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, Params weight,
    Params bias, const float* __restrict__ drop,
    const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ part,
    long long hw, int c, int groups, int cpb, int ctiles, int chunks, int rows) {
  __shared__ float l1[kBlock * VEC], l2[kBlock * VEC];
  const Place p = gn_place<VEC>(hw, c, cpb, ctiles, chunks, rows);
  float s1[VEC] = {}, s2[VEC] = {};
  if (p.in) {
    float mu[VEC], a[VEC], b[VEC];
    const int cpg = c / groups;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const long long s = p.image * groups + (p.c0 + i) / cpg;
      mu[i] = mean[s];
      a[i] = rstd[s] * weight.at(p.c0 + i, 1.f);
      b[i] = bias.at(p.c0 + i, 0.f);
    }
    const float keep = drop ? drop[p.image] : 1.f;
    const long long off = p.image * hw * c + p.c0;
    for (long long r = p.r0 + p.rg; r < p.r1; r += p.nrg) {
      const DfdVec<T, VEC> v = dfd_vload<T, VEC>(x + off + r * c);
      const DfdVec<T, VEC> u = dfd_vload<T, VEC>(dy + off + r * c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = DfdCvt<T>::to_f32(v.v[i]) - mu[i];
        const float g = DfdCvt<T>::to_f32(u.v[i]) * keep * act_bwd(d * a[i] + b[i], ACT);
        s1[i] += g;
        s2[i] += g * d;
      }
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
    const long long chunk = blockIdx.x / ctiles;
    float* out = part + chunk * 2 * c + p.c0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      out[i] = l1[t * VEC + i];
      out[c + i] = l2[t * VEC + i];
    }
  }
}

// One wave a group: k[image][group] = (A / m, B rstd / m), so that
// dx = rstd (weight g - k.x - (x - mean) k.y).
__global__ __launch_bounds__(kBlock) void gn_bwd_group_kernel(
    const float* __restrict__ part, Params weight,
    const float* __restrict__ rstd, float2* __restrict__ k, long long total, long long hw,
    int c, int groups, int chunks) {
  const long long id = (long long)blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
  if (id >= total) return;
  const int lane = threadIdx.x % kWave;
  const int cpg = c / groups;
  const long long image = id / groups;
  const int g = (int)(id - image * groups);
  const float* src = part + image * chunks * 2 * c + (long long)g * cpg;
  float a = 0.f, b = 0.f;
  for (int e = lane; e < chunks * cpg; e += kWave) {
    const int ch = e / cpg, j = e - ch * cpg;
    const float w = weight.at(g * cpg + j, 1.f);
    a += w * src[(long long)ch * 2 * c + j];
    b += w * src[(long long)ch * 2 * c + c + j];
  }
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) {
    a += __shfl_xor(a, off);
    b += __shfl_xor(b, off);
  }
  if (lane == 0) {
    const float m = (float)hw * (float)cpg;
    const float r = rstd[id];
    k[id] = make_float2(a / m, b * r * r / m);
  }
}

// dweight[c], dbias[c]: 32 channels a block, 8 threads for each of them.
__global__ __launch_bounds__(kBlock) void gn_bwd_params_kernel(
    const float* __restrict__ part, const float* __restrict__ rstd,
    float* __restrict__ dweight, float* __restrict__ dbias, long long n, int c, int groups,
    int chunks) {
  __shared__ float l1[kBlock], l2[kBlock];
  const int t = threadIdx.x;
  const int ch = blockIdx.x * 32 + t % 32;
  float s1 = 0.f, s2 = 0.f;
  if (ch < c) {
    const int g = ch / (c / groups);
    for (long long e = t / 32; e < n * chunks; e += 8) {
      const float* src = part + e * 2 * c + ch;
      s1 += src[0];
      s2 += src[c] * rstd[e / chunks * groups + g];
    }
  }
  l1[t] = s1;
  l2[t] = s2;
  __syncthreads();
  if (t < 32 && ch < c) {
    for (int i = 1; i < 8; ++i) {
      s1 += l1[t + 32 * i];
      s2 += l2[t + 32 * i];
    }
    if (dbias) dbias[ch] = s1;
    if (dweight) dweight[ch] = s2;
  }
}

template <typename T, int VEC, Act ACT>
__global__ __launch_bounds__(kBlock) void gn_bwd_dx_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, Params weight,
    Params bias, const float* __restrict__ drop,
    const float* __restrict__ mean, const float* __restrict__ rstd,
    const float2* __restrict__ k, T* __restrict__ dx, long long hw, int c, int groups,
    int cpb, int ctiles, int chunks, int rows) {
  const Place p = gn_place<VEC>(hw, c, cpb, ctiles, chunks, rows);
  if (!p.in) return;
  float mu[VEC], a[VEC], b[VEC], k0[VEC], k1[VEC];
  const int cpg = c / groups;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const long long s = p.image * groups + (p.c0 + i) / cpg;
    const float r = rstd[s];
    const float2 kk = k[s];
    mu[i] = mean[s];
    a[i] = r * weight.at(p.c0 + i, 1.f);
    b[i] = bias.at(p.c0 + i, 0.f);
    k0[i] = r * kk.x;
    k1[i] = r * kk.y;
  }
  const float keep = drop ? drop[p.image] : 1.f;
  const long long off = p.image * hw * c + p.c0;
  for (long long r = p.r0 + p.rg; r < p.r1; r += p.nrg) {
    const DfdVec<T, VEC> v = dfd_vload<T, VEC>(x + off + r * c);
    const DfdVec<T, VEC> u = dfd_vload<T, VEC>(dy + off + r * c);
    DfdVec<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float d = DfdCvt<T>::to_f32(v.v[i]) - mu[i];
      const float g = DfdCvt<T>::to_f32(u.v[i]) * keep * act_bwd(d * a[i] + b[i], ACT);
      o.v[i] = DfdCvt<T>::from_f32(g * a[i] - k0[i] - d * k1[i]);
    }
    dfd_vstore<T, VEC>(dx + off + r * c, o);
  }
}

#define GN_VEC(VAL, ...)                                    \
  switch (VAL) {                                            \
    case 8: { constexpr int V = 8; __VA_ARGS__; break; }    \
    case 4: { constexpr int V = 4; __VA_ARGS__; break; }    \
    case 2: { constexpr int V = 2; __VA_ARGS__; break; }    \
    default: { constexpr int V = 1; __VA_ARGS__; break; }   \
  }
#define GN_TYPE(VAL, ...)                                            \
  switch (VAL) {                                                     \
    case GnType::kF32: { using T = float; __VA_ARGS__; break; }      \
    case GnType::kBf16: { using T = __hip_bfloat16; __VA_ARGS__; break; } \
    case GnType::kF16: { using T = __half; __VA_ARGS__; break; }     \
  }
#define GN_ACT(VAL, ...)                                                      \
  switch (static_cast<Act>(VAL)) {                                            \
    case Act::kRelu: { constexpr Act A = Act::kRelu; __VA_ARGS__; break; }    \
    case Act::kSilu: { constexpr Act A = Act::kSilu; __VA_ARGS__; break; }    \
    default: { constexpr Act A = Act::kNone; __VA_ARGS__; break; }            \
  }

}  // namespace

long long gn_fwd_ws(const GnArgs& a) { return a.n * gn_plan(a).chunks * a.c * 2; }

long long gn_bwd_ws(const GnArgs& a) {
  return a.n * gn_plan(a).chunks * a.c * 2 + a.n * a.groups * 2;
}

hipError_t gn_fwd(const GnArgs& a, hipStream_t stream) {
  const GnPlan p = gn_plan(a);
  const Params weight = {a.weight, a.ptype}, bias = {a.bias, a.ptype};
  const dim3 grid((unsigned)(a.n * p.chunks * p.ctiles));
  const long long groups = a.n * a.groups;
  const dim3 waves((unsigned)((groups + 3) / 4));
  GN_TYPE(a.type, GN_VEC(p.vec, {
            const T* x = static_cast<const T*>(a.x);
            gn_stats_kernel<T, V><<<grid, kBlock, 0, stream>>>(
                x, reinterpret_cast<float2*>(a.ws), a.hw, a.c, p.cpb, p.ctiles, p.chunks,
                p.rows_per_chunk);
            gn_finalize_kernel<<<waves, kBlock, 0, stream>>>(
                reinterpret_cast<const float2*>(a.ws), a.mean, a.rstd, groups, a.hw, a.c,
                a.groups, p.chunks, p.rows_per_chunk, a.eps);
            GN_ACT(a.act, gn_apply_kernel<T, V, A><<<grid, kBlock, 0, stream>>>(
                              x, weight, bias, static_cast<const T*>(a.residual), a.drop,
                              static_cast<T*>(a.y), a.mean, a.rstd, a.hw, a.c, a.groups, p.cpb,
                              p.ctiles, p.chunks, p.rows_per_chunk));
          }));
  return hipGetLastError();
}

hipError_t gn_bwd(const GnArgs& a, hipStream_t stream) {
  const GnPlan p = gn_plan(a);
  const Params weight = {a.weight, a.ptype}, bias = {a.bias, a.ptype};
  const dim3 grid((unsigned)(a.n * p.chunks * p.ctiles));
  const long long groups = a.n * a.groups;
  const dim3 waves((unsigned)((groups + 3) / 4));
  float2* k = reinterpret_cast<float2*>(a.ws + a.n * p.chunks * a.c * 2);
  GN_TYPE(a.type, GN_VEC(p.vec, GN_ACT(a.act, {
            const T* x = static_cast<const T*>(a.x);
            const T* dy = static_cast<const T*>(a.dy);
            gn_bwd_sums_kernel<T, V, A><<<grid, kBlock, 0, stream>>>(
                dy, x, weight, bias, a.drop, a.mean, a.rstd, a.ws, a.hw, a.c, a.groups,
                p.cpb, p.ctiles, p.chunks, p.rows_per_chunk);
            if (a.dweight || a.dbias)
              gn_bwd_params_kernel<<<dim3((a.c + 31) / 32), kBlock, 0, stream>>>(
                  a.ws, a.rstd, a.dweight, a.dbias, a.n, a.c, a.groups, p.chunks);
            if (a.dx) {
              gn_bwd_group_kernel<<<waves, kBlock, 0, stream>>>(
                  a.ws, weight, a.rstd, k, groups, a.hw, a.c, a.groups, p.chunks);
              gn_bwd_dx_kernel<T, V, A><<<grid, kBlock, 0, stream>>>(
                  dy, x, weight, bias, a.drop, a.mean, a.rstd, k,
                  static_cast<T*>(a.dx), a.hw, a.c, a.groups, p.cpb, p.ctiles, p.chunks,
                  p.rows_per_chunk);
            }
          })));
  return hipGetLastError();
}
