// What the group norm kernels share (group_norm.hip, group_norm_slab.hip).
#pragma once

#include "common.h"
#include "group_norm.h"

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
  template <int N>
  DFD_DEV void load(int i, float otherwise, float (&out)[N]) const {
    if (p == nullptr) {
#pragma unroll
      for (int e = 0; e < N; ++e) out[e] = otherwise;
    } else if (type == GnType::kF32) {
#pragma unroll
      for (int e = 0; e < N; ++e) out[e] = static_cast<const float*>(p)[i + e];
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) out[e] = at(i + e, otherwise);
    }
  }
};

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
  const float w = b.n * __builtin_amdgcn_rcpf(n);
  return {n, a.mean + d * w, a.m2 + b.m2 + d * d * a.n * w};
}

// Values from another lane of a row of 16, and from lane L to all.
template <int CTRL>
DFD_DEV float lane_move(float v) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int L>
DFD_DEV float lane_of(float v) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), L));
}
constexpr int kQuadXor1 = 0xb1, kQuadXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;

// Sums and joins over L lanes, 16 or the whole wave, always in the same order:
// right in the first lane of each L.
template <int L>
DFD_DEV float lanes_sum(float v) {
  v += lane_move<kQuadXor1>(v);
  v += lane_move<kQuadXor2>(v);
  v += lane_move<kHalfMirror>(v);
  v += lane_move<kMirror>(v);
  if constexpr (L == kWave)
    v = (lane_of<0>(v) + lane_of<16>(v)) + (lane_of<32>(v) + lane_of<48>(v));
  return v;
}

template <int CTRL>
DFD_DEV Moments moved(const Moments& m) {
  return {lane_move<CTRL>(m.n), lane_move<CTRL>(m.mean), lane_move<CTRL>(m.m2)};
}
template <int FROM>
DFD_DEV Moments moments_of(const Moments& m) {
  return {lane_of<FROM>(m.n), lane_of<FROM>(m.mean), lane_of<FROM>(m.m2)};
}

template <int L>
DFD_DEV Moments lanes_join(Moments m) {
  m = join(m, moved<kQuadXor1>(m));
  m = join(m, moved<kQuadXor2>(m));
  m = join(m, moved<kHalfMirror>(m));
  m = join(m, moved<kMirror>(m));
  if constexpr (L == kWave)
    m = join(join(moments_of<0>(m), moments_of<16>(m)),
             join(moments_of<32>(m), moments_of<48>(m)));
  return m;
}

// n / d for 0 <= n < 2^21 by one product: the quotient's error, n / d * 2^-22
// at most, is less than the half step of 1 / d that the half keeps it away
// from the next whole number.
DFD_DEV int div_small(int n, float inv_d) { return (int)(((float)n + 0.5f) * inv_d); }

// Two values a column: over the rows of the block's threads, then over each
// group's columns. Either sums, or the mean and the squares about it.
struct Columns {
  static constexpr int NV = 2;
  float* raw;   // [NV][nrg * cols], as the threads wrote them
  float* part;  // [NV][parts * cols]
  float* sums;  // [NV][groups of the slab]
  float* counts;  // [parts]
  int cols, nrg, cpg, groups, parts;  // cpg: columns a group
  float inv_cpg;

  DFD_DEV Columns(float* lds, int cols_, int nrg_, int cpg_)
      : raw(lds), cols(cols_), nrg(nrg_), cpg(cpg_) {
    inv_cpg = 1.f / (float)cpg;
    groups = div_small(cols, inv_cpg);
    parts = div_small(blockDim.x, 1.f / (float)cols);
    if (parts > nrg) parts = nrg;
    if (parts < 1) parts = 1;
    part = raw + NV * nrg * cols;
    sums = part + NV * parts * cols;
    counts = sums + NV * groups;
  }

  // Sums over rows: part[v][p][col].
  DFD_DEV void over_rows() {
    __syncthreads();
    // without a part for each thread the columns are more than the threads
    const int p0 = cols > (int)blockDim.x ? 0 : div_small(threadIdx.x, 1.f / (float)cols);
    if (p0 < parts)
      for (int col = threadIdx.x - p0 * cols; col < cols; col += blockDim.x) {
        float s[NV] = {};
        for (int r = p0; r < nrg; r += parts)
#pragma unroll
          for (int v = 0; v < NV; ++v) s[v] += raw[(v * nrg + r) * cols + col];
#pragma unroll
        for (int v = 0; v < NV; ++v) part[(v * parts + p0) * cols + col] = s[v];
      }
    __syncthreads();
  }

  // The thread's moments of its N channels: n rows, and for each channel the
  // sum a and the squares b about a pivot. One column if `whole`, or else N.
  template <int N>
  DFD_DEV void put(int rg, int slot, bool whole, float n, const float (&pivot)[N],
                   float (&a)[N], float (&b)[N]) {
    const float inv = n > 0.f ? __builtin_amdgcn_rcpf(n) : 0.f;
    float* to = raw + rg * cols;
    const int second = nrg * cols;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float m2 = b[i] - a[i] * a[i] * inv;
      b[i] = m2 < 0.f ? 0.f : m2;  // a NaN stays one
      a[i] = n > 0.f ? pivot[i] + a[i] * inv : 0.f;
    }
    if (whole) {
      float m = a[0], m2 = b[0];
#pragma unroll
      for (int i = 1; i < N; ++i) m += a[i];
      m *= 1.f / N;
#pragma unroll
      for (int i = 1; i < N; ++i) m2 += b[i];
#pragma unroll
      for (int i = 0; i < N; ++i) m2 += n * (a[i] - m) * (a[i] - m);
      to[slot] = m;
      to[second + slot] = m2;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        to[slot * N + i] = a[i];
        to[second + slot * N + i] = b[i];
      }
    }
  }

  // As over_rows, of moments; `each` values a row went into a column, and
  // thread row r of nrg took every nrg-th of hw.
  DFD_DEV float row_count(int r, int hw, int each) const {
    return (float)(div_small(hw - 1 - r + nrg, 1.f / (float)nrg) * each);
  }

  DFD_DEV void join_rows(int hw, int each) {
    __syncthreads();
    const int p0 = cols > (int)blockDim.x ? 0 : div_small(threadIdx.x, 1.f / (float)cols);
    if (p0 < parts)
      for (int col = threadIdx.x - p0 * cols; col < cols; col += blockDim.x) {
        Moments m = {0.f, 0.f, 0.f};
        for (int r = p0; r < nrg; r += parts)
          m = join(m, {row_count(r, hw, each), raw[r * cols + col], raw[(nrg + r) * cols + col]});
        part[p0 * cols + col] = m.mean;
        part[(parts + p0) * cols + col] = m.m2;
        if (col == 0) counts[p0] = m.n;
      }
    __syncthreads();
  }

  // The moments of columns c0 .. c0 + n, by L lanes.
  template <int L>
  DFD_DEV Moments join_columns(int c0, int n) const {
    Moments m = {0.f, 0.f, 0.f};
    const float inv_n = 1.f / (float)n;
    for (int e = threadIdx.x % L; e < parts * n; e += L) {
      const int p = div_small(e, inv_n);
      const int col = c0 + (e - p * n);
      m = join(m, {counts[p], part[p * cols + col], part[(parts + p) * cols + col]});
    }
    return lanes_join<L>(m);
  }

  // Many small groups are taken by 16 lanes each, a few large ones by a wave.
  DFD_DEV bool small_groups(int count) const { return count * kWave > (int)blockDim.x; }

  // sums[0][group] = mean, sums[1][group] = 1 / sqrt(variance + eps).
  template <int L>
  DFD_DEV void join_groups_by(float eps) {
    for (int g = threadIdx.x / L; g < groups; g += blockDim.x / L) {
      const Moments m = join_columns<L>(g * cpg, cpg);
      if (threadIdx.x % L == 0) {
        sums[g] = m.mean;
        sums[groups + g] = rsqrtf(m.m2 / m.n + eps);
      }
    }
  }
  DFD_DEV void join_groups(float eps) {
    if (small_groups(groups)) join_groups_by<16>(eps);
    else join_groups_by<kWave>(eps);
    __syncthreads();
  }

  // Sums over the columns of a group: sums[v][group].
  template <int L, typename W>
  DFD_DEV void over_groups_by(W weight) {
    for (int g = threadIdx.x / L; g < groups; g += blockDim.x / L) {
      float s[NV] = {};
      for (int e = threadIdx.x % L; e < parts * cpg; e += L) {
        const int p = div_small(e, inv_cpg);
        const int col = g * cpg + (e - p * cpg);
        const float w = weight(col);
#pragma unroll
        for (int v = 0; v < NV; ++v) s[v] += w * part[(v * parts + p) * cols + col];
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        s[v] = lanes_sum<L>(s[v]);
        if (threadIdx.x % L == 0) sums[v * groups + g] = s[v];
      }
    }
  }
  template <typename W>
  DFD_DEV void over_groups(W weight) {
    if (small_groups(groups)) over_groups_by<16>(weight);
    else over_groups_by<kWave>(weight);
    __syncthreads();
  }
};

// The bytes of LDS that Columns takes; a partial tile of fewer columns takes no
// more.
static inline int columns_lds(int threads, int nrg, int cols) {
  const int part = threads > cols ? threads : cols;  // at least parts * cols
  return 8 * (nrg * cols + part + cols) + 4 * threads;
}

// The activation and its derivative at z. The sigmoid's reciprocal is one
// instruction, off by one step of fp32; a division costs ten and made the
// streaming kernels wait for arithmetic.
DFD_DEV float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

DFD_DEV float gn_act(float z, Act act) {
  switch (act) {
    case Act::kRelu: return z > 0.f ? z : z != z ? z : 0.f;
    case Act::kSilu: return z * gn_sigmoid(z);
    default: return z;
  }
}

DFD_DEV float gn_act_slope(float z, Act act) {
  switch (act) {
    case Act::kRelu: return z > 0.f ? 1.f : 0.f;
    case Act::kSilu: {
      const float s = gn_sigmoid(z);
      return s * (1.f + z * (1.f - s));
    }
    default: return 1.f;
  }
}

// A store past the caches: they keep what the pass reads again.
template <typename T, int VEC>
DFD_DEV void gn_store_once(T* p, const DfdVec<T, VEC>& x) {
  if constexpr (VEC * sizeof(T) == 16) {
    typedef unsigned Words __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(*reinterpret_cast<const Words*>(&x), reinterpret_cast<Words*>(p));
  } else {
    dfd_vstore<T, VEC>(p, x);
  }
}

// The widest vector of channels, at most 16 bytes, that divides the channels
// and that every tensor's address allows.
static inline int gn_elem(GnType t) { return t == GnType::kF32 ? 4 : 2; }

static inline int gn_vec(const GnArgs& a) {
  const int es = gn_elem(a.type);
  int vec = dfd_pick_vec(a.c, es);
  const void* ptrs[] = {a.x, a.y, a.residual, a.dy, a.dx};
  for (const void* p : ptrs)
    while (vec > 1 && reinterpret_cast<unsigned long long>(p) % (vec * es) != 0) vec >>= 1;
  return vec;
}

#define GN_VEC(VAL, ...)                                    \
  switch (VAL) {                                            \
    case 8: {                                               \
      if constexpr (sizeof(T) == 2) {                       \
        constexpr int V = 8;                                \
        __VA_ARGS__;                                        \
      }                                                     \
      break;                                                \
    }                                                       \
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

