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

// (count, mean, sum of squares about the mean) of a set of values: sets can be
// put together without losing anything to a large common offset, as plain sums
// of squares would.
struct Moments {
  float n, mean, m2;
};

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

// The sum over L lanes (1, 16 or the wave), the same bits in each of them.
template <int L>
DFD_DEV float lanes_sum(float v) {
  if constexpr (L > 1) {
    v += lane_move<kQuadXor1>(v);
    v += lane_move<kQuadXor2>(v);
    v += lane_move<kHalfMirror>(v);
    v += lane_move<kMirror>(v);
  }
  if constexpr (L == kWave)
    v = (lane_of<0>(v) + lane_of<16>(v)) + (lane_of<32>(v) + lane_of<48>(v));
  return v;
}

// The moments of n sets together, get(0) .. get(n - 1), by L lanes: the mean
// first and the squares about it after, where what rounding left the mean
// beside the true one is seen and taken out. Two short loops of sums are
// faster than one of joins, each of which waits for the one before.
template <int L, typename F>
DFD_DEV Moments gather(int n, F get) {
  const int lane = L > 1 ? threadIdx.x % L : 0;
  float cnt = 0.f, sum = 0.f;
  for (int e = lane; e < n; e += L) {
    const Moments m = get(e);
    cnt += m.n;
    sum += m.n * m.mean;
  }
  cnt = lanes_sum<L>(cnt);
  const float inv = cnt > 0.f ? __builtin_amdgcn_rcpf(cnt) : 0.f;
  const float mean = lanes_sum<L>(sum) * inv;
  float by = 0.f, m2 = 0.f;
  for (int e = lane; e < n; e += L) {
    const Moments m = get(e);
    const float d = m.mean - mean;
    by += m.n * d;
    m2 += m.m2 + m.n * d * d;
  }
  by = lanes_sum<L>(by);
  m2 = lanes_sum<L>(m2) - by * by * inv;
  return {cnt, mean + by * inv, m2 < 0.f ? 0.f : m2};  // a NaN stays one
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
    part = raw + NV * (nrg * cols > 32 ? nrg * cols : 32);
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
    // the first `longer` of the threads' rows took `most` rows, the others one less
    const int most = div_small(hw - 1 + nrg, 1.f / (float)nrg);
    const int longer = hw - (most - 1) * nrg;
    const float inv_parts = 1.f / (float)parts;
    __syncthreads();
    const int p0 = cols > (int)blockDim.x ? 0 : div_small(threadIdx.x, 1.f / (float)cols);
    if (p0 < parts)
      for (int col = threadIdx.x - p0 * cols; col < cols; col += blockDim.x) {
        const Moments m = gather<1>(div_small(nrg - 1 - p0 + parts, inv_parts), [&](int e) {
          const int r = p0 + e * parts;
          const float n = (float)((r < longer ? most : most - 1) * each);
          return Moments{n, raw[r * cols + col], raw[(nrg + r) * cols + col]};
        });
        part[p0 * cols + col] = m.mean;
        part[(parts + p0) * cols + col] = m.m2;
        if (col == 0) counts[p0] = m.n;
      }
    __syncthreads();
  }

  // The moments of columns c0 .. c0 + n, by L lanes; of `of` waves that share
  // the work, the one numbered `wave`.
  template <int L>
  DFD_DEV Moments join_columns(int c0, int n, int wave = 0, int of = 1) const {
    const float inv_n = 1.f / (float)n;
    const int all = parts * n;
    const int each = of == 1 ? all : (all + of - 1) / of;  // a wave's entries
    const int from = wave * each;
    const int count = all - from < each ? all - from : each;
    return gather<L>(count, [&](int i) {
      const int e = from + i;
      const int p = div_small(e, inv_n);
      const int col = c0 + (e - p * n);
      return Moments{counts[p], part[p * cols + col], part[(parts + p) * cols + col]};
    });
  }

  // Many small groups are taken by 16 lanes each, a few large ones by a wave
  // each or by several.
  DFD_DEV bool small_groups(int count) const { return count * kWave > (int)blockDim.x; }
  DFD_DEV int waves_a_group() const {
    const int w = (int)(blockDim.x / kWave) / groups;
    return w < 1 ? 1 : w;
  }

  // sums[0][group] = mean, sums[1][group] = 1 / sqrt(variance + eps).
  DFD_DEV void join_groups(float eps) {
    auto store = [&](int g, const Moments& m) {
      sums[g] = m.mean;
      sums[groups + g] = rsqrtf(m.m2 * __builtin_amdgcn_rcpf(m.n) + eps);
    };
    if (small_groups(groups)) {
      for (int g = threadIdx.x / 16; g < groups; g += blockDim.x / 16) {
        const Moments m = join_columns<16>(g * cpg, cpg);
        if (threadIdx.x % 16 == 0) store(g, m);
      }
    } else {
      const int per = waves_a_group();
      const int g = threadIdx.x / kWave / per, w = threadIdx.x / kWave - g * per;
      if (g < groups) {
        const Moments m = join_columns<kWave>(g * cpg, cpg, w, per);
        if (threadIdx.x % kWave == 0) {
          if (per == 1) {
            store(g, m);
          } else {
            float* to = raw + 3 * (g * per + w);  // the rows' sums have been read
            to[0] = m.n;
            to[1] = m.mean;
            to[2] = m.m2;
          }
        }
      }
      if (per > 1) {
        __syncthreads();
        const int h = threadIdx.x / 16;
        if (h < groups) {
          const Moments m = gather<16>(per, [&](int e) {
            const float* from = raw + 3 * (h * per + e);
            return Moments{from[0], from[1], from[2]};
          });
          if (threadIdx.x % 16 == 0) store(h, m);
        }
      }
    }
    __syncthreads();
  }

  // Sums over the columns of a group, weighted: sums[v][group].
  template <int L, typename W>
  DFD_DEV void group_sum(int g, int wave, int of, W weight, float (&s)[NV]) const {
    const int all = parts * cpg;
    const int each = of == 1 ? all : (all + of - 1) / of;
    const int end = (wave + 1) * each < all ? (wave + 1) * each : all;
    for (int e = wave * each + threadIdx.x % L; e < end; e += L) {
      const int p = div_small(e, inv_cpg);
      const int col = g * cpg + (e - p * cpg);
      const float w = weight(col);
#pragma unroll
      for (int v = 0; v < NV; ++v) s[v] += w * part[(v * parts + p) * cols + col];
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) s[v] = lanes_sum<L>(s[v]);
  }

  template <typename W>
  DFD_DEV void over_groups(W weight) {
    if (small_groups(groups)) {
      for (int g = threadIdx.x / 16; g < groups; g += blockDim.x / 16) {
        float s[NV] = {};
        group_sum<16>(g, 0, 1, weight, s);
        if (threadIdx.x % 16 == 0)
#pragma unroll
          for (int v = 0; v < NV; ++v) sums[v * groups + g] = s[v];
      }
    } else {
      const int per = waves_a_group();
      const int g = threadIdx.x / kWave / per, w = threadIdx.x / kWave - g * per;
      if (g < groups) {
        float s[NV] = {};
        group_sum<kWave>(g, w, per, weight, s);
        if (threadIdx.x % kWave == 0)
#pragma unroll
          for (int v = 0; v < NV; ++v) (per == 1 ? sums[v * groups + g] : raw[NV * (g * per + w) + v]) = s[v];
      }
      if (per > 1) {
        __syncthreads();  // raw: the rows' sums have been read
        if ((int)threadIdx.x < groups)
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            float s = 0.f;
            for (int e = 0; e < per; ++e) s += raw[NV * (threadIdx.x * per + e) + v];
            sums[v * groups + threadIdx.x] = s;
          }
      }
    }
    __syncthreads();
  }
};

// The bytes of LDS that Columns takes; a partial tile of fewer columns takes no
// more.
static inline int columns_lds(int threads, int nrg, int cols) {
  const int part = threads > cols ? threads : cols;  // at least parts * cols
  const int raw = nrg * cols > 32 ? nrg * cols : 32;  // also what 16 waves share
  return 8 * (raw + part + cols) + 4 * threads;
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

// The widest vector of channels, at most 16 bytes, that divides the channels
// and that every tensor's address allows.
static inline int gn_elem(GnType t) { return t == GnType::kF32 ? 4 : 2; }

static inline bool gn_too_many(long long blocks, int threads) {
  return blocks * threads >= 1ll << 32;
}

static inline int gcd_of(int a, int b) { return b ? gcd_of(b, a % b) : a; }

static inline bool gn_aligned(const GnArgs& a, int vec) {
  const void* ptrs[] = {a.x, a.y, a.residual, a.dy, a.dx};
  for (const void* p : ptrs)
    if (reinterpret_cast<unsigned long long>(p) % (vec * gn_elem(a.type)) != 0) return false;
  return true;
}

static inline int gn_vec(const GnArgs& a) {
  int vec = dfd_pick_vec(a.c, gn_elem(a.type));
  while (vec > 1 && !gn_aligned(a, vec)) vec >>= 1;
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

