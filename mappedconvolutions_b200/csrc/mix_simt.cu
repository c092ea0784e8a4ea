// Channel mixing on the CUDA cores: products of (pixels, channels) matrices in float32 and float64, any layout, size and
// alignment.
//
// 128 x 128 outputs per block of 256 threads, 8 x 8 per thread (rows and columns in two groups of four, 64 apart), so
// that a thread's two column groups are a gate and its factor where a block holds 64 columns of each.  The operands'
// next slices are in registers while the present ones are multiplied from shared memory.
#include "mix.cuh"

namespace mc {
namespace mix {

constexpr int TM = 128, TN = 128, PITCH = 132;
template <typename T> struct Depth { static constexpr int BK = 16; };
template <> struct Depth<double> { static constexpr int BK = 8; };

template <typename CT>
struct Tile {
  static constexpr int BK = Depth<CT>::BK;
  CT v[2][2][BK][PITCH];  // buffer, operand, slice, row
};

// one slice of an operand: 128 x BK elements, BK / 2 per thread; consecutive threads walk the contiguous direction
template <typename CT, int BK, typename Get>
__device__ __forceinline__ void fetch(CT (&r)[BK / 2], bool kfast, Get get) {
#pragma unroll
  for (int i = 0; i < BK / 2; ++i) {
    const int e = threadIdx.x + 256 * i;
    r[i] = kfast ? get(e / BK, e % BK) : get(e % 128, e / 128);
  }
}
template <typename CT, int BK>
__device__ __forceinline__ void put(CT (*dst)[PITCH], const CT (&r)[BK / 2], bool kfast) {
#pragma unroll
  for (int i = 0; i < BK / 2; ++i) {
    const int e = threadIdx.x + 256 * i;
    if (kfast) dst[e % BK][e / BK] = r[i];
    else dst[e / 128][e % 128] = r[i];
  }
}
template <typename CT, int BK>
__device__ __forceinline__ void multiply(const CT (*a)[PITCH], const CT (*b)[PITCH], CT (&acc)[8][8], int tx, int ty) {
#pragma unroll
  for (int k = 0; k < BK; ++k) {
    CT av[8], bv[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      av[i] = a[k][ty * 4 + i], av[4 + i] = a[k][64 + ty * 4 + i];
      bv[i] = b[k][tx * 4 + i], bv[4 + i] = b[k][64 + tx * 4 + i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] += av[i] * bv[j];
  }
}

template <typename T, int EPI>
__global__ void __launch_bounds__(256) rows_kernel(const RowsArgs a, const PixDiv pd, bool a_kfast, bool w_kfast) {
  typedef typename Traits<T>::CT CT;
  constexpr int BK = Depth<CT>::BK;
  extern __shared__ __align__(16) unsigned char raw[];
  Tile<CT>& sm = *reinterpret_cast<Tile<CT>*>(raw);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const long long p0 = (long long)blockIdx.x * TM;
  constexpr int WIDE = EPI == EPI_GATE ? 64 : 128;  // output columns of a block
  const int n0 = blockIdx.y * WIDE;
  const T* ap = (const T*)a.a.ptr;
  const T* wp = (const T*)a.w;

  int kk = 0;
  const auto load_a = [&](int r, int k) -> CT {
    const long long p = p0 + r;
    if (p >= a.P || kk + k >= a.K) return CT(0);
    uint32_t b, s;
    pd.split((uint32_t)p, b, s);
    return ldv(ap + b * a.a.img + s * a.a.pix + (long long)(kk + k) * a.a.ch);
  };
  const auto load_w = [&](int r, int k) -> CT {
    int n;
    bool in;
    if (EPI == EPI_GATE) {
      n = n0 + (r & 63);
      in = n < a.N;
      n += r >= 64 ? a.N : 0;
    } else {
      n = n0 + r;
      in = n < a.N;
    }
    if (!in || kk + k >= a.K) return CT(0);
    return ldv(wp + (long long)n * a.wn + (long long)(kk + k) * a.wk);
  };

  CT acc[8][8] = {};
  CT ra[BK / 2], rb[BK / 2];
  fetch<CT, BK>(ra, a_kfast, load_a);
  fetch<CT, BK>(rb, w_kfast, load_w);
  int buf = 0;
  for (;;) {
    put<CT, BK>(sm.v[buf][0], ra, a_kfast);
    put<CT, BK>(sm.v[buf][1], rb, w_kfast);
    __syncthreads();
    kk += BK;
    if (kk < a.K) {
      fetch<CT, BK>(ra, a_kfast, load_a);
      fetch<CT, BK>(rb, w_kfast, load_w);
    }
    multiply<CT, BK>(sm.v[buf][0], sm.v[buf][1], acc, tx, ty);
    if (kk >= a.K) break;
    buf ^= 1;
  }

  const T* bias = (const T*)a.bias;
  const T* res = (const T*)a.res.ptr;
  T* y = (T*)a.y.ptr;
  T* z = (T*)a.z.ptr;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long long p = p0 + (i < 4 ? 0 : 60) + ty * 4 + i;
    if (p >= a.P) continue;
    uint32_t b, s;
    pd.split((uint32_t)p, b, s);
    const long long ro = b * a.res.img + s * a.res.pix, yo = b * a.y.img + s * a.y.pix, zo = b * a.z.img + s * a.z.pix;
#pragma unroll
    for (int j = 0; j < (EPI == EPI_GATE ? 4 : 8); ++j) {
      const int n = n0 + (j < 4 ? 0 : 60) + tx * 4 + j;
      if (n >= a.N) continue;
      if (EPI == EPI_LAYER) {
        const CT v = acc[i][j] + (bias ? (CT)ldv(bias + n) : CT(0));
        if (z) stv(z + zo + n * a.z.ch, v);
        CT o = act_value<CT>(a.act, v);
        if (res) o += (CT)ldv(res + ro + n * a.res.ch);
        stv(y + yo + n * a.y.ch, o);
      } else if (EPI == EPI_GATE) {
        const CT g = acc[i][j] + (bias ? (CT)ldv(bias + n) : CT(0));
        const CT u = acc[i][j + 4] + (bias ? (CT)ldv(bias + a.N + n) : CT(0));
        if (z) {
          stv(z + zo + n * a.z.ch, g);
          stv(z + zo + (long long)(a.N + n) * a.z.ch, u);
        }
        stv(y + yo + n * a.y.ch, act_value<CT>(a.act, g) * u);
      } else {
        const CT g = ldv(res + ro + n * a.res.ch), u = ldv(res + ro + (long long)(a.N + n) * a.res.ch);
        stv(y + yo + n * a.y.ch, acc[i][j] * u * act_slope<CT>(a.act, g));
        stv(y + yo + (long long)(a.N + n) * a.y.ch, acc[i][j] * act_value<CT>(a.act, g));
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) outer_kernel(const OuterArgs a, const PixDiv pd, bool g_kfast, bool x_kfast) {
  typedef typename Traits<T>::CT CT;
  constexpr int BK = Depth<CT>::BK;
  extern __shared__ __align__(16) unsigned char raw[];
  Tile<CT>& sm = *reinterpret_cast<Tile<CT>*>(raw);
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int m0 = blockIdx.x * TM, n0 = blockIdx.y * TN;
  const long long begin = blockIdx.z * a.share, end = begin + a.share < a.P ? begin + a.share : a.P;
  const T* gp = (const T*)a.g.ptr;
  const T* xp = (const T*)a.x.ptr;
  long long kk = begin;
  const auto load = [&](const T* base, const View& v, int c, int C, int k) -> CT {
    const long long p = kk + k;
    if (p >= end || c >= C) return CT(0);
    uint32_t b, s;
    pd.split((uint32_t)p, b, s);
    return ldv(base + b * v.img + s * v.pix + c * v.ch);
  };
  const auto load_g = [&](int r, int k) -> CT { return load(gp, a.g, m0 + r, a.M, k); };
  const auto load_x = [&](int r, int k) -> CT { return load(xp, a.x, n0 + r, a.N, k); };
  CT acc[8][8] = {};
  CT col = CT(0);
  CT ra[BK / 2], rb[BK / 2];
  fetch<CT, BK>(ra, g_kfast, load_g);
  fetch<CT, BK>(rb, x_kfast, load_x);
  int buf = 0;
  for (;;) {
    put<CT, BK>(sm.v[buf][0], ra, g_kfast);
    put<CT, BK>(sm.v[buf][1], rb, x_kfast);
    __syncthreads();
    kk += BK;
    if (kk < end) {
      fetch<CT, BK>(ra, g_kfast, load_g);
      fetch<CT, BK>(rb, x_kfast, load_x);
    }
    multiply<CT, BK>(sm.v[buf][0], sm.v[buf][1], acc, tx, ty);
    if (blockIdx.y == 0 && threadIdx.x < 128) {
      CT s = CT(0);
#pragma unroll
      for (int k = 0; k < BK; ++k) s += sm.v[buf][0][k][threadIdx.x];
      col += s;
    }
    if (kk >= end) break;
    buf ^= 1;
  }
  CT* part = (CT*)a.part + (long long)blockIdx.z * a.M * a.N;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int m = m0 + (i < 4 ? 0 : 60) + ty * 4 + i;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = n0 + (j < 4 ? 0 : 60) + tx * 4 + j;
      if (n < a.N) part[(long long)m * a.N + n] = acc[i][j];
    }
  }
  if (blockIdx.y == 0 && threadIdx.x < 128 && m0 + threadIdx.x < a.M)
    ((CT*)a.csum)[(long long)blockIdx.z * a.M + m0 + threadIdx.x] = col;
}

template <typename Kern>
static bool opt_in(Kern kern, size_t smem) {
  return smem <= 48 * 1024 ||
         cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess;
}

template <typename T>
static int rows_typed(Epilogue epi, const RowsArgs& a, cudaStream_t st) {
  typedef typename Traits<T>::CT CT;
  const size_t smem = sizeof(Tile<CT>);
  const int wide = epi == EPI_GATE ? 64 : 128;
  const dim3 grid((unsigned)((a.P + TM - 1) / TM), (unsigned)((a.N + wide - 1) / wide));
  const bool akf = a.a.ch == 1, wkf = a.wk == 1;
  const PixDiv pd((uint32_t)a.S);
#define MC_ROWS(E)                                                     \
  if (!opt_in(rows_kernel<T, E>, smem)) return MC_ERR_LAUNCH;          \
  rows_kernel<T, E><<<grid, 256, smem, st>>>(a, pd, akf, wkf), MC_COUNT(1)
  switch (epi) {
    case EPI_LAYER: MC_ROWS(EPI_LAYER); break;
    case EPI_GATE: MC_ROWS(EPI_GATE); break;
    default: MC_ROWS(EPI_GATE_BWD); break;
  }
#undef MC_ROWS
  MC_CHECK_LAUNCH();
  return MC_OK;
}
int simt_rows_launch(int dtype, Epilogue epi, const RowsArgs& a, cudaStream_t st) {
  return dtype == MC_F64 ? rows_typed<double>(epi, a, st) : rows_typed<float>(epi, a, st);
}

template <typename T>
static int outer_typed(const OuterArgs& a, cudaStream_t st) {
  typedef typename Traits<T>::CT CT;
  const size_t smem = sizeof(Tile<CT>);
  if (!opt_in(outer_kernel<T>, smem)) return MC_ERR_LAUNCH;
  const dim3 grid((a.M + TM - 1) / TM, (a.N + TN - 1) / TN, a.splits);
  outer_kernel<T><<<grid, 256, smem, st>>>(a, PixDiv((uint32_t)a.S), a.g.pix == 1 && a.g.ch != 1,
                                           a.x.pix == 1 && a.x.ch != 1), MC_COUNT(1);
  MC_CHECK_LAUNCH();
  return MC_OK;
}
int simt_outer_launch(int dtype, const OuterArgs& a, cudaStream_t st) {
  return dtype == MC_F64 ? outer_typed<double>(a, st) : outer_typed<float>(a, st);
}

}  // namespace mix
}  // namespace mc
