// Channel mixing on the CUDA cores: products of (pixels, channels) matrices in float32 and float64, any layout, size and
// alignment.
//
// Bound: the FMA units (float32: 148 SMs x 128 per cycle, 72 TFLOP/s at 1.9 GHz).  128 pixels x TN channels per block of
// 256 threads, 8 x TN / 16 per thread from shared memory, which asynchronous copies of single elements fill three slices
// ahead: element by element because nothing promises alignment (an icosphere has 10 * 4^l + 2 vertices, so that a channel
// of an NCHW tensor starts on any multiple of 8 bytes), and because a copy can then land transposed.  A thread's rows lie
// at one distance from each other, so that a copy costs an addition and a comparison.  4 x 128 x 256 pixels in NCHW, 50 -> 99
// channels, SiLU: layer 90 us, input gradient 52 us, weight and bias gradient 64 us (30 - 50 % of the FMA peak, padding
// counted).
#include "mix.cuh"

namespace mc {
namespace mix {

constexpr int TM = 128, STAGES = 3;
template <typename T> struct Depth { static constexpr int BK = 16; };
template <> struct Depth<double> { static constexpr int BK = 8; };

template <typename T, int TN>
struct Slice {  // (pitches: whole 16-byte groups, and rows that start on different banks)
  T a[Depth<T>::BK][TM + 4], b[Depth<T>::BK][TN + 4];
};

template <typename T>
__device__ __forceinline__ void copy_async(T* dst, const T* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
               "n"(sizeof(T)), "r"(there ? (int)sizeof(T) : 0)
               : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_landed() { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory"); }

// One operand's slices of R rows x BK: this thread copies NI elements of each, `step` apart in memory.  Consecutive
// threads walk the contiguous direction.
template <typename T, int R>
struct Stream {
  static constexpr int BK = Depth<T>::BK, NI = R * BK / 256;
  const T *p, *any;      // any: an address that exists
  long long step, next;  // between a thread's elements; from slice to slice
  int r, k, left;        // first element; of its R rows, how many exist
  bool kfast;
  // at(row) + kstride * k is element (row, k)
  template <typename At>
  __device__ Stream(bool kf, int rows, long long rstride, long long kstride, const At& at) : kfast(kf), left(rows) {
    r = kf ? threadIdx.x / BK : threadIdx.x % R;
    k = kf ? threadIdx.x % BK : threadIdx.x / R;
    step = kf ? rstride * (256 / BK) : kstride * (256 / R);
    next = kstride * BK;
    any = at(0);
    p = at(r) + kstride * k;
  }
  // remaining: elements along k from this slice on.  half, jump: rows from `half` on are `jump` elements further away
  template <typename Row>
  __device__ __forceinline__ void fetch(Row* dst, long long remaining, int half, long long jump) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int ri = kfast ? r + 256 / BK * i : r, ki = kfast ? k : k + 256 / R * i;
      const bool up = ri >= half;
      const bool there = ki < remaining && (up ? ri - half : ri) < left;
      copy_async(&dst[ki][ri], there ? p + i * step + (kfast && up ? jump : 0) : any, there);
    }
    p += next;
  }
};

template <typename T, int W>
struct alignas(sizeof(T) * W) Run {
  T v[W];
};

// two accumulators at once: one issue slot for a pair of float32 FMAs
__device__ __forceinline__ void fma_pair(float* acc, float a, const float* b) {
  const float2 av = make_float2(a, a), bv = make_float2(b[0], b[1]);
  float2 c = make_float2(acc[0], acc[1]);
  asm("fma.rn.f32x2 %0, %1, %2, %0;"
      : "+l"(reinterpret_cast<unsigned long long&>(c))
      : "l"(reinterpret_cast<const unsigned long long&>(av)), "l"(reinterpret_cast<const unsigned long long&>(bv)));
  acc[0] = c.x, acc[1] = c.y;
}
__device__ __forceinline__ void fma_pair(double* acc, double a, const double* b) {
  acc[0] += a * b[0], acc[1] += a * b[1];
}

// acc[i][j] += a[k][pixel i] b[k][channel j]; pixels tp * 4 + {0 .. 3} and 64 more, channels tc * W + {0 .. W - 1} and
// TN / 2 more
template <typename T, int TN>
__device__ __forceinline__ void multiply(const Slice<T, TN>& s, T (&acc)[8][TN / 16], int tp, int tc) {
  constexpr int W = TN / 32;
#pragma unroll
  for (int k = 0; k < Depth<T>::BK; ++k) {
    T a[8], b[2 * W];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (sizeof(T) == 4) {
        *reinterpret_cast<Run<T, 4>*>(a + 4 * h) = *reinterpret_cast<const Run<T, 4>*>(&s.a[k][64 * h + 4 * tp]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e += 2)
          *reinterpret_cast<Run<T, 2>*>(a + 4 * h + e) = *reinterpret_cast<const Run<T, 2>*>(&s.a[k][64 * h + 4 * tp + e]);
      }
      constexpr int V = W * sizeof(T) > 16 ? 16 / sizeof(T) : W;
#pragma unroll
      for (int e = 0; e < W; e += V)
        *reinterpret_cast<Run<T, V>*>(b + W * h + e) = *reinterpret_cast<const Run<T, V>*>(&s.b[k][TN / 2 * h + W * tc + e]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 2 * W; j += 2) fma_pair(acc[i] + j, a[i], b + j);
  }
}

// n values of a run; in one access where it is whole and aligned
template <typename T, int W>
__device__ __forceinline__ void store_run(T* p, long long step, const T (&v)[W], int n, bool vec) {
  if (W > 1 && vec && n >= W) {
    constexpr int V = W * sizeof(T) > 16 ? 16 / sizeof(T) : W;
#pragma unroll
    for (int e = 0; e < W; e += V) *reinterpret_cast<Run<T, V>*>(p + e) = *reinterpret_cast<const Run<T, V>*>(v + e);
    return;
  }
#pragma unroll
  for (int e = 0; e < W; ++e)
    if (e < n) p[e * step] = v[e];
}
template <typename T, int W>
__device__ __forceinline__ void load_run(const T* p, long long step, T (&v)[W], int n, bool vec) {
  if (W > 1 && vec && n >= W) {
    constexpr int V = W * sizeof(T) > 16 ? 16 / sizeof(T) : W;
#pragma unroll
    for (int e = 0; e < W; e += V) *reinterpret_cast<Run<T, V>*>(v + e) = *reinterpret_cast<const Run<T, V>*>(p + e);
    return;
  }
#pragma unroll
  for (int e = 0; e < W; ++e) v[e] = e < n ? p[e * step] : T(0);
}

template <typename T, int W>
__device__ __forceinline__ void act_run(int act, const T (&v)[W], T (&o)[W]) {
  Values<T, W> z;
#pragma unroll
  for (int e = 0; e < W; ++e) z.v[e] = v[e];
  if (act) z = act_value_call<T, W>(act, z);
#pragma unroll
  for (int e = 0; e < W; ++e) o[e] = z.v[e];
}

struct RowsFlags {
  bool a_kfast, w_kfast;   // which direction of a and w is contiguous
  bool vec_y, vec_z, vec_r;  // runs of y, z, res are aligned (see aligned_runs)
};

// PIX: consecutive threads hold consecutive pixels (outputs in NCHW) instead of channels.
template <typename T, int EPI, int TN, bool PIX>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 1) rows_kernel(const RowsArgs a, const PixDiv pd, const RowsFlags f) {
  constexpr int BK = Depth<T>::BK, W = TN / 32;
  extern __shared__ __align__(16) unsigned char raw[];
  Slice<T, TN>* sm = reinterpret_cast<Slice<T, TN>*>(raw);
  const int tp = PIX ? threadIdx.x % 16 : threadIdx.x / 16, tc = PIX ? threadIdx.x / 16 : threadIdx.x % 16;
  const long long p0 = (long long)blockIdx.x * TM;
  constexpr int WIDE = EPI == EPI_GATE ? TN / 2 : TN;  // output channels of a block
  const int n0 = blockIdx.y * WIDE;
  const int pixels = a.P - p0 < TM ? (int)(a.P - p0) : TM, channels = a.N - n0 < WIDE ? a.N - n0 : WIDE;

  // (rows of a that are contiguous along k lie pix apart across images too: img = S * pix)
  Stream<T, TM> sa(f.a_kfast, pixels, a.a.pix, a.a.ch, [&](int r) {
    uint32_t b, s;
    pd.split((uint32_t)(p0 + (r < pixels ? r : 0)), b, s);
    return (const T*)a.a.ptr + b * a.a.img + s * a.a.pix;
  });
  // rows of a gate's block: TN / 2 of the gate, TN / 2 of its factor N rows further down
  constexpr int HALF = EPI == EPI_GATE ? TN / 2 : 1 << 20;
  Stream<T, TN> sw(f.w_kfast, channels, a.wn, a.wk, [&](int r) {
    long long n = r;
    if (EPI == EPI_GATE && !f.w_kfast && r >= HALF) n += a.N - HALF;
    return (const T*)a.w + (n0 + n) * a.wn;
  });
  const long long jump = EPI == EPI_GATE ? (long long)(a.N - HALF) * a.wn : 0;

  T acc[8][2 * W] = {};
  const int slices = (a.K + BK - 1) / BK;
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (i < slices) {
      sa.fetch(sm[i].a, a.K - i * BK, 1 << 20, 0);
      sw.fetch(sm[i].b, a.K - i * BK, HALF, jump);
    }
    copies_issued();
  }
  for (int i = 0; i < slices; ++i) {
    copies_landed();
    __syncthreads();  // (everybody's copies, and everybody is done with the slice that is overwritten next)
    const int n = i + STAGES - 1;
    if (n < slices) {
      sa.fetch(sm[n % STAGES].a, a.K - n * BK, 1 << 20, 0);
      sw.fetch(sm[n % STAGES].b, a.K - n * BK, HALF, jump);
    }
    copies_issued();
    multiply<T, TN>(sm[i % STAGES], acc, tp, tc);
  }

  const T* bias = (const T*)a.bias;
  const T* res = (const T*)a.res.ptr;
  T* y = (T*)a.y.ptr;
  T* z = (T*)a.z.ptr;
  if (EPI == EPI_LAYER && PIX) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r0 = 64 * h + 4 * tp;
      uint32_t b, s;
      pd.split((uint32_t)(p0 + (r0 < pixels ? r0 : 0)), b, s);
      // four pixels of one image at once, or one by one where an image or the tensor ends
      const bool whole = r0 + 4 <= pixels && s + 4 <= pd.S;
#pragma unroll
      for (int j = 0; j < 2 * W; ++j) {
        const int n = j / W * (TN / 2) + W * tc + j % W;
        if (n >= channels) continue;
        const T bj = bias ? bias[n0 + n] : T(0);
        T v[4], o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[4 * h + e][j] + bj;
        act_run(a.act, v, o);
        if (whole) {
          const long long c = n0 + n;
          if (z) store_run(z + b * a.z.img + s * a.z.pix + c * a.z.ch, a.z.pix, v, 4, f.vec_z);
          if (res) {
            T q[4];
            load_run(res + b * a.res.img + s * a.res.pix + c * a.res.ch, a.res.pix, q, 4, f.vec_r);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += q[e];
          }
          store_run(y + b * a.y.img + s * a.y.pix + c * a.y.ch, a.y.pix, o, 4, f.vec_y);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (r0 + e >= pixels) continue;
            uint32_t be, se;
            pd.split((uint32_t)(p0 + r0 + e), be, se);
            const long long c = n0 + n;
            if (z) z[be * a.z.img + se * a.z.pix + c * a.z.ch] = v[e];
            if (res) o[e] += res[be * a.res.img + se * a.res.pix + c * a.res.ch];
            y[be * a.y.img + se * a.y.pix + c * a.y.ch] = o[e];
          }
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i / 4 * 64 + 4 * tp + i % 4;
    if (r >= pixels) continue;
    uint32_t b, s;
    pd.split((uint32_t)(p0 + r), b, s);
    const T* rr = res + b * a.res.img + s * a.res.pix;
    T *yr = y + b * a.y.img + s * a.y.pix, *zr = z + b * a.z.img + s * a.z.pix;
#pragma unroll
    for (int h = 0; h < (EPI == EPI_GATE ? 1 : 2); ++h) {
      const int n = TN / 2 * h + W * tc, left = channels - n;
      if (left <= 0) continue;
      const long long c = n0 + n;
      T v[W], o[W];
      if (EPI == EPI_LAYER) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          v[e] = acc[i][W * h + e] + (bias && e < left ? bias[c + e] : T(0));
        }
        act_run(a.act, v, o);
        if (z) store_run(zr + c * a.z.ch, a.z.ch, v, left, f.vec_z);
        if (res) {
          T q[W];
          load_run(rr + c * a.res.ch, a.res.ch, q, left, f.vec_r);
#pragma unroll
          for (int e = 0; e < W; ++e) o[e] += q[e];
        }
        store_run(yr + c * a.y.ch, a.y.ch, o, left, f.vec_y);
      } else if (EPI == EPI_GATE) {
        T u[W];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          v[e] = acc[i][e] + (bias && e < left ? bias[c + e] : T(0));
          u[e] = acc[i][W + e] + (bias && e < left ? bias[a.N + c + e] : T(0));
        }
        act_run(a.act, v, o);
#pragma unroll
        for (int e = 0; e < W; ++e) o[e] *= u[e];
        if (z) {
          store_run(zr + c * a.z.ch, a.z.ch, v, left, f.vec_z);
          store_run(zr + (a.N + c) * a.z.ch, a.z.ch, u, left, f.vec_z);
        }
        store_run(yr + c * a.y.ch, a.y.ch, o, left, f.vec_y);
      } else {
        T g[W], u[W];
        load_run(rr + c * a.res.ch, a.res.ch, g, left, f.vec_r);
        load_run(rr + (a.N + c) * a.res.ch, a.res.ch, u, left, f.vec_r);
        Values<T, W> z;
#pragma unroll
        for (int e = 0; e < W; ++e) z.v[e] = g[e];
        const ActBoth<T, W> both = act_both_call<T, W>(a.act, z);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          v[e] = acc[i][W * h + e] * u[e] * both.slope.v[e];
          o[e] = acc[i][W * h + e] * both.value.v[e];
        }
        store_run(yr + c * a.y.ch, a.y.ch, v, left, f.vec_y);
        store_run(yr + (a.N + c) * a.y.ch, a.y.ch, o, left, f.vec_y);
      }
    }
  }
}

// Block (m tile, n tile, share).
template <typename T, int TN>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 1) outer_kernel(const OuterArgs a) {
  constexpr int BK = Depth<T>::BK, W = TN / 32;
  extern __shared__ __align__(16) unsigned char raw[];
  Slice<T, TN>* sm = reinterpret_cast<Slice<T, TN>*>(raw);
  const int tp = threadIdx.x / 16, tc = threadIdx.x % 16;
  const int m0 = blockIdx.x * TM, n0 = blockIdx.y * TN;
  const int first = blockIdx.z / a.per_image * a.group, last = first + a.group < a.B ? first + a.group : a.B;
  const long long begin = blockIdx.z % a.per_image * a.share;
  const long long len = a.S - begin < a.share ? a.S - begin : a.share;
  const int rows = a.M - m0 < TM ? a.M - m0 : TM, cols = a.N - n0 < TN ? a.N - n0 : TN;
  const int slices = (int)((len + BK - 1) / BK);
  T acc[8][2 * W] = {};
  T col = T(0);
  for (int image = first; image < last; ++image) {
    Stream<T, TM> sg(a.g.pix == 1 && a.g.ch != 1, rows, a.g.ch, a.g.pix, [&](int r) {
      return (const T*)a.g.ptr + image * a.g.img + begin * a.g.pix + (m0 + (r < rows ? r : 0)) * a.g.ch;
    });
    Stream<T, TN> sx(a.x.pix == 1 && a.x.ch != 1, cols, a.x.ch, a.x.pix, [&](int r) {
      return (const T*)a.x.ptr + image * a.x.img + begin * a.x.pix + (n0 + (r < cols ? r : 0)) * a.x.ch;
    });
    __syncthreads();
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      if (i < slices) {
        sg.fetch(sm[i].a, len - i * BK, 1 << 20, 0);
        sx.fetch(sm[i].b, len - i * BK, 1 << 20, 0);
      }
      copies_issued();
    }
    for (int i = 0; i < slices; ++i) {
      copies_landed();
      __syncthreads();
      const int n = i + STAGES - 1;
      if (n < slices) {
        sg.fetch(sm[n % STAGES].a, len - (long long)n * BK, 1 << 20, 0);
        sx.fetch(sm[n % STAGES].b, len - (long long)n * BK, 1 << 20, 0);
      }
      copies_issued();
      multiply<T, TN>(sm[i % STAGES], acc, tp, tc);
      if (blockIdx.y == 0 && threadIdx.x < TM) {
        T s = T(0);
#pragma unroll
        for (int k = 0; k < BK; ++k) s += sm[i % STAGES].a[k][threadIdx.x];
        col += s;
      }
    }
  }
  T* part = (T*)a.part + (long long)blockIdx.z * a.M * a.N;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int m = i / 4 * 64 + 4 * tp + i % 4;
    if (m >= rows) continue;
#pragma unroll
    for (int j = 0; j < 2 * W; ++j) {
      const int n = j / W * (TN / 2) + W * tc + j % W;
      if (n < cols) part[(long long)(m0 + m) * a.N + n0 + n] = acc[i][j];
    }
  }
  if (blockIdx.y == 0 && threadIdx.x < rows) ((T*)a.csum)[(long long)blockIdx.z * a.M + m0 + threadIdx.x] = col;
}

template <typename Kern>
static bool opt_in(Kern kern, size_t smem) {
  return smem <= 48 * 1024 ||
         cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess;
}

// Runs of W elements along the contiguous direction start on multiples of their size: the base, and every stride that
// leads to a run.
template <typename T>
static bool aligned_runs(const View& v, int W, bool pix, long long other) {
  const long long run = W * sizeof(T) > 16 ? 16 / sizeof(T) : W;
  const long long c = pix ? v.pix : v.ch, s = pix ? v.ch : v.pix;
  return c == 1 && s % run == 0 && v.img % run == 0 && other % run == 0 && ((uintptr_t)v.ptr & (run * sizeof(T) - 1)) == 0;
}

template <typename T, int EPI, int TN, bool PIX>
static int rows_go(const RowsArgs& a, cudaStream_t st) {
  const size_t smem = STAGES * sizeof(Slice<T, TN>);
  const int wide = EPI == EPI_GATE ? TN / 2 : TN, W = TN / 32;
  const dim3 grid((unsigned)((a.P + TM - 1) / TM), (unsigned)((a.N + wide - 1) / wide));
  // runs: four pixels of an image that starts anywhere, or W channels (gate: of both halves of 2 N)
  const long long other = PIX ? a.S : EPI == EPI_LAYER ? 0 : a.N;
  const RowsFlags f{a.a.ch == 1, a.wk == 1, aligned_runs<T>(a.y, PIX ? 4 : W, PIX, other),
                    aligned_runs<T>(a.z, PIX ? 4 : W, PIX, other), aligned_runs<T>(a.res, PIX ? 4 : W, PIX, other)};
  if (!opt_in(rows_kernel<T, EPI, TN, PIX>, smem)) return MC_ERR_LAUNCH;
  rows_kernel<T, EPI, TN, PIX><<<grid, 256, smem, st>>>(a, PixDiv((uint32_t)a.S), f), MC_COUNT(1);
  MC_CHECK_LAUNCH();
  return MC_OK;
}
template <typename T, int EPI, bool PIX>
static int rows_width(const RowsArgs& a, cudaStream_t st) {
  // The width that pads least, the widest of equals.  (128: an FMA per 1.1 bytes from shared memory, 32: per 2.5.)
  const int n = EPI == EPI_GATE ? 2 * a.N : a.N;
  const auto padded = [&](int w) { return (n + w - 1) / w * w; };
  if (padded(128) <= padded(64)) return rows_go<T, EPI, 128, PIX>(a, st);
  if (padded(64) <= padded(32)) return rows_go<T, EPI, 64, PIX>(a, st);
  return rows_go<T, EPI, 32, PIX>(a, st);
}
template <typename T>
static int rows_typed(Epilogue epi, const RowsArgs& a, cudaStream_t st) {
  switch (epi) {
    case EPI_LAYER:
      return a.y.pix == 1 && a.y.ch != 1 ? rows_width<T, EPI_LAYER, true>(a, st) : rows_width<T, EPI_LAYER, false>(a, st);
    case EPI_GATE: return rows_width<T, EPI_GATE, false>(a, st);
    default: return rows_width<T, EPI_GATE_BWD, false>(a, st);
  }
}
int simt_rows_launch(int dtype, Epilogue epi, const RowsArgs& a, cudaStream_t st) {
  return dtype == MC_F64 ? rows_typed<double>(epi, a, st) : rows_typed<float>(epi, a, st);
}

template <typename T, int TN>
static int outer_go(const OuterArgs& a, cudaStream_t st) {
  const size_t smem = STAGES * sizeof(Slice<T, TN>);
  if (!opt_in(outer_kernel<T, TN>, smem)) return MC_ERR_LAUNCH;
  const dim3 grid((a.M + TM - 1) / TM, (a.N + TN - 1) / TN, a.splits);
  outer_kernel<T, TN><<<grid, 256, smem, st>>>(a), MC_COUNT(1);
  MC_CHECK_LAUNCH();
  return MC_OK;
}
template <typename T>
static int outer_typed(const OuterArgs& a, cudaStream_t st) {
  const auto padded = [&](int w) { return (a.N + w - 1) / w * w; };
  if (padded(128) <= padded(64)) return outer_go<T, 128>(a, st);
  if (padded(64) <= padded(32)) return outer_go<T, 64>(a, st);
  return outer_go<T, 32>(a, st);
}
int simt_outer_launch(int dtype, const OuterArgs& a, cudaStream_t st) {
  return dtype == MC_F64 ? outer_typed<double>(a, st) : outer_typed<float>(a, st);
}

}  // namespace mix
}  // namespace mc
