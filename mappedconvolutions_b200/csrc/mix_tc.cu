// Channel mixing on the tensor cores (bf16 operands, float32 sums in TMEM).
//
// rows kernel:  tiles of 128 pixels x BN channels.  One warp fetches operand tiles by TMA, one thread issues the MMAs into
// two accumulator sets in turn.  Each set has four read-out warps of its own (a tile's latencies - TMEM loads, elementary
// functions, hand-over of the staged tiles - overlap with the other set's), which apply the epilogue and leave bf16 tiles
// in shared memory, from where an I/O thread stores them by TMA; the same slots receive the tiles that an epilogue adds
// or multiplies (residual, grad_output) beforehand.  Where all weights that a block needs fit beside the rings they stay
// in shared memory and the block keeps its channel tile; otherwise they travel with the pixels.
//
// outer kernel: parameter gradients, both operands read along the pixels (MN-major); every block sums a share of the
// pixels for one tile of the gradient and writes float32 partial sums, which are added in order afterwards.  The eight
// read-out warps, idle meanwhile, sum the columns of the first operand in shared memory (the bias gradient).
#include <cuda.h>

#include "mix.cuh"
#include "tc_common.cuh"

namespace mc {
namespace mix {
using namespace tc;

constexpr int TILE = 128;       // pixels per tile
constexpr int KB = 64;          // channels per pipeline stage: one 128-byte swizzle row
constexpr int A_BYTES = TILE * KB * 2;
constexpr int THREADS = 384;    // loader, MMA, two I/O warps, eight read-out warps
constexpr int MAX_STAGES = 12;
constexpr int CH_BYTES = TILE * 64 * 2;  // a staged tile
constexpr int SMEM_LIMIT = 226 * 1024;  // of 227 KB, the rest is static

// ---- activations: fast forms, relative error below 2^-16 (half a bf16 step is 2^-9), two values at a time -----------------
// (packed float32 instructions: the read-out warps are short of issue slots, not of arithmetic)
__device__ __forceinline__ unsigned long long& bits(float2& v) { return reinterpret_cast<unsigned long long&>(v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(bits(d)) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(bits(d)) : "l"(bits(a)), "l"(bits(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(bits(d)) : "l"(bits(a)), "l"(bits(b)));
  return d;
}
__device__ __forceinline__ float2 two(float v) { return make_float2(v, v); }
__device__ __forceinline__ float rcp_(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float exp2_(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float2 rcp2(float2 v) { return make_float2(rcp_(v.x), rcp_(v.y)); }
__device__ __forceinline__ float2 exp2_2(float2 v) { return make_float2(exp2_(v.x), exp2_(v.y)); }
// 1 / (1 + 2^v): the logistic function of z for v = -z log2(e)
__device__ __forceinline__ float2 logistic2(float2 v) { return rcp2(add2(exp2_2(v), two(1.f))); }
constexpr float LOG2E = 1.44269504f;
struct ActNone {
  __device__ static float2 value(float2 z) { return z; }
  __device__ static void both(float2 z, float2& v, float2& s) { v = z, s = two(1.f); }
};
struct ActRelu {
  __device__ static float value1(float z) { return z < 0.f ? 0.f : z; }  // (NaN stays NaN)
  __device__ static float slope1(float z) { return z > 0.f ? 1.f : (z == z ? 0.f : z); }
  __device__ static float2 value(float2 z) { return make_float2(value1(z.x), value1(z.y)); }
  __device__ static void both(float2 z, float2& v, float2& s) {
    v = value(z), s = make_float2(slope1(z.x), slope1(z.y));
  }
};
struct ActGelu {
  // Phi(z), and e = exp(-z^2 / 2).  With x = |z| / sqrt(2), t = 1 / (1 + 0.44 x): exp(x^2) erfc(x) / 2 = t q(t), q a
  // least-squares fit of the relative error over x in [0, 10] (at most 5.2e-6; e alone decays beyond).
  __device__ static float2 phi(float2 z, float2& e) {
    const float2 t = rcp2(fma2(two(0.31112698f), make_float2(fabsf(z.x), fabsf(z.y)), two(1.f)));
    e = exp2_2(mul2(mul2(z, two(-0.5f * LOG2E)), z));
    float2 q = fma2(two(-0.07305045425891876f), t, two(0.1753196418285370f));
    q = fma2(q, t, two(0.020372465252876282f));
    q = fma2(q, t, two(0.1317897737026215f));
    q = fma2(q, t, two(0.12128554284572601f));
    q = fma2(q, t, two(0.12428044527769089f));
    const float2 c = mul2(mul2(q, t), e), d = fma2(c, two(-1.f), two(1.f));
    return make_float2(z.x < 0.f ? c.x : d.x, z.y < 0.f ? c.y : d.y);
  }
  __device__ static float2 value(float2 z) {
    float2 e;
    return mul2(z, phi(z, e));
  }
  __device__ static void both(float2 z, float2& v, float2& s) {
    float2 e;
    const float2 p = phi(z, e);
    v = mul2(z, p);
    s = fma2(mul2(z, two(0.39894228f)), e, p);
  }
};
struct ActGeluTanh {  // (1 + tanh(a)) / 2 is the logistic function of 2 a
  __device__ static float2 part(float2 z) {
    return logistic2(mul2(mul2(z, two(-1.59576912f * LOG2E)), fma2(mul2(z, two(0.044715f)), z, two(1.f))));
  }
  __device__ static float2 value(float2 z) { return mul2(z, part(z)); }
  __device__ static void both(float2 z, float2& v, float2& s) {
    const float2 p = part(z);
    v = mul2(z, p);
    s = fma2(mul2(v, fma2(p, two(-1.f), two(1.f))), fma2(mul2(z, two(1.59576912f * 0.134145f)), z, two(1.59576912f)), p);
  }
};
struct ActSilu {
  __device__ static float2 value(float2 z) { return mul2(z, logistic2(mul2(z, two(-LOG2E)))); }
  __device__ static void both(float2 z, float2& v, float2& s) {
    const float2 p = logistic2(mul2(z, two(-LOG2E)));
    v = mul2(z, p);
    s = fma2(v, fma2(p, two(-1.f), two(1.f)), p);
  }
};
struct ActSigmoid {
  __device__ static float2 value(float2 z) { return logistic2(mul2(z, two(-LOG2E))); }
  __device__ static void both(float2 z, float2& v, float2& s) {
    v = value(z), s = mul2(v, fma2(v, two(-1.f), two(1.f)));
  }
};
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {  // one branch per 32 columns, not per value
  switch (act) {
    case MC_ACT_RELU: f(ActRelu()); break;
    case MC_ACT_GELU: f(ActGelu()); break;
    case MC_ACT_GELU_TANH: f(ActGeluTanh()); break;
    case MC_ACT_SILU: f(ActSilu()); break;
    case MC_ACT_SIGMOID: f(ActSigmoid()); break;
    default: f(ActNone()); break;
  }
}

template <int N>
__device__ __forceinline__ float2 pair_of(const uint32_t (&v)[N], int j) {
  return make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
}
__device__ __forceinline__ float2 bias2(const float* b, int j) { return reinterpret_cast<const float2*>(b)[j]; }

// ---- TMA ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"((uint64_t)tm), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* tm, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"((uint64_t)tm), "r"(x),
               "r"(y), "r"(src)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  int ok = 1;
  if (threadIdx.x % 32 == 0) ok = mbar_wait(bar, parity, abort_flag, code) ? 1 : 0;
  return __shfl_sync(~0u, ok, 0) != 0;
}

// ---- rows kernel ---------------------------------------------------------------------------------------
enum Mode {
  LAYER = 0,     // y = act(A B^T + bias) + r; two A B^T pairs can be summed
  GATE = 1,      // y = act(g) u, [g|u] = A B^T + bias: rows n and N + n of B
  GATE_BWD = 2,  // [g|u] as above from the first operands, gh from the second: y0 = gh u act'(g), y1 = gh act(g)
  ACT_BWD = 3    // y = r act'(A B^T + bias)
};
// BN: channels of a tile; it is staged 64 channels (128 swizzled bytes a row) at a time.
template <int MODE, int BN> struct Cfg {
  static constexpr int N0 = MODE == GATE || MODE == GATE_BWD ? 2 * BN : BN;  // columns of the first product
  static constexpr int N1 = MODE == GATE_BWD ? BN : N0;                      // and of the second
  static constexpr int OFF1 = MODE == GATE_BWD ? N0 : 0;                     // its first accumulator column
  static constexpr int NCH = MODE == GATE_BWD ? 2 : BN / 64;                 // staged tiles
  static constexpr int BMAX = (N0 > N1 ? N0 : N1) * KB * 2;
};

struct alignas(64) GemmArgs {
  CUtensorMap a[2], b[2], r, y[2];
  const bf16* bias;  // null: none
  int m_tiles, n_tiles, N, kb[2], act;
  int up;            // distance between a gate's row of b[0] and bias and its factor's
  int res;           // r is read
  int resident, stages, slots;
};

constexpr int ROWS_BARS = 2 * MAX_STAGES + 1 + 4 + 8 + 1 + 2;

struct TileWalk {  // this block's tiles
  long long t, step, end;
  int n_tiles, n;
  bool fixed;
  // from the `first`-th tile on, every `every`-th one
  __device__ TileWalk(const GemmArgs& a, int first = 0, int every = 1) : n_tiles(a.n_tiles), fixed(a.resident) {
    if (fixed) {
      n = blockIdx.x % n_tiles;
      t = blockIdx.x / n_tiles, step = gridDim.x / n_tiles, end = a.m_tiles;
    } else {
      t = blockIdx.x, step = gridDim.x, end = (long long)a.m_tiles * n_tiles;
    }
    t += step * first;
    step *= every;
  }
  __device__ bool more() const { return t < end; }
  __device__ void next() { t += step; }
  __device__ int m() const { return (int)(fixed ? t : t / n_tiles); }
  __device__ int nt() const { return fixed ? n : (int)(t % n_tiles); }
};

template <int MODE, int BN, bool BMN>
__device__ __forceinline__ void load_b(const GemmArgs& g, int seg, uint32_t dst, int k, int n0, uint32_t bar) {
  typedef Cfg<MODE, BN> C;
  if (MODE == GATE || (MODE == GATE_BWD && seg == 0)) {
    tma_load(dst, &g.b[0], k, n0, bar);
    tma_load(dst + BN * 128, &g.b[0], k, g.up + n0, bar);
  } else if (BMN || MODE == GATE_BWD) {  // 64 channels x 64 rows along k per box
#pragma unroll
    for (int i = 0; i < C::N1 / 64; ++i) tma_load(dst + i * 8192, &g.b[seg], n0 + 64 * i, k, bar);
  } else {
    tma_load(dst, &g.b[seg], k, n0, bar);
  }
}

template <int MODE, int BN, bool BMN>
__global__ void __launch_bounds__(THREADS, 1) rows_tc_kernel(const __grid_constant__ GemmArgs g) {
  typedef Cfg<MODE, BN> C;
  extern __shared__ unsigned char raw[];
  __shared__ volatile int abort_flag_s;
  unsigned char* sm = (unsigned char*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  volatile int* abort_flag = &abort_flag_s;
  const uint32_t out0 = smem_u32(sm);
  const uint32_t a0 = out0 + 2 * g.slots * CH_BYTES;
  const uint32_t b0 = a0 + g.stages * A_BYTES;
  const int bbytes = g.resident ? g.kb[0] * C::N0 * 128 + g.kb[1] * C::N1 * 128 : g.stages * C::BMAX;
  float* bias_s = (float*)(sm + (b0 - out0) + bbytes);  // two tiles' worth per set
  const uint32_t bar0 = smem_u32(bias_s + 4 * 256);
  uint32_t* tmem_s = (uint32_t*)((unsigned char*)(bias_s + 4 * 256) + ROWS_BARS * 8);
  const auto full = [&](uint32_t s) { return bar0 + 8 * s; };
  const auto empty = [&](uint32_t s) { return bar0 + 8 * (MAX_STAGES + s); };
  const uint32_t bfull = bar0 + 8 * (2 * MAX_STAGES);
  const auto tfull = [&](uint32_t s) { return bfull + 8 + 8 * s; };
  const auto tempty = [&](uint32_t s) { return bfull + 24 + 8 * s; };
  const auto ready = [&](int set, uint32_t s) { return bfull + 40 + 8 * (2 * set + s); };
  const auto done = [&](int set, uint32_t s) { return bfull + 72 + 8 * (2 * set + s); };
  const uint32_t drain = bfull + 104;
  const auto biased = [&](int set) { return bfull + 112 + 8 * set; };

  if (threadIdx.x == 0) {
    abort_flag_s = 0;
    for (int i = 0; i < g.stages; ++i) mbar_init(full(i), 1), mbar_init(empty(i), 1);
    mbar_init(bfull, 1);
    mbar_init(drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull(i), 1);
      mbar_init(tempty(i), 4);
      mbar_init(biased(i), 4);
      for (int s = 0; s < 2; ++s) mbar_init(ready(i, s), 1), mbar_init(done(i, s), 4);
    }
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_s), 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_s;

  if (warp == 0) {
    // ---- loader.  (Loader and MMA warp run converged, one elected lane issues: addresses and descriptors then live in
    // uniform registers.  In a branch of a single lane each of them is moved there for every instruction, and the
    // issuing thread, not the tensor core, sets the pace: 240 instead of 128 cycles per MMA of 256 columns.)
    const bool leader = elect_one();
    TileWalk w(g);
    if (g.resident && w.more() && leader) {
      mbar_expect_tx(bfull, bbytes);
      const int n0 = w.nt() * BN;
      uint32_t dst = b0;
      for (int seg = 0; seg < 2; ++seg)
        for (int k = 0; k < g.kb[seg]; ++k) {
          load_b<MODE, BN, BMN>(g, seg, dst, k * KB, n0, bfull);
          dst += (seg ? C::N1 : C::N0) * 128;
        }
    }
    __syncwarp();
    uint32_t st = 0, ph = 0;
    bool ok = true;
    for (; w.more() && ok; w.next()) {
      const int m0 = w.m() * TILE, n0 = w.nt() * BN;
      for (int seg = 0; seg < 2 && ok; ++seg)
        for (int k = 0; k < g.kb[seg]; ++k) {
          ok = mbar_wait(empty(st), ph ^ 1, abort_flag, 0x101);
          if (!__all_sync(~0u, ok)) {
            ok = false;
            break;
          }
          if (leader) {
            mbar_expect_tx(full(st), A_BYTES + (g.resident ? 0 : (seg ? C::N1 : C::N0) * 128));
            tma_load(a0 + st * A_BYTES, &g.a[seg], k * KB, m0, full(st));
            if (!g.resident) load_b<MODE, BN, BMN>(g, seg, b0 + st * C::BMAX, k * KB, n0, full(st));
          }
          __syncwarp();
          if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
        }
    }
  } else if (warp == 1) {
    // ---- MMA issuer
    const bool leader = elect_one();
    uint32_t st = 0, ph = 0, it = 0;
    TileWalk w(g);
    bool ok = true;
    if (g.resident && w.more()) ok = __all_sync(~0u, mbar_wait(bfull, 0, abort_flag, 0x111));
    for (; w.more() && ok; w.next(), ++it) {
      const uint32_t acc = it & 1, aph = (it >> 1) & 1;
      ok = __all_sync(~0u, mbar_wait(tempty(acc), aph ^ 1, abort_flag, 0x112));
      if (!ok) break;
      tc_fence_after_sync();
      uint32_t bres = b0;
#pragma unroll
      for (int seg = 0; seg < 2; ++seg) {
        constexpr uint32_t HI = desc_sw128_hi(1024);
        const bool mn = MODE == GATE_BWD ? seg == 1 : BMN;
        const uint32_t idesc = make_idesc_bf16(TILE, seg ? C::N1 : C::N0, 0, mn ? 1 : 0);
        const uint32_t d = tmem + acc * 256 + (seg ? C::OFF1 : 0);
        const uint32_t bstep = mn ? 128 : 2;  // sixteen rows along k, or 32 bytes
        for (int k = 0; k < g.kb[seg] && ok; ++k) {
          ok = __all_sync(~0u, mbar_wait(full(st), ph, abort_flag, 0x113));
          if (!ok) break;
          const uint32_t ad = desc_sw128_lo(a0 + st * A_BYTES, 16);
          const uint32_t bd = desc_sw128_lo(g.resident ? bres : b0 + st * C::BMAX, mn ? 8192 : 16);
          if (leader) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              mma_bf16_ss_lo(d, ad + 2 * j, HI, bd + bstep * j, HI, idesc, (k | j) != 0 || (seg && C::OFF1 == 0));
            mma_commit(empty(st));
          }
          __syncwarp();
          bres += (seg ? C::N1 : C::N0) * 128;
          if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
        }
      }
      if (ok && leader) mma_commit(tfull(acc));
      __syncwarp();
    }
    if (leader) {
      mma_commit(drain);
      mbar_wait(drain, 0, abort_flag, 0x114);
    }
    __syncwarp();
  } else if (warp < 4) {
    // ---- I/O of one set's staged tiles: fill the slots ahead (residual), store what the read-out warps leave in them
    if (lane == 0) {
      const int set = warp - 2;
      TileWalk lead(g, set, 2);
      int lead_c = 0;
      uint32_t lead_i = 0;
      const uint32_t buf = out0 + set * g.slots * CH_BYTES;
      const auto column = [&](const TileWalk& w, int c) { return w.nt() * BN + (MODE == GATE_BWD ? 0 : c * 64); };
      const auto advance = [&]() {
        if (!lead.more()) return;
        const uint32_t s = lead_i % g.slots;
        const int col = column(lead, lead_c);
        if (g.res && col < g.N) {
          mbar_expect_tx(ready(set, s), CH_BYTES);
          tma_load(buf + s * CH_BYTES, &g.r, col, lead.m() * TILE, ready(set, s));
        } else {
          mbar_arrive(ready(set, s));
        }
        ++lead_i;
        if (++lead_c == C::NCH) lead_c = 0, lead.next();
      };
      for (int i = 0; i < g.slots; ++i) advance();
      bool ok = true;
      uint32_t i = 0;
      for (TileWalk w(g, set, 2); w.more() && ok; w.next())
        for (int c = 0; c < C::NCH; ++c, ++i) {
          const uint32_t s = i % g.slots;
          ok = mbar_wait(done(set, s), (i / g.slots) & 1, abort_flag, 0x121);
          if (!ok) break;
          const int col = column(w, c);
          if (col < g.N) {
            tma_store(&g.y[MODE == GATE_BWD ? c : 0], col, w.m() * TILE, buf + s * CH_BYTES);
            bulk_commit();
            bulk_wait_read();
          }
          advance();
        }
      bulk_wait_all();
    }
    __syncwarp();
  } else {
    // ---- read-out: thread = pixel, 32 channels at a time
    const int set = (warp - 4) / 4, q = warp & 3, row = q * 32 + lane;
    const uint32_t buf = out0 + set * g.slots * CH_BYTES;
    const uint32_t t0 = tmem + ((uint32_t)(q * 32) << 16) + set * 256;
    // 16-byte piece j of this row of a staged tile
    const auto piece = [&](uint32_t slot, int j) { return buf + slot * CH_BYTES + row * 128 + ((j ^ (row & 7)) << 4); };
    const auto slot_ready = [&](uint32_t i) { return warp_wait(ready(set, i % g.slots), (i / g.slots) & 1, abort_flag, 0x132); };
    const auto slot_done = [&](uint32_t i) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(done(set, i % g.slots));
    };
    const auto accumulators_free = [&]() {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty(set));
    };
    uint32_t it = 0, i = 0;
    bool ok = true;
    for (TileWalk w(g, set, 2); w.more() && ok; w.next(), ++it) {
      float* bs = bias_s + set * 512 + (g.resident ? 0 : (it & 1) * 256);
      if (it == 0 || !g.resident) {
        // (the other half is still being read by warps that are a tile behind; nobody is two behind)
        const int n0 = w.nt() * BN;
#pragma unroll
        for (int e = row; e < C::N0; e += 128) {
          const int n = n0 + e % BN + (e >= BN ? g.up : 0);
          bs[e] = g.bias && n0 + e % BN < g.N
                      ? __bfloat162float(__ushort_as_bfloat16(__ldg((const unsigned short*)g.bias + n)))
                      : 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(biased(set));
        ok = warp_wait(biased(set), it & 1, abort_flag, 0x133);  // (a bounded wait, unlike bar.sync)
        if (!ok) break;
      }
      ok = warp_wait(tfull(set), it & 1, abort_flag, 0x131);
      if (!ok) break;
      tc_fence_after_sync();
      if constexpr (MODE == GATE_BWD) {
        uint32_t pu[2][16];  // the second result, packed, until its slot is free
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t vg[32], vu[32], vh[32];
          tmem_ld_32x32(t0 + 32 * k, vg);
          tmem_ld_32x32(t0 + BN + 32 * k, vu);
          tmem_ld_32x32(t0 + C::OFF1 + 32 * k, vh);
          tmem_ld_wait();
          if (k == 1) accumulators_free();
          with_act(g.act, [&](auto a) {
            typedef decltype(a) Act;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float2 v, s;
              Act::both(add2(pair_of(vg, j), bias2(bs, 16 * k + j)), v, s);
              const float2 gh = pair_of(vh, j), u = add2(pair_of(vu, j), bias2(bs + BN, 16 * k + j));
              const float2 og = mul2(mul2(gh, u), s), ou = mul2(gh, v);
              vg[j] = pack_bf16x2(og.x, og.y);
              pu[k][j] = pack_bf16x2(ou.x, ou.y);
            }
          });
          if (k == 0) ok = slot_ready(i);
          if (!ok) break;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sts16(piece(i % g.slots, 4 * k + j), make_uint4(vg[4 * j], vg[4 * j + 1], vg[4 * j + 2], vg[4 * j + 3]));
        }
        if (!ok) break;
        slot_done(i++);
        ok = slot_ready(i);
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t* v = &pu[j / 4][j % 4 * 4];
          sts16(piece(i % g.slots, j), make_uint4(v[0], v[1], v[2], v[3]));
        }
        slot_done(i++);
      } else {
#pragma unroll 1
        for (int c = 0; c < C::NCH && ok; ++c) {
          const uint32_t s = i % g.slots;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t v[32], u[32];
            tmem_ld_32x32(t0 + 64 * c + 32 * k, v);
            if (MODE == GATE) tmem_ld_32x32(t0 + BN + 64 * c + 32 * k, u);
            tmem_ld_wait();
            if (c == C::NCH - 1 && k == 1) accumulators_free();
            const float* b = bs + 64 * c + 32 * k;
            with_act(g.act, [&](auto a) {
              typedef decltype(a) Act;
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 z = add2(pair_of(v, j), bias2(b, j));
                float2 o;
                if (MODE == ACT_BWD) {
                  float2 val;
                  Act::both(z, val, o);
                } else {
                  o = Act::value(z);
                  if (MODE == GATE) o = mul2(o, add2(pair_of(u, j), bias2(b + BN, j)));
                }
                if (MODE == GATE) v[j] = pack_bf16x2(o.x, o.y);
                else v[2 * j] = __float_as_uint(o.x), v[2 * j + 1] = __float_as_uint(o.y);
              }
            });
            if (k == 0) ok = slot_ready(i);
            if (!ok) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t at = piece(s, 4 * k + j);
              if (MODE == GATE) {
                sts16(at, make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
                continue;
              }
              float2 f[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) f[e] = pair_of(v, 4 * j + e);
              if (MODE == ACT_BWD || (MODE == LAYER && g.res)) {
                const uint4 r = lds16(at);
                const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 w = make_float2(__uint_as_float(rw[e] << 16), __uint_as_float(rw[e] & 0xFFFF0000u));
                  f[e] = MODE == ACT_BWD ? mul2(f[e], w) : add2(f[e], w);
                }
              }
              sts16(at, make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y), pack_bf16x2(f[2].x, f[2].y),
                                   pack_bf16x2(f[3].x, f[3].y)));
            }
          }
          if (ok) slot_done(i++);
        }
      }
    }
  }
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {  // given up: copies still in flight land within microseconds
    const long long c = clock64();
    while (clock64() - c < 4000000) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ---- outer kernel ----------------------------------------------------------------------------------------
struct alignas(64) OuterTcArgs {
  CUtensorMap g[2], x;
  float *part, *csum;  // [split][M total][ldn], [split][M total]
  int M, segs, N, ldn; // rows of one of the (one or two) first operands
  int m_tiles, n_tiles;
  int kblocks, per;    // 64-pixel blocks in all, and of a share
  int stages;
};
constexpr int OUTER_BARS = 2 * MAX_STAGES + 1;

// MT: groups of 128 channels of the first operand, BN: channels of the second
template <int MT, int BN>
__global__ void __launch_bounds__(THREADS, 1) outer_tc_kernel(const __grid_constant__ OuterTcArgs g) {
  constexpr int GB = MT * A_BYTES, STAGE = GB + BN * 128;
  extern __shared__ unsigned char raw[];
  __shared__ volatile int abort_flag_s;
  __shared__ uint64_t bars[OUTER_BARS];
  __shared__ uint32_t tmem_s;
  unsigned char* sm = (unsigned char*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  volatile int* abort_flag = &abort_flag_s;
  const uint32_t s0 = smem_u32(sm), bar0 = smem_u32(bars);
  const auto full = [&](uint32_t s) { return bar0 + 8 * s; };
  const auto empty = [&](uint32_t s) { return bar0 + 8 * (MAX_STAGES + s); };
  const uint32_t done = bar0 + 16 * MAX_STAGES;
  const int tiles = g.segs * g.m_tiles * g.n_tiles;
  const int split = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  const int nt = tile % g.n_tiles, mt = tile / g.n_tiles % g.m_tiles, seg = tile / g.n_tiles / g.m_tiles;
  const int m0 = mt * MT * 128, n0 = nt * BN;
  const int k0 = split * g.per, k1 = min(g.kblocks, k0 + g.per);
  const bool sums = nt == 0;

  if (threadIdx.x == 0) {
    abort_flag_s = 0;
    for (int i = 0; i < g.stages; ++i) mbar_init(full(i), 1), mbar_init(empty(i), sums ? 9 : 1);
    mbar_init(done, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_s), MT * BN < 32 ? 32 : MT * BN);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_s;

  if (warp == 0) {  // (converged, one elected lane issues: see the rows kernel)
    const bool leader = elect_one();
    uint32_t st = 0, ph = 0;
    for (int k = k0; k < k1; ++k) {
      if (!__all_sync(~0u, mbar_wait(empty(st), ph ^ 1, abort_flag, 0x141))) break;
      if (leader) {
        mbar_expect_tx(full(st), STAGE);
        const uint32_t dst = s0 + st * STAGE;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) tma_load(dst + i * 8192, &g.g[seg], m0 + 64 * i, k * KB, full(st));
#pragma unroll
        for (int i = 0; i < BN / 64; ++i) tma_load(dst + GB + i * 8192, &g.x, n0 + 64 * i, k * KB, full(st));
      }
      __syncwarp();
      if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    constexpr uint32_t idesc = make_idesc_bf16(128, BN, 1, 1), HI = desc_sw128_hi(1024);
    uint32_t st = 0, ph = 0;
    for (int k = k0; k < k1; ++k) {
      if (!__all_sync(~0u, mbar_wait(full(st), ph, abort_flag, 0x142))) break;
      if (leader) {
        const uint32_t bd = desc_sw128_lo(s0 + st * STAGE + GB, 8192), ad = desc_sw128_lo(s0 + st * STAGE, 8192);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j)  // sixteen pixels each
            mma_bf16_ss_lo(tmem + m * BN, ad + m * (A_BYTES >> 4) + 128 * j, HI, bd + 128 * j, HI, idesc, k != k0 || j != 0);
        mma_commit(empty(st));
      }
      __syncwarp();
      if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
    }
    if (leader) mma_commit(done);
    __syncwarp();
  } else if (warp >= 4) {
    const int ew = warp - 4, q = warp & 3;
    bool ok = true;
    if (sums) {
      // columns of the first operand: 2 MT 16-byte pieces (8 channels each) per warp, 16 / MT pixels at a time
      constexpr int PC = 2 * MT, PX = 32 / PC;
      const int piece = ew * PC + lane % PC, box = piece / 8, j = piece % 8;
      float acc[8] = {};
      uint32_t st = 0, ph = 0;
      for (int k = k0; k < k1; ++k) {
        ok = warp_wait(full(st), ph, abort_flag, 0x143);
        if (!ok) break;
        const uint32_t base = s0 + st * STAGE + box * 8192;
#pragma unroll
        for (int p = lane / PC; p < KB; p += PX) {
          const uint4 r = lds16(base + p * 128 + ((j ^ (p & 7)) << 4));
          const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[2 * e] += __uint_as_float(w[e] << 16);
            acc[2 * e + 1] += __uint_as_float(w[e] & 0xFFFF0000u);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(st));
        if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int o = 16; o >= PC; o >>= 1) acc[e] += __shfl_xor_sync(~0u, acc[e], o);
        const int m = m0 + piece * 8 + e;
        if (lane < PC && m < g.M) g.csum[((size_t)split * g.segs + seg) * g.M + m] = acc[e];
      }
    }
    if (ok) ok = warp_wait(done, 0, abort_flag, 0x144);
    if (ok && k1 > k0) {
      tc_fence_after_sync();
#pragma unroll 1
      for (int t = ew / 4; t < MT * BN / 32; t += 2) {  // 32 columns each
        uint32_t v[32];
        tmem_ld_32x32(tmem + ((uint32_t)(q * 32) << 16) + t * 32, v);
        tmem_ld_wait();
        const int m = m0 + t * 32 / BN * 128 + q * 32 + lane, n = n0 + t * 32 % BN;
        float* out = g.part + (((size_t)split * g.segs + seg) * g.M + m) * g.ldn + n;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (m < g.M && n + 4 * j < g.ldn)
            *reinterpret_cast<float4*>(out + 4 * j) =
                make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 2]),
                            __uint_as_float(v[4 * j + 3]));
        __syncwarp();
      }
      tc_fence_before_sync();
    }
  }
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {
    const long long c = clock64();
    while (clock64() - c < 4000000) __nanosleep(1000);
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, MT * BN < 32 ? 32 : MT * BN);
}

// ---- host ------------------------------------------------------------------------------------------------
// boxes of 64 channels x box_r rows, 128-byte swizzle
static bool encode(CUtensorMap* tm, const TcRows& t, int box_r) {
  static std::atomic<void*> fn{nullptr};
  void* f = fn.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess || !f)
      return false;
    fn.store(f, std::memory_order_release);
  }
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  const cuuint64_t dims[2] = {(cuuint64_t)t.cols, (cuuint64_t)t.rows}, strides[1] = {(cuuint64_t)t.ld * 2};
  const cuuint32_t box[2] = {KB, (cuuint32_t)box_r}, es[2] = {1, 1};
  for (int attempt = 0; attempt < 2; ++attempt) {
    if (((Encode)f)(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(t.p), dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS)
      return true;
    // A thread whose first CUDA call this is (autograd's, with all memory cached) has no context yet; selecting its
    // device makes one current.
    int dev = 0;
    if (attempt || cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) break;
  }
  return false;
}
static int sm_total() {
  static std::atomic<int> n{0};
  int v = n.load();
  if (!v) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    n.store(v);
  }
  return v;
}
template <typename Kern>
static bool allow_smem(Kern kern) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT) == cudaSuccess;
}

template <int MODE, int BN, bool BMN>
static int launch_rows(GemmArgs& g, int n_cover, cudaStream_t st) {
  typedef Cfg<MODE, BN> C;
  g.n_tiles = (n_cover + BN - 1) / BN;
  const int fixed_bytes = 1024 + 4 * 256 * 4 + ROWS_BARS * 8 + 16 + 64;
  const int b_all = g.kb[0] * C::N0 * 128 + g.kb[1] * C::N1 * 128;
  const int sms = sm_total();
  g.slots = 2;
  int left = SMEM_LIMIT - fixed_bytes - 2 * g.slots * CH_BYTES;
  // Weights stay where at least three stages of pixels fit beside them and every channel tile gets a block.
  g.resident = g.n_tiles <= sms && b_all + 3 * A_BYTES <= left;
  if (!g.resident && g.n_tiles <= sms) {  // one slot per set makes room for 128 KB of them
    const int one = left + 2 * CH_BYTES;
    if (b_all + 3 * A_BYTES <= one) g.slots = 1, left = one, g.resident = 1;
  }
  g.stages = g.resident ? (left - b_all) / A_BYTES : left / (A_BYTES + C::BMAX);
  if (g.stages > MAX_STAGES) g.stages = MAX_STAGES;
  const size_t smem = fixed_bytes + 2 * g.slots * CH_BYTES + (size_t)g.stages * A_BYTES +
                      (g.resident ? b_all : g.stages * C::BMAX);
  long long grid;
  if (g.resident) {
    grid = sms / g.n_tiles;
    if (grid > g.m_tiles) grid = g.m_tiles;
    grid *= g.n_tiles;
  } else {
    grid = (long long)g.m_tiles * g.n_tiles;
    if (grid > sms) grid = sms;
  }
  if (!allow_smem(rows_tc_kernel<MODE, BN, BMN>)) return MC_ERR_LAUNCH;
  rows_tc_kernel<MODE, BN, BMN><<<(unsigned)grid, THREADS, smem, st>>>(g), MC_COUNT(1);
  MC_CHECK_LAUNCH();
  return MC_OK;
}

// Channels of a tile: the smallest of 64, 128, 256 that holds all of them, else the one that pads least.
static int tile_width(int n) {
  if (n <= 64) return 64;
  if (n <= 128) return 128;
  return (n + 255) / 256 * 256 <= (n + 127) / 128 * 128 + 64 ? 256 : 128;
}
static int kblocks(int c) { return (c + KB - 1) / KB; }
static int tiles_of(long long P) { return (int)((P + TILE - 1) / TILE); }

static GemmArgs base_args(const TcRows& a, const TcRows& y, const bf16* bias, int act) {
  GemmArgs g{};
  g.bias = bias;
  g.m_tiles = tiles_of(a.rows);
  g.N = y.cols;
  g.kb[0] = kblocks(a.cols);
  g.act = act;
  return g;
}

int tc_layer(const TcRows& a, const TcRows& w, const bf16* bias, int act, const TcRows& r, const TcRows& y,
             bool backward, cudaStream_t st) {
  GemmArgs g = base_args(a, y, bias, act);
  g.res = r.p != nullptr;
  const int bn = tile_width(y.cols);
  if (!encode(&g.a[0], a, TILE) || !encode(&g.b[0], w, bn) || !encode(&g.y[0], y, TILE)) return MC_ERR_LAUNCH;
  if (g.res && !encode(&g.r, r, TILE)) return MC_ERR_LAUNCH;
  if (backward) {
    if (bn == 64) return launch_rows<ACT_BWD, 64, false>(g, y.cols, st);
    if (bn == 128) return launch_rows<ACT_BWD, 128, false>(g, y.cols, st);
    return launch_rows<ACT_BWD, 256, false>(g, y.cols, st);
  }
  if (bn == 64) return launch_rows<LAYER, 64, false>(g, y.cols, st);
  if (bn == 128) return launch_rows<LAYER, 128, false>(g, y.cols, st);
  return launch_rows<LAYER, 256, false>(g, y.cols, st);
}

int tc_input_grad(const TcRows& g0, const TcRows& w0, const TcRows& g1, const TcRows& w1, const TcRows& gx,
                  cudaStream_t st) {
  GemmArgs g = base_args(g0, gx, nullptr, MC_ACT_NONE);
  const int bn = tile_width(gx.cols);
  if (!encode(&g.a[0], g0, TILE) || !encode(&g.b[0], w0, 64) || !encode(&g.y[0], gx, TILE)) return MC_ERR_LAUNCH;
  if (g1.p) {
    g.kb[1] = kblocks(g1.cols);
    if (!encode(&g.a[1], g1, TILE) || !encode(&g.b[1], w1, 64)) return MC_ERR_LAUNCH;
  }
  if (bn == 64) return launch_rows<LAYER, 64, true>(g, gx.cols, st);
  if (bn == 128) return launch_rows<LAYER, 128, true>(g, gx.cols, st);
  return launch_rows<LAYER, 256, true>(g, gx.cols, st);
}

int tc_gate(const TcRows& x, const TcRows& w_in, const bf16* b_in, int act, const TcRows& h, cudaStream_t st) {
  GemmArgs g = base_args(x, h, b_in, act);
  g.up = h.cols;
  if (!encode(&g.a[0], x, TILE) || !encode(&g.b[0], w_in, 128) || !encode(&g.y[0], h, TILE)) return MC_ERR_LAUNCH;
  return launch_rows<GATE, 128, false>(g, h.cols, st);
}

int tc_gate_bwd(const TcRows& x, const TcRows& w_in, const bf16* b_in, int act, const TcRows& gy, const TcRows& w_out,
                const TcRows& gg, const TcRows& gu, cudaStream_t st) {
  GemmArgs g = base_args(x, gg, b_in, act);
  g.up = gg.cols;
  g.kb[1] = kblocks(gy.cols);
  if (!encode(&g.a[0], x, TILE) || !encode(&g.b[0], w_in, 64) || !encode(&g.a[1], gy, TILE) ||
      !encode(&g.b[1], w_out, 64) || !encode(&g.y[0], gg, TILE) || !encode(&g.y[1], gu, TILE))
    return MC_ERR_LAUNCH;
  return launch_rows<GATE_BWD, 64, false>(g, gg.cols, st);
}

// Blocks per gradient tile: as many as fill the SMs once or a whole number of times with equal shares.
struct OuterPlan {
  int mt, bn, m_tiles, n_tiles, splits, per;
};
static OuterPlan outer_plan(long long P, int M, int segs, int N) {
  OuterPlan p;
  p.mt = M > 128 ? 2 : 1;
  p.bn = N <= 64 ? 64 : N <= 128 ? 128 : 256;
  p.m_tiles = (M + 128 * p.mt - 1) / (128 * p.mt);
  p.n_tiles = (N + p.bn - 1) / p.bn;
  const long long tiles = (long long)segs * p.m_tiles * p.n_tiles, kb = (P + KB - 1) / KB;
  double best = 1e30;
  p.splits = 1, p.per = (int)kb;
  for (long long s = 1; s <= 148 && s <= (kb + 3) / 4; ++s) {
    const long long per = (kb + s - 1) / s;
    const double waves = (double)((tiles * s + 147) / 148);
    // a block's stages, and what it costs to write its sums and to add them up again
    const double t = waves * (per + 8.0) + 0.05 * tiles * s;
    if (t < best) best = t, p.splits = (int)((kb + per - 1) / per), p.per = (int)per;
  }
  return p;
}
size_t tc_outer_floats(long long P, int M, int segs, int N, int* splits, int* ldn) {
  const OuterPlan p = outer_plan(P, M, segs, N);
  *splits = p.splits;
  *ldn = (N + 3) / 4 * 4;
  return (size_t)p.splits * segs * M * *ldn;
}

template <int MT, int BN>
static int launch_outer(OuterTcArgs& g, const OuterPlan& p, cudaStream_t st) {
  constexpr int STAGE = MT * A_BYTES + BN * 128;
  g.stages = (SMEM_LIMIT - 2048) / STAGE;
  if (g.stages > MAX_STAGES) g.stages = MAX_STAGES;
  if (!allow_smem(outer_tc_kernel<MT, BN>)) return MC_ERR_LAUNCH;
  outer_tc_kernel<MT, BN><<<g.segs * p.m_tiles * p.n_tiles * p.splits, THREADS, 1024 + g.stages * STAGE, st>>>(g), MC_COUNT(1);
  MC_CHECK_LAUNCH();
  return MC_OK;
}
int tc_outer(const TcRows& g0, const TcRows& g1, const TcRows& x, float* part, float* csum, cudaStream_t st) {
  OuterTcArgs g{};
  g.segs = g1.p ? 2 : 1;
  const OuterPlan p = outer_plan(x.rows, g0.cols, g.segs, x.cols);
  if (!encode(&g.g[0], g0, KB) || (g1.p && !encode(&g.g[1], g1, KB)) || !encode(&g.x, x, KB)) return MC_ERR_LAUNCH;
  g.part = part, g.csum = csum;
  g.M = g0.cols, g.N = x.cols, g.ldn = (x.cols + 3) / 4 * 4;
  g.m_tiles = p.m_tiles, g.n_tiles = p.n_tiles;
  g.kblocks = (int)((x.rows + KB - 1) / KB), g.per = p.per;
  if (p.mt == 1) {
    if (p.bn == 64) return launch_outer<1, 64>(g, p, st);
    if (p.bn == 128) return launch_outer<1, 128>(g, p, st);
    return launch_outer<1, 256>(g, p, st);
  }
  if (p.bn == 64) return launch_outer<2, 64>(g, p, st);
  if (p.bn == 128) return launch_outer<2, 128>(g, p, st);
  return launch_outer<2, 256>(g, p, st);
}

int tc_status_read(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, tc::g_status, sizeof(int)) != cudaSuccess) return MC_ERR_LAUNCH;
  if (reset && v != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(tc::g_status, &z, sizeof(int));
  }
  return v;
}

}  // namespace mix
}  // namespace mc
