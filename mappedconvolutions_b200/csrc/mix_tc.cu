// Channel mixing on the tensor cores (bf16 operands, float32 sums in TMEM).
//
// Two blocks of a cluster work on one MMA (cta_group::2): each holds its own 128 pixels and half of the weights' rows,
// the leader issues.  What bounds a block alone is its shared memory: TMA writes and operand reads share 128 bytes a
// cycle, and a 128 x 256 tile asks for 96 + 96 of them at the tensor core's pace.  Halving the weights' part takes that
// to 64 + 64.
//
// rows kernel: tiles of 2 x 128 pixels x BN channels.  One warp fetches operand tiles by TMA, one thread issues the MMAs
// into two or four accumulators in turn.  Every second tile has four read-out warps of its own (a tile's latencies - TMEM
// loads, elementary functions, hand-over of the staged tiles - overlap with the other set's), which apply the epilogue and
// leave bf16 tiles in shared memory, from where an I/O thread stores them by TMA; the same slots receive the tiles that an
// epilogue adds or multiplies (residual, grad_output) beforehand.  Where all weights that a block needs fit beside the
// rings they stay in shared memory and the block keeps its channel tile; otherwise they travel with the pixels.
// 1024 -> 1024 channels at 655 488 pixels: 1281 TFLOP/s without an epilogue, 1094 with GELU, 1005 with GELU and residual
// (first launches; over a second, with the clock held down by the power limit, 1118, 958 and 874; a library product of
// these sizes 1338 and 1170).  128 -> 256 channels with residual, 655 488 pixels: 78 % of the copy bandwidth.
//
// outer kernel: parameter gradients, both operands read along the pixels (MN-major); every block sums a share of the
// pixels for one tile of the gradient and writes float32 partial sums, which are added in order afterwards.  The eight
// read-out warps, idle meanwhile, sum the columns of the first operand in shared memory (the bias gradient).
// 2048 x 256 and 256 x 1024 gradients over 655 488 pixels: 954 us together, 1080 TFLOP/s.
#include <cuda.h>

#include "act_pairs.cuh"
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
constexpr int SMEM_LIMIT = 226 * 1024;  // of 227 KB, the rest is static

// ---- activations: the fast forms of act_pairs.cuh, sixteen values at a time
constexpr int NV = 8;
typedef float2 Pairs[NV];
#define MC_EACH _Pragma("unroll") for (int j = 0; j < NV; ++j)
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {  // one branch per read-out warp
  switch (act) {
    case MC_ACT_RELU: f(ActRelu()); break;
    case MC_ACT_GELU: f(ActGelu()); break;
    case MC_ACT_GELU_TANH: f(ActGeluTanh()); break;
    case MC_ACT_SILU: f(ActSilu()); break;
    case MC_ACT_SIGMOID: f(ActSigmoid()); break;
    default: f(ActNone()); break;
  }
}

// 32 lanes x 16 columns of accumulators
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
template <int N>
__device__ __forceinline__ float2 pair_of(const uint32_t (&v)[N], int j) {
  return make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
}
__device__ __forceinline__ float2 bias2(const float* b, int j) { return reinterpret_cast<const float2*>(b)[j]; }

// Has the phase completed?  Never suspends the thread, so that the answer for the next stage can be on its way while this
// stage's MMAs are issued.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// The kernels here may be launched while the one before them is still running: what they set up first touches no memory of
// others, and here they wait until all of it is written.  (The next kernel may start likewise.)
__device__ __forceinline__ void behind_previous_kernel() {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- pairs of blocks -----------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// the address that a barrier of the leader has from both blocks
__device__ __forceinline__ uint32_t of_leader(uint32_t a) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void arrive_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pair_alloc(uint32_t result_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(result_smem), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// D (256 rows, 128 in each block's TMEM) (+)= A (128 rows in each block) B (half of the columns in each block)
__device__ __forceinline__ void pair_mma(uint32_t d, uint32_t alo, uint32_t ahi, uint32_t blo, uint32_t bhi, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n\t}"
      :
      : "r"(d), "r"(alo), "r"(ahi), "r"(blo), "r"(bhi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// one arrival at this barrier of both blocks when all MMAs issued so far have finished
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"((uint16_t)3)
               : "memory");
}
// the same at this barrier of the issuing block alone
__device__ __forceinline__ void leader_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// ---- TMA ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"((uint64_t)tm), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// into this block's shared memory, counted by a barrier of the leader
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst),
      "l"((uint64_t)tm), "r"(x), "r"(y), "r"(leader_bar)
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
  ACT_BWD = 3,   // y = r act'(A B^T + bias)
  SCORE_SUM = 4, // softmax sums of z = A B^T + bias over the tile's columns, the label's z
  SCORE_GRAD = 5,// y = scale exp(z - top - rest), the label's scale (e^-loss - 1)
  FLOATS = 6     // y = A B^T in float32
};
// Products of float32 values in three bf16 parts each, 0 the largest: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0).  The others are below
// 2^-24 of the product.  Small ones come first: the accumulators truncate, up to 2^-23 of what they hold for every MMA.
constexpr int PRODUCTS = 6;
__device__ __forceinline__ int part_a(int product) { return 0x052 >> 2 * product & 3; }
__device__ __forceinline__ int part_b(int product) { return 0x118 >> 2 * product & 3; }
// Where the second operand stays in shared memory with all its parts, the first one passes four times, not six: part 2 for (2,0), 1 for
// (1,1) (1,0), 0 for (0,2) (0,1), and 0 again for (0,0), which comes last as before.  (Input gradient of 131 072 pixels, 99 -> 50: 46 us
// with six, 34.6 with four; the two kernels that read scores out, 29 -> 28 and 49 -> 48.)
constexpr int PASSES = 4;
__device__ __forceinline__ int pass_a(int pass) { return 0x06 >> 2 * pass & 3; }
__device__ __forceinline__ int pass_b(int pass) { return 0x24 >> 2 * pass & 3; }  // of the first product
__device__ __forceinline__ bool pass_twice(int pass) { return pass == 1 || pass == 2; }  // the next smaller number is the second's
// BN: channels of a tile.  It is staged CW channels (128 or 64 swizzled bytes a row) at a time; the two results of
// GATE_BWD side by side, in smaller tiles because its weights leave little room.
template <int MODE, int BN> struct Cfg {
  static constexpr int N0 = MODE == GATE || MODE == GATE_BWD ? 2 * BN : BN;  // columns of the first product
  static constexpr int N1 = MODE == GATE_BWD ? BN : N0;                      // and of the second
  static constexpr int OFF1 = MODE == GATE_BWD ? N0 : 0;                     // its first accumulator column
  static constexpr int CW = MODE == GATE_BWD ? 32 : 64;
  static constexpr int NCH = (MODE == GATE_BWD ? 2 : 1) * BN / CW;           // staged tiles
  static constexpr int CH_BYTES = TILE * CW * 2;
  // 2^SLOT_BITS slots for staged tiles in each set.  (The gate's gradients with two: 11 % slower.  One, where that makes room
  // for weights that stay: 512 -> 512 channels with residual, 163 872 pixels 146 us instead of 115.)
  static constexpr int SLOT_BITS = MODE == GATE_BWD ? 2 : 1;
  // Accumulators in TMEM: as many as fit, since an epilogue's latencies are hidden by the tiles behind it.
  static constexpr int NACC = MODE == GATE_BWD || N0 > 128 ? 2 : 4, ACC = 512 / NACC;
  static constexpr int B0 = N0 / 2 * KB * 2, B1 = N1 / 2 * KB * 2;           // a block's weights per stage
  static constexpr int BMAX = B0 > B1 ? B0 : B1;
};

struct alignas(64) GemmArgs {
  CUtensorMap a[2], b[2], r, y[2];
  const bf16* bias;  // null: none
  int m_pairs, rows; // pairs of tiles; pixels
  int a_across[2], y_across;  // blocks next to each other where a tensor lies in blocks, else 0
  int per;           // stages of a product of parts where operands are in parts, else 0
  int kw;            // stages of b[0] that stay
  float* floats;     // FLOATS: y, rows of ld values or (ld == 0) planes
  long long ld;
  int n_tiles, N, kb[2], act;
  int up;            // distance between a gate's row of b[0] and bias and its factor's
  int res;           // r is read
  // LAYER: y in NCHW, written by the read-out warps themselves, whose lanes are neighbouring pixels.  (A residual comes as
  // rows all the same: read here from planes, a piece ahead, its latency made the kernel twice as slow.)
  bf16* planes;
  PixDiv pd;
  Scores sc;         // SCORE_*
  int group;         // channel tiles of a pair of blocks whose weights stay in shared memory, 0: none do
  int stages;
};

constexpr int ROWS_BARS = 2 * MAX_STAGES + 1 + 8 + 16 + 1 + 2;

// The tiles of a pair of blocks, from the `first`-th on, every `every`-th one.  With resident weights a pair keeps its
// group of channel tiles and takes every so many pixel tiles; otherwise the channel tiles of a pixel tile are next to
// each other among the pairs.  Either way what is read of the pixels at one time is shared through L2.
struct TileWalk {
  uint32_t t, step, end, per, base;  // t = pixel tile * per + channel tile - base
  __device__ TileWalk(const GemmArgs& a, int first = 0, int every = 1) {
    const uint32_t pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    if (a.group) {
      const uint32_t groups = a.n_tiles / a.group;
      base = pair % groups * a.group;
      per = a.group;
      m0 = pair / groups, mstep = pairs / groups;
      end = ((uint32_t)a.m_pairs - m0 + mstep - 1) / mstep * per;
      t = 0, step = 1;
    } else {
      base = 0, per = a.n_tiles, m0 = 0, mstep = 1;
      t = pair, step = pairs, end = (uint32_t)a.m_pairs * per;
    }
    t += step * first;
    step *= every;
  }
  uint32_t m0, mstep;
  __device__ bool more() const { return t < end; }
  __device__ void next() { t += step; }
  __device__ uint32_t local_n() const { return t % per; }
  __device__ int nt() const { return (int)(base + t % per); }
  __device__ int m() const { return (int)(m0 + t / per * mstep); }  // pair of pixel tiles
};

// this block's half of the weights of one stage; boxes are half a product's columns (or one of gate and factor) high
template <int MODE, int BN>
__device__ __forceinline__ void load_b(const GemmArgs& g, int seg, uint32_t rank, uint32_t dst, int k, int n0, uint32_t bar) {
  typedef Cfg<MODE, BN> C;
  int row = n0;
  if (MODE == GATE || (MODE == GATE_BWD && seg == 0)) row += rank ? g.up : 0;
  else row += rank * (C::N1 / 2);
  tma_load_pair(dst, &g.b[seg], k, row, bar);
}

// Offsets of the barriers behind bfull.
constexpr uint32_t BAR_TFULL = 8, BAR_TEMPTY = 40, BAR_READY = 72, BAR_DONE = 136, BAR_DRAIN = 200, BAR_BIASED = 208;

// Read-out warps of one accumulator set: thread = pixel.  Sixteen channels at a time in a loop that is not unrolled: the
// code of a whole tile does not stay in the instruction cache, and then fetching it takes longer than running it.
template <int MODE, int BN, typename Act>
__device__ __forceinline__ void read_out(const GemmArgs& g, int set, uint32_t rank, float* bias_s, uint32_t out0,
                                         uint32_t bfull, volatile int* abort_flag) {
  typedef Cfg<MODE, BN> C;
  constexpr int NP = BN / 16, PER = C::CW / 16;  // pieces of a tile, and of a staged tile
  const int lane = threadIdx.x % 32, q = threadIdx.x / 32 & 3, row = q * 32 + lane;
  const uint32_t buf = out0 + (set << C::SLOT_BITS) * C::CH_BYTES, mask = (1u << C::SLOT_BITS) - 1;
  const uint32_t tempty0 = of_leader(bfull + BAR_TEMPTY);
  // 16-byte piece j of this row of a staged tile
  const uint32_t at0 = buf + row * C::CW * 2, swizzle = (C::CW == 64 ? row & 7 : (row >> 1) & 3) << 4;
  const auto slot = [&](uint32_t i) { return at0 + (i & mask) * C::CH_BYTES; };
  const auto bar_of = [&](uint32_t base, uint32_t i) { return bfull + base + 32 * set + 8 * (i & mask); };
  const auto slot_ready = [&](uint32_t i) {
    return warp_wait(bar_of(BAR_READY, i), i >> C::SLOT_BITS & 1, abort_flag, 0x132);
  };
  const auto slot_done = [&](uint32_t i) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_of(BAR_DONE, i));
  };
  uint32_t it = 0, i = 0;
  for (TileWalk w(g, set, 2); w.more(); w.next(), ++it) {
    float* bs = bias_s + set * 512 + (g.group == 1 ? 0 : (it & 1) * 256);
    if (it == 0 || g.group != 1) {
      // (the other half is still being read by warps that are a tile behind; nobody is two behind)
      const int n0 = w.nt() * BN;
      for (int e = row; e < C::N0; e += 128) {
        const int n = n0 + e % BN + (e >= BN ? g.up : 0);
        bs[e] = g.bias && n0 + e % BN < g.N
                    ? __bfloat162float(__ushort_as_bfloat16(__ldg((const unsigned short*)g.bias + n)))
                    : 0.f;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bfull + BAR_BIASED + 8 * set);
      if (!warp_wait(bfull + BAR_BIASED + 8 * set, it & 1, abort_flag, 0x133)) return;  // (bounded, unlike bar.sync)
    }
    long long plane0 = -1;  // this pixel of channel n0 of the NCHW output
    if (MODE == LAYER && g.planes) {
      const uint32_t p = (w.m() * 2 + rank) * TILE + row;
      if (p < (uint32_t)g.rows) {
        uint32_t im, s;
        g.pd.split(p, im, s);
        plane0 = ((long long)im * g.N + w.nt() * BN) * g.pd.S + s;
      }
    }
    constexpr int NL = MODE == GATE_BWD ? 3 : MODE == GATE ? 2 : 1;
    uint32_t v[2][NL][16];
    const uint32_t tile = 2 * it + set, acc = tile % C::NACC;  // (the pair's tile, and where it is)
    const uint32_t t0 = ((uint32_t)(q * 32) << 16) + acc * C::ACC;
    if (!warp_wait(bfull + BAR_TFULL + 8 * acc, tile / C::NACC & 1, abort_flag, 0x131)) return;
    tc_fence_after_sync();
    const auto fetch = [&](uint32_t (&d)[NL][16], int p) {
      tmem_ld_32x16(t0 + 16 * p, d[0]);
      if (NL > 1) tmem_ld_32x16(t0 + BN + 16 * p, d[NL > 1 ? 1 : 0]);
      if (NL > 2) tmem_ld_32x16(t0 + C::OFF1 + 16 * p, d[NL > 2 ? 2 : 0]);
    };
    // pieces with channels that exist; whether staged tiles are handed over at all
    // (the gate's kernels read out whole tiles: the tests cost them 4 - 10 %, and their tiles are seldom that empty)
    int live = NP;
    if (MODE == LAYER || MODE == ACT_BWD) {
      const int left = (g.N - w.nt() * BN + 15) / 16;
      if (left < NP) live = left;
    }
    const bool turns = !(MODE == LAYER && g.planes) || g.res;
    // one piece, while the next one is on its way
    const auto step = [&](int now, int p) -> bool {
      uint32_t(&cur)[NL][16] = v[now];
      if (p < live) tmem_ld_wait();
      if (p + 1 < live) fetch(v[now ^ 1], p + 1);
      if (p + 1 == NP) {  // the accumulators are free
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_leader(tempty0 + 8 * acc);
      }
      if (p >= live) {  // (the staged tile takes its turn all the same)
        if (p % PER == 0 && turns && (!slot_ready(i) || (MODE == GATE_BWD && !slot_ready(i + 1)))) return false;
        if (p % PER == PER - 1 && turns) {
          slot_done(i++);
          if (MODE == GATE_BWD) slot_done(i++);
        }
        return true;
      }
      const float* b = bs + 16 * p;
      Pairs z, o;
      MC_EACH z[j] = add2(pair_of(cur[0], j), bias2(b, j));
      if (MODE == ACT_BWD || MODE == GATE_BWD) Act::both(z, o);
      else Act::value(z);
      uint32_t r0[8], r1[8];
      if (MODE == GATE) MC_EACH z[j] = mul2(z[j], add2(pair_of(cur[NL > 1 ? 1 : 0], j), bias2(b + BN, j)));
      if (MODE == GATE_BWD) MC_EACH {
        const float2 gh = pair_of(cur[NL > 2 ? 2 : 0], j), u = add2(pair_of(cur[NL > 1 ? 1 : 0], j), bias2(b + BN, j));
        o[j] = mul2(mul2(gh, u), o[j]);
        z[j] = mul2(gh, z[j]);
        r1[j] = pack_bf16x2(z[j].x, z[j].y);
      }
      const uint32_t j0 = p % PER * 2;
      const bool staged = !(MODE == LAYER && g.planes);
      if (p % PER == 0 && (staged || g.res)) {
        if (!slot_ready(i)) return false;
        if (MODE == GATE_BWD && !slot_ready(i + 1)) return false;
      }
      const uint32_t at[2] = {slot(i) + ((j0 << 4) ^ swizzle), slot(i) + (((j0 + 1) << 4) ^ swizzle)};
      if (MODE == ACT_BWD || (MODE == LAYER && g.res)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 r = lds16(at[h]);
          const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = make_float2(__uint_as_float(rw[e] << 16), __uint_as_float(rw[e] & 0xFFFF0000u));
            if (MODE == ACT_BWD) o[4 * h + e] = mul2(o[4 * h + e], f);
            else z[4 * h + e] = add2(z[4 * h + e], f);
          }
        }
      }
      if (!staged) {
        if (plane0 >= 0) {
          const int left = g.N - w.nt() * BN - 16 * p;
          bf16* to = g.planes + plane0 + 16ll * p * g.pd.S;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (j < left) to[(long long)j * g.pd.S] = __float2bfloat16_rn(j & 1 ? z[j / 2].y : z[j / 2].x);
        }
        if (g.res && p % PER == PER - 1) slot_done(i++);
        return true;
      }
      if (MODE == ACT_BWD || MODE == GATE_BWD) MC_EACH r0[j] = pack_bf16x2(o[j].x, o[j].y);
      else MC_EACH r0[j] = pack_bf16x2(z[j].x, z[j].y);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sts16(at[h], make_uint4(r0[4 * h], r0[4 * h + 1], r0[4 * h + 2], r0[4 * h + 3]));
        if (MODE == GATE_BWD)
          sts16(at[h] - slot(i) + slot(i + 1), make_uint4(r1[4 * h], r1[4 * h + 1], r1[4 * h + 2], r1[4 * h + 3]));
      }
      if (p % PER == PER - 1) {
        slot_done(i++);
        if (MODE == GATE_BWD) slot_done(i++);
      }
      return true;
    };
    fetch(v[0], 0);
#pragma unroll 1
    for (int p = 0; p < NP; p += 2)
      if (!step(0, p) || !step(1, p + 1)) return;
  }
}

// Read-out warps of a classifier: thread = pixel, 32 classes at a time (sixteen: 304 and 328 us instead of 297 and 294
// for 40 968 pixels x 10 242 classes x 256 channels).
// SCORE_SUM keeps the running maximum and sum of the tile's classes; SCORE_GRAD leaves bf16 gradients of the scores in the
// staged tiles.  Classes behind the last one have a bias of -infinity: exp makes zeros of them.
template <int MODE, int BN>
__device__ __forceinline__ void read_scores(const GemmArgs& g, int set, uint32_t rank, float* bias_s, uint32_t out0,
                                            uint32_t bfull, volatile int* abort_flag) {
  typedef Cfg<MODE, BN> C;
  constexpr int PW = 32, NP = BN / PW, PER = C::CW / PW;
#define MC_HALF _Pragma("unroll") for (int j = 0; j < PW / 2; ++j)
  const int lane = threadIdx.x % 32, q = threadIdx.x / 32 & 3, row = q * 32 + lane;
  const uint32_t mask = (1u << C::SLOT_BITS) - 1;
  const uint32_t at0 = out0 + (set << C::SLOT_BITS) * C::CH_BYTES + row * C::CW * 2, swizzle = (row & 7) << 4;
  const auto bar_of = [&](uint32_t base, uint32_t i) { return bfull + base + 32 * set + 8 * (i & mask); };
  const uint32_t tempty0 = of_leader(bfull + BAR_TEMPTY);
  // (few classes take narrow tiles; a test for them in the widest took 388 us instead of 315 for 40 968 pixels x 10 242 classes)
  const int second = BN == 64 ? g.sc.second : 0;
  float scale = 0.f;
  if (MODE == SCORE_GRAD) scale = g.sc.count ? (float)((double)*g.sc.grad / *g.sc.count) : *g.sc.grad;
  uint32_t it = 0, i = 0;
  // labels and what is kept of a tile are fetched a tile ahead
  long long t_next = 0;
  float top_next = INFINITY, rest_next = 0.f, miss_next = 0.f;
  const auto fetch_pixel = [&](const TileWalk& w) {
    const uint32_t p = (w.m() * 2 + rank) * TILE + row;
    if (!w.more() || p >= (uint32_t)g.rows) return;
    t_next = __ldg((const long long*)g.sc.target + p);
    if (MODE == SCORE_GRAD) top_next = __ldg(g.sc.kept.top + p), rest_next = __ldg(g.sc.kept.rest + p), miss_next = __ldg(g.sc.kept.miss + p);
  };
  fetch_pixel(TileWalk(g, set, 2));
  for (TileWalk w(g, set, 2); w.more(); w.next(), ++it) {
    float* bs = bias_s + set * 512 + (g.group == 1 ? 0 : (it & 1) * 256);
    const int n0 = w.nt() * BN;
    if (it == 0 || g.group != 1) {
      // (the other half is still being read by warps that are a tile behind; nobody is two behind)
      for (int e = row; e < BN; e += 128) {
        float b = n0 + e < g.N ? 0.f : -INFINITY;
        if (g.bias && n0 + e < g.N) b = __bfloat162float(__ushort_as_bfloat16(__ldg((const unsigned short*)g.bias + n0 + e)));
        if (g.sc.bias32 && n0 + e < g.N) b = __ldg(g.sc.bias32 + n0 + e);
        bs[e] = b;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bfull + BAR_BIASED + 8 * set);
      if (!warp_wait(bfull + BAR_BIASED + 8 * set, it & 1, abort_flag, 0x153)) return;  // (bounded, unlike bar.sync)
    }
    const int tile0 = (w.m() * 2 + rank) * TILE;
    const uint32_t p = tile0 + row;
    const bool in = p < (uint32_t)g.rows;
    int label = -1;  // of this tile's columns
    float kept = INFINITY, rest = 0.f, miss = 0.f;  // (kept: the largest score of all)
    if (in) {
      const long long t = t_next;
      if (t >= n0 && t < n0 + BN && t < g.N && t != g.sc.ignore) label = (int)(t - n0);
      if (MODE == SCORE_GRAD) kept = top_next, rest = rest_next, miss = miss_next;
    }
    TileWalk ahead = w;
    ahead.next();
    fetch_pixel(ahead);
    const bool dead = kept == INFINITY;
    int live = (g.N - n0 + PW - 1) / PW;  // pieces with classes; a staged tile is filled up with zeros
    if (MODE == SCORE_GRAD) live = second ? 1 : (live + PER - 1) / PER * PER;
    if (live > NP) live = NP;
    uint32_t v[2][PW];
    const uint32_t tile = 2 * it + set, acc = tile % C::NACC;
    const uint32_t t0 = ((uint32_t)(q * 32) << 16) + acc * C::ACC;
    if (!warp_wait(bfull + BAR_TFULL + 8 * acc, tile / C::NACC & 1, abort_flag, 0x151)) return;
    tc_fence_after_sync();
    float top = -INFINITY, sum = 0.f, hit = 0.f;
    const auto step = [&](int now, int pc) -> bool {
      uint32_t(&cur)[PW] = v[now];
      if (pc < live) tmem_ld_wait();
      if (pc + 1 < live) tmem_ld_32x32(t0 + PW * (pc + 1), v[now ^ 1]);
      if (pc + 1 == NP) {  // the accumulators are free
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_leader(tempty0 + 8 * acc);
      }
      const bool staged = MODE == SCORE_GRAD && !g.sc.gz;
      const bool turn = staged && pc % PER == 0, done = staged && pc % PER == PER - 1;
      if (turn && !warp_wait(bar_of(BAR_READY, i), i >> C::SLOT_BITS & 1, abort_flag, 0x152)) return false;
      if (pc < live) {
        float2 z[PW / 2];
        MC_HALF z[j] = add2(pair_of(cur, j), bias2(bs + PW * pc, j));
        // (a branch of the whole warp: few pieces hold a label of its pixels)
        const int here = (label >> 5) == pc ? label & 31 : -1;
        const bool any = __any_sync(~0u, here >= 0);
        if (MODE == SCORE_SUM) {
          if (any) MC_HALF hit = here == 2 * j ? z[j].x : here == 2 * j + 1 ? z[j].y : hit;
          float t[PW / 2];
          MC_HALF t[j] = fmaxf(z[j].x, z[j].y);
#pragma unroll
          for (int o = PW / 4; o; o /= 2)
#pragma unroll
            for (int j = 0; j < o; ++j) t[j] = fmaxf(t[j], t[j + o]);
          const float m = fmaxf(top, t[0]);
          const float base = m == -INFINITY ? 0.f : m;  // (nothing but ruled-out classes so far: sums of zeros)
          // (differences first: they lose nothing, and the largest score's exponential is one, its products with log2(e) rounded or not)
          sum *= exp2_((top - base) * LOG2E);
          MC_HALF z[j] = exp2_2(mul2(add2(z[j], two(-base)), two(LOG2E)));
#pragma unroll
          for (int o = PW / 4; o; o /= 2)
#pragma unroll
            for (int j = 0; j < o; ++j) z[j] = add2(z[j], z[j + o]);
          sum += z[0].x + z[0].y;
          top = m;
        } else {
          MC_HALF z[j] = exp2_2(fma2(add2(z[j], two(-kept)), two(LOG2E), two(-rest)));
          if (any) MC_HALF z[j] = make_float2(here == 2 * j ? miss : z[j].x, here == 2 * j + 1 ? miss : z[j].y);
          MC_HALF z[j] = dead ? two(0.f) : mul2(z[j], two(scale));
          if (staged) {
            const uint32_t at = at0 + (i & mask) * C::CH_BYTES, j0 = pc % PER * (PW / 8);
            uint32_t r[PW / 2];
            // gz is rounded to bf16 here for the products that read it.  More than 32 classes have this one part: gx and gW are then 0.20 % off
            // 64 bits and gb 0.30 % where the results' own rounding is 0.16 % (40 968 pixels x 10 242 classes; norms).  A second part
            // would double both products (475 us of 1207).  gb alone from the values before they are rounded, 32 columns of 32 pixels
            // added up by shuffles, 0.16 %, took 415 us instead of 320 here.
            MC_HALF r[j] = pack_bf16x2(z[j].x, z[j].y);
#pragma unroll
            for (int h = 0; h < PW / 8; ++h)
              if (!second || h < second) sts16(at + (((j0 + h) << 4) ^ swizzle), make_uint4(r[4 * h], r[4 * h + 1], r[4 * h + 2], r[4 * h + 3]));
            if (second) {  // (the first 32 columns are all there are)
              MC_HALF {
                z[j] = add2(z[j], make_float2(-__uint_as_float(r[j] << 16), -__uint_as_float(r[j] & 0xFFFF0000u)));
                r[j] = pack_bf16x2(z[j].x, z[j].y);
              }
#pragma unroll
              for (int h = 0; h < PW / 8; ++h)
                if (h < second)
                  sts16(at + (((second + h) << 4) ^ swizzle), make_uint4(r[4 * h], r[4 * h + 1], r[4 * h + 2], r[4 * h + 3]));
            }
          } else if (tile0 < g.rows) {
            // 64 bytes of this pixel's row in the block of each part
            bf16* to = g.sc.gz + (((long long)(tile0 / TILE) * g.y_across + (n0 + PW * pc) / KB) * TILE + row) * KB + PW * pc % KB;
#pragma unroll
            for (int part = 0; part < 3; ++part, to += (long long)(g.y_across / 3) * TILE * KB) {
              uint32_t r[PW / 2];
              MC_HALF {
                r[j] = pack_bf16x2(z[j].x, z[j].y);
                z[j] = add2(z[j], make_float2(-__uint_as_float(r[j] << 16), -__uint_as_float(r[j] & 0xFFFF0000u)));
              }
#pragma unroll
              for (int h = 0; h < PW / 8; ++h)
                *reinterpret_cast<uint4*>(to + 8 * h) = make_uint4(r[4 * h], r[4 * h + 1], r[4 * h + 2], r[4 * h + 3]);
            }
          }
        }
      }
      if (done) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_of(BAR_DONE, i));
        ++i;
      }
      return true;
    };
    tmem_ld_32x32(t0, v[0]);
#pragma unroll 1
    for (int pc = 0; pc < NP; pc += 2)
      if (!step(0, pc) || !step(1, pc + 1)) return;
    if (MODE == SCORE_SUM && in) {
      g.sc.part[(long long)w.nt() * g.rows + p] = make_float2(top, sum);
      if (label >= 0) g.sc.hit[p] = hit;
    }
  }
}
#undef MC_HALF

// Read-out warps of a product in float32: thread = pixel, sixteen columns at a time.
template <int BN>
__device__ __forceinline__ void read_floats(const GemmArgs& g, int set, uint32_t rank, uint32_t bfull, volatile int* abort_flag) {
  typedef Cfg<FLOATS, BN> C;
  const int lane = threadIdx.x % 32, q = threadIdx.x / 32 & 3, row = q * 32 + lane;
  const uint32_t tempty0 = of_leader(bfull + BAR_TEMPTY);
  uint32_t it = 0;
  for (TileWalk w(g, set, 2); w.more(); w.next(), ++it) {
    const uint32_t p = (w.m() * 2 + rank) * TILE + row, tile = 2 * it + set, acc = tile % C::NACC;
    const int n0 = w.nt() * BN, left = g.N - n0, live = left < BN ? (left + 15) / 16 : BN / 16;
    const bool in = p < (uint32_t)g.rows;
    long long step = 1;
    float* to = g.floats;
    if (in && g.ld) to += p * g.ld + n0;
    if (in && !g.ld) {
      uint32_t im, s;
      g.pd.split(p, im, s);
      to += ((long long)im * g.N + n0) * g.pd.S + s, step = g.pd.S;
    }
    if (!warp_wait(bfull + BAR_TFULL + 8 * acc, tile / C::NACC & 1, abort_flag, 0x161)) return;
    tc_fence_after_sync();
    const uint32_t t0 = ((uint32_t)(q * 32) << 16) + acc * C::ACC;
#pragma unroll 1
    for (int pc = 0; pc < live; ++pc) {
      uint32_t v[16];
      tmem_ld_32x16(t0 + 16 * pc, v);
      tmem_ld_wait();
      if (in) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (16 * pc + j < left) to[(16 * pc + j) * step] = __uint_as_float(v[j]);
      }
      __syncwarp();
    }
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) arrive_leader(tempty0 + 8 * acc);
  }
}

template <int MODE, int BN>
__global__ void __launch_bounds__(THREADS, 1) rows_tc_kernel(const __grid_constant__ GemmArgs g) {
  typedef Cfg<MODE, BN> C;
  constexpr bool PARTS = MODE == SCORE_SUM || MODE == SCORE_GRAD || MODE == FLOATS;  // can come in parts
  extern __shared__ unsigned char raw[];
  __shared__ volatile int abort_flag_s;
  unsigned char* sm = (unsigned char*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  volatile int* abort_flag = &abort_flag_s;
  const uint32_t out0 = smem_u32(sm);
  const uint32_t a0 = out0 + (2 << C::SLOT_BITS) * C::CH_BYTES;
  const uint32_t b0 = a0 + g.stages * A_BYTES;
  const uint32_t btile = g.kw * C::B0 + g.kb[1] * C::B1;  // a channel tile's weights
  const int bbytes = g.group ? g.group * btile : g.stages * C::BMAX;
  const uint32_t rank = cluster_rank();
  float* bias_s = (float*)(sm + (b0 - out0) + bbytes);  // two tiles' worth per set
  const uint32_t bar0 = smem_u32(bias_s + 4 * 256);
  uint32_t* tmem_s = (uint32_t*)((unsigned char*)(bias_s + 4 * 256) + ROWS_BARS * 8);
  const auto full = [&](uint32_t s) { return bar0 + 8 * s; };
  const auto empty = [&](uint32_t s) { return bar0 + 8 * (MAX_STAGES + s); };
  const uint32_t bfull = bar0 + 8 * (2 * MAX_STAGES);
  const auto tfull = [&](uint32_t s) { return bfull + BAR_TFULL + 8 * s; };
  const auto tempty = [&](uint32_t s) { return bfull + BAR_TEMPTY + 8 * s; };
  const auto ready = [&](int set, uint32_t s) { return bfull + BAR_READY + 8 * (4 * set + s); };
  const auto done = [&](int set, uint32_t s) { return bfull + BAR_DONE + 8 * (4 * set + s); };
  const uint32_t drain = bfull + BAR_DRAIN;
  const auto biased = [&](int set) { return bfull + BAR_BIASED + 8 * set; };

  if (threadIdx.x == 0) {
    abort_flag_s = 0;
    for (int i = 0; i < g.stages; ++i) mbar_init(full(i), 1), mbar_init(empty(i), 1);
    mbar_init(bfull, 1);
    mbar_init(drain, 1);
    for (int i = 0; i < C::NACC; ++i) {
      mbar_init(tfull(i), 1);
      mbar_init(tempty(i), 8);  // (the leader's: four warps of each block)
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(biased(i), 4);
      for (int s = 0; s < 4; ++s) mbar_init(ready(i, s), 1), mbar_init(done(i, s), 4);
    }
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) pair_alloc(smem_u32(tmem_s), 512);
  behind_previous_kernel();
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc_fence_after_sync();
  constexpr uint32_t tmem = 0;  // (all columns are allocated; a constant stays in uniform registers)

  if (warp == 0) {
    // ---- loader.  (Loader and MMA warp run converged, one elected lane issues: addresses and descriptors then live in
    // uniform registers.  In a branch of a single lane each of them is moved there for every instruction, and the
    // issuing thread, not the tensor core, sets the pace: 240 instead of 128 cycles per MMA of 256 columns.)
    const bool elected = elect_one();
    TileWalk w(g);
    if (g.group && w.more() && elected) {
      const uint32_t bar = of_leader(bfull);
      if (rank == 0) mbar_expect_tx(bfull, 2 * bbytes);
      uint32_t dst = b0;
      for (int n = 0; n < g.group; ++n)
        for (int seg = 0; seg < 2; ++seg)
          for (int k = 0; k < (seg ? g.kb[1] : g.kw); ++k) {
            load_b<MODE, BN>(g, seg, rank, dst, k * KB, (w.base + n) * BN, bar);
            dst += seg ? C::B1 : C::B0;
          }
    }
    __syncwarp();
    uint32_t st = 0, ph = 0;
    bool ok = true;
    for (; w.more() && ok; w.next()) {
      const int m0 = (w.m() * 2 + rank) * TILE, n0 = w.nt() * BN;
      for (int seg = 0; seg < 2 && ok; ++seg)
        for (int k = 0; k < g.kb[seg]; ++k) {
          ok = __all_sync(~0u, mbar_wait(empty(st), ph ^ 1, abort_flag, 0x101));
          if (!ok) break;
          if (elected) {
            const uint32_t bar = of_leader(full(st));
            if (rank == 0) mbar_expect_tx(full(st), 2 * (A_BYTES + (g.group ? 0 : seg ? C::B1 : C::B0)));
            const int across = MODE == LAYER || MODE == FLOATS ? g.a_across[seg] : 0;
            int ka = k, kb = k;
            if (PARTS && g.per && g.group) ka = pass_a(k / g.per) * g.per + k % g.per;
            else if (PARTS && g.per) ka = part_a(k / g.per) * g.per + k % g.per, kb = part_b(k / g.per) * g.per + k % g.per;
            tma_load_pair(a0 + st * A_BYTES, &g.a[seg], across ? 0 : ka * KB, across ? m0 * across + ka * TILE : m0, bar);
            if (!g.group) load_b<MODE, BN>(g, seg, rank, b0 + st * C::BMAX, kb * KB, n0, bar);
          }
          __syncwarp();
          if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
        }
    }
    // Every arrival that the leader's commits send here is waited for: a block that left before one came would have its
    // shared memory written behind it.
    for (int i = 0; i < g.stages && ok; ++i) {
      ok = __all_sync(~0u, mbar_wait(empty(st), ph ^ 1, abort_flag, 0x102));
      if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
    }
  } else if (warp == 1) {
    // ---- MMA issuer, in the leader only
    if (rank == 0) {
      const bool elected = elect_one();
      uint32_t st = 0, ph = 0;
      TileWalk w(g);
      uint32_t n = w.local_n();
      const uint32_t a_lo = desc_sw128_lo(a0, 16), b_lo = desc_sw128_lo(b0, 16);
      bool ok = true, there = false;
      if (g.group && w.more()) ok = __all_sync(~0u, mbar_wait(bfull, 0, abort_flag, 0x111));
      for (uint32_t it = 0; w.more() && ok; w.next(), ++it) {
        const uint32_t acc = it % C::NACC, aph = it / C::NACC & 1;
        ok = __all_sync(~0u, mbar_wait(tempty(acc), aph ^ 1, abort_flag, 0x112));
        if (!ok) break;
        tc_fence_after_sync();
        uint32_t bres = b_lo + n * (btile >> 4);
        if (++n == (uint32_t)g.group) n = 0;
#pragma unroll
        for (int seg = 0; seg < 2; ++seg) {
          constexpr uint32_t HI = desc_sw128_hi(1024);
          const uint32_t idesc = make_idesc_bf16(2 * TILE, seg ? C::N1 : C::N0, 0, 0);
          const uint32_t d = acc * C::ACC + (seg ? C::OFF1 : 0);
          int pass = 0, kp = 0;  // of the first operand, where it passes several times; stage of the pass
          for (int k = 0; k < g.kb[seg]; ++k) {
            if (!there) {
              ok = __all_sync(~0u, mbar_wait(full(st), ph, abort_flag, 0x113));
              if (!ok) break;
            }
            const bool passes = PARTS && g.per && g.group;
            const uint32_t cur = st, ad = a_lo + st * (A_BYTES >> 4);
            const uint32_t bd = !g.group ? b_lo + st * (C::BMAX >> 4)
                                         : passes ? bres + (pass_b(pass) * g.per + kp) * (C::B0 >> 4) : bres;
            if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
            const bool next = mbar_test(full(st), ph);
            if (elected) {
#pragma unroll
              for (int j = 0; j < 4; ++j)  // sixteen channels, 32 bytes each
                pair_mma(d, ad + 2 * j, HI, bd + 2 * j, HI, idesc, (k | j) != 0 || (seg && C::OFF1 == 0));
              if (passes && pass_twice(pass)) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  pair_mma(d, ad + 2 * j, HI, bd - g.per * (C::B0 >> 4) + 2 * j, HI, idesc, true);
              }
              pair_commit(empty(cur));
            }
            if (!passes) bres += (seg ? C::B1 : C::B0) >> 4;
            else if (++kp == g.per) kp = 0, ++pass;
            there = __all_sync(~0u, next);
          }
          if (!ok) break;
        }
        if (ok && elected) pair_commit(tfull(acc));
        __syncwarp();
      }
      if (elected) {
        leader_commit(drain);  // (nobody in the other block waits for it)
        mbar_wait(drain, 0, abort_flag, 0x114);
      }
      __syncwarp();
    }
  } else if (warp < 4) {
    // ---- I/O of one set's staged tiles: fill the slots ahead (residual), store what the read-out warps leave in them
    if (lane == 0 && MODE != SCORE_SUM && MODE != FLOATS && !(MODE == SCORE_GRAD && g.sc.gz) &&
        !(MODE == LAYER && g.planes && !g.res)) {
      const int set = warp - 2;
      TileWalk lead(g, set, 2);
      int lead_c = 0;
      uint32_t lead_i = 0;
      const uint32_t buf = out0 + (set << C::SLOT_BITS) * C::CH_BYTES, slots = 1u << C::SLOT_BITS;
      const auto column = [&](const TileWalk& w, int c) { return w.nt() * BN + (MODE == GATE_BWD ? c / 2 : c) * C::CW; };
      const auto advance = [&]() {
        if (!lead.more()) return;
        const uint32_t s = lead_i & (slots - 1);
        const int col = column(lead, lead_c);
        if (g.res && col < g.N && (lead.m() * 2 + rank) * TILE < g.rows) {
          mbar_expect_tx(ready(set, s), C::CH_BYTES);
          tma_load(buf + s * C::CH_BYTES, &g.r, col, (lead.m() * 2 + rank) * TILE, ready(set, s));
        } else {
          mbar_arrive(ready(set, s));
        }
        ++lead_i;
        if (++lead_c == C::NCH) lead_c = 0, lead.next();
      };
      for (int i = 0; i < (int)slots; ++i) advance();
      bool ok = true;
      uint32_t i = 0;
      for (TileWalk w(g, set, 2); w.more() && ok; w.next())
        for (int c = 0; c < C::NCH; ++c, ++i) {
          const uint32_t s = i & (slots - 1);
          ok = mbar_wait(done(set, s), i >> C::SLOT_BITS & 1, abort_flag, 0x121);
          if (!ok) break;
          const int col = column(w, c), m0 = (w.m() * 2 + rank) * TILE;
          if (col < g.N && m0 < g.rows && !(MODE == LAYER && g.planes)) {
            if (MODE == SCORE_GRAD && g.y_across) tma_store(&g.y[0], 0, m0 * g.y_across + col / KB * TILE, buf + s * C::CH_BYTES);
            else tma_store(&g.y[MODE == GATE_BWD ? c % 2 : 0], col, m0, buf + s * C::CH_BYTES);
            bulk_commit();
            bulk_wait_read();
          }
          advance();
        }
      bulk_wait_all();
    }
    __syncwarp();
  } else {
    // ---- read-out
    if constexpr (MODE == SCORE_SUM || MODE == SCORE_GRAD) {
      read_scores<MODE, BN>(g, (warp - 4) / 4, rank, bias_s, out0, bfull, abort_flag);
    } else if constexpr (MODE == FLOATS) {
      read_floats<BN>(g, (warp - 4) / 4, rank, bfull, abort_flag);
    } else {
      with_act(g.act, [&](auto act) {
        read_out<MODE, BN, decltype(act)>(g, (warp - 4) / 4, rank, bias_s, out0, bfull, abort_flag);
      });
    }
  }
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {  // given up: copies still in flight land within microseconds
    const long long c = clock64();
    while (clock64() - c < 4000000) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();  // (no block leaves while the other's MMAs, copies or arrivals still reach it)
  if (warp == 1) pair_dealloc(tmem, 512);
}

// ---- outer kernel ----------------------------------------------------------------------------------------
struct alignas(64) OuterTcArgs {
  CUtensorMap g[2], x;
  float *part, *csum;  // [split][M total][ldn], [split][M total]
  int M, segs, N, ldn; // rows of one of the (one or two) first operands
  int m_tiles, n_tiles;
  int kblocks, per;    // 64-pixel blocks in all, and of a share
  int stages;
  int across;          // blocks next to each other where the first operand lies in blocks, else 0
  int g_part, x_part;  // columns from part to part
};
constexpr int OUTER_BARS = 3 * MAX_STAGES + 1;

// MT: groups of 2 x 128 channels of the first operand, BN: channels of the second.  A block holds half of either.
// PARTS: of values in three parts.  A stage has all parts of both operands (each was fetched for each product before: 82 us instead of
// 58 for 131 072 pixels, 99 x 50 channels), and the five small products have an accumulator of their own.
template <int MT, int BN, bool PARTS>
__global__ void __launch_bounds__(THREADS, 1) outer_tc_kernel(const __grid_constant__ OuterTcArgs g) {
  constexpr int NP = PARTS ? 3 : 1, GB = MT * A_BYTES, XB = BN / 2 * 128, STAGE = NP * (GB + XB), COLS = MT * BN * (PARTS ? 2 : 1);
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
  const auto landed = [&](uint32_t s) { return bar0 + 8 * (2 * MAX_STAGES + s); };  // (full is the leader's alone)
  const uint32_t done = bar0 + 24 * MAX_STAGES;
  const int tiles = g.segs * g.m_tiles * g.n_tiles;
  const uint32_t rank = cluster_rank();
  const int split = blockIdx.x / 2 / tiles, tile = blockIdx.x / 2 % tiles;
  const int nt = tile % g.n_tiles, mt = tile / g.n_tiles % g.m_tiles, seg = tile / g.n_tiles / g.m_tiles;
  // channel group m of this block starts at m0 + 256 m
  const int m0 = mt * MT * 256 + rank * 128, n0 = nt * BN;
  const int k0 = split * g.per, k1 = min(g.kblocks, k0 + g.per), steps = k1 > k0 ? k1 - k0 : 0;
  const bool sums = nt == 0;

  if (threadIdx.x == 0) {
    abort_flag_s = 0;
    for (int i = 0; i < g.stages; ++i) mbar_init(full(i), 1), mbar_init(landed(i), 1), mbar_init(empty(i), sums ? 9 : 1);
    mbar_init(done, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) pair_alloc(smem_u32(&tmem_s), COLS);
  behind_previous_kernel();
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_s;

  if (warp == 0) {  // (converged, one elected lane issues: see the rows kernel)
    const bool elected = elect_one();
    uint32_t st = 0, ph = 0;
    bool ok = true;
    // Boxes of 64 channels without a channel are not fetched: whatever lies there makes sums that nobody reads.  (But one of either
    // block always is: the leader must not take up a stage that the other block's warps have not left yet.)
    const auto has_g = [&](int i, int r) { return i == 0 || mt * MT * 256 + r * 128 + i / 2 * 256 + i % 2 * 64 < g.M; };
    const auto has_x = [&](int i, int r) { return n0 + r * (BN / 2) + 64 * i < g.N; };
    int boxes = 0;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) boxes += has_g(i, r);
#pragma unroll
      for (int i = 0; i < BN / 128; ++i) boxes += has_x(i, r);
    }
    for (int k = k0; k < k0 + steps && ok; ++k) {
      ok = __all_sync(~0u, mbar_wait(empty(st), ph ^ 1, abort_flag, 0x141));
      if (!ok) break;
      if (elected) {
        const uint32_t bar = of_leader(full(st)), dst = s0 + st * STAGE;
        const int row = k * KB;
        if (rank == 0) mbar_expect_tx(full(st), boxes * NP * 8192);
#pragma unroll
        for (int part = 0; part < NP; ++part) {
#pragma unroll
          for (int i = 0; i < 2 * MT; ++i) {
            const int col = part * g.g_part + m0 + i / 2 * 256 + i % 2 * 64;
            const uint32_t to = dst + part * GB + i * 8192;
            if (!has_g(i, rank)) continue;
            if (g.across) tma_load_pair(to, &g.g[seg], 0, (row / TILE * g.across + col / KB) * TILE + row % TILE, bar);
            else tma_load_pair(to, &g.g[seg], col, row, bar);
          }
#pragma unroll
          for (int i = 0; i < BN / 128; ++i)
            if (has_x(i, rank))
              tma_load_pair(dst + NP * GB + part * XB + i * 8192, &g.x, part * g.x_part + n0 + rank * (BN / 2) + 64 * i, row, bar);
        }
      }
      __syncwarp();
      if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
    }
    for (int i = 0; i < g.stages && ok; ++i) {  // (no arrival of the leader's commits is left behind)
      ok = __all_sync(~0u, mbar_wait(empty(st), ph ^ 1, abort_flag, 0x145));
      if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool elected = elect_one();
      constexpr uint32_t idesc = make_idesc_bf16(256, BN, 1, 1), HI = desc_sw128_hi(1024);
      uint32_t st = 0, ph = 0;
      bool there = false;
      for (int i = 0; i < steps; ++i) {
        if (!there && !__all_sync(~0u, mbar_wait(full(st), ph, abort_flag, 0x142))) break;
        const uint32_t cur = st;
        if (++st == (uint32_t)g.stages) st = 0, ph ^= 1;
        const bool next = mbar_test(full(st), ph);
        if (elected) {
          const uint32_t bd = desc_sw128_lo(s0 + cur * STAGE + NP * GB, 8192), ad = desc_sw128_lo(s0 + cur * STAGE, 8192);
#pragma unroll
          for (int t = 0; t < (PARTS ? PRODUCTS : 1); ++t) {
            const int pa = PARTS ? part_a(t) * (GB >> 4) : 0, pb = PARTS ? part_b(t) * (XB >> 4) : 0;
            const bool small = PARTS && t + 1 < PRODUCTS, more = PARTS && t > 0 && small;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int j = 0; j < 4; ++j)  // sixteen pixels each
                pair_mma(tmem + (small ? MT * BN : 0) + m * BN, ad + pa + m * (A_BYTES >> 4) + 128 * j, HI, bd + pb + 128 * j, HI, idesc,
                         i != 0 || j != 0 || more);
          }
          pair_commit(empty(cur));
          if (sums) pair_commit(landed(cur));
        }
        there = __all_sync(~0u, next);
      }
      if (elected) pair_commit(done);
      __syncwarp();
    }
  } else if (warp >= 4) {
    const int ew = warp - 4, q = warp & 3;
    bool ok = true;
    if (sums) {
      // columns of the first operand: 2 MT 16-byte pieces (8 channels each) per warp, 16 / MT pixels at a time
      constexpr int PC = 2 * MT, PX = 32 / PC;
      const int piece = ew * PC + lane % PC, box = piece / 8, j = piece % 8;
      float acc[8] = {};
      uint32_t st = 0, ph = 0;
      for (int i = 0; i < steps; ++i) {
        ok = warp_wait(landed(st), ph, abort_flag, 0x143);
        if (!ok) break;
        const uint32_t base = s0 + st * STAGE + box * 8192;
#pragma unroll
        for (int part = NP - 1; part >= 0; --part) {
#pragma unroll
          for (int p = lane / PC; p < KB; p += PX) {
            const uint4 r = lds16(base + part * GB + p * 128 + ((j ^ (p & 7)) << 4));
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              acc[2 * e] += __uint_as_float(w[e] << 16);
              acc[2 * e + 1] += __uint_as_float(w[e] & 0xFFFF0000u);
            }
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
        const int m = m0 + piece / 16 * 256 + piece % 16 * 8 + e;
        if (lane < PC && m < g.M) g.csum[((size_t)split * g.segs + seg) * g.M + m] = acc[e];
      }
    }
    if (ok) ok = warp_wait(done, 0, abort_flag, 0x144);
    if (ok && steps) {
      tc_fence_after_sync();
#pragma unroll 1
      for (int t = ew / 4; t < MT * BN / 32; t += 2) {  // 32 columns each
        uint32_t v[32];
        tmem_ld_32x32(tmem + ((uint32_t)(q * 32) << 16) + t * 32, v);
        if (PARTS) {
          uint32_t small[32];
          tmem_ld_32x32(tmem + ((uint32_t)(q * 32) << 16) + MT * BN + t * 32, small);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(small[j]));
        } else {
          tmem_ld_wait();
        }
        const int m = m0 + t * 32 / BN * 256 + q * 32 + lane, n = n0 + t * 32 % BN;
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
  cluster_sync();
  if (warp == 1) pair_dealloc(tmem, COLS);
}

// ---- host ------------------------------------------------------------------------------------------------
// boxes of 64 channels x box_r rows, 128-byte swizzle (32 channels: 64-byte)
static bool encode(CUtensorMap* tm, const TcRows& t, int box_r, int box_c = KB) {
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
  cuuint64_t dims[2] = {(cuuint64_t)t.cols, (cuuint64_t)t.rows}, strides[1] = {(cuuint64_t)t.ld * 2};
  if (t.parts > 1) dims[0] = (cuuint64_t)t.across() * KB;
  if (t.blocks) dims[0] = KB, dims[1] = t.block_bytes() / (KB * 2), strides[0] = KB * 2;
  const cuuint32_t box[2] = {(cuuint32_t)box_c, (cuuint32_t)box_r}, es[2] = {1, 1};
  for (int attempt = 0; attempt < 2; ++attempt) {
    if (((Encode)f)(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(t.p), dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, box_c == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
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
// Once per kernel and device: the limit belongs to the kernel, not to a call.
template <auto kern>
static bool allow_smem() {
  static std::atomic<uint64_t> done{0};  // a bit per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

// Blocks in clusters of two.
template <auto kern, typename Args>
static int launch_pairs(unsigned pairs, size_t smem, const Args& args, cudaStream_t st) {
  if (!allow_smem<kern>()) return MC_ERR_LAUNCH;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, args) != cudaSuccess) return MC_ERR_LAUNCH;
  MC_COUNT(1);
  return MC_OK;
}

struct RowsPlan {
  int bn, n_tiles, group, stages;
  unsigned pairs;  // of blocks that are launched
  size_t smem;
};
template <int MODE, int BN>
static RowsPlan plan_rows(int m_pairs, int N, int kb0, int kb1, int sms, int kw = 0) {  // kw: stages of the first weights that stay, if not kb0
  typedef Cfg<MODE, BN> C;
  RowsPlan p{};
  p.bn = BN;
  p.n_tiles = (N + BN - 1) / BN;
  const int fixed_bytes = 1024 + 4 * 256 * 4 + ROWS_BARS * 8 + 16 + 64;
  const int b_tile = (kw ? kw : kb0) * C::B0 + kb1 * C::B1, pairs = sms / 2;
  const int left = SMEM_LIMIT - fixed_bytes - (2 << C::SLOT_BITS) * C::CH_BYTES;
  // Weights stay in shared memory where at least three stages of pixels fit beside them.  us at 655 488 pixels, weights that
  // stay / that travel: without activation 96 -> 96 channels 63 / 70, 64 -> 64 49.6 / 50.4, 128 -> 256 114 / 113; ReLU and
  // residual 128 -> 256 167 / 166, 256 -> 256 180 / 183; GELU 64 -> 64 63 / 66, 256 -> 256 198 / 197, 320 -> 320 312 / 277,
  // 192 -> 768 559 / 539; the gate with 64 -> 64 -> 64 108 / 111, 256 -> 1024 -> 256 1092 / 1114, 128 -> 512 -> 128 482 / 484.
  // Few channels gain, three channel tiles lose: groups of pairs leave two pairs idle, several tiles a pair round its share
  // up (72 -> 328 at 40 962 pixels: 30.5 / 25.7).
  // How many channel tiles a pair keeps: the number that leaves the fewest pairs without work; fewer than four stages count
  // as 7 % of them (128 -> 768, one tile with seven stages / three tiles with three: 322 / 320, GELU 544 / 526; 256 -> 384
  // 227 / 234, GELU 310 / 316).  The gate's gradients, two operands of pixels and small tiles, need the room for stages (256 ->
  // 1024 channels, 163 872 pixels: 380 us, 451 us with weights that stay).
  // Where a pair has a tile or two only, weights that stay are weights that are waited for (2 562 pixels, 680 -> 256
  // channels, 44 tiles: 11.6 us, 9.0 us if they travel with the pixels; 128 -> 512, 88 tiles: 9.7 and 6.9; the gate with
  // 64 -> 256 channels, 82 tiles: 18.8 and 20.5 for the block).
  const bool stay = MODE != GATE_BWD && (long long)m_pairs * p.n_tiles > (MODE == GATE ? 1 : 2) * pairs;
  // (a classifier's many channel tiles seldom divide the pairs: 41 tiles kept by 41 of 74 pairs took 1.7 times as long)
  double best = MODE == SCORE_SUM || MODE == SCORE_GRAD ? 0.95 : 0;
  for (int group = 1; stay && group <= p.n_tiles; ++group) {
    const int groups = p.n_tiles / group;
    if (p.n_tiles % group || groups > pairs) continue;
    if ((long long)group * b_tile + 3 * A_BYTES > left) break;
    const int stages = (left - group * b_tile) / A_BYTES;
    const double used = (double)(pairs / groups * groups) / pairs * (stages >= 4 ? 1.0 : 0.93);
    if (used > best + 1e-9) best = used, p.group = group;
  }
  p.stages = p.group ? (left - p.group * b_tile) / A_BYTES : left / (A_BYTES + C::BMAX);
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  p.smem = fixed_bytes + (2 << C::SLOT_BITS) * C::CH_BYTES + (size_t)p.stages * A_BYTES +
                      (p.group ? p.group * b_tile : p.stages * C::BMAX);
  long long n;
  if (p.group) {
    const int groups = p.n_tiles / p.group;
    n = pairs / groups;
    if (n > m_pairs) n = m_pairs;
    n *= groups;
  } else {
    n = (long long)m_pairs * p.n_tiles;
    if (n > pairs) n = pairs;
  }
  p.pairs = (unsigned)n;
  return p;
}

template <int MODE, int BN>
static int launch_rows(GemmArgs& g, cudaStream_t st) {
  const RowsPlan p = plan_rows<MODE, BN>(g.m_pairs, g.N, g.kb[0], g.kb[1], sm_total(), 3 * g.per);
  g.n_tiles = p.n_tiles, g.group = p.group, g.stages = p.stages;
  g.kw = g.per ? 3 * g.per : g.kb[0];
  if (g.per && g.group) g.kb[0] = PASSES * g.per;
  return launch_pairs<rows_tc_kernel<MODE, BN>>(p.pairs, p.smem, g, st);
}

// Channels of a tile, for `pairs` pixel tiles, n channels, kb stages: the least estimated time.  A tile costs its MMAs
// (half a cycle per column and 16 channels, not less than its stages' hand-over), its read-out and a start; many pixels
// want wide tiles, few pixels so many tiles that every pair of blocks has one (680 -> 256 channels at 2 562 pixels, 11
// pixel tiles: 9.8 us with tiles of 64, 15.6 with 256).  Against the best of the three widths, at 642 to 655 488 pixels and
// eleven pairs of channel counts from 16 -> 8 to 1024 -> 1024: 1.7 % more time on average, at most 23 % (10 242 pixels, 64 ->
// 160: 9.6 us with 128, 7.8 with 64), 9 - 19 % for seven shapes of 10 242 and 40 962 pixels that take 256 where 128 is faster.
static int tile_width(long long pairs, int n, int kb, int sms) {
  const int all = sms / 2;
  int best = 64;
  double least = 1e300;
  for (int w = 64; w <= 256; w *= 2) {
    const double tiles = (double)pairs * ((n + w - 1) / w), waves = tiles <= all ? 1 : tiles / all;
    const double t = waves * (1500 + kb * (w > 150 ? 2.0 * w : 300.0) + 16.0 * w);
    if (t < least) least = t, best = w;
  }
  return best;
}
// The same for a long sum over a classifier's classes: a tile is nothing but its MMAs then, and a last wave that is not full
// counts in whole.  (Narrow tiles read more of the pixels for each MMA.)
static int long_tile_width(long long pairs, int n, int sms) {
  const int all = sms / 2;
  int best = 64;
  double least = 1e300;
  for (int w = 64; w <= 256; w *= 2) {
    const long long tiles = pairs * ((n + w - 1) / w);
    const double t = (double)((tiles + all - 1) / all) * (w > 150 ? w : w > 100 ? 1.15 * w : 1.6 * w);
    if (t < least) least = t, best = w;
  }
  return best;
}
static int kblocks(int c) { return (c + KB - 1) / KB; }

static GemmArgs base_args(const TcRows& a, const TcRows& y, const bf16* bias, int act) {
  GemmArgs g{};
  g.bias = bias;
  g.rows = (int)a.rows;
  g.m_pairs = (int)((a.rows + 2 * TILE - 1) / (2 * TILE));
  g.N = y.cols;
  g.kb[0] = kblocks(a.cols);
  g.act = act;
  return g;
}
template <int MODE>
static int launch_wide(GemmArgs& g, int bn, cudaStream_t st) {
  if (bn == 64) return launch_rows<MODE, 64>(g, st);
  if (bn == 128) return launch_rows<MODE, 128>(g, st);
  return launch_rows<MODE, 256>(g, st);
}

int tc_layer(const TcRows& a, const TcRows& w, const bf16* bias, int act, const TcRows& r, const TcRows& y,
             bool backward, cudaStream_t st) {
  GemmArgs g = base_args(a, y, bias, act);
  g.res = r.p != nullptr;
  const int bn = tile_width(g.m_pairs, y.cols, g.kb[0], sm_total());
  if (!encode(&g.a[0], a, TILE) || !encode(&g.b[0], w, bn / 2)) return MC_ERR_LAUNCH;
  if (y.ld == 0) g.planes = (bf16*)y.p, g.pd = PixDiv((uint32_t)y.S);
  else if (!encode(&g.y[0], y, TILE)) return MC_ERR_LAUNCH;
  if (g.res && !encode(&g.r, r, TILE)) return MC_ERR_LAUNCH;
  return backward ? launch_wide<ACT_BWD>(g, bn, st) : launch_wide<LAYER>(g, bn, st);
}

int tc_input_grad(const TcRows& g0, const TcRows& w0, const TcRows& g1, const TcRows& w1, const TcRows& gx,
                  cudaStream_t st) {
  GemmArgs g = base_args(g0, gx, nullptr, MC_ACT_NONE);
  if (g1.p) g.kb[1] = kblocks(g1.cols);
  if (g0.blocks) g.a_across[0] = g0.across();
  const int bn = g0.blocks ? long_tile_width(g.m_pairs, gx.cols, sm_total())
                           : tile_width(g.m_pairs, gx.cols, g.kb[0] + g.kb[1], sm_total());
  if (!encode(&g.a[0], g0, TILE) || !encode(&g.b[0], w0, bn / 2)) return MC_ERR_LAUNCH;
  if (gx.ld == 0) g.planes = (bf16*)gx.p, g.pd = PixDiv((uint32_t)gx.S);
  else if (!encode(&g.y[0], gx, TILE)) return MC_ERR_LAUNCH;
  if (g1.p && (!encode(&g.a[1], g1, TILE) || !encode(&g.b[1], w1, bn / 2))) return MC_ERR_LAUNCH;
  return launch_wide<LAYER>(g, bn, st);
}

static int stages_of(const TcRows& a) { return a.parts > 1 ? PRODUCTS * a.part_blocks() : kblocks(a.cols); }
int tc_scores_tiles(long long P, int C, int V, int parts) {
  const int bn = tile_width((P + 2 * TILE - 1) / (2 * TILE), V, stages_of(TcRows{nullptr, P, C, 0, 0, false, parts}), sm_total());
  return (V + bn - 1) / bn;
}
static GemmArgs score_args(const TcRows& x, int classes, const bf16* bias, const Scores& s) {
  GemmArgs g = base_args(x, TcRows{nullptr, x.rows, classes, 0}, bias, MC_ACT_NONE);
  g.sc = s;
  g.kb[0] = stages_of(x);
  if (x.parts > 1) g.per = x.part_blocks();
  return g;
}
int tc_scores_sum(const TcRows& x, const TcRows& w, const bf16* bias, const Scores& s, cudaStream_t st) {
  GemmArgs g = score_args(x, (int)w.rows, bias, s);
  const int bn = tile_width(g.m_pairs, g.N, g.kb[0], sm_total());
  if (!encode(&g.a[0], x, TILE) || !encode(&g.b[0], w, bn / 2)) return MC_ERR_LAUNCH;
  return launch_wide<SCORE_SUM>(g, bn, st);
}
int tc_scores_grad(const TcRows& x, const TcRows& w, const bf16* bias, const Scores& s, const TcRows& gz, cudaStream_t st) {
  GemmArgs g = score_args(x, (int)w.rows, bias, s);
  g.y_across = gz.blocks ? gz.across() : 0;
  if (gz.parts > 1) g.sc.gz = (bf16*)const_cast<void*>(gz.p);
  const int bn = s.second ? 64 : tile_width(g.m_pairs, g.N, g.kb[0], sm_total());
  if (!encode(&g.a[0], x, TILE) || !encode(&g.b[0], w, bn / 2) || (!g.sc.gz && !encode(&g.y[0], gz, TILE))) return MC_ERR_LAUNCH;
  return launch_wide<SCORE_GRAD>(g, bn, st);
}
int tc_input_grad32(const TcRows& gz, const TcRows& w, float* gx, long long ld, long long S, cudaStream_t st) {
  GemmArgs g = base_args(gz, TcRows{nullptr, gz.rows, (int)w.rows, 0}, nullptr, MC_ACT_NONE);
  g.kb[0] = stages_of(gz), g.per = gz.part_blocks(), g.a_across[0] = gz.across();
  g.floats = gx, g.ld = ld;
  if (!ld) g.pd = PixDiv((uint32_t)S);
  const int bn = long_tile_width(g.m_pairs, g.N, sm_total());
  if (!encode(&g.a[0], gz, TILE) || !encode(&g.b[0], w, bn / 2)) return MC_ERR_LAUNCH;
  return launch_wide<FLOATS>(g, bn, st);
}

// 128 hidden channels a tile of the gate, 64 where that pads less: 38 hidden channels take half the time (wide blocks 4 % more)
static int gate_width(int hidden) { return hidden <= 256 && (hidden + 63) / 64 % 2 ? 64 : 128; }

int tc_gate(const TcRows& x, const TcRows& w_in, const bf16* b_in, int act, const TcRows& h, cudaStream_t st) {
  GemmArgs g = base_args(x, h, b_in, act);
  g.up = h.cols;
  const int wide = gate_width(h.cols);
  if (!encode(&g.a[0], x, TILE) || !encode(&g.b[0], w_in, wide) || !encode(&g.y[0], h, TILE)) return MC_ERR_LAUNCH;
  return wide == 64 ? launch_rows<GATE, 64>(g, st) : launch_rows<GATE, 128>(g, st);
}

int tc_gate_bwd(const TcRows& x, const TcRows& w_in, const bf16* b_in, int act, const TcRows& gy, const TcRows& w_out_t,
                const TcRows& gg, const TcRows& gu, cudaStream_t st) {
  GemmArgs g = base_args(x, gg, b_in, act);
  g.up = gg.cols;
  g.kb[1] = kblocks(gy.cols);
  if (!encode(&g.a[0], x, TILE) || !encode(&g.b[0], w_in, 64) || !encode(&g.a[1], gy, TILE) ||
      !encode(&g.b[1], w_out_t, 32) || !encode(&g.y[0], gg, TILE, 32) || !encode(&g.y[1], gu, TILE, 32))
    return MC_ERR_LAUNCH;
  return launch_rows<GATE_BWD, 64>(g, st);
}

// Blocks per gradient tile: as many as fill the SMs once or a whole number of times with equal shares, of 2^17 pixels at most:
// the accumulators truncate, up to 2^-23 of the sum for every sixteen pixels, which does not cancel where all terms have one
// sign (2^30 pixels, 8 x 8 channels: 9 % off with 74 shares; 2^17 pixels: 2^-10, a quarter of half a bf16 step).
constexpr int MOST_PER = (1 << 17) / KB;
struct OuterPlan {
  int mt, bn, m_tiles, n_tiles, splits, per;
};
// Of float32 values in parts: 2^10 pixels, 2^-18 of a sum of one sign at most.
constexpr int MOST_PER_PARTS = (1 << 10) / KB;
static OuterPlan outer_plan(long long P, int M, int segs, int N, int sms, int parts = 1) {
  OuterPlan p;
  p.mt = M > 256 && parts == 1 ? 2 : 1;  // (stages of parts are large)
  p.bn = N <= 128 ? 128 : 256;
  p.m_tiles = (M + 256 * p.mt - 1) / (256 * p.mt);
  p.n_tiles = (N + p.bn - 1) / p.bn;
  const long long tiles = (long long)segs * p.m_tiles * p.n_tiles, kb = (P + KB - 1) / KB;
  double best = 1e30;
  const int pairs = sms / 2;
  const int most_per = parts > 1 ? MOST_PER_PARTS : MOST_PER, products = parts > 1 ? PRODUCTS : 1;
  const long long least = (kb + most_per - 1) / most_per;
  p.splits = 1, p.per = (int)kb;
  for (long long s = least; s < least + pairs && s <= (kb + 3) / 4; ++s) {
    const long long per = (kb + s - 1) / s;
    const double waves = (double)((tiles * s + pairs - 1) / pairs);
    // a pair's stages, and what it costs to write its sums and to add them up again (against eight other numbers of shares,
    // at 642 to 655 488 pixels and ten pairs of channel counts: 1.6 % more time on average, at most 10 %)
    const double t = waves * (products * per + 8.0) + 0.05 * tiles * s;
    if (t < best) best = t, p.splits = (int)((kb + per - 1) / per), p.per = (int)per;
  }
  return p;
}
size_t tc_outer_floats(long long P, int M, int segs, int N, int* splits, int* ldn, int parts) {
  const OuterPlan p = outer_plan(P, M, segs, N, sm_total(), parts);
  *splits = p.splits;
  *ldn = (N + 3) / 4 * 4;
  return (size_t)p.splits * segs * M * *ldn;
}

template <int MT, int BN, bool PARTS>
static int launch_outer(OuterTcArgs& g, const OuterPlan& p, cudaStream_t st) {
  constexpr int STAGE = (PARTS ? 3 : 1) * (MT * A_BYTES + BN / 2 * 128);
  g.stages = (SMEM_LIMIT - 2048) / STAGE;
  if (g.stages > MAX_STAGES) g.stages = MAX_STAGES;
  return launch_pairs<outer_tc_kernel<MT, BN, PARTS>>(g.segs * p.m_tiles * p.n_tiles * p.splits, 1024 + g.stages * STAGE, g, st);
}
int tc_outer(const TcRows& g0, const TcRows& g1, const TcRows& x, float* part, float* csum, cudaStream_t st) {
  OuterTcArgs g{};
  g.segs = g1.p ? 2 : 1;
  g.across = g0.blocks ? g0.across() : 0;
  const OuterPlan p = outer_plan(x.rows, g0.cols, g.segs, x.cols, sm_total(), g0.parts);
  g.g_part = g0.part_blocks() * KB, g.x_part = x.part_blocks() * KB;
  if (!encode(&g.g[0], g0, KB) || (g1.p && !encode(&g.g[1], g1, KB)) || !encode(&g.x, x, KB)) return MC_ERR_LAUNCH;
  g.part = part, g.csum = csum;
  g.M = g0.cols, g.N = x.cols, g.ldn = (x.cols + 3) / 4 * 4;
  g.m_tiles = p.m_tiles, g.n_tiles = p.n_tiles;
  g.kblocks = (int)((x.rows + KB - 1) / KB), g.per = p.per;
  if (g0.parts > 1) return p.bn == 128 ? launch_outer<1, 128, true>(g, p, st) : launch_outer<1, 256, true>(g, p, st);
  if (p.mt == 1) return p.bn == 128 ? launch_outer<1, 128, false>(g, p, st) : launch_outer<1, 256, false>(g, p, st);
  return p.bn == 128 ? launch_outer<2, 128, false>(g, p, st) : launch_outer<2, 256, false>(g, p, st);
}

// ---- what the rules above choose ------------------------------------------------------------------------------
template <int MODE>
static RowsPlan plan_wide(int m_pairs, int N, int kb0, int kb1, int sms) {
  const int bn = tile_width(m_pairs, N, kb0 + kb1, sms);
  return bn == 64 ? plan_rows<MODE, 64>(m_pairs, N, kb0, kb1, sms)
         : bn == 128 ? plan_rows<MODE, 128>(m_pairs, N, kb0, kb1, sms) : plan_rows<MODE, 256>(m_pairs, N, kb0, kb1, sms);
}
bool tc_plan(const mc_mix_desc* d, int product, int sms, int32_t* out) {
  if (sms == 0) sms = sm_total();
  const long long P = d->B * d->S;
  const int m = (int)((P + 2 * TILE - 1) / (2 * TILE)), H = d->hidden;
  const int ki = kblocks(d->C_in), ko = kblocks(d->C_out), kh = kblocks(H ? H : 1);
  if (sms < 2 || sms > 4096) return false;
  RowsPlan p{};
  OuterPlan o{};
  switch (product) {
    case MC_MIX_OUTPUT: p = plan_wide<LAYER>(m, d->C_out, H ? kh : ki, 0, sms); break;
    case MC_MIX_GATE:
      if (!H) return false;
      p = gate_width(H) == 64 ? plan_rows<GATE, 64>(m, H, ki, 0, sms) : plan_rows<GATE, 128>(m, H, ki, 0, sms);
      break;
    case MC_MIX_ACT_GRAD:
      if (!H && d->act == MC_ACT_NONE) return false;
      p = H ? plan_rows<GATE_BWD, 64>(m, H, ki, ko, sms) : plan_wide<ACT_BWD>(m, d->C_out, ki, 0, sms);
      break;
    case MC_MIX_INPUT_GRAD: p = plan_wide<LAYER>(m, d->C_in, H ? kh : ko, H ? kh : 0, sms); break;
    case MC_MIX_WEIGHT_GRAD: o = H ? outer_plan(P, H, 2, d->C_in, sms) : outer_plan(P, d->C_out, 1, d->C_in, sms); break;
    case MC_MIX_WEIGHT_OUT_GRAD:
      if (!H) return false;
      o = outer_plan(P, d->C_out, 1, H, sms);
      break;
    default: return false;
  }
  if (o.mt) {
    const int v[6] = {256 * o.mt, o.bn, o.m_tiles * (product == MC_MIX_WEIGHT_GRAD && H ? 2 : 1), o.n_tiles, o.splits, o.per};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
  } else {
    const int v[6] = {p.bn, p.n_tiles, m, p.group, (int)p.pairs, p.stages};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
  }
  return true;
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

// The waits' self-test on this file's status word.
constexpr int SELFTEST_STATUS = 0x7F2;

}  // namespace mix
}  // namespace mc

extern "C" int mc_selftest_mix_wait_expiry(int32_t* observed_dev, void* stream) {
  using namespace mc;
  tc::wait_expiry_selftest_kernel<<<1, 32, 0, (cudaStream_t)stream>>>(mix::SELFTEST_STATUS, 2000000LL, observed_dev),
      MC_COUNT(1);
  MC_CHECK_LAUNCH();
  return MC_OK;
}
