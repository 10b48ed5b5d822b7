// The norms around a block, with its gate and residual scale, in one pass:
//
//   u = post ? delta * r1 * post : delta       r1 = rsqrt(mean(delta^2) + eps)
//   y = x + scale * gate * u                    (rounded to the residual's type)
//   h = y * r2 * pre                            r2 = rsqrt(mean(y^2) + eps)
//
// and its backward pass from dy (the gradient of y itself) and dh:
//
//   g  = dh * pre,  yhat = y * r2
//   dt = dy + r2 * (g - yhat * mean(g * yhat))             -> dx
//   dpre = sum_rows dh * yhat,  dgate = scale * dt * u     (summed over what the gate broadcasts over)
//   w  = scale * dt * gate * post,  dhat = delta * r1
//   ddelta = r1 * (w - dhat * mean(w * dhat)),  dpost = sum_rows scale * dt * gate * dhat
//
// Both are bound by memory: forward reads x and delta and writes y and h, backward
// reads y, delta, dy and dh and writes dx and ddelta, each element once, held in
// registers between the two reductions. Sums are fp32; the only rounding on the
// way is y's, which the next block reads in the residual's type anyway
// (round_branch adds that of u, as separate norm and add launches have it).
//
// A row's sums are taken in one fixed order whatever the batch: eight neighbours
// of a thread in turn, then a butterfly over 32 such groups, then one over the
// group sums. It is the order of add_rmsnorm_kernel, whose results these equal
// bit for bit.
#include "b200_elem.cuh"
#include "b200_train.h"

namespace b200 {

enum GateKind : int { kGateNone = 0, kGateChannel = 1, kGateRow = 2, kGateElement = 3 };

struct BlockNormArgs {
  const void *x, *delta;    // [T, H]
  const void *post, *pre;   // [H] or null
  const void* gate;         // [H], [T] or [T, H] by gate_kind
  void *y, *h;              // forward outputs (h null without pre)
  float *r1, *r2;           // [T] reciprocal RMS, or null
  const void *dy, *dh;      // backward inputs (either may be null: zero)
  void *dx, *ddelta;
  void* dgate;              // row: [T], element: [T, H] in the residual's type; channel: in `part`
  float* part;              // [n][grid][H] column sums of dpost, dpre, dgate (those wanted, in this order)
  int64_t ldx, ldd, ldg, ldy, ldh, lddy, lddh, ldo;  // row strides; ldo: dx, ddelta and dgate
  int64_t T;
  int H;
  int gate_kind;
  int want_post, want_pre, want_gate;
  int offset_one, round_branch;
  int slots;  // backward: rows that a stage holds (delta, and dy, y, dh, gate where given)
  float eps, scale;
};

// Column of element j of a thread's v-th group of E. Aligned rows: E neighbours
// (16- or 32-byte accesses); others: one column a lane, so that a warp's access is
// contiguous.
template <bool VEC, int E>
__device__ __forceinline__ int column(int v, int j, int threads) {
  return VEC ? (v * threads + (int)threadIdx.x) * E + j : (v * E + j) * threads + (int)threadIdx.x;
}
template <typename T, bool VEC, int E>
__device__ __forceinline__ void load_group(Group<T, E>& p, const T* row, int v, int threads, int H) {
  if constexpr (VEC) {
    const int c = column<true, E>(v, 0, threads);
    if (c < H) p.load(row + c);
    else p.zero();
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int c = column<false, E>(v, j, threads);
      p.e[j] = c < H ? row[c] : from_f32<T>(0.f);
    }
  }
}
template <typename T, bool VEC, int E>
__device__ __forceinline__ void store_group(T* row, const Group<T, E>& p, int v, int threads, int H) {
  if constexpr (VEC) {
    const int c = column<true, E>(v, 0, threads);
    if (c < H) p.store(row + c);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int c = column<false, E>(v, j, threads);
      if (c < H) row[c] = p.e[j];
    }
  }
}
// A group of factors along the columns: p + one, or `none` throughout without p.
template <typename W, bool VEC, int E>
__device__ __forceinline__ void factors(float* w, const void* p, float one, float none, int v, int threads, int H) {
  if (p) {
    Group<W, E> q;
    load_group<W, VEC, E>(q, reinterpret_cast<const W*>(p), v, threads, H);
    q.unpack(w);
    if (one != 0.f) {
#pragma unroll
      for (int j = 0; j < E; ++j) w[j] += one;
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) w[j] = none;
  }
}

// Sums of four values over the warp, six shuffles: lanes 8 g .. 8 g + 7 get the sum of
// v[g]. Each sum is taken in the order of warp_sum's butterfly (partners 16, 8, 4, 2,
// 1 lanes apart), whose bits it has.
__device__ __forceinline__ float warp_sum4(const float (&v)[4]) {
  const int lane = threadIdx.x & 31;
  const bool hi = lane & 16, odd = lane & 8;
  float a = hi ? v[2] : v[0], b = hi ? v[3] : v[1];
  a += __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[2], 16);
  b += __shfl_xor_sync(0xffffffffu, hi ? v[1] : v[3], 16);
  float s = odd ? b : a;
  s += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// Sum over the block of NV group sums a thread (1 or 4): a butterfly over the lanes
// for each group index, then one over the at most 32 warp sums, in index order.
// `red`: 32 floats that no other reduction of the same row uses.
template <int NV>
__device__ __forceinline__ float row_sum(const float (&s)[NV], float* red) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if constexpr (NV == 4) {
    const float t = warp_sum4(s);
    if ((lane & 7) == 0) red[(lane >> 3) * nw + wid] = t;
  } else {
    const float t = warp_sum(s[0]);
    if (lane == 0) red[wid] = t;
  }
  __syncthreads();
  return warp_sum(lane < NV * nw ? red[lane] : 0.f);
}

// u rounded to the residual's type or not, gated, scaled and added: y and the sums of
// its squares.
template <typename T, bool VEC, int NV, int NS, bool GATED, bool ROUND>
__device__ __forceinline__ void add_branch(Group<T, 8> (&x)[NV], const float* u, float grow, const void* gate, float scale,
                                           int v, int n, int H, float (&s)[NS]) {
  float f[8], g[8];
  x[v].unpack(f);
  if (GATED) factors<T, VEC, 8>(g, gate, 0.f, grow, v, n, H);
  float b[8];
  if (ROUND) {
    Group<T, 8> r;
    r.pack(u);
    r.unpack(b);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = u[j];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] += scale * (GATED ? b[j] * g[j] : b[j]);
  x[v].pack(f);
  x[v].unpack(f);
#pragma unroll
  for (int j = 0; j < 8; ++j) s[NS == 1 ? 0 : v] += f[j] * f[j];
}

// One row a CTA. NV groups of eight a thread; SEQ: rows above 8192 columns add a
// thread's groups one after the other, shorter ones sum each group on its own.
template <typename T, typename W, bool VEC, int NV, bool SEQ, bool GATED>
__global__ void __launch_bounds__(1024, 1) block_norms_kernel(const BlockNormArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float red[2][32];
  constexpr int NS = SEQ ? 1 : NV;
  const int64_t row = blockIdx.x;
  const int n = blockDim.x, H = a.H;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  const T* dr = reinterpret_cast<const T*>(a.delta) + row * a.ldd;
  Group<T, 8> x[NV], d[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) load_group<T, VEC, 8>(d[v], dr, v, n, H);
#pragma unroll
  for (int v = 0; v < NV; ++v) load_group<T, VEC, 8>(x[v], xr, v, n, H);
  const float one = a.offset_one ? 1.f : 0.f;
  float r1 = 1.f;
  if (a.post) {
    float s[NS] = {};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[8];
      d[v].unpack(f);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[SEQ ? 0 : v] += f[j] * f[j];
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) d[v].hold();
    r1 = rsqrtf(row_sum(s, red[0]) / (float)H + a.eps);
  }
  const float grow = GATED && a.gate_kind == kGateRow ? to_f32(reinterpret_cast<const T*>(a.gate)[row]) : 1.f;
  const void* gate = nullptr;  // a gate along the columns
  if (GATED && a.gate_kind == kGateChannel) gate = a.gate;
  if (GATED && a.gate_kind == kGateElement) gate = reinterpret_cast<const T*>(a.gate) + row * a.ldg;
  T* yr = reinterpret_cast<T*>(a.y) + row * a.ldy;
  float s[NS] = {};
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float u[8];
    d[v].unpack(u);
    if (a.post) {
      float w[8];
      factors<W, VEC, 8>(w, a.post, one, 1.f, v, n, H);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = u[j] * r1 * w[j];
    }
    if (a.round_branch) add_branch<T, VEC, NV, NS, GATED, true>(x, u, grow, gate, a.scale, v, n, H, s);
    else add_branch<T, VEC, NV, NS, GATED, false>(x, u, grow, gate, a.scale, v, n, H, s);
    store_group<T, VEC, 8>(yr, x[v], v, n, H);
  }
  if (threadIdx.x == 0 && a.r1) a.r1[row] = r1;
  if (!a.pre) return;
#pragma unroll
  for (int v = 0; v < NV; ++v) x[v].hold();
  const float r2 = rsqrtf(row_sum(s, red[1]) / (float)H + a.eps);
  if (threadIdx.x == 0 && a.r2) a.r2[row] = r2;
  T* hr = reinterpret_cast<T*>(a.h) + row * a.ldh;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float f[8], w[8];
    factors<W, VEC, 8>(w, a.pre, one, 1.f, v, n, H);
    x[v].unpack(f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = f[j] * r2 * w[j];
    x[v].pack(f);
    store_group<T, VEC, 8>(hr, x[v], v, n, H);
  }
}

// Backward: a CTA walks the rows blockIdx.x, + gridDim.x, ... and keeps its
// columns' weight-gradient sums in registers, so that they cost gridDim.x partial
// rows instead of T. `part` is summed over the CTAs afterwards, in order.
//
// Both means come from one round of sums: with c = gate * post * dhat and
// b = dy + r2 g, mean(w * dhat) = scale * (sum c b - r2 m sum c yhat) / H where
// m = mean(g * yhat), so neither waits for the other.
//
// STAGES > 0: the rows arrive in shared memory by bulk copies, STAGES of them under
// way at a time, so that a row's loads run under the sums of those before it and cost
// no registers; those hold the weights instead. 0 (unaligned rows, and rows too wide
// for two stages): straight from global memory. 8192 x 4096 bf16 (403 MB): 95 us from
// global memory, 81 us (5.0 TB/s) staged, bound by the sums' round trips between rows.
// The other instantiations pay for registers: at 64 a thread the unstaged ones and the staged
// gated ones of 1024 threads spill 40 - 164 bytes, and rows of more than 1024 groups (above 8192
// columns of 16 bits, 4096 of fp32), four or eight groups a thread, 0.8 - 1.4 KB: 4096 x 5120
// fp32 815 us (0.6 TB/s) where 4096 x 4096 takes 79, 4096 x 12288 bf16 946 us.
template <typename T, bool VEC, int E, int STAGES>
struct BwdRows {
  const BlockNormArgs& a;
  int n, tid;
  uint32_t ring, bars;  // shared memory: [STAGES][slots][row bytes], [STAGES] barriers
  int slots, row_bytes;
  bool dead = false;
  uint32_t at = 0;      // the current row's stage
  int64_t row = 0;

  __device__ __forceinline__ BwdRows(const BlockNormArgs& args, uint8_t* smem)
      : a(args), n(blockDim.x), tid(threadIdx.x), ring(smem_u32(smem)), bars(0), slots(args.slots),
        row_bytes(args.H * (int)sizeof(T)) {
    if constexpr (STAGES > 0) {
      bars = ring + STAGES * slots * row_bytes;
      if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(bars + 8 * i, 1);
        fence_barrier_init();
      }
      __syncthreads();
    }
  }
  // The k-th row of this CTA into its stage (one thread).
  __device__ __forceinline__ void fetch(int k) {
    const int64_t r = blockIdx.x + (int64_t)k * gridDim.x;
    if (r >= a.T) return;
    const uint32_t dst = ring + (k % (STAGES > 0 ? STAGES : 1)) * slots * row_bytes, bar = bars + 8 * (k % (STAGES > 0 ? STAGES : 1));
    const uint64_t pol = l2_policy_evict_first();
    mbar_arrive_expect_tx(bar, (uint32_t)(slots * row_bytes));
    int s = 0;
    auto get = [&](const void* p, int64_t ld) {
      bulk_g2s(dst + row_bytes * s++, reinterpret_cast<const T*>(p) + r * ld, (uint32_t)row_bytes, bar, pol);
    };
    get(a.delta, a.ldd);
    if (a.dy) get(a.dy, a.lddy);
    if (a.dh) {
      get(a.y, a.ldy);
      get(a.dh, a.lddh);
    }
    if (a.gate_kind == kGateElement) get(a.gate, a.ldg);
  }
  __device__ __forceinline__ void begin(int k, int64_t r) {
    row = r;
    if constexpr (STAGES > 0) {
      at = ring + (k % STAGES) * slots * row_bytes;
      // after a wait that ran out (the status word says so) the rows go by unread waits, so that the kernel ends
      if (!dead) dead = !mbar_wait(bars + 8 * (k % STAGES), (k / STAGES) & 1, kErrGemmWait);
    }
  }
  __device__ __forceinline__ void load(Group<T, E>& g, int slot, const void* p, int64_t ld, int v) const {
    if constexpr (STAGES > 0) {
      const int c = column<true, E>(v, 0, n);
      if (c < a.H) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&g);
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(at + slot * row_bytes + c * (int)sizeof(T)));
      } else {
        g.zero();
      }
    } else {
      load_group<T, VEC, E>(g, reinterpret_cast<const T*>(p) + row * ld, v, n, a.H);
    }
  }
  __device__ __forceinline__ void delta(Group<T, E>& g, int v) const { load(g, 0, a.delta, a.ldd, v); }
  __device__ __forceinline__ void dy(Group<T, E>& g, int v) const {
    if (a.dy) load(g, 1, a.dy, a.lddy, v);
    else g.zero();
  }
  __device__ __forceinline__ void y(Group<T, E>& g, int v) const {
    if (a.dh) load(g, 1 + (a.dy != nullptr), a.y, a.ldy, v);
    else g.zero();
  }
  __device__ __forceinline__ void dh(Group<T, E>& g, int v) const {
    if (a.dh) load(g, 2 + (a.dy != nullptr), a.dh, a.lddh, v);
    else g.zero();
  }
  // Gate along the columns (1 where there is none), times `by`.
  __device__ __forceinline__ void gate(float* w, float by, int v) const {
    if (a.gate_kind == kGateElement) {
      Group<T, E> g;
      load(g, slots - 1, a.gate, a.ldg, v);
      g.unpack(w);
    } else {
      factors<T, VEC, E>(w, a.gate_kind == kGateChannel ? a.gate : nullptr, 0.f, by, v, n, a.H);
    }
  }
};

template <typename T, typename W, bool VEC, int NV, bool GATED, int MAXT, int STAGES>
__global__ void __launch_bounds__(MAXT, STAGES > 0 ? 1 : 1024 / MAXT) block_norms_bwd_kernel(const BlockNormArgs a) {
  constexpr int E = 16 / sizeof(T);  // 16-byte groups
  extern __shared__ __align__(128) uint8_t bwd_smem[];
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float red[2][4][32];
  const int n = blockDim.x, H = a.H, lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = n >> 5;
  const float one = a.offset_one ? 1.f : 0.f, inv_h = 1.f / (float)H;
  const void* pre = a.dh ? a.pre : nullptr;
  float cpost[NV][E] = {}, cpre[NV][E] = {}, cgate[GATED ? NV : 1][E] = {};
  int flip = 0, k = 0;
  BwdRows<T, VEC, E, STAGES> rows(a, bwd_smem);
  if (STAGES > 0 && threadIdx.x == 0)
    for (int i = 0; i < STAGES; ++i) rows.fetch(i);
  auto r1_of = [&](int64_t row) { return a.post && row < a.T ? a.r1[row] : 1.f; };
  auto r2_of = [&](int64_t row) { return a.dh && row < a.T ? a.r2[row] : 0.f; };
  float next_r1 = r1_of(blockIdx.x), next_r2 = r2_of(blockIdx.x);
  // the weights stay in registers where the rows do not need them
  float wpost[STAGES > 0 ? E : 1], wpre[STAGES > 0 ? E : 1];
  if constexpr (STAGES > 0) {
    factors<W, VEC, E>(wpost, a.post, one, 1.f, 0, n, H);
    factors<W, VEC, E>(wpre, pre, one, 0.f, 0, n, H);
  }
  auto post_w = [&](float* w, int v) {
    if constexpr (STAGES > 0) {
#pragma unroll
      for (int j = 0; j < E; ++j) w[j] = wpost[j];
    } else {
      factors<W, VEC, E>(w, a.post, one, 1.f, v, n, H);
    }
  };
  for (int64_t row = blockIdx.x; row < a.T; row += gridDim.x, flip ^= 1, ++k) {
    // the sums' buffers alternate between rows: a thread may be writing the next
    // row's while a slower one still reads this row's
    const float r1 = next_r1, r2 = next_r2;
    next_r1 = r1_of(row + gridDim.x);
    next_r2 = r2_of(row + gridDim.x);
    const float grow = GATED && a.gate_kind == kGateRow ? to_f32(reinterpret_cast<const T*>(a.gate)[row]) : 1.f;
    rows.begin(k, row);
    Group<T, E> y[NV], d[NV];
    // r1 and r2 are factored out of the sums and of what the second loop repeats:
    //   q = r2 dh pre, b = dy + q, c = delta post (gate);  dt = b - y r2^2 (sum q y) / H
    float s[4] = {}, b[NV][E];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float c[E], w[E], f[E], t[E];
      Group<T, E> in;
      rows.delta(d[v], v);
      d[v].unpack(c);
      post_w(w, v);
#pragma unroll
      for (int j = 0; j < E; ++j) c[j] *= w[j];
      if (GATED) {
        rows.gate(w, 1.f, v);
#pragma unroll
        for (int j = 0; j < E; ++j) c[j] *= w[j];
      }
      rows.dy(in, v);
      in.unpack(b[v]);
      rows.y(y[v], v);
      y[v].unpack(f);
      rows.dh(in, v);
      in.unpack(t);
      if constexpr (STAGES > 0) {
#pragma unroll
        for (int j = 0; j < E; ++j) w[j] = wpre[j];
      } else {
        factors<W, VEC, E>(w, pre, one, 0.f, v, n, H);
      }
#pragma unroll
      for (int j = 0; j < E; ++j) {
        t[j] *= r2;
        cpre[v][j] += t[j] * f[j];
        const float q = t[j] * w[j];
        b[v][j] += q;
        s[0] += q * f[j];
        s[1] += c[j] * b[v][j];
        s[2] += c[j] * f[j];
      }
      if (STAGES == 0) {
        y[v].hold();
        d[v].hold();
      }
    }
    const float t = warp_sum4(s);
    if ((lane & 7) == 0) red[flip][lane >> 3][wid] = t;
    __syncthreads();
    // every thread is done with the row before this one: its stage takes the row STAGES - 1 ahead
    if (STAGES > 0 && threadIdx.x == 0 && k > 0) rows.fetch(k - 1 + STAGES);
    float q[4];
#pragma unroll
    for (int k = 0; k < 3; ++k) q[k] = lane < nw ? red[flip][k][lane] : 0.f;
    q[3] = 0.f;
    const float total = warp_sum4(q);
    const float s1 = __shfl_sync(0xffffffffu, total, 0), s2 = __shfl_sync(0xffffffffu, total, 8),
                s3 = __shfl_sync(0xffffffffu, total, 16);
    const float mr2 = s1 * inv_h * r2 * r2;
    const float k1 = r1 * a.scale;
    const float along = k1 * (s2 - mr2 * s3);  // sum of scale * dt * dhat * post, without a row gate
    const float k2 = a.post ? r1 * r1 * (along * grow * inv_h) : 0.f;
    if (GATED && a.gate_kind == kGateRow && a.dgate && threadIdx.x == 0)
      reinterpret_cast<T*>(a.dgate)[row] = from_f32<T>(along);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float w[E], f[E];
      Group<T, E> o;
      if (STAGES > 0) {  // again from the stage rather than held over the sums
        rows.y(y[v], v);
        rows.delta(d[v], v);
      }
      y[v].unpack(f);
#pragma unroll
      for (int j = 0; j < E; ++j) b[v][j] -= f[j] * mr2;  // dt
      if (a.dx) {
        o.pack(b[v]);
        store_group<T, VEC, E>(reinterpret_cast<T*>(a.dx) + row * a.ldo, o, v, n, H);
      }
      post_w(w, v);
      d[v].unpack(f);
#pragma unroll
      for (int j = 0; j < E; ++j) b[v][j] *= k1;
      if (GATED) {
        float g[E], dg[E];
        rows.gate(g, grow, v);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          dg[j] = b[v][j] * f[j] * w[j];
          cgate[v][j] += dg[j];
          b[v][j] *= g[j];
        }
        if (a.gate_kind == kGateElement && a.dgate) {
          o.pack(dg);
          store_group<T, VEC, E>(reinterpret_cast<T*>(a.dgate) + row * a.ldo, o, v, n, H);
        }
      }
#pragma unroll
      for (int j = 0; j < E; ++j) {
        cpost[v][j] += b[v][j] * f[j];
        b[v][j] = b[v][j] * w[j] - k2 * f[j];
      }
      if (a.ddelta) {
        o.pack(b[v]);
        store_group<T, VEC, E>(reinterpret_cast<T*>(a.ddelta) + row * a.ldo, o, v, n, H);
      }
    }
  }
  float* part = a.part;
  auto put = [&](const float (&c)[E], int v) {
    float* r = part + (int64_t)blockIdx.x * H;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int col = column<VEC, E>(v, j, n);
      if (col < H) r[col] = c[j];
    }
  };
  const int64_t next = (int64_t)gridDim.x * H;
  if (a.want_post) {
#pragma unroll
    for (int v = 0; v < NV; ++v) put(cpost[v], v);
    part += next;
  }
  if (a.want_pre) {
#pragma unroll
    for (int v = 0; v < NV; ++v) put(cpre[v], v);
    part += next;
  }
  if constexpr (GATED) {
    if (a.want_gate && a.gate_kind == kGateChannel) {
#pragma unroll
      for (int v = 0; v < NV; ++v) put(cgate[v], v);
    }
  }
}

struct ColSumArgs {
  const float* part;  // [n][G][H]
  void* out[3];       // [H] each
  int type[3];
  int G, H;
};

// out[k][c] = sum over g of part[k][g][c]: 32 columns a CTA, 32 rows of threads
// that each add every 32nd partial, then a tree over them; a fixed order.
__global__ void __launch_bounds__(1024) col_sum_kernel(ColSumArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float t[32][33];
  const int lane = threadIdx.x & 31, r = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const float* p = a.part + (int64_t)blockIdx.y * a.G * a.H;
  float s = 0.f;
  if (c < a.H)
    for (int g = r; g < a.G; g += 32) s += p[(int64_t)g * a.H + c];
  t[r][lane] = s;
  __syncthreads();
  s = warp_sum(t[lane][r]);  // thread (r, lane): partial row `lane` of column r
  const int oc = blockIdx.x * 32 + r;
  if (lane == 0 && oc < a.H) store_elem(a.out[blockIdx.y], a.type[blockIdx.y], oc, s);
}

static inline int round32(int v) { return (v + 31) / 32 * 32; }

// Groups of eight a thread, forward. Rows above 8192 columns need more than one for
// each of 1024 threads. Below, one keeps a few rows' latency low and four leave room
// for four times the rows on an SM, whose loads then overlap the others' sums; both add
// in the same order. bf16 rows of 4096, one group against four: 64 rows 2.7 us against
// 3.7, 592 rows 4.8 against 5.0, 1184 rows 8.3 against 6.5, 8192 rows 55 against 44 (6.1
// TB/s). Unaligned rows are dealt to the lanes by the thread count, so there the choice
// goes by the width alone.
constexpr int kFewRows = 4;  // rows an SM
template <typename T, typename W, bool VEC, bool GATED>
static int launch_fwd_gate(const BlockNormArgs& a, int num_sms, cudaStream_t st) {
  const int groups = (a.H + 7) / 8;
  const dim3 grid((unsigned)a.T);
  cudaError_t e;
  if (groups > 1024)
    e = launch_k(block_norms_kernel<T, W, VEC, 4, true, GATED>, grid, dim3(1024), 0, st, 1, a);
  else if (VEC && a.T <= (int64_t)kFewRows * num_sms)
    e = launch_k(block_norms_kernel<T, W, VEC, 1, false, GATED>, grid, dim3(round32(groups)), 0, st, 1, a);
  else
    e = launch_k(block_norms_kernel<T, W, VEC, 4, false, GATED>, grid, dim3(round32((groups + 3) / 4)), 0, st, 1, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
template <typename T, typename W, bool VEC>
static int launch_fwd(const BlockNormArgs& a, int num_sms, cudaStream_t st) {
  return a.gate_kind == kGateNone ? launch_fwd_gate<T, W, VEC, false>(a, num_sms, st)
                                  : launch_fwd_gate<T, W, VEC, true>(a, num_sms, st);
}

// Backward: a 16-byte group a thread up to 1024 threads, more groups for wider rows.
static inline int bwd_threads(int H, int type) {
  const int g = type == kElemF32 ? (H + 3) / 4 : (H + 7) / 8;
  return round32(g < 1024 ? g : 1024);
}
// CTAs an SM by their registers a thread: 64, and at most 112 where the weights stay in
// registers beside staged rows (512 threads or fewer).
static inline int ctas_per_sm(int threads, int regs) {
  const int c = 65536 / (regs * threads);
  return c > 16 ? 16 : c < 1 ? 1 : c;
}
// Launches with at most `most` CTAs; returns their number in *grid.
template <auto Kernel>
static int launch_bwd_one(const BlockNormArgs& a, int64_t most, int threads, int smem, int* grid, cudaStream_t st) {
  if (smem > 0)
    if (int e = smem_attr_once<Kernel>(smem)) return e;
  *grid = (int)(a.T < most ? a.T : most);
  const cudaError_t e = launch_k(Kernel, dim3(*grid), dim3(threads), smem, st, 1, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
template <typename T, typename W, bool VEC, bool GATED>
static int launch_bwd_gate(const BlockNormArgs& a, int num_sms, int* grid, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T), kWide = 32 / E;  // kWide x 1024 groups cover the widest row
  const int groups = (a.H + E - 1) / E;
  const int threads = round32(groups < 1024 ? groups : 1024);
  const int64_t plain = (int64_t)ctas_per_sm(threads, 64) * num_sms;
  if (groups > 1024) return launch_bwd_one<block_norms_bwd_kernel<T, W, VEC, kWide, GATED, 1024, 0>>(a, plain, threads, 0, grid, st);
  if constexpr (VEC) {
    // four stages where they fit beside the SM's other CTAs, else two
    const int per_sm = ctas_per_sm(threads, groups > 512 ? 64 : 112);
    const int64_t most = (int64_t)per_sm * num_sms;
    const int stage = a.slots * a.H * (int)sizeof(T), room = 220 * 1024 / per_sm - 1024;
    if (4 * (stage + 8) <= room)
      return groups > 512 ? launch_bwd_one<block_norms_bwd_kernel<T, W, VEC, 1, GATED, 1024, 4>>(a, most, threads, 4 * (stage + 8), grid, st)
                          : launch_bwd_one<block_norms_bwd_kernel<T, W, VEC, 1, GATED, 512, 4>>(a, most, threads, 4 * (stage + 8), grid, st);
    if (2 * (stage + 8) <= room)
      return groups > 512 ? launch_bwd_one<block_norms_bwd_kernel<T, W, VEC, 1, GATED, 1024, 2>>(a, most, threads, 2 * (stage + 8), grid, st)
                          : launch_bwd_one<block_norms_bwd_kernel<T, W, VEC, 1, GATED, 512, 2>>(a, most, threads, 2 * (stage + 8), grid, st);
  }
  return groups > 512 ? launch_bwd_one<block_norms_bwd_kernel<T, W, VEC, 1, GATED, 1024, 0>>(a, plain, threads, 0, grid, st)
                      : launch_bwd_one<block_norms_bwd_kernel<T, W, VEC, 1, GATED, 512, 0>>(a, plain, threads, 0, grid, st);
}
template <typename T, typename W, bool VEC>
static int launch_bwd(const BlockNormArgs& a, int num_sms, int* grid, cudaStream_t st) {
  return a.gate_kind == kGateNone ? launch_bwd_gate<T, W, VEC, false>(a, num_sms, grid, st)
                                  : launch_bwd_gate<T, W, VEC, true>(a, num_sms, grid, st);
}

// f(T, W, VEC) for the element type, the weights' type (that or fp32) and alignment.
template <typename F>
static int by_type(int type, int w_type, bool vec, F f) {
  auto pick = [&](auto t, auto w) { return vec ? f(t, w, std::true_type{}) : f(t, w, std::false_type{}); };
  if (type == kElemF32) return pick(float{}, float{});
  if (type == kElemBf16) return w_type == kElemF32 ? pick(__nv_bfloat16{}, float{}) : pick(__nv_bfloat16{}, __nv_bfloat16{});
  return w_type == kElemF32 ? pick(__half{}, float{}) : pick(__half{}, __half{});
}

}  // namespace b200

using namespace b200;

extern "C" {

// Widest row: four groups of eight columns for each of 1024 threads.
int b200_block_norms_max_width() { return 4 * 1024 * 8; }

// CTAs of the backward pass (rows of its partial sums) for T rows of H columns: what
// fits on the SMs at 64 registers a thread.
int b200_block_norms_bwd_grid(int64_t T, int H, int type, int num_sms) {
  const int64_t most = (int64_t)ctas_per_sm(bwd_threads(H, type), 64) * num_sms;
  return (int)(T < most ? T : most);
}

// Forward. type: ElemType of x, delta, gate, y and h; w_type: of post and pre, that or fp32.
// y may be x. Returns 0, a CUDA error code, or -1 for arguments out of range.
int b200_block_norms(const void* x, int64_t ldx, const void* delta, int64_t ldd, const void* post, const void* pre,
                     int w_type, const void* gate, int64_t ldg, int gate_kind, void* y, int64_t ldy, void* h,
                     int64_t ldh, float* r1, float* r2, int64_t T, int H, int type, float eps, float scale,
                     int offset_one, int round_branch, int num_sms, cudaStream_t st) {
  if (T < 0 || H < 1 || H > b200_block_norms_max_width() || T > 0x7FFFFFFFll || type < 0 || type > 2 || w_type < 0 ||
      w_type > 2 || (w_type != type && w_type != kElemF32) || gate_kind < 0 || gate_kind > 3 || (gate_kind && !gate))
    return -1;
  if (T == 0) return 0;
  BlockNormArgs a = {};
  a.x = x;
  a.delta = delta;
  a.post = post;
  a.pre = pre;
  a.gate = gate;
  a.y = y;
  a.h = h;
  a.r1 = r1;
  a.r2 = r2;
  a.ldx = ldx;
  a.ldd = ldd;
  a.ldg = ldg;
  a.ldy = ldy;
  a.ldh = ldh;
  a.T = T;
  a.H = H;
  a.gate_kind = gate_kind;
  a.eps = eps;
  a.scale = scale;
  a.offset_one = offset_one;
  a.round_branch = round_branch;
  const int size = type == kElemF32 ? 4 : 2;
  auto rows16 = [&](const void* p, int64_t ld) { return (((uintptr_t)p | (uintptr_t)(ld * size)) & 15) == 0; };
  const bool vec = H % 8 == 0 && rows16(x, ldx) && rows16(delta, ldd) && rows16(y, ldy) && rows16(h, ldh) &&
                   rows16(post, 0) && rows16(pre, 0) && (gate_kind == kGateRow || rows16(gate, gate_kind == kGateElement ? ldg : 0));
  return by_type(type, w_type, vec, [&](auto t, auto w, auto v) {
    return launch_fwd<decltype(t), decltype(w), decltype(v)::value>(a, num_sms, st);
  });
}

// Backward from y, delta and the saved r1 / r2. dy or dh may be null (zero); dx,
// ddelta, dgate, dpost and dpre are null where not wanted. dx, ddelta and an
// element gate's gradient have rows of H elements. part: fp32
// [number of dpost, dpre and channel dgate wanted][b200_block_norms_bwd_grid][H].
int b200_block_norms_bwd(const void* y, int64_t ldy, const void* delta, int64_t ldd, const void* post, const void* pre,
                         int w_type, const void* gate, int64_t ldg, int gate_kind, const float* r1, const float* r2,
                         const void* dy, int64_t lddy, const void* dh, int64_t lddh, void* dx, void* ddelta,
                         void* dgate, void* dpost, void* dpre, float* part, int64_t T, int H, int type, float scale,
                         int offset_one, int num_sms, cudaStream_t st) {
  if (T < 0 || H < 1 || H > b200_block_norms_max_width() || T > 0x7FFFFFFFll || type < 0 || type > 2 || w_type < 0 ||
      w_type > 2 || (w_type != type && w_type != kElemF32) || gate_kind < 0 || gate_kind > 3 || (gate_kind && !gate) || (dh && !pre) || (dpre && !dh))
    return -1;
  if (T == 0) return 0;
  BlockNormArgs a = {};
  a.y = const_cast<void*>(y);
  a.delta = delta;
  a.post = post;
  a.pre = pre;
  a.gate = gate;
  a.r1 = const_cast<float*>(r1);
  a.r2 = const_cast<float*>(r2);
  a.dy = dy;
  a.dh = dh;
  a.dx = dx;
  a.ddelta = ddelta;
  a.dgate = gate_kind == kGateChannel ? nullptr : dgate;
  a.part = part;
  a.ldy = ldy;
  a.ldd = ldd;
  a.ldg = ldg;
  a.lddy = lddy;
  a.lddh = lddh;
  a.ldo = H;
  a.T = T;
  a.H = H;
  a.gate_kind = gate_kind;
  a.scale = scale;
  a.offset_one = offset_one;
  a.slots = 1 + (dy != nullptr) + 2 * (dh != nullptr) + (gate_kind == kGateElement);
  a.want_post = dpost != nullptr;
  a.want_pre = dpre != nullptr;
  a.want_gate = dgate != nullptr;
  const int size = type == kElemF32 ? 4 : 2;
  auto rows16 = [&](const void* p, int64_t ld) { return (((uintptr_t)p | (uintptr_t)(ld * size)) & 15) == 0; };
  const bool vec = H % 8 == 0 && rows16(y, ldy) && rows16(delta, ldd) && rows16(dy, lddy) && rows16(dh, lddh) &&
                   rows16(dx, 0) && rows16(ddelta, 0) && rows16(post, 0) && rows16(pre, 0) &&
                   (gate_kind == kGateRow ||
                    (rows16(gate, gate_kind == kGateElement ? ldg : 0) && (gate_kind != kGateElement || rows16(dgate, 0))));
  int grid = 0;
  const int e = by_type(type, w_type, vec, [&](auto t, auto w, auto v) {
    return launch_bwd<decltype(t), decltype(w), decltype(v)::value>(a, num_sms, &grid, st);
  });
  if (e) return e;
  ColSumArgs c = {};
  int k = 0;
  auto add = [&](void* out, int t) {
    if (!out) return;
    c.out[k] = out;
    c.type[k++] = t;
  };
  add(dpost, w_type);
  add(dpre, w_type);
  add(gate_kind == kGateChannel ? dgate : nullptr, type);
  if (!k) return 0;
  c.part = part;
  c.G = grid;
  c.H = H;
  cudaError_t ce = launch_k(col_sum_kernel, dim3((H + 31) / 32, k), dim3(1024), 0, st, 1, c);
  return ce != cudaSuccess ? (int)ce : (int)cudaGetLastError();
}

}  // extern "C"

B200_STATUS_ACCESSORS(block_norms)
