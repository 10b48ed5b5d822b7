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
  int gate_kind, w_type;
  int want_post, want_pre, want_gate;
  int offset_one, round_branch;
  float eps, scale;
};

// Column of element j of a thread's v-th group of eight. Aligned rows: eight
// neighbours (one 16- or 32-byte access); others: one column a lane, so that a
// warp's access is contiguous.
template <bool VEC>
__device__ __forceinline__ int column(int v, int j, int threads) {
  return VEC ? (v * threads + (int)threadIdx.x) * 8 + j : (v * 8 + j) * threads + (int)threadIdx.x;
}

template <typename T, bool VEC>
__device__ __forceinline__ Pack8<T> load_group(const T* row, int v, int threads, int H) {
  Pack8<T> p;
  if constexpr (VEC) {
    const int c = column<true>(v, 0, threads);
    if (c < H) return load_pack(row + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) p.e[j] = from_f32<T>(0.f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<false>(v, j, threads);
      p.e[j] = c < H ? row[c] : from_f32<T>(0.f);
    }
  }
  return p;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_group(T* row, const Pack8<T>& p, int v, int threads, int H) {
  if constexpr (VEC) {
    const int c = column<true>(v, 0, threads);
    if (c < H) store_pack(row + c, p);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<false>(v, j, threads);
      if (c < H) row[c] = p.e[j];
    }
  }
}
// Eight weights (0 past the row's end).
template <bool VEC>
__device__ __forceinline__ void load_weights(float* w, const void* p, int type, int v, int threads, int H) {
  if (VEC && column<true>(v, 0, threads) < H) {
    const int c = column<true>(v, 0, threads);
    if (type == kElemF32) {
      const Pack8<float> q = load_pack(reinterpret_cast<const float*>(p) + c);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = q.e[j];
    } else if (type == kElemBf16) {
      const Pack8<__nv_bfloat16> q = load_pack(reinterpret_cast<const __nv_bfloat16*>(p) + c);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = to_f32(q.e[j]);
    } else {
      const Pack8<__half> q = load_pack(reinterpret_cast<const __half*>(p) + c);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = to_f32(q.e[j]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = column<VEC>(v, j, threads);
    w[j] = !VEC && c < H ? load_elem(p, type, c) : 0.f;
  }
}

// Sum over the block of NV group sums a thread: a butterfly over the lanes for
// each group index, then one over the at most 32 warp sums, in index order.
// `red`: 32 floats that no other reduction of the same row uses.
template <int NV>
__device__ __forceinline__ float row_sum(const float (&s)[NV], float* red) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const float t = warp_sum(s[v]);
    if (lane == 0) red[v * nw + wid] = t;
  }
  __syncthreads();
  return warp_sum(lane < NV * nw ? red[lane] : 0.f);
}

// One row a CTA. NV groups of eight a thread; SEQ: rows above 8192 columns add a
// thread's groups one after the other, shorter ones sum each group on its own.
template <typename T, bool VEC, int NV, bool SEQ>
__global__ void __launch_bounds__(1024) block_norms_kernel(BlockNormArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float red[2][32];
  constexpr int NS = SEQ ? 1 : NV;
  const int64_t row = blockIdx.x;
  const int n = blockDim.x, H = a.H;
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  const T* dr = reinterpret_cast<const T*>(a.delta) + row * a.ldd;
  Pack8<T> x[NV], d[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) d[v] = load_group<T, VEC>(dr, v, n, H);
#pragma unroll
  for (int v = 0; v < NV; ++v) x[v] = load_group<T, VEC>(xr, v, n, H);
  const float one = a.offset_one ? 1.f : 0.f;
  float r1 = 1.f;
  if (a.post) {
    float s[NS] = {};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = to_f32(d[v].e[j]);
        s[SEQ ? 0 : v] += f * f;
      }
    r1 = rsqrtf(row_sum(s, red[0]) / (float)H + a.eps);
  }
  const float grow = a.gate_kind == kGateRow ? to_f32(reinterpret_cast<const T*>(a.gate)[row]) : 1.f;
  T* yr = reinterpret_cast<T*>(a.y) + row * a.ldy;
  float s[NS] = {};
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float w[8], g[8];
    if (a.post) load_weights<VEC>(w, a.post, a.w_type, v, n, H);
    if (a.gate_kind == kGateChannel) load_weights<VEC>(g, a.gate, sizeof(T) == 4 ? kElemF32 : (std::is_same<T, __half>::value ? kElemF16 : kElemBf16), v, n, H);
    if (a.gate_kind == kGateElement) {
      const Pack8<T> q = load_group<T, VEC>(reinterpret_cast<const T*>(a.gate) + row * a.ldg, v, n, H);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = to_f32(q.e[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float u = to_f32(d[v].e[j]);
      if (a.post) u = u * r1 * (w[j] + one);
      if (a.round_branch) u = to_f32(from_f32<T>(u));
      if (a.gate_kind == kGateRow) u *= grow;
      else if (a.gate_kind != kGateNone) u *= g[j];
      x[v].e[j] = from_f32<T>(to_f32(x[v].e[j]) + a.scale * u);
      const float f = to_f32(x[v].e[j]);
      s[SEQ ? 0 : v] += f * f;
    }
    store_group<T, VEC>(yr, x[v], v, n, H);
  }
  if (threadIdx.x == 0 && a.r1) a.r1[row] = r1;
  if (!a.pre) return;
  const float r2 = rsqrtf(row_sum(s, red[1]) / (float)H + a.eps);
  if (threadIdx.x == 0 && a.r2) a.r2[row] = r2;
  T* hr = reinterpret_cast<T*>(a.h) + row * a.ldh;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float w[8];
    load_weights<VEC>(w, a.pre, a.w_type, v, n, H);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[v].e[j] = from_f32<T>(to_f32(x[v].e[j]) * r2 * (w[j] + one));
    store_group<T, VEC>(hr, x[v], v, n, H);
  }
}

// Backward: a CTA walks the rows blockIdx.x, + gridDim.x, ... and keeps its
// columns' weight-gradient sums in registers, so that they cost gridDim.x
// partial rows instead of T. `part` is summed over the CTAs afterwards, in order.
template <typename T, bool VEC, int NV>
__global__ void __launch_bounds__(1024) block_norms_bwd_kernel(BlockNormArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float red[2][3][32];
  const int n = blockDim.x, H = a.H;
  const float one = a.offset_one ? 1.f : 0.f;
  float cpost[NV][8] = {}, cpre[NV][8] = {}, cgate[NV][8] = {};
  constexpr int kT = sizeof(T) == 4 ? kElemF32 : (std::is_same<T, __half>::value ? kElemF16 : kElemBf16);
  int flip = 0;
  for (int64_t row = blockIdx.x; row < a.T; row += gridDim.x, flip ^= 1) {
    // the reductions' buffers alternate between rows: a thread may be writing the
    // next row's sums while a slower one still reads this row's
    Pack8<T> y[NV], d[NV], ty[NV], th[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (a.dh) {
        y[v] = load_group<T, VEC>(reinterpret_cast<const T*>(a.y) + row * a.ldy, v, n, H);
        th[v] = load_group<T, VEC>(reinterpret_cast<const T*>(a.dh) + row * a.lddh, v, n, H);
      }
      if (a.dy) ty[v] = load_group<T, VEC>(reinterpret_cast<const T*>(a.dy) + row * a.lddy, v, n, H);
      d[v] = load_group<T, VEC>(reinterpret_cast<const T*>(a.delta) + row * a.ldd, v, n, H);
    }
    float dt[NV][8];
    if (a.dh) {
      const float r2 = a.r2[row];
      float s[1] = {0.f};
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float w[8];
        load_weights<VEC>(w, a.pre, a.w_type, v, n, H);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float yh = to_f32(y[v].e[j]) * r2, g = to_f32(th[v].e[j]);
          cpre[v][j] += g * yh;
          dt[v][j] = g * (w[j] + one);
          s[0] += dt[v][j] * yh;
        }
      }
      const float m = row_sum(s, red[flip][0]) / (float)H;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          dt[v][j] = r2 * (dt[v][j] - to_f32(y[v].e[j]) * r2 * m) + (a.dy ? to_f32(ty[v].e[j]) : 0.f);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) dt[v][j] = a.dy ? to_f32(ty[v].e[j]) : 0.f;
    }
    T* dxr = reinterpret_cast<T*>(a.dx) + row * a.ldo;
    const float r1 = a.post ? a.r1[row] : 1.f;
    const float grow = a.gate_kind == kGateRow ? to_f32(reinterpret_cast<const T*>(a.gate)[row]) : 1.f;
    float s[1] = {0.f}, sg[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (a.dx) {
        Pack8<T> o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o.e[j] = from_f32<T>(dt[v][j]);
        store_group<T, VEC>(dxr, o, v, n, H);
      }
      float w[8], g[8];
      if (a.post) load_weights<VEC>(w, a.post, a.w_type, v, n, H);
      if (a.gate_kind == kGateChannel) load_weights<VEC>(g, a.gate, kT, v, n, H);
      if (a.gate_kind == kGateElement) {
        const Pack8<T> q = load_group<T, VEC>(reinterpret_cast<const T*>(a.gate) + row * a.ldg, v, n, H);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = to_f32(q.e[j]);
      }
      Pack8<T> og;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float dhat = to_f32(d[v].e[j]) * r1;
        const float wj = a.post ? w[j] + one : 1.f;
        float du = a.scale * dt[v][j];
        if (a.gate_kind != kGateNone) {
          const float dg = du * dhat * wj;
          cgate[v][j] += dg;
          sg[0] += dg;
          og.e[j] = from_f32<T>(dg);
          du *= a.gate_kind == kGateRow ? grow : g[j];
        }
        cpost[v][j] += du * dhat;
        dt[v][j] = du * wj;  // gradient of dhat
        s[0] += dt[v][j] * dhat;
      }
      if (a.gate_kind == kGateElement && a.dgate)
        store_group<T, VEC>(reinterpret_cast<T*>(a.dgate) + row * a.ldo, og, v, n, H);
    }
    if (a.gate_kind == kGateRow && a.dgate) {
      const float t = row_sum(sg, red[flip][1]);
      if (threadIdx.x == 0) reinterpret_cast<T*>(a.dgate)[row] = from_f32<T>(t);
    }
    if (a.ddelta) {
      const float m = a.post ? row_sum(s, red[flip][2]) / (float)H : 0.f;
      T* ddr = reinterpret_cast<T*>(a.ddelta) + row * a.ldo;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        Pack8<T> o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o.e[j] = from_f32<T>(r1 * (dt[v][j] - to_f32(d[v].e[j]) * r1 * m));
        store_group<T, VEC>(ddr, o, v, n, H);
      }
    }
  }
  float* part = a.part;
  auto put = [&](const float (&c)[NV][8]) {
    float* r = part + (int64_t)blockIdx.x * H;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int col = column<VEC>(v, j, n);
        if (col < H) r[col] = c[v][j];
      }
    part += (int64_t)gridDim.x * H;
  };
  if (a.want_post) put(cpost);
  if (a.want_pre) put(cpre);
  if (a.want_gate && a.gate_kind == kGateChannel) put(cgate);
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

template <typename T, bool VEC>
static int launch_fwd(const BlockNormArgs& a, cudaStream_t st) {
  const int groups = (a.H + 7) / 8;
  const int full = round32(groups < 1024 ? groups : 1024);  // threads at one group each
  const dim3 grid((unsigned)a.T);
  cudaError_t e;
  if (groups > 2048)
    e = launch_k(block_norms_kernel<T, VEC, 4, true>, grid, dim3(1024), 0, st, 1, a);
  else if (groups > 1024)
    e = launch_k(block_norms_kernel<T, VEC, 2, true>, grid, dim3(1024), 0, st, 1, a);
  else
    e = launch_k(block_norms_kernel<T, VEC, 1, false>, grid, dim3(full), 0, st, 1, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

template <typename T, bool VEC>
static int launch_bwd(const BlockNormArgs& a, int grid, cudaStream_t st) {
  const int groups = (a.H + 7) / 8;
  const int full = round32(groups < 1024 ? groups : 1024);
  cudaError_t e;
  if (groups > 2048)
    e = launch_k(block_norms_bwd_kernel<T, VEC, 4>, dim3(grid), dim3(1024), 0, st, 1, a);
  else if (groups > 1024)
    e = launch_k(block_norms_bwd_kernel<T, VEC, 2>, dim3(grid), dim3(1024), 0, st, 1, a);
  else
    e = launch_k(block_norms_bwd_kernel<T, VEC, 1>, dim3(grid), dim3(full), 0, st, 1, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace b200

using namespace b200;

extern "C" {

// Widest row: four groups of eight columns for each of 1024 threads.
int b200_block_norms_max_width() { return 4 * 1024 * 8; }

// CTAs of the backward pass (rows of its partial sums) for T rows of H columns.
int b200_block_norms_bwd_grid(int64_t T, int H, int num_sms) {
  const int threads = round32((H + 7) / 8 < 1024 ? (H + 7) / 8 : 1024);
  int per_sm = 1024 / threads;
  per_sm = per_sm > 16 ? 16 : per_sm < 1 ? 1 : per_sm;
  const int64_t most = (int64_t)per_sm * num_sms;
  return (int)(T < most ? T : most);
}

// Forward. type: ElemType of x, delta, gate, y and h; w_type: of post and pre.
// y may be x. Returns 0, a CUDA error code, or -1 for arguments out of range.
int b200_block_norms(const void* x, int64_t ldx, const void* delta, int64_t ldd, const void* post, const void* pre,
                     int w_type, const void* gate, int64_t ldg, int gate_kind, void* y, int64_t ldy, void* h,
                     int64_t ldh, float* r1, float* r2, int64_t T, int H, int type, float eps, float scale,
                     int offset_one, int round_branch, cudaStream_t st) {
  if (T < 0 || H < 1 || H > b200_block_norms_max_width() || T > 0x7FFFFFFFll || type < 0 || type > 2 || w_type < 0 ||
      w_type > 2 || gate_kind < 0 || gate_kind > 3 || (gate_kind && !gate))
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
  a.w_type = w_type;
  a.eps = eps;
  a.scale = scale;
  a.offset_one = offset_one;
  a.round_branch = round_branch;
  const int size = type == kElemF32 ? 4 : 2;
  auto rows16 = [&](const void* p, int64_t ld) { return (((uintptr_t)p | (uintptr_t)(ld * size)) & 15) == 0; };
  const bool vec = H % 8 == 0 && rows16(x, ldx) && rows16(delta, ldd) && rows16(y, ldy) && rows16(h, ldh) &&
                   rows16(post, 0) && rows16(pre, 0) && (gate_kind == kGateRow || rows16(gate, gate_kind == kGateElement ? ldg : 0));
  if (type == kElemBf16) return vec ? launch_fwd<__nv_bfloat16, true>(a, st) : launch_fwd<__nv_bfloat16, false>(a, st);
  if (type == kElemF16) return vec ? launch_fwd<__half, true>(a, st) : launch_fwd<__half, false>(a, st);
  return vec ? launch_fwd<float, true>(a, st) : launch_fwd<float, false>(a, st);
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
      w_type > 2 || gate_kind < 0 || gate_kind > 3 || (gate_kind && !gate) || (dh && !pre) || (dpre && !dh))
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
  a.w_type = w_type;
  a.scale = scale;
  a.offset_one = offset_one;
  a.want_post = dpost != nullptr;
  a.want_pre = dpre != nullptr;
  a.want_gate = dgate != nullptr;
  const int size = type == kElemF32 ? 4 : 2;
  auto rows16 = [&](const void* p, int64_t ld) { return (((uintptr_t)p | (uintptr_t)(ld * size)) & 15) == 0; };
  const bool vec = H % 8 == 0 && rows16(y, ldy) && rows16(delta, ldd) && rows16(dy, lddy) && rows16(dh, lddh) &&
                   rows16(dx, 0) && rows16(ddelta, 0) && rows16(post, 0) && rows16(pre, 0) &&
                   (gate_kind == kGateRow ||
                    (rows16(gate, gate_kind == kGateElement ? ldg : 0) && (gate_kind != kGateElement || rows16(dgate, 0))));
  const int grid = b200_block_norms_bwd_grid(T, H, num_sms);
  int e;
  if (type == kElemBf16) e = vec ? launch_bwd<__nv_bfloat16, true>(a, grid, st) : launch_bwd<__nv_bfloat16, false>(a, grid, st);
  else if (type == kElemF16) e = vec ? launch_bwd<__half, true>(a, grid, st) : launch_bwd<__half, false>(a, grid, st);
  else e = vec ? launch_bwd<float, true>(a, grid, st) : launch_bwd<float, false>(a, grid, st);
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
