// Residual update of a block fused with the norms before and after it:
//
//   z = out                                          or, with a norm after the block,
//   z = out / sqrt(mean(out^2) + eps) * (1 + post_gamma)
//   y = x + scale * z * sigmoid(gate)                (no gate: factor 1)
//   n = bf16(y / sqrt(mean(y^2) + eps) * (1 + gamma))
//
// i.e. rt_gate_residual / rt_residual_add followed by the next block's
// rt_rms_norm (confluence/confluence/layers.py:16-30, 170-174, 219-238) with
// y kept in registers between the two. x, y fp32, out / gate / n bf16; all
// sums and statistics fp32; n, d_out and d_gate are rounded once, when stored
// (they feed bf16 matmuls). Without a norm after the block the arithmetic is
// that of the separate kernels, operation for operation: both give the same
// bits where a warp takes a row in both (widths up to 512, multiples of 8);
// beyond, the row's sums are added in another order.
//
// Backward, r = rstd(y), yh = y r, a = dn (1 + gamma), s = sigmoid(gate):
//   dx = dy + r (a - yh mean(a yh)),   dgamma = sum over rows of dn yh
//   dz = dx scale s,                   dgate = dx scale z s (1 - s)
//   d_out = dz, or with ro = rstd(out), oh = out ro, c = dz (1 + post_gamma):
//   d_out = ro (c - oh mean(c oh)),    dpost_gamma = sum over rows of dz oh
//
// Memory-bound: forward 14 bytes per element (12 without gate), backward 22
// (18). A row belongs to a team of 32 to 1024 threads, which holds it in
// registers, so each tensor is read once; a thread moves 8 columns at a time
// (16 bytes of bf16, 32 of fp32). 32768 x 512 with gate: forward 38 us (94 % of
// the measured copy bandwidth), backward 71 us (80 %, the separate kernels'
// blocks kept for their bits); 32768 x 1024 with gate: 71 and 120 us (102 %,
// 94 %). Rows of a width that is no multiple of 8
// start anywhere: there the groups of 8 begin at the row's first 16-byte
// boundary (of the bf16 tensors, hence of the fp32 ones), and the up to 14
// columns before and behind them go to one thread each. A team's rows all
// start at the same remainder, so that a thread's columns, and its sums of
// dgamma and dpost_gamma over rows, stay the same ones.

namespace rt {
namespace layer {

constexpr int kResMaxD = 8192;  // 1024 threads x 8 columns
// Threads of a block: one team or several.
__host__ __device__ constexpr int res_threads(int tpr) { return tpr > 256 ? tpr : 256; }
constexpr int kResGate = 1, kResPost = 2;  // MODE bits: a gate, a norm after the block
// Blocks of the backward per SM, by what its registers hold, and the grid is
// just those: four without a gate, three with one, or at widths that are no
// multiple of 8, two with two groups a thread. (A warp per row keeps the
// separate kernels' two, for their bits.) Backward, us: 32768 x 1024 with a
// norm after the block 2 per SM in two waves 120, 4 in one 103; with a gate 4,
// which spill, 127, 3 120 (16384 x 2048 132 and 120); with both 2 129, 3 120,
// 4 163; 16000 x 1999 without gate and norm 2 144, 3 117. Spills remain where
// fewer blocks are slower or the team takes the whole block: up to 116 bytes a
// thread at widths that are no multiple of 8 (16000 x 1999 with both 2 178, 3
// 166, with 72 bytes; but 30000 x 1001 with both 145 and 153, so 2), and with
// 1024 threads, 64 registers each (72 bytes at widths of 8, 200 at others).
__host__ __device__ constexpr int res_bwd_per_sm(int tpr, int groups, int mode, bool edge) {
  const bool gated = (mode & kResGate) != 0, both = mode == (kResGate | kResPost);
  if (tpr > 256) return 1;
  if (tpr == 32 || groups > 1 || (both && edge && tpr < 256)) return 2;
  return gated || edge ? 3 : 4;
}

// The columns of one thread of a team: groups of 8 from `head` on, and with
// EDGE at most one column outside them (-1: none).
template <bool EDGE>
struct Columns {
  int head, groups, edge;
  __device__ __forceinline__ Columns(size_t row_start, int d, int t) {
    head = EDGE ? min(d, (int)((8 - row_start % 8) % 8)) : 0;
    groups = (d - head) / 8;
    const int outside = d - groups * 8;
    edge = !EDGE || t >= outside ? -1 : t < head ? t : t + groups * 8;
  }
};

__device__ __forceinline__ float bf16_at(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
__device__ __forceinline__ void put_bf16(uint16_t* p, float v) { *p = __bfloat16_as_ushort(__float2bfloat16_rn(v)); }

// gamma of columns c .. c + 7. With EDGE c is any column: 16-byte loads from
// the boundary before it on and a shift, the same for the whole team, instead
// of eight loads whose lanes are 32 bytes apart (9999 x 509, gate and both norms: forward
// 22 -> 16 us, backward 50 -> 46 us).
template <bool EDGE>
__device__ __forceinline__ F8 load_gamma(const float* g, int c, int d) {
  if (!EDGE) return load_f32x8(g + c);
  const int s = c & 3;
  const float4* q = reinterpret_cast<const float4*>(g + c - s);
  const float4 a = __ldg(q), b = __ldg(q + 1);
  if (s == 0) return F8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  float4 n = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c - s + 12 <= d) {
    n = __ldg(q + 2);
  } else {  // the last columns: none behind d
    n.x = __ldg(g + c - s + 8);
    if (s > 1) n.y = __ldg(g + c - s + 9);
    if (s > 2) n.z = __ldg(g + c - s + 10);
  }
  if (s == 1) return F8{{a.y, a.z, a.w, b.x, b.y, b.z, b.w, n.x}};
  if (s == 2) return F8{{a.z, a.w, b.x, b.y, b.z, b.w, n.x, n.y}};
  return F8{{a.w, b.x, b.y, b.z, b.w, n.x, n.y, n.z}};
}

// Sum over the TPR threads of a team; every thread gets it. The team's threads
// all call it together. `slot` alternates between calls, so that the next sum
// does not overwrite the one still being read.
template <int TPR>
__device__ __forceinline__ float team_sum(float v, float (*s_red)[res_threads(TPR) / 32], int slot) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  if (TPR == 32) return v;
  const int first = threadIdx.x / TPR * (TPR / 32);  // the team's first warp
  if ((threadIdx.x & 31) == 0) s_red[slot][threadIdx.x >> 5] = v;
  if (TPR == res_threads(TPR)) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / TPR), "n"(TPR) : "memory");
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < TPR / 32; ++w) t += s_red[slot][first + w];
  return t;
}

template <int TPR, int G, int MODE, bool EDGE>
__global__ void __launch_bounds__(res_threads(TPR)) residual_norm_kernel(
    const float* __restrict__ x, const uint16_t* __restrict__ out, const uint16_t* __restrict__ gate,
    const float* __restrict__ gamma, const float* __restrict__ post_gamma, long long rows, int d, float scale,
    float eps, float* __restrict__ y, uint16_t* __restrict__ n, float* __restrict__ rstd) {
  pdl_wait();  // the previous kernel on the stream has completed (launch_pdl)
  pdl_trigger();
  __shared__ float s_red[2][res_threads(TPR) / 32];
  constexpr bool gated = (MODE & kResGate) != 0, post = (MODE & kResPost) != 0;
  const int t = threadIdx.x % TPR;
  const long long row = (long long)blockIdx.x * (res_threads(TPR) / TPR) + threadIdx.x / TPR;
  if (row >= rows) return;  // a whole team
  const size_t start = (size_t)row * d;
  const Columns<EDGE> col(start, d, t);
  const size_t at = start + col.head;
  F8 xv[G], ov[G], gv[G];
  float xe = 0.f, oe = 0.f, ge = 0.f;
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const int c = t + TPR * j;
    if (c < col.groups) {
      xv[j] = load_f32x8(x + at + c * 8);
      ov[j] = load_bf16x8(out + at + c * 8);
      if (gated) gv[j] = load_bf16x8(gate + at + c * 8);
    }
  }
  if (EDGE && col.edge >= 0) {
    xe = x[start + col.edge];
    oe = bf16_at(out + start + col.edge);
    if (gated) ge = bf16_at(gate + start + col.edge);
  }
  if (post) {
    float so = EDGE ? oe * oe : 0.f;
#pragma unroll
    for (int j = 0; j < G; ++j)
      if (t + TPR * j < col.groups)
#pragma unroll
        for (int e = 0; e < 8; ++e) so = fmaf(ov[j].v[e], ov[j].v[e], so);
    const float ro = rsqrtf(team_sum<TPR>(so, s_red, 0) / (float)d + eps);
    if (t == 0) rstd[rows + row] = ro;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int c = t + TPR * j;
      if (c < col.groups) {
        const F8 pg = load_gamma<EDGE>(post_gamma, col.head + c * 8, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) ov[j].v[e] = ov[j].v[e] * ro * (1.f + pg.v[e]);
      }
    }
    if (EDGE && col.edge >= 0) oe = oe * ro * (1.f + post_gamma[col.edge]);
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const int c = t + TPR * j;
    if (c < col.groups) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xv[j].v[e] = gated ? xv[j].v[e] + scale * ov[j].v[e] * sigmoidf_(gv[j].v[e])
                           : xv[j].v[e] + scale * ov[j].v[e];
        ss = fmaf(xv[j].v[e], xv[j].v[e], ss);
      }
      store_f32x8(y + at + c * 8, xv[j]);
    }
  }
  if (EDGE && col.edge >= 0) {
    xe = gated ? xe + scale * oe * sigmoidf_(ge) : xe + scale * oe;
    ss = fmaf(xe, xe, ss);
    y[start + col.edge] = xe;
  }
  const float r = rsqrtf(team_sum<TPR>(ss, s_red, 1) / (float)d + eps);
  if (t == 0) rstd[row] = r;
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const int c = t + TPR * j;
    if (c < col.groups) {
      const F8 gm = load_gamma<EDGE>(gamma, col.head + c * 8, d);
      F8 o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o.v[e] = xv[j].v[e] * r * (1.f + gm.v[e]);
      store_bf16x8(n + at + c * 8, o);
    }
  }
  if (EDGE && col.edge >= 0) put_bf16(n + start + col.edge, xe * r * (1.f + gamma[col.edge]));
}

// Gradients of one column: from a = dn (1 + gamma) and yh to dx, d_gate and
// either d_out or the pair (oh, c) that d_out is made of.
struct ColumnGrad {
  float dx, d_gate, d_out, oh, c, dz;
};
template <bool gated, bool post>
__device__ __forceinline__ ColumnGrad column_grad(float a, float yh, float mdot, float r, bool has_dy, float dy, float o,
                                                  float gate, float ro, float pg, float scale) {
  ColumnGrad g;
  g.dx = r * (a - yh * mdot);
  if (has_dy) g.dx = __fadd_rn(dy, g.dx);  // not contracted: the sum of the two gradients of y
  const float s = gated ? sigmoidf_(gate) : 1.f;
  g.oh = post ? o * ro : 0.f;
  const float z = post ? g.oh * (1.f + pg) : o;
  g.dz = gated ? g.dx * scale * s : g.dx * scale;
  g.d_gate = gated ? g.dx * scale * z * s * (1.f - s) : 0.f;
  g.d_out = g.dz;
  g.c = post ? g.dz * (1.f + pg) : 0.f;
  return g;
}

// Rows blockIdx.x, + gridDim.x, ... (in units of the teams of a block); a
// block leaves the sums over its rows of dgamma in part[block][d] and, with a
// norm after the block, of dpost_gamma in part[gridDim.x + block][d]. All of a
// row's loads are issued before its first sum.
template <int TPR, int G, int MODE, bool EDGE>
__global__ void __launch_bounds__(res_threads(TPR), res_bwd_per_sm(TPR, G, MODE, EDGE))
    residual_norm_bwd_kernel(
    const float* __restrict__ dy, const uint16_t* __restrict__ dn, const float* __restrict__ y,
    const uint16_t* __restrict__ out, const uint16_t* __restrict__ gate, const float* __restrict__ gamma,
    const float* __restrict__ post_gamma, const float* __restrict__ rstd, long long rows, int d, float scale,
    float* __restrict__ dx, uint16_t* __restrict__ d_out, uint16_t* __restrict__ d_gate, float* __restrict__ part) {
  pdl_wait();  // the previous kernel on the stream has completed (launch_pdl)
  pdl_trigger();
  constexpr bool gated = (MODE & kResGate) != 0, post = (MODE & kResPost) != 0;
  constexpr int kTeams = res_threads(TPR) / TPR;
  extern __shared__ float s_sum[];  // [d], the block's sums at the end
  __shared__ float s_red[2][res_threads(TPR) / 32];
  const int t = threadIdx.x % TPR, team = threadIdx.x / TPR;
  const bool has_dy = dy != nullptr;
  F8 dg[G], dp[post ? G : 1];
  float dge = 0.f, dpe = 0.f;
#pragma unroll
  for (int j = 0; j < G; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      dg[j].v[e] = 0.f;
      if (post) dp[j].v[e] = 0.f;
    }
  const long long first = (long long)blockIdx.x * kTeams + team;
  const Columns<EDGE> col((size_t)first * d, d, t);
  for (long long row = first; row < rows; row += (long long)gridDim.x * kTeams) {
    const size_t start = (size_t)row * d, at = start + col.head;
    const float r = rstd[row];
    const float ro = post ? rstd[rows + row] : 0.f;
    F8 yh[G], a[G], up[G];
    uint4 ob[G], gb[G];
    float yhe = 0.f, ae = 0.f;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int c = t + TPR * j;
      if (c < col.groups) {
        yh[j] = load_f32x8(y + at + c * 8);
        a[j] = load_bf16x8(dn + at + c * 8);
        ob[j] = *reinterpret_cast<const uint4*>(out + at + c * 8);
        if (gated) gb[j] = *reinterpret_cast<const uint4*>(gate + at + c * 8);
        if (has_dy) up[j] = load_f32x8(dy + at + c * 8);
      }
    }
    float dot = 0.f;
    if (EDGE && col.edge >= 0) {
      const float g = bf16_at(dn + start + col.edge);
      yhe = y[start + col.edge] * r;
      ae = g * (1.f + gamma[col.edge]);
      dot = ae * yhe;
      dge = fmaf(g, yhe, dge);
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int c = t + TPR * j;
      if (c < col.groups) {
        const F8 gm = load_gamma<EDGE>(gamma, col.head + c * 8, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          yh[j].v[e] *= r;
          const float g = a[j].v[e];
          a[j].v[e] = g * (1.f + gm.v[e]);
          dot = fmaf(a[j].v[e], yh[j].v[e], dot);
          dg[j].v[e] = fmaf(g, yh[j].v[e], dg[j].v[e]);
        }
      }
    }
    const float mdot = team_sum<TPR>(dot, s_red, 0) / (float)d;
    float dot2 = 0.f;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int c = t + TPR * j;
      if (c < col.groups) {
        const size_t p = at + c * 8;
        F8 o, gt, w, pg, gx, gg, go;
        o = unpack8(ob[j]);
        if (gated) gt = unpack8(gb[j]);
        if (has_dy) w = up[j];
        if (post) pg = load_gamma<EDGE>(post_gamma, col.head + c * 8, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const ColumnGrad g = column_grad<gated, post>(a[j].v[e], yh[j].v[e], mdot, r, has_dy, has_dy ? w.v[e] : 0.f,
                                                        o.v[e], gated ? gt.v[e] : 0.f, ro, post ? pg.v[e] : 0.f, scale);
          gx.v[e] = g.dx;
          gg.v[e] = g.d_gate;
          go.v[e] = g.d_out;
          if (post) {
            yh[j].v[e] = g.oh;  // the pair (oh, c) takes the place of (yh, a)
            a[j].v[e] = g.c;
            dot2 = fmaf(g.c, g.oh, dot2);
            dp[j].v[e] = fmaf(g.dz, g.oh, dp[j].v[e]);
          }
        }
        store_f32x8(dx + p, gx);
        if (gated) store_bf16x8(d_gate + p, gg);
        if (!post) store_bf16x8(d_out + p, go);
      }
    }
    if (EDGE && col.edge >= 0) {
      const size_t p = start + col.edge;
      const ColumnGrad g = column_grad<gated, post>(ae, yhe, mdot, r, has_dy, has_dy ? dy[p] : 0.f, bf16_at(out + p),
                                                    gated ? bf16_at(gate + p) : 0.f, ro,
                                                    post ? post_gamma[col.edge] : 0.f, scale);
      dx[p] = g.dx;
      if (gated) put_bf16(d_gate + p, g.d_gate);
      if (!post) put_bf16(d_out + p, g.d_out);
      if (post) {
        yhe = g.oh;
        ae = g.c;
        dot2 = fmaf(g.c, g.oh, dot2);
        dpe = fmaf(g.dz, g.oh, dpe);
      }
    }
    if (post) {
      const float mdot2 = team_sum<TPR>(dot2, s_red, 1) / (float)d;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const int c = t + TPR * j;
        if (c < col.groups) {
          F8 o;
#pragma unroll
          for (int e = 0; e < 8; ++e) o.v[e] = ro * (a[j].v[e] - yh[j].v[e] * mdot2);
          store_bf16x8(d_out + at + c * 8, o);
        }
      }
      if (EDGE && col.edge >= 0) put_bf16(d_out + start + col.edge, ro * (ae - yhe * mdot2));
    } else if (TPR > 32) {  // s_red[0] is rewritten by the next row
      if (kTeams == 1) __syncthreads();
      else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(TPR) : "memory");
    }
  }
  // the block's sums over its rows, its teams' added in order
  for (int which = 0; which < (post ? 2 : 1); ++which) {
    float* dst = part + ((size_t)which * gridDim.x + blockIdx.x) * d;
    const float ge = which ? dpe : dge;
    for (int k = 0; k < kTeams; ++k) {
      if (team == k) {
        auto put = [&](int c, float v) {
          if (kTeams == 1) dst[c] = v;
          else s_sum[c] = k == 0 ? v : s_sum[c] + v;
        };
#pragma unroll
        for (int j = 0; j < G; ++j)
          if (t + TPR * j < col.groups)
#pragma unroll
            for (int e = 0; e < 8; ++e) put(col.head + (t + TPR * j) * 8 + e, which ? dp[post ? j : 0].v[e] : dg[j].v[e]);
        if (EDGE && col.edge >= 0) put(col.edge, ge);
      }
      if (kTeams > 1) __syncthreads();
    }
    if (kTeams > 1) {
      for (int c = threadIdx.x; c < d; c += res_threads(TPR)) dst[c] = s_sum[c];
      __syncthreads();
    }
  }
}

// dgamma / dpost_gamma from the blocks' partial sums, as sum_partials_kernel
// (a fixed order): blockIdx.y = which.
__global__ void __launch_bounds__(256) sum_gamma_partials_kernel(const float* __restrict__ part, int nparts, int d,
                                                                 float* __restrict__ dgamma,
                                                                 float* __restrict__ dpost_gamma) {
  pdl_wait();  // the previous kernel on the stream has completed (launch_pdl)
  pdl_trigger();
  __shared__ float sw[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  part += (size_t)blockIdx.y * nparts * d;
  float s = 0.f;
  if (c < d)
    for (int p = warp; p < nparts; p += 8) s += part[(size_t)p * d + c];
  sw[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < d) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += sw[w][lane];
    (blockIdx.y ? dpost_gamma : dgamma)[c] = t;
  }
}

// Threads of a row's team, and the groups of 8 columns a thread holds: one
// group a thread, because the backward's registers (five tensors and one or
// two sums) limit the loads in flight -- except where a warp takes up to 512
// columns as the separate kernels do, to give their bits.
// Backward, us: 32768 x 1024 with a norm after the block 250 for a warp per
// row (4 groups), 104 for 128 threads; 4096 x 8192 with gate 214 for 256
// threads (4 groups), 133 for 1024; but 8192 x 4096 132 for 256 threads (2
// groups), 167 for 512: two blocks per SM overlap one's sums with the other's
// loads. 9999 x 509 with both norms: a warp (2 groups) 46, 64 threads 34.
struct RowShape {
  int tpr, groups;
};
inline RowShape res_shape(int d, int mode, bool backward) {
  if (d <= 256) return {32, 1};
  if (d <= 512) {  // forward of 32768 x 512 with a norm after the block: 34.7 a warp, 37.5 64 threads
    const bool own_bits = (mode & kResPost) == 0, light = !backward && mode == kResPost;
    return (own_bits || light) && d % 8 == 0 ? RowShape{32, 2} : RowShape{64, 1};
  }
  if (d <= 1024) return {128, 1};
  if (d <= 2048) return {256, 1};
  if (d <= 4096) return backward ? RowShape{256, 2} : RowShape{512, 1};
  return {1024, 1};
}

// Blocks of the backward, which fix the order in which dgamma is summed: where
// a warp takes a row, those of rms_norm_bwd. At widths that are no multiple of
// 8 a multiple of 8, so that a team's rows start at one remainder.
inline int res_bwd_blocks(int64_t rows, int d, int mode) {
  const RowShape sh = res_shape(d, mode, true);
  const bool edge = d % 8 != 0;
  const int64_t teams = res_threads(sh.tpr) / sh.tpr;
  int most = 148 * res_bwd_per_sm(sh.tpr, sh.groups, mode, edge);
  if (edge) most -= most % 8;
  static_assert(kNormBwdBlocks == 2 * 148, "a warp per row: the separate kernel's blocks");
  return (int)std::min<int64_t>(std::max<int64_t>((rows + teams - 1) / teams, 1), most);
}

// Calls f with a shape's constants <TPR, G, MODE, EDGE>.
template <int TPR, int G, bool EDGE, typename F>
int with_mode(int mode, const F& f) {
  using std::integral_constant;
  auto pick = [&](auto m) {
    return f(integral_constant<int, TPR>(), integral_constant<int, G>(), m, integral_constant<bool, EDGE>());
  };
  switch (mode) {
    case 0: return pick(integral_constant<int, 0>());
    case 1: return pick(integral_constant<int, 1>());
    case 2: return pick(integral_constant<int, 2>());
    default: return pick(integral_constant<int, 3>());
  }
}
template <int TPR, int G, typename F>
int with_mode(int mode, bool edge, const F& f) {
  return edge ? with_mode<TPR, G, true>(mode, f) : with_mode<TPR, G, false>(mode, f);
}
template <bool BACKWARD, typename F>
int with_row_shape(int d, int mode, const F& f) {
  const bool edge = d % 8 != 0;
  const RowShape sh = res_shape(d, mode, BACKWARD);
  switch (sh.tpr) {
    case 32: {
      if (sh.groups == 1) return with_mode<32, 1>(mode, edge, f);
      constexpr std::integral_constant<int, 32> tpr;
      constexpr std::integral_constant<int, 2> groups;
      if (mode == kResGate) return f(tpr, groups, std::integral_constant<int, kResGate>(), std::false_type());
      if constexpr (!BACKWARD)
        if (mode == kResPost) return f(tpr, groups, std::integral_constant<int, kResPost>(), std::false_type());
      return f(tpr, groups, std::integral_constant<int, 0>(), std::false_type());
    }
    case 64: {  // a multiple of 8 with a norm after the block, in the forward a gate as well
      if (edge) return with_mode<64, 1, true>(mode, f);
      constexpr std::integral_constant<int, 64> tpr;
      constexpr std::integral_constant<int, 1> groups;
      if constexpr (BACKWARD)
        if (mode == kResPost) return f(tpr, groups, std::integral_constant<int, kResPost>(), std::false_type());
      return f(tpr, groups, std::integral_constant<int, kResGate | kResPost>(), std::false_type());
    }
    case 128: return with_mode<128, 1>(mode, edge, f);
    case 256:
      if constexpr (BACKWARD)
        if (sh.groups == 2) return with_mode<256, 2>(mode, edge, f);
      return with_mode<256, 1>(mode, edge, f);
    case 512:
      if constexpr (!BACKWARD) return with_mode<512, 1>(mode, edge, f);
      [[fallthrough]];
    default: return with_mode<1024, 1>(mode, edge, f);
  }
}

}  // namespace layer
}  // namespace rt

extern "C" int rt_residual_norm(const float* x, const uint16_t* out, const uint16_t* gate, const float* gamma,
                                const float* post_gamma, int64_t rows, int32_t d, float scale, float eps, float* y,
                                uint16_t* n, float* rstd, void* stream) {
  using namespace rt;
  if (rows < 0 || rows > INT32_MAX || d <= 0 || d > layer::kResMaxD || !(eps >= 0.f) || !std::isfinite(scale))
    return RT_ERR_INVALID_ARGUMENT;
  if (rows == 0) return RT_OK;
  if (!ok16(x) || !ok16(out) || (gate && !ok16(gate)) || !ok16(gamma) || (post_gamma && !ok16(post_gamma)) ||
      !ok16(y) || !ok16(n) || !ok16(rstd))
    return RT_ERR_INVALID_ARGUMENT;
  DeviceGuard guard(x);
  if (guard.status() != RT_OK) return guard.status();
  const int mode = (gate ? layer::kResGate : 0) | (post_gamma ? layer::kResPost : 0);
  return layer::with_row_shape<false>(d, mode, [&](auto tpr, auto g, auto m, auto edge) {
    constexpr int threads = layer::res_threads(tpr.value), per = threads / tpr.value;
    return launch_pdl("residual_norm_kernel launch",
                      layer::residual_norm_kernel<tpr.value, g.value, m.value, edge.value>, dim3((unsigned)((rows + per - 1) / per)), dim3(threads), 0,
                      static_cast<cudaStream_t>(stream), x, out, gate, gamma, post_gamma, rows, d, scale, eps, y, n,
                      rstd);
  });
}

extern "C" size_t rt_residual_norm_bwd_workspace_bytes(int64_t rows, int32_t d) {
  if (rows < 0 || d <= 0) return 0;
  int blocks = 0;
  for (int mode = 0; mode < 4; ++mode) blocks = std::max(blocks, rt::layer::res_bwd_blocks(rows, d, mode));
  return 2 * sizeof(float) * (size_t)blocks * (size_t)d;
}

extern "C" int rt_residual_norm_bwd(const float* dy, const uint16_t* dn, const float* y, const uint16_t* out,
                                    const uint16_t* gate, const float* gamma, const float* post_gamma,
                                    const float* rstd, int64_t rows, int32_t d, float scale, float* dx,
                                    uint16_t* d_out, uint16_t* d_gate, float* dgamma, float* dpost_gamma,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  using namespace rt;
  if (rows < 0 || rows > INT32_MAX || d <= 0 || d > layer::kResMaxD || !std::isfinite(scale))
    return RT_ERR_INVALID_ARGUMENT;
  if (!dgamma || (post_gamma != nullptr) != (dpost_gamma != nullptr) || (gate != nullptr) != (d_gate != nullptr))
    return RT_ERR_INVALID_ARGUMENT;
  if (!ok16(workspace)) return RT_ERR_INVALID_ARGUMENT;
  if (rows > 0 && ((dy && !ok16(dy)) || !ok16(dn) || !ok16(y) || !ok16(out) || (gate && !ok16(gate)) || !ok16(gamma) ||
                   (post_gamma && !ok16(post_gamma)) || !ok16(rstd) || !ok16(dx) || !ok16(d_out) ||
                   (d_gate && !ok16(d_gate))))
    return RT_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < rt_residual_norm_bwd_workspace_bytes(rows, d)) return RT_ERR_WORKSPACE;
  DeviceGuard guard(dgamma);
  if (guard.status() != RT_OK) return guard.status();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int mode = (gate ? layer::kResGate : 0) | (post_gamma ? layer::kResPost : 0);
  const int blocks = layer::res_bwd_blocks(rows, d, mode);  // no rows: one block leaves zeros
  float* part = static_cast<float*>(workspace);
  const int st = layer::with_row_shape<true>(d, mode, [&](auto tpr, auto g, auto m, auto edge) {
    constexpr int threads = layer::res_threads(tpr.value);
    // a team keeps its columns from row to row: its rows have to start at one remainder
    const int64_t at_once = (int64_t)blocks * (threads / tpr.value);
    if (edge.value && rows > at_once && at_once % 8 != 0) return (int)RT_ERR_INVALID_ARGUMENT;
    const size_t smem = tpr.value < threads ? sizeof(float) * (size_t)d : 0;
    return launch_pdl("residual_norm_bwd_kernel launch",
                      layer::residual_norm_bwd_kernel<tpr.value, g.value, m.value, edge.value>, dim3(blocks),
                      dim3(threads), smem, s, dy, dn, y, out, gate, gamma, post_gamma, rstd, rows,
                      d, scale, dx, d_out, d_gate, part);
  });
  if (st != RT_OK) return st;
  return launch_pdl("sum_gamma_partials_kernel launch", layer::sum_gamma_partials_kernel,
                    dim3((d + 31) / 32, post_gamma ? 2 : 1), dim3(256), 0, s, part, blocks, d, dgamma, dpost_gamma);
}
