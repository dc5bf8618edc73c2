// Cross entropy of up to eight tokens in f32 whose rows of x fit FEW_SHARED bytes
// (8 x 6136, 4 x 12280, 1 x 49144): the weights stream through the CUDA cores. (Part
// of om_loss.cu.)
//
//   few_rows_kernel  a warp takes four rows of w at a time and their dot products
//                    with every token (x in shared memory); forward: the running
//                    maximum and sum per token, backward: dz of the rows.
//   few_outer_kernel a thread has four columns of w, a block a range of rows:
//                    dw_v = sum_n dz_nv x_n is written as w_v is read, and
//                    dx_n += dz_nv w_v stays in registers until the block's end.
//
// Bound by HBM: w is read once forward, twice backward, and dw written once,
// where the tensor cores' products make and read three planes of w. Sums are
// formed in one order. Measured with gradients: 3 x 1344 x 11307 93 us (tensor
// cores 202), 8 x 2048 x 32000 341 us (nine tokens, on the tensor cores, 617: eight is
// what the kernels are compiled for, not where the two forms cross). In
// 16 bits, where w needs no planes, the tensor cores win even for one token (8 x
// 2048 x 32000 bf16: 149 us against 418 in this form).
#pragma once

constexpr int FEW = 8;                     // tokens
constexpr int FEW_ROWS = 4;                // of w per warp and turn
constexpr int FEW_SHARED = 192 * 1024;     // bytes of x, rows rounded up to few_of

struct FewArgs {
  int N;
  int64_t D, V;
  const float* x;
  int64_t xd, xn;
  const float* w;
  int64_t wd, wv;
  const void* targets;
  int t64;
  // forward
  float2* part;  // [block][N]
  float* hit;
  // backward
  const float *lse, *dloss;
  float* dz;     // [V][NN]
  float* dw;
  int64_t dwd, dwv;
  float* acc;    // [block][N][D]
};

// 16 bytes of a row as f32
__device__ __forceinline__ void load_part(const float* p, float (&v)[4]) {
  const float4 u = __ldg(reinterpret_cast<const float4*>(p));
  v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
}

// VEC: rows of w are contiguous and 16-byte aligned
template <int NN, bool VEC, bool BWD>
__global__ void __launch_bounds__(256) few_rows_kernel(const __grid_constant__ FewArgs p) {
  extern __shared__ __align__(16) float xs[];  // [NN][Dp]
  constexpr int E = 4, R = FEW_ROWS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = (int)p.D, Dp = (D + E - 1) / E * E;
  for (int n = 0; n < NN; ++n)
    for (int d = threadIdx.x; d < Dp; d += 256)
      xs[n * Dp + d] = n < p.N && d < D ? p.x[n * p.xn + d * p.xd] : 0.f;
  // lane n has token n
  const int64_t target = lane < p.N ? target_of(p.targets, p.t64, lane) : -1;
  const bool counts = target >= 0 && target < p.V;
  float lse = 0.f, g = 0.f, m = -INFINITY, s = 0.f;
  if (BWD && lane < p.N) {
    lse = counts ? p.lse[lane] : 0.f;
    g = counts ? p.dloss[lane] : 0.f;
  }
  __syncthreads();
  const int64_t turns = (p.V + R - 1) / R;
  for (int64_t t = (int64_t)blockIdx.x * 8 + warp; t < turns; t += (int64_t)gridDim.x * 8) {
    const int64_t v0 = t * R;
    float acc[R][NN];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NN; ++n) acc[r][n] = 0.f;
    const float* row[R];
#pragma unroll
    for (int r = 0; r < R; ++r) row[r] = p.w + min(v0 + r, p.V - 1) * p.wv;
    if constexpr (VEC) {
      const int whole = D / E * E;
#pragma unroll 2
      for (int d = lane * E; d < whole; d += 32 * E) {
        float w[R][E];
#pragma unroll
        for (int r = 0; r < R; ++r) load_part(row[r] + d, w[r]);
#pragma unroll
        for (int n = 0; n < NN; ++n) {
          if (NN > 1 && n >= p.N) break;
          const float4 x = *reinterpret_cast<const float4*>(xs + n * Dp + d);
#pragma unroll
          for (int r = 0; r < R; ++r)
            acc[r][n] += w[r][0] * x.x + w[r][1] * x.y + w[r][2] * x.z + w[r][3] * x.w;
        }
      }
      for (int d = whole + lane; d < D; d += 32)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float w = row[r][d];
#pragma unroll
          for (int n = 0; n < NN; ++n) acc[r][n] += w * xs[n * Dp + d];
        }
    } else {
#pragma unroll 4
      for (int d = lane; d < D; d += 32) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float w = row[r][d * p.wd];
#pragma unroll
          for (int n = 0; n < NN; ++n) acc[r][n] += w * xs[n * Dp + d];
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float z = 0.f;  // of this lane's token
#pragma unroll
      for (int n = 0; n < NN; ++n) {
        if (NN > 1 && n >= p.N) break;
        float a = acc[r][n];
#pragma unroll
        for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        if (lane == n) z = a;
      }
      if (v0 + r >= p.V) break;
      if constexpr (!BWD) {
        merge(m, s, z, 1.f);
        if (target == v0 + r) p.hit[lane] = z;
      } else if (lane < NN) {
        const float q = exp2_fast((z - lse) * LOG2E) - (target == v0 + r ? 1.f : 0.f);
        p.dz[(v0 + r) * NN + lane] = counts ? g * q : 0.f;
      }
    }
  }
  if constexpr (!BWD) {
    __shared__ float2 part[8][FEW];
    if (lane < FEW) part[warp][lane] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.x < p.N) {
      for (int i = 1; i < 8; ++i) merge(m, s, part[i][lane].x, part[i][lane].y);
      p.part[(int64_t)blockIdx.x * p.N + lane] = make_float2(m, s);
    }
  }
}

// VEC: rows of w and dw are contiguous and 16-byte aligned, a thread has E
// neighbouring columns; else E columns a block's width apart
template <int NN, bool VEC>
__global__ void __launch_bounds__(256) few_outer_kernel(const __grid_constant__ FewArgs p) {
  constexpr int E = 4, ROWS = 128, AHEAD = 8;  // rows whose dz is in shared memory at a time
  __shared__ float dz[ROWS][NN];
  const int64_t v0 = p.V * blockIdx.x / gridDim.x, v1 = p.V * (blockIdx.x + 1) / gridDim.x;
  const int64_t first = (int64_t)blockIdx.y * 256 * E;
  int64_t col[E];
  float x[NN][E], acc[NN][E];
#pragma unroll
  for (int e = 0; e < E; ++e)
    col[e] = first + (VEC ? (int64_t)threadIdx.x * E + e : (int64_t)e * 256 + threadIdx.x);
#pragma unroll
  for (int n = 0; n < NN; ++n) {
    bool counts = n < p.N;
    if (counts) {
      const int64_t t = target_of(p.targets, p.t64, n);
      counts = t >= 0 && t < p.V;  // whatever another row holds reaches no gradient
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[n][e] = counts && col[e] < p.D ? p.x[n * p.xn + col[e] * p.xd] : 0.f;
      acc[n][e] = 0.f;
    }
  }
  const bool whole = VEC && col[E - 1] < p.D;
  for (int64_t v = v0; v < v1; v += ROWS) {
    const int rows = (int)min((int64_t)ROWS, v1 - v);
    __syncthreads();
    for (int i = threadIdx.x; i < rows * NN; i += 256) (&dz[0][0])[i] = p.dz[v * NN + i];
    __syncthreads();
    for (int r0 = 0; r0 < rows; r0 += AHEAD) {
      float a[AHEAD][E];  // the rows' loads are all under way before the first is used
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const float* w = p.w + min(v + r0 + u, v1 - 1) * p.wv;
        if (whole) {
          load_part(w + col[0], a[u]);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) a[u][e] = col[e] < p.D ? w[col[e] * p.wd] : 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (r0 + u >= rows) break;
        float* dw = p.dw + (v + r0 + u) * p.dwv;
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
        for (int n = 0; n < NN; ++n) {
          const float g = dz[r0 + u][n];  // zero for tokens that do not exist
#pragma unroll
          for (int e = 0; e < E; ++e) {
            acc[n][e] += g * a[u][e];
            o[e] += g * x[n][e];
          }
        }
        if (whole) {
          __stcs(reinterpret_cast<float4*>(dw + col[0]), make_float4(o[0], o[1], o[2], o[3]));
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (col[e] < p.D) dw[col[e] * p.dwd] = o[e];
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NN; ++n) {
    if (n >= p.N) break;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (col[e] < p.D) p.acc[((int64_t)blockIdx.x * p.N + n) * p.D + col[e]] = acc[n][e];
  }
}

// dx = sum of the blocks, 32 columns by 8 groups of blocks per block
__global__ void few_join(const float* __restrict__ acc, int blocks, int64_t total, int64_t D,
                         Counted counted, float* __restrict__ dx, int64_t dxd, int64_t dxn) {
  __shared__ float part[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t i = blockIdx.x * (int64_t)32 + tx;
  float s = 0.f;
  if (i < total)
#pragma unroll 8
    for (int k = ty; k < blocks; k += 8) s += __ldcg(acc + (int64_t)k * total + i);
  part[ty][tx] = s;
  __syncthreads();
  if (ty || i >= total) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += part[k][tx];
  dx[i / D * dxn + i % D * dxd] = counted.out(i / D) ? 0.f : s;
}

// tokens that the kernels are compiled for
constexpr int few_of(int64_t n) { return n == 1 ? 1 : n <= 4 ? 4 : FEW; }
bool few_tokens(const LossArgs& p) {
  return p.N <= FEW && few_of(p.N) * (p.D + 8) * 4 <= FEW_SHARED;
}

template <int NN, bool BWD>
int launch_few_rows(om_backend* be, const FewArgs& a, int blocks) {
  constexpr int E = 4;
  const bool vec = a.wd == 1 && !((uintptr_t)a.w & 15) && a.wv * 4 % 16 == 0;
  const int smem = (int)(NN * ((a.D + E - 1) / E * E) * 4);
  auto kernel = vec ? few_rows_kernel<NN, true, BWD> : few_rows_kernel<NN, false, BWD>;
  if (smem > PLAIN_SHARED) OM_TRY(allow_shared(be, (const void*)kernel, smem, "loss"));
  ProfScope prof(be, BWD ? "loss_few_dlogits" : "loss_few_logits");
  kernel<<<blocks, 256, smem, be->stream>>>(a);
  note_launch();
  return check_cuda(cudaGetLastError(), "loss launch");
}

template <int NN>
int few_forward(om_backend* be, FewArgs a, const LossArgs& p, float* loss, float* lse) {
  const int blocks = (int)std::min<int64_t>((p.V + 8 * FEW_ROWS - 1) / (8 * FEW_ROWS), (int64_t)be->num_sms * 3);
  Scratch ws;
  OM_TRY(ws.alloc(be, (size_t)blocks * p.N * 8 + p.N * 4));
  a.part = (float2*)ws.ptr;
  a.hit = (float*)(a.part + (int64_t)blocks * p.N);
  OM_TRY((launch_few_rows<NN, false>(be, a, blocks)));
  ProfScope prof(be, "loss_join_stats");
  join_stats<<<1, 256, 0, be->stream>>>(a.part, blocks, p.N, p.targets, p.target64, p.V, a.hit, loss, lse);
  note_launch();
  return check_cuda(cudaGetLastError(), "loss join launch");
}

template <int NN>
int few_backward(om_backend* be, FewArgs a, const LossArgs& p, const float* lse,
                 const float* dloss, float* dx, int64_t dxd, int64_t dxn, float* dw, int64_t dwd, int64_t dwv) {
  constexpr int E = 4;
  const int blocks = (int)std::min<int64_t>((p.V + 8 * FEW_ROWS - 1) / (8 * FEW_ROWS), (int64_t)be->num_sms * 3);
  // ranges of 64 rows at least, which outweigh the block's part of dx
  const unsigned segments = (unsigned)((p.D + 256 * E - 1) / (256 * E));
  const int64_t fill = std::max<int64_t>(1, (int64_t)be->num_sms * 4 / segments);
  const int ranges = (int)std::max<int64_t>(1, std::min<int64_t>(p.V / 64, fill));
  Scratch ws;
  const int64_t nd = p.N * p.D;
  OM_TRY(ws.alloc(be, ((size_t)p.V * NN + (size_t)ranges * nd) * 4));
  a.lse = lse, a.dloss = dloss;
  a.dz = (float*)ws.ptr;
  a.acc = a.dz + p.V * NN;
  a.dw = dw, a.dwd = dwd, a.dwv = dwv;
  OM_TRY((launch_few_rows<NN, true>(be, a, blocks)));
  const bool vec = a.wd == 1 && dwd == 1 && !(((uintptr_t)a.w | (uintptr_t)dw) & 15) &&
                   a.wv * 4 % 16 == 0 && dwv * 4 % 16 == 0;
  {
    ProfScope prof(be, "loss_few_gradients");
    if (vec) few_outer_kernel<NN, true><<<dim3(ranges, segments), 256, 0, be->stream>>>(a);
    else few_outer_kernel<NN, false><<<dim3(ranges, segments), 256, 0, be->stream>>>(a);
    note_launch();
  }
  ProfScope prof(be, "loss_join_splits");
  few_join<<<(unsigned)((nd + 31) / 32), 256, 0, be->stream>>>(a.acc, ranges, nd, p.D, counted_of(p), dx, dxd, dxn);
  note_launch();
  return check_cuda(cudaGetLastError(), "loss backward launch");
}

FewArgs few_args(const LossArgs& p) {
  FewArgs a{};
  a.N = (int)p.N, a.D = p.D, a.V = p.V;
  a.x = (const float*)p.x, a.xd = p.xd, a.xn = p.xn;
  a.w = (const float*)p.w, a.wd = p.wd, a.wv = p.wv;
  a.targets = p.targets, a.t64 = p.target64;
  return a;
}
