// pd_weights.cu -- attention weights of one decode step added to running sums (sm_100a).
//
// The decode kernel's scores variant leaves every score s (log2 units) of the step and each (row, q head)'s
// maximum m and normaliser l = sum exp2(s - m). This kernel adds to row b, kv head h, token j
//   sum over the group's q heads of exp2(s - m) / l,
// which needs m and l of the whole row, so it is a second launch; it is a programmatic dependent one, whose
// CTAs are resident when the decode's last one ends. A (row, kv head)'s sums have one writer per token: no atomics.
//
// Bound by memory where it is not by its launch: 4 bytes per (token, q head), just written and so mostly in L2,
// and 8 per (token, kv head), next to 4 * head_dim of K and V in the decode itself. 32 rows of 2048 tokens, 16 heads on
// 8: the decode 46.5 us, this launch 4.3 more.
#include "pd_internal.h"

namespace pd {

namespace {

constexpr int THREADS = 256;
constexpr int AHEAD = 4;  // tokens of a thread in flight

// G: q heads per kv head where vector loads fit, or 0 (any).
template <int G>
__global__ void __launch_bounds__(THREADS) pd_weights_kernel(const WeightsParams p) {
  const int h = blockIdx.y, b = blockIdx.z;
  griddep_wait();  // (the next decode is not let in before this kernel is through: its CTAs would take the SMs)
  int len = __ldg(p.seqlen + b);
  len = len < 0 ? 0 : (len > p.capacity ? p.capacity : len);
  const int group = G ? G : p.group;
  const int64_t item = int64_t(b) * p.n_kv_head + h;
  const float* scores = p.scores + item * p.capacity * group;
  const float *m = p.m + item * group, *l = p.l + item * group;
  float* w = p.weights + int64_t(b) * p.w_sb + int64_t(h) * p.w_sh;
  constexpr int N = G ? G : 1;
  float mg[N], inv[N];
  if constexpr (G != 0) {
    if (int(blockIdx.x) * THREADS * AHEAD >= len) return;
#pragma unroll
    for (int g = 0; g < N; ++g) {
      mg[g] = __ldg(m + g);
      inv[g] = 1.f / __ldg(l + g);
    }
  }
  for (int j0 = int(blockIdx.x) * THREADS * AHEAD; j0 < len; j0 += int(gridDim.x) * THREADS * AHEAD) {
    float sum[AHEAD], old[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int j = j0 + i * THREADS + int(threadIdx.x);
      old[i] = sum[i] = 0.f;
      if (j >= len) continue;
      old[i] = w[j];
      const float* s = scores + int64_t(j) * group;
      if constexpr (G == 0) {
        for (int g = 0; g < group; ++g) sum[i] += exp2f(s[g] - __ldg(m + g)) / __ldg(l + g);
      } else {
        float x[N];
        if constexpr (G >= 4) {
#pragma unroll
          for (int g = 0; g < N; g += 4) {
            const float4 v = *reinterpret_cast<const float4*>(s + g);
            x[g] = v.x;
            x[g + 1] = v.y;
            x[g + 2] = v.z;
            x[g + 3] = v.w;
          }
        } else if constexpr (G == 2) {
          const float2 v = *reinterpret_cast<const float2*>(s);
          x[0] = v.x;
          x[1] = v.y;
        } else {
          x[0] = s[0];
        }
#pragma unroll
        for (int g = 0; g < N; ++g) sum[i] = fmaf(exp2f(x[g] - mg[g]), inv[g], sum[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int j = j0 + i * THREADS + int(threadIdx.x);
      if (j < len) w[j] = old[i] + sum[i];
    }
  }
}

}  // namespace

cudaError_t launch_weights(const WeightsParams& p0, cudaStream_t stream) {
  WeightsParams p = p0;
  // CTAs per (row, head): enough to cover the table, at most about 16 per SM in all
  const int64_t items = int64_t(p.batch) * p.n_kv_head;
  int64_t x = (int64_t(p.capacity) + THREADS * AHEAD - 1) / (THREADS * AHEAD);
  const int64_t most = 16 * int64_t(p.sms) / items;
  if (x > most) x = most;
  if (x < 1) x = 1;
  void (*fn)(WeightsParams) = pd_weights_kernel<0>;
  switch (p.group) {
    case 1: fn = pd_weights_kernel<1>; break;
    case 2: fn = pd_weights_kernel<2>; break;
    case 4: fn = pd_weights_kernel<4>; break;
    case 8: fn = pd_weights_kernel<8>; break;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  // rows in parts that fit a grid's third dimension
  const int batch = p.batch, most_rows = 65535;
  for (int b0 = 0; b0 < batch; b0 += most_rows) {
    p.batch = batch - b0 < most_rows ? batch - b0 : most_rows;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(x), unsigned(p.n_kv_head), unsigned(p.batch));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, p);
    if (e != cudaSuccess) return e;
    const int64_t heads = int64_t(p.batch) * p.n_kv_head * p.group;
    p.scores += heads * p.capacity;
    p.m += heads;
    p.l += heads;
    p.seqlen += p.batch;
    p.weights += int64_t(p.batch) * p.w_sb;
  }
  return cudaSuccess;
}

}  // namespace pd
