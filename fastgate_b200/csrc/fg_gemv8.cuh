// int8 x int8 GEMV for one or two token rows (fg_linear_w8a8).
//
// A call of this size is a stream of the weight and the latencies around it: one warp takes R weight rows, its lanes stride
// over k in 16-byte pieces, four dp4a per piece and token row, one integer reduction across the warp at the end.  No
// ring, no partial tiles, no tickets: nothing stands between the last byte and the output.  The first pieces of the weight
// are asked for before the previous kernel of the stream has finished (it may not be that kernel's output; the activations
// are read after griddepcontrol.wait, through L1: every warp of an SM reads the same ones).
// Measured on B200 (us, one / two token rows, weights from memory, call after call): 1024 x 1024 1.6 / 1.8, 4096 x 4096 4.7 / 5.4,
// 11008 x 4096 8.9 / 10.0, 8192 x 8192 12.1 / 13.4, 28672 x 8192 35.7 / 38.8 (the weight at the measured copy bandwidth: 35.9; a weight
// of 17 MB that stays in L2: 3.7).  Four token rows took 7 to 52, against 8 to 38 in the tensor-core kernel: L1 cannot deliver the
// activations that often.
// Weights above 60 MB: a warp with two weight rows halves the reads of x (8192 x 8192 12.1 / 13.4, with one row 14.4 / 16.9;
// 28672 x 8192 35.7 / 38.8 and 36.1 / 38.9).  Below, one weight row a warp spreads the few rows wider (4096 x 4096 4.7 / 5.4, with two
// 5.0 / 5.7; 11008 x 4096 8.9 / 10.0 and 9.7 / 11.8; 4096 x 11008 alone gains with two tokens, 10.5 / 12.0 and 10.7 / 11.7).
#pragma once
#include "fg_w8a8.cuh"

namespace fg {

constexpr int kGemv8Warps = 4;
constexpr int kGemv8MaxM = 2;
constexpr int kGemv8Pieces = 4;                          // 16-byte pieces of each of its rows that a lane has in flight
constexpr long long kGemv8TwoRowBytes = 60LL * 1000 * 1000;  // larger weights: two rows per warp

struct Gemv8Params {
  const int8_t* x;           // [M, K]
  const int8_t* W;           // [N, K]
  W8A8Params out;
};

template <int M, int R>
__global__ void __launch_bounds__(kGemv8Warps * 32) fg_gemv8_kernel(const Gemv8Params p) {
  const int lane = threadIdx.x & 31;
  const long long wid = static_cast<long long>(blockIdx.x) * kGemv8Warps + (threadIdx.x >> 5);
  const int K = p.out.K, N = p.out.N;
  const bool gated = p.out.act == kActSiluGate;
  // Rows of this warp: n0, n0 + step, ...: neighbours, or with the SiLU gate R/2 gate rows and the matching up rows 64 further.
  const int first = static_cast<int>(wid * R);
  int n[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    n[r] = gated && R > 1 ? gate_row(first / 2 + r / 2) + (r & 1) * 64 : first + r;
  }
  if (first >= N) return;
  const int pieces = K / 16;
  const uint4* w[R];
#pragma unroll
  for (int r = 0; r < R; ++r) w[r] = reinterpret_cast<const uint4*>(p.W + static_cast<size_t>(n[r]) * K);
  const uint4* x = reinterpret_cast<const uint4*>(p.x);
  int acc[R][M];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) acc[r][m] = 0;

  uint4 q[kGemv8Pieces][R];
  auto load = [&](int at) {
#pragma unroll
    for (int i = 0; i < kGemv8Pieces; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r) q[i][r] = at + 32 * i < pieces ? __ldcs(w[r] + at + 32 * i) : make_uint4(0, 0, 0, 0);
  };
  load(lane);
  griddep_wait();
  griddep_launch_dependents();
  for (int at = lane; at < pieces;) {
#pragma unroll
    for (int i = 0; i < kGemv8Pieces; ++i) {
      if (at + 32 * i < pieces) {
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const uint4 v = x[static_cast<size_t>(m) * pieces + at + 32 * i];
#pragma unroll
          for (int r = 0; r < R; ++r) {
            acc[r][m] = __dp4a(static_cast<int>(q[i][r].x), static_cast<int>(v.x), acc[r][m]);
            acc[r][m] = __dp4a(static_cast<int>(q[i][r].y), static_cast<int>(v.y), acc[r][m]);
            acc[r][m] = __dp4a(static_cast<int>(q[i][r].z), static_cast<int>(v.z), acc[r][m]);
            acc[r][m] = __dp4a(static_cast<int>(q[i][r].w), static_cast<int>(v.w), acc[r][m]);
          }
        }
      }
    }
    at += 32 * kGemv8Pieces;
    if (at - lane < pieces) load(at);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) acc[r][m] = __reduce_add_sync(0xffffffffu, acc[r][m]);
  // lane r M + m finishes output (m, n[r]); the gated pair (rows 2 i, 2 i + 1) is finished by the gate row's lane
  auto value = [&](int r, int m) {
    return w8a8_value(acc[r][m], x_scale(p.out, m), p.out.w_scales ? __half2float(p.out.w_scales[n[r]]) : 1.f,
                      p.out.bias ? __half2float(p.out.bias[n[r]]) : 0.f);
  };
  auto store = [&](int m, int width, int col, float y) {
    const size_t at = static_cast<size_t>(m) * width + col;
    if (p.out.residual != nullptr) y = __fadd_rn(y, __half2float(p.out.residual[at]));
    p.out.C[at] = __float2half_rn(y);
  };
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      if (lane != r * M + m) continue;
      if (gated) {
        if (R > 1 && (r & 1) == 0) store(m, N / 2, first / 2 + r / 2, w8a8_gate(value(r, m), value(r + (R > 1), m)));
      } else {
        with_act(p.out.act, [&](auto tag) { store(m, N, n[r], w8a8_act<decltype(tag)::value>(value(r, m))); });
      }
    }
}

}  // namespace fg
