// Rotary positions of several axes (MI355X, gfx950), forwards and back.
//
// Pair p of a head's dims belongs to one axis and turns by pos[axis(p)] * f(p):
//   y0 = x0 cos - x1 sin,  y1 = x0 sin + x1 cos  (inverse: the angle's negative, which
// is also the map's gradient, a rotation's transpose being its inverse).
// Pairs are neighbours (2p, 2p + 1) or halves (p, P + p) of the first 2P dims; the
// other dims pass through.
//
// HBM bound: 4 bytes of each value, 3 flop. An angle is formed as a number of turns in
// 64 bits (a position of 10^6 times a frequency has 20 bits before the point; fp32
// would leave 4 behind it), reduced to half a turn each way there, and only then
// rounded to fp32. That is done once for a token's pairs, into LDS; a thread keeps the 8
// cosines and sines of its 16 dims in registers over all heads it visits, the next of
// which it loads while it turns one. 2 x 8192 tokens of 48 heads: 75 us, 5.4 TB/s (84 us
// with four tokens in a workgroup, 77 without the loads ahead).
#include <limits.h>

#include "mm_common.hpp"

namespace mm {
namespace rope {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;

struct Args {
  char* x[2];                // q, k
  char* y[2];
  long long x_s[2][3], y_s[2][3];  // batch, position, head; elements
  const int* pos;
  long long pos_s[3];        // axis, batch, position
  const double* turns;       // [pairs]: turns per position
  const int* axes;           // [pairs]
  long long tokens;          // B * S
  int S, heads[2], pairs, n_axes, halves, inverse;
};

struct Chunk {
  u32x4 lo, hi;  // a thread's two runs of 8 dims
};

// Heads of TOKENS tokens that a workgroup visits at once, 16 dims for each thread.
constexpr int heads_at_once(int D, int tokens) { return kThreads / (D / 16 * tokens); }

template <int D, int TOKENS>
__global__ __launch_bounds__(kThreads) void rope_kernel(const Args a) {
  constexpr int kChunks = D / 16, kHeads = heads_at_once(D, TOKENS);
  __shared__ float2 sh[TOKENS][kMaxPairs];
  const int tid = threadIdx.x, c = tid % kChunks, t = tid / kChunks % TOKENS;
  const long long tok0 = (long long)blockIdx.x * TOKENS;
  const auto place = [&](int i, long long& b, long long& s) {  // the last token in place of those past it
    const long long tok = min(tok0 + i, a.tokens - 1);
    b = tok / a.S;
    s = tok - b * a.S;
  };
  long long b, s;
  place(t, b, s);
  // Byte offsets of the thread's two runs of 8 dims.
  const bool turned = 8 * c < a.pairs;
  const int d0 = 2 * (turned && a.halves ? 8 * c : 16 * c);
  const int d1 = turned && a.halves ? d0 + 2 * a.pairs : d0 + 16;
  const int all = a.heads[0] + a.heads[1], step = kHeads * gridDim.y;
  const auto at = [&](int h, char* const (&base)[2], const long long (&st)[2][3]) {
    const int w = h >= a.heads[0];
    return base[w] + 2 * (b * st[w][0] + s * st[w][1] + (w ? h - a.heads[0] : h) * st[w][2]);
  };
  const auto load = [&](int h) {
    const char* x = at(min(h, all - 1), a.x, a.x_s);
    return Chunk{*reinterpret_cast<const u32x4*>(x + d0), *reinterpret_cast<const u32x4*>(x + d1)};
  };
  // The first head's dims are on their way while the angles are formed.
  int h = blockIdx.y * kHeads + tid / (kChunks * TOKENS);
  Chunk x = load(h);
  for (int i = tid; i < a.pairs * TOKENS; i += kThreads) {
    const int p = TOKENS == 1 ? i : i % a.pairs, u = TOKENS == 1 ? 0 : i / a.pairs;
    const int ax = min(max(a.axes[p], 0), a.n_axes - 1);
    long long bu, su;
    place(u, bu, su);
    const double turn = (double)a.pos[ax * a.pos_s[0] + bu * a.pos_s[1] + su * a.pos_s[2]] * a.turns[p];
    float sn, cs;
    sincospif(2.f * (float)(turn - rint(turn)), &sn, &cs);
    sh[u][p] = float2{cs, a.inverse ? -sn : sn};
  }
  __syncthreads();
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 y = turned ? sh[t][8 * c + e] : float2{1.f, 0.f};
    cs[e] = y.x;
    sn[e] = y.y;
  }
  for (; h < all && tok0 + t < a.tokens; h += step) {
    const Chunk next = load(h + step);
    Chunk y = x;
    if (turned) {
      const auto val = [](uint32_t pair, bool up) {
        return __builtin_bit_cast(float, up ? pair & 0xFFFF0000u : pair << 16);
      };
      if (a.halves) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float u[2], v[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = val(x.lo[i], e), q = val(x.hi[i], e);
            u[e] = p * cs[2 * i + e] - q * sn[2 * i + e];
            v[e] = p * sn[2 * i + e] + q * cs[2 * i + e];
          }
          y.lo[i] = pack2_bf16_canon<kRTNE>(u[0], u[1]);
          y.hi[i] = pack2_bf16_canon<kRTNE>(v[0], v[1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t pair = i < 4 ? x.lo[i & 3] : x.hi[i & 3];
          const float p = val(pair, false), q = val(pair, true);
          const uint32_t r = pack2_bf16_canon<kRTNE>(p * cs[i] - q * sn[i], p * sn[i] + q * cs[i]);
          if (i < 4) y.lo[i & 3] = r;
          else y.hi[i & 3] = r;
        }
      }
    }
    char* to = at(h, a.y, a.y_s);
    *reinterpret_cast<u32x4*>(to + d0) = y.lo;
    *reinterpret_cast<u32x4*>(to + d1) = y.hi;
    x = next;
  }
}

}  // namespace rope
}  // namespace mm

extern "C" {

int launch_rope_axes(const void* q, const void* k, void* q_out, void* k_out, const void* positions, const void* turns,
                     const void* axes, int B, int S, int Hq, int Hk, int head_dim, int n_pairs, int n_axes, int halves,
                     int inverse, const long long* strides, void* stream) {
  using namespace mm::rope;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return -2;
  if (Hq < 1 || Hk < 0) return -3;
  if (B < 0 || S < 0) return -4;
  if (n_pairs < 8 || n_pairs % 8 != 0 || 2 * n_pairs > head_dim || n_axes < 1) return -5;
  if (B == 0 || S == 0) return 0;
  if (!q || !q_out || !positions || !turns || !axes || !strides || (Hk > 0 && (!k || !k_out))) return -6;
  Args a{};
  a.x[0] = (char*)q;
  a.x[1] = (char*)k;
  a.y[0] = (char*)q_out;
  a.y[1] = (char*)k_out;
  for (int i = 0; i < 3; ++i) {
    a.x_s[0][i] = strides[i];
    a.x_s[1][i] = strides[3 + i];
    a.y_s[0][i] = strides[6 + i];
    a.y_s[1][i] = strides[9 + i];
    a.pos_s[i] = strides[12 + i];
  }
  a.pos = (const int*)positions;
  a.turns = (const double*)turns;
  a.axes = (const int*)axes;
  a.tokens = (long long)B * S;
  a.S = S;
  a.heads[0] = Hq;
  a.heads[1] = Hk;
  a.pairs = n_pairs;
  a.n_axes = n_axes;
  a.halves = halves != 0;
  a.inverse = inverse != 0;
  if ((long long)Hq + Hk > INT_MAX / 2) return -8;
  // A token for each workgroup, or four where its heads would leave half the threads idle.
  const int all = Hq + Hk, tokens = (long long)all * (head_dim / 16) > kThreads / 2 ? 1 : 4;
  const long long grid = (a.tokens + tokens - 1) / tokens;
  if (grid > UINT_MAX / kThreads) return -8;
  // Few tokens: the heads are shared out over more workgroups, up to two for each CU.
  const int once = heads_at_once(head_dim, tokens);
  const long long visits = (all + (long long)once - 1) / once;
  const long long parts = 512 / grid < 1 ? 1 : 512 / grid < visits ? 512 / grid : visits;
  void (*kern)(Args) = tokens == 1
                           ? (head_dim == 64    ? rope_kernel<64, 1>
                              : head_dim == 128 ? rope_kernel<128, 1>
                                                : rope_kernel<256, 1>)
                           : (head_dim == 64    ? rope_kernel<64, 4>
                              : head_dim == 128 ? rope_kernel<128, 4>
                                                : rope_kernel<256, 4>);
  hipLaunchKernelGGL(kern, dim3((unsigned)grid, (unsigned)parts), dim3(kThreads), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}

}  // extern "C"
