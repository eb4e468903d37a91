// Decode attention of grouped query heads over a paged K/V cache (MI355X, gfx950).
//
// For each request b of S cached tokens, query position t of q_len and query head
// h (kv head h / G, G = Hq / Hkv):
//   o = sum_j softmax_j(scale * q . k_j) v_j   over the tokens j < S - q_len + t + 1,
// zeros where that leaves no token, with lse = ln sum_j exp(scale * q . k_j).
//
// A task is one request, kv head and block of 16 * NT query rows (row t * G + g):
// its rows share every K and V element read. The tasks' 128-token tiles, in order,
// are cut into equal runs, one for each workgroup; a task that a cut divides leaves fp32
// records (O, m, l) that a second kernel joins. So the work is even whatever the
// lengths are, they are read on the device, and the workspace depends on neither.
//
// Within a workgroup the four waves take 32-token steps of a tile in turn, each with
// its own running maximum and sum (one pass over the data); they are joined in LDS
// at the end of a task.
//
// No operand passes through LDS. 16x16x32 MFMAs compute S^T = K Q^T and
// O^T = V^T P^T, so a lane keeps one query row (lane % 16) throughout:
//  - K, the A operand, wants 8 dims of token lane % 16: 16-byte loads.
//  - S^T gives lane group g = lane / 16 tokens 4g..4g+3 of each 16; these are taken
//    as the k indices 8g..8g+7 of the second product, so P needs no exchange.
//  - V^T wants 8 tokens of one dim. A lane loads the same D / 16 dims of its 8
//    tokens (16 lanes read a whole row) and transposes them in registers: one
//    v_perm for two elements. MFMA j's row i is dim (D / 16) i + j.
// What bf16 leaves of P goes through a second MFMA: the kernel is HBM bound and the
// matrix cores are idle, and the output is then off by its own rounding only.
#include <limits.h>

#include "gqa_common.hpp"

namespace mm {
namespace gqa {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kStep = 32;               // tokens of one wave's step
constexpr int kTile = kStep * kWaves;   // tokens of one workgroup's tile
constexpr int kMaxQLen = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DecodeArgs {
  const char* q;         // [B, q_len, Hq, D] bf16 by strides
  Cache k, v;
  char* out;             // [B, q_len, Hq, D] bf16 by strides
  float* lse;            // [B, q_len, Hq] contiguous, or null
  const int* seq_lens;   // [B]
  const int* table;      // [B, width] by table_s
  float* rec_o;          // [2 * grid][16 * NT][D]
  float* rec_ml;         // [2 * grid][16 * NT][2]
  int4* joins;           // [grid]: the task that ends in this workgroup's run and began before it
  long long q_s[3], out_s[3];  // batch, position, head; elements
  long long table_s;
  int B, q_len, Hq, Hkv, G, rows, row_blocks;
  int num_blocks, width, page_shift;
  float scale2;          // softmax scale * log2(e)
};

__device__ __forceinline__ float xor16_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto pr = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)pr[0]), __builtin_bit_cast(float, (uint32_t)pr[1]));
}
__device__ __forceinline__ float xor16_sum(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto pr = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)pr[0]) + __builtin_bit_cast(float, (uint32_t)pr[1]);
}

// Lengths and page ids are wave-uniform and do not change during a launch: through
// the scalar cache, beside the waits of the vector loads.
typedef const __attribute__((address_space(4))) int* ConstInts;

__device__ __forceinline__ int clamped_len(const DecodeArgs& a, int b) {
  const long long most = (long long)a.width << a.page_shift;
  const int n = a.seq_lens[b];
  return n < 0 ? 0 : (n > most ? (int)most : n);
}
__device__ __forceinline__ int tiles_of(int len) { return (len >> 7) + ((len & 127) != 0); }
static_assert(kTile == 128, "tiles_of counts 128-token tiles");

// What one 32-token step of a wave reads: two 16-token halves, each within a page.
template <int D, bool FP8>
struct Step {
  static constexpr int kRow = FP8 ? D : 2 * D;        // bytes of a row
  static constexpr int kKLoads = kRow / 64;           // 16-byte loads of K per lane and half
  static constexpr int kVWords = kRow / 64;           // dwords of V per lane and token
  u32x4 k[2][kKLoads];
  uint32_t v[8][kVWords];
  f32x4 ks[2], vs[2];
};

// The pages of a step's halves (wave-uniform, through the scalar cache).
struct Pages {
  int id[2];
};
__device__ __forceinline__ Pages step_pages(const DecodeArgs& a, ConstInts row, int tok) {
  Pages p;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = min((tok + 16 * i) >> a.page_shift, a.width - 1);
    const int id = row[at];
    p.id[i] = min(max(id, 0), a.num_blocks - 1);
  }
  return p;
}

template <int D, bool FP8>
__device__ __forceinline__ void load_k(const DecodeArgs& a, Step<D, FP8>& s, const Pages& pg, int tok, int head,
                                       int lane) {
  constexpr int kElem = FP8 ? 1 : 2;
  const uint32_t off = (uint32_t)(lane & 15) * (uint32_t)(a.k.row_s * kElem) + 16u * (lane >> 4);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = (tok + 16 * i) & ((1 << a.page_shift) - 1);
    const char* kb = a.k.base + (pg.id[i] * a.k.block_s + head * a.k.head_s + row * a.k.row_s) * kElem;
#pragma unroll
    for (int c = 0; c < Step<D, FP8>::kKLoads; ++c) s.k[i][c] = *reinterpret_cast<const u32x4*>(kb + off + 64 * c);
    if constexpr (FP8)
      s.ks[i] = *reinterpret_cast<const f32x4*>(a.k.scale + pg.id[i] * a.k.sblock_s + head * a.k.shead_s + row +
                                                4 * (lane >> 4));
  }
}

template <int D, bool FP8>
__device__ __forceinline__ void load_v(const DecodeArgs& a, Step<D, FP8>& s, const Pages& pg, int tok, int head,
                                       int lane) {
  using S = Step<D, FP8>;
  constexpr int kElem = FP8 ? 1 : 2;
  const uint32_t off = 4u * (lane >> 4) * (uint32_t)(a.v.row_s * kElem) + (uint32_t)(S::kVWords * 4 * (lane & 15));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = (tok + 16 * i) & ((1 << a.page_shift) - 1);
    const char* vb = a.v.base + (pg.id[i] * a.v.block_s + head * a.v.head_s + row * a.v.row_s) * kElem;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const char* p = vb + r * (a.v.row_s * kElem) + off;
      uint32_t* to = s.v[4 * i + r];
      if constexpr (S::kVWords == 1) {
        to[0] = *reinterpret_cast<const uint32_t*>(p);
      } else if constexpr (S::kVWords == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        to[0] = x[0];
        to[1] = x[1];
      } else {
#pragma unroll
        for (int c = 0; c < S::kVWords / 4; ++c) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(p + 16 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) to[4 * c + e] = x[e];
        }
      }
    }
    if constexpr (FP8)
      s.vs[i] = *reinterpret_cast<const f32x4*>(a.v.scale + pg.id[i] * a.v.sblock_s + head * a.v.shead_s + row +
                                                4 * (lane >> 4));
  }
}

// A wave's state: its query rows and what it has summed for them.
template <int D, int NT>
struct Rows {
  bf16x8 q[NT][D / 32];
  f32x4 o[NT][D / 16];   // o[nt][j][r]: row lane % 16, dim (D / 16) * (4 g + r) + j
  float m[NT], l[NT];    // log2 domain; l over this lane's tokens only
  int pos[NT];           // the row's query position
};

// P is held as two bf16: its upper half and the rest, 2^-16 of it lost. The rest of a
// P above zero is kept above zero, so that an infinity in V is not met by 0 * inf.
__device__ __forceinline__ float rest(float p, float upper) {
  return fmaxf(p - upper, fminf(p, kMinScale));
}

// Two bf16 pairs (one of token e, one of e + 1) -> the pair of their `hi` elements.
__device__ __forceinline__ uint32_t zip(uint32_t even, uint32_t odd, bool hi) {
  return __builtin_amdgcn_perm(odd, even, hi ? 0x07060302u : 0x05040100u);
}

// O^T += V^T P^T for one step's 32 tokens. TAIL: tokens of `end` and above are
// hidden from query position `only` and must not reach it even as 0 * NaN.
template <int D, bool FP8, int NT, bool TAIL>
__device__ __forceinline__ void add_pv(Rows<D, NT>& w, const Step<D, FP8>& s, const bf16x8 (&hi)[NT],
                                       const bf16x8 (&lo)[NT], int tok0, int end, int only) {
  using S = Step<D, FP8>;
  constexpr int kPerWord = FP8 ? 4 : 2;  // elements of one dword of V
#pragma unroll
  for (int c = 0; c < S::kVWords; ++c) {
    uint32_t x[8][kPerWord / 2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t word = s.v[e][c];
      if constexpr (TAIL) word = tok0 + (e & 3) + 16 * (e >> 2) < end ? word : 0u;
      if constexpr (FP8) {
        const u32x2 y = fp8x4_to_bf16(word);
        x[e][0] = y[0];
        x[e][1] = y[1];
      } else {
        x[e][0] = word;
      }
    }
#pragma unroll
    for (int h = 0; h < kPerWord; ++h) {
      u32x4 f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = zip(x[2 * e][h / 2], x[2 * e + 1][h / 2], h & 1);
      const bf16x8 vf = __builtin_bit_cast(bf16x8, f);
      const int j = c * kPerWord + h;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        f32x4 acc = mfma16(vf, hi[nt], w.o[nt][j]);
        acc = mfma16(vf, lo[nt], acc);
        if constexpr (TAIL) {
#pragma unroll
          for (int r = 0; r < 4; ++r) w.o[nt][j][r] = w.pos[nt] == only ? acc[r] : w.o[nt][j][r];
        } else {
          w.o[nt][j] = acc;
        }
      }
    }
  }
}

// One step's 32 tokens. Without TAIL every query position sees them all, and each
// operand's registers take the next step's loads as soon as the products have read
// them, so about a step (16 KB for 128 bf16 dims) is in flight for each wave at any time.
template <int D, bool FP8, int NT, bool TAIL>
__device__ __forceinline__ void compute_step(const DecodeArgs& a, Rows<D, NT>& w, Step<D, FP8>& s, int tok, int len,
                                             const Pages& pg, int next, int head, int lane) {
  using S = Step<D, FP8>;
  const int tok0 = tok + 4 * (lane >> 4);  // this lane's tokens: tok0 + r and tok0 + 16 + r
  bf16x8 hi[NT], lo[NT];
  f32x4 sc[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) sc[nt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int c = 0; c < S::kKLoads; ++c) {
      if constexpr (FP8) {
        // 16 dims of a load feed two MFMAs: Q is laid out to match.
        bf16x8 kf[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x2 x = fp8x4_to_bf16(s.k[i][c][2 * h]), y = fp8x4_to_bf16(s.k[i][c][2 * h + 1]);
          kf[h] = __builtin_bit_cast(bf16x8, u32x4{x[0], x[1], y[0], y[1]});
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[nt][i] = mfma16(kf[0], w.q[nt][2 * c], sc[nt][i]);
          sc[nt][i] = mfma16(kf[1], w.q[nt][2 * c + 1], sc[nt][i]);
        }
      } else {
        const bf16x8 kf = __builtin_bit_cast(bf16x8, s.k[i][c]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][i] = mfma16(kf, w.q[nt][c], sc[nt][i]);
      }
    }
  }
  const f32x4 ks[2] = {s.ks[0], s.ks[1]};
  if constexpr (!TAIL) load_k<D, FP8>(a, s, pg, next, head, lane);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int end = len - a.q_len + w.pos[nt] + 1;  // the row sees the tokens before it
    float mx = w.m[nt];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = sc[nt][i][r] * a.scale2;
        if constexpr (FP8) x *= ks[i][r];
        if constexpr (TAIL) x = tok0 + 16 * i + r < end ? x : -__builtin_inff();
        sc[nt][i][r] = x;
        mx = fmaxf(mx, x);
      }
    mx = xor32_max(xor16_max(mx));
    // Nothing to rescale unless some row's maximum rose.
    if (__any(mx > w.m[nt])) {
      const float f = __builtin_amdgcn_exp2f(w.m[nt] - mx);
      w.l[nt] *= f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) w.o[nt][j][r] *= f;
      w.m[nt] = mx;
    }
    float p[8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = __builtin_amdgcn_exp2f(sc[nt][i][r] - mx);
        sum += x;
        if constexpr (FP8) x *= s.vs[i][r];
        if constexpr (TAIL) x = tok0 + 16 * i + r < end ? x : 0.f;  // a hidden row's scale may be NaN
        p[4 * i + r] = x;
      }
    w.l[nt] += sum;
    u32x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      h[e] = pack2_bf16<kRTZ>(p[2 * e], p[2 * e + 1]);
      l[e] = pack2_bf16<kRTNE>(rest(p[2 * e], bf16_lo(h[e])), rest(p[2 * e + 1], bf16_hi(h[e])));
    }
    hi[nt] = __builtin_bit_cast(bf16x8, h);
    lo[nt] = __builtin_bit_cast(bf16x8, l);
  }
  if constexpr (TAIL) {
    // Query positions see different numbers of these tokens: each adds its own.
    for (int t = 0; t < a.q_len; ++t) add_pv<D, FP8, NT, true>(w, s, hi, lo, tok0, len - a.q_len + t + 1, t);
  } else {
    add_pv<D, FP8, NT, false>(w, s, hi, lo, tok0, 0, 0);
    load_v<D, FP8>(a, s, pg, next, head, lane);
  }
}

__device__ __forceinline__ long long uniform(long long x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (long long)((uint64_t)hi << 32 | lo);
}

// The runs: tile i of `total` belongs to run w where start(w) <= i < start(w + 1),
// start(w) = floor(w * total / runs). No run is empty: there are at most `total`.
__device__ __forceinline__ long long run_start(long long total, int runs, int w) {
  return total / runs * w + total % runs * w / runs;
}

// A workgroup's run, and the request in which its first tile lies with the number
// of tiles before that. Every thread calls it.
struct Run {
  long long total;
  long long start, end;   // tiles of all tasks, in order
  long long before;       // tiles before request b
  int runs, b;
};
__device__ Run find_run(const DecodeArgs& a, int wg, int grid, long long* sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = a.Hkv * a.row_blocks;
  long long mine = 0;
  for (int b = tid; b < a.B; b += kThreads) mine += (long long)tiles_of(clamped_len(a, b));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) mine += __shfl_xor(mine, d);
  if (lane == 0) sh[wave] = mine;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) total += sh[i];
  __syncthreads();
  Run run;
  run.total = total = uniform(total * per);
  run.runs = (int)min((long long)grid, total);
  run.start = run.end = run.before = 0;
  run.b = a.B;
  if (wg >= run.runs) return run;
  run.start = run_start(total, run.runs, wg);
  run.end = run_start(total, run.runs, wg + 1);
  // Requests in groups of 256: a prefix sum finds the one that holds `start`.
  long long base = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + tid;
    const long long n = b < a.B ? (long long)tiles_of(clamped_len(a, b)) * per : 0;
    long long incl = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const long long x = __shfl_up(incl, d);
      if (lane >= d) incl += x;
    }
    if (lane == 63) sh[wave] = incl;
    __syncthreads();
    long long ahead = base, sum = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) ahead += sh[i];
      sum += sh[i];
    }
    if (n > 0 && run.start >= ahead + incl - n && run.start < ahead + incl) {
      sh[kWaves] = b;
      sh[kWaves + 1] = ahead + incl - n;
    }
    __syncthreads();
    if (run.start < base + sum) {
      run.b = __builtin_amdgcn_readfirstlane((int)sh[kWaves]);
      run.before = uniform(sh[kWaves + 1]);
      __syncthreads();
      return run;
    }
    base += sum;
    __syncthreads();
  }
  return run;
}

// Workgroups of a CU: as many as the registers of their waves allow (512 of a SIMD).
template <int D, int NT>
constexpr int kPerCu = D * NT <= 128 ? 2 : 1;

template <int D, bool FP8, int NT>
__global__ __launch_bounds__(kThreads, (kPerCu<D, NT>)) void gqa_decode_kernel(const DecodeArgs a, const int split) {
  constexpr int kRows = 16 * NT;
  constexpr int kPitch = D + 4;  // floats: rows of the join start on different banks
  __shared__ float sh_o[kWaves][16][kPitch];
  __shared__ float sh_ml[kWaves][kRows][2];
  __shared__ long long sh_plan[kWaves + 2];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grid = gridDim.x;
  const int wg = xcd_remap(blockIdx.x, grid);
  const int per = a.Hkv * a.row_blocks;

  Run run{};
  if (split) {
    run = find_run(a, wg, grid, sh_plan);
    if (tid == 0) a.joins[wg] = int4{-1, 0, 0, 0};
  } else {  // a whole task for each workgroup
    run.b = wg / per;
    const int n = tiles_of(clamped_len(a, run.b));
    run.before = 0;
    run.start = (long long)(wg % per) * n;
    run.end = run.start + n;
  }
  bool first = true;
  int b = run.b;
  long long at = run.start, before = run.before;
  while (at < run.end && b < a.B) {
    const int len = __builtin_amdgcn_readfirstlane(clamped_len(a, b));
    const int tiles = tiles_of(len);
    if (at - before >= (long long)tiles * per) {  // done with request b
      before += (long long)tiles * per;
      ++b;
      continue;
    }
    const int task = __builtin_amdgcn_readfirstlane((int)((at - before) / tiles));
    const int tile0 = __builtin_amdgcn_readfirstlane((int)((at - before) - (long long)task * tiles));
    const int tile1 = __builtin_amdgcn_readfirstlane((int)min((long long)tiles, tile0 + (run.end - at)));
    const int head = task / a.row_blocks, row0 = (task % a.row_blocks) * kRows;
    const int rows = min(kRows, a.rows - row0);
    const ConstInts table = (ConstInts)(uintptr_t)(a.table + (long long)b * a.table_s);

    Rows<D, NT> w;
    const int n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + 16 * nt + n;
      const bool live = 16 * nt + n < rows;
      const int t = live ? r / a.G : a.q_len - 1;
      w.pos[nt] = t;
      w.m[nt] = kNegFltMax;
      w.l[nt] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) w.o[nt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      const char* qr = a.q + 2 * (b * a.q_s[0] + t * a.q_s[1] + (head * a.G + (live ? r - t * a.G : 0)) * a.q_s[2]);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        // dims of MFMA c for lane group g, as K's loads have them
        const int d = FP8 ? 64 * (c / 2) + 16 * g + 8 * (c & 1) : 32 * c + 8 * g;
        u32x4 x = *reinterpret_cast<const u32x4*>(qr + 2 * d);
        if (!live) x = u32x4{0u, 0u, 0u, 0u};
        w.q[nt][c] = __builtin_bit_cast(bf16x8, x);
      }
    }

    // This wave's steps: every fourth one. Only the last can hold a token that some
    // position does not see (q_len - 1 + 31 tokens lie in two steps at most, of two
    // waves). Loads past the last step repeat it: one under a branch would make the
    // compiler wait for all of them.
    int st = tile0 * kWaves + wave;
    const int s_end = min(tile1 * kWaves, (len + kStep - 1) / kStep);
    if (st < s_end) {
      const int s_last = st + (s_end - 1 - st) / kWaves * kWaves;
      const int s_full = (len - a.q_len + 1) >> 5;  // steps before it are seen by all
      static_assert(kStep == 32, "s_full counts 32-token steps");
      Step<D, FP8> s;
      Pages pg = step_pages(a, table, st * kStep);
      load_k<D, FP8>(a, s, pg, st * kStep, head, lane);
      load_v<D, FP8>(a, s, pg, st * kStep, head, lane);
      int next = min(st + kWaves, s_last);
      pg = step_pages(a, table, next * kStep);
      for (; st <= s_last && st < s_full; st += kWaves) {
        const int after = min(next + kWaves, s_last);
        const Pages pa = step_pages(a, table, after * kStep);
        compute_step<D, FP8, NT, false>(a, w, s, st * kStep, len, pg, next * kStep, head, lane);
        pg = pa;
        next = after;
      }
      if (st <= s_last) compute_step<D, FP8, NT, true>(a, w, s, st * kStep, len, pg, 0, head, lane);
    }

    // Join the waves.
    const bool whole = tile0 == 0 && tile1 == tiles;
    const int rec = 2 * wg + (first ? 0 : 1);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      w.l[nt] = xor32_sum(xor16_sum(w.l[nt]));
      if (g == 0) {
        sh_ml[wave][16 * nt + n][0] = w.m[nt];
        sh_ml[wave][16 * nt + n][1] = w.l[nt];
      }
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (16 * nt < rows) {
        {
          float top = sh_ml[0][16 * nt + n][0];
#pragma unroll
          for (int i = 1; i < kWaves; ++i) top = fmaxf(top, sh_ml[i][16 * nt + n][0]);
          const float f = __builtin_amdgcn_exp2f(w.m[nt] - top);
          // A lane's dims (D / 16) * 4 g .. + D / 4 of its row, in order.
          float* to = &sh_o[wave][n][D / 4 * g];
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < D / 16; j += 4)
              *reinterpret_cast<f32x4*>(to + (D / 16) * r + j) =
                  f32x4{w.o[nt][j][r] * f, w.o[nt][j + 1][r] * f, w.o[nt][j + 2][r] * f, w.o[nt][j + 3][r] * f};
        }
        __syncthreads();
        {
          // 16 threads for each row, D / 16 dims each.
          constexpr int kPer = D / 16;
          const int r = tid >> 4, d0 = (tid & 15) * kPer, row = 16 * nt + r;
          if (row < rows) {
            float top = sh_ml[0][row][0];
#pragma unroll
            for (int i = 1; i < kWaves; ++i) top = fmaxf(top, sh_ml[i][row][0]);
            float l = 0.f;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) l += sh_ml[i][row][1] * __builtin_amdgcn_exp2f(sh_ml[i][row][0] - top);
            float o[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
              o[j] = 0.f;
#pragma unroll
              for (int i = 0; i < kWaves; ++i) o[j] += sh_o[i][r][d0 + j];
            }
            if (whole) {
              const int R = row0 + row, t = R / a.G, h = head * a.G + R - t * a.G;
              const bool none = len - a.q_len + t + 1 <= 0;  // the row sees no token
              const float inv = 1.f / l;
              char* to = a.out + 2 * (b * a.out_s[0] + t * a.out_s[1] + h * a.out_s[2] + d0);
#pragma unroll
              for (int j = 0; j < kPer; j += 4) {
                u32x2 x;
                x[0] = pack2_bf16_canon<kRTNE>(o[j] * inv, o[j + 1] * inv);
                x[1] = pack2_bf16_canon<kRTNE>(o[j + 2] * inv, o[j + 3] * inv);
                if (none) x = u32x2{0u, 0u};
                *reinterpret_cast<u32x2*>(to + 2 * j) = x;
              }
              if (a.lse && (tid & 15) == 0)
                a.lse[((long long)b * a.q_len + t) * a.Hq + h] =
                    none ? -__builtin_inff() : kLn2 * (top + __builtin_amdgcn_logf(l));
            } else {
              float* to = a.rec_o + ((long long)rec * kRows + row) * D + d0;
#pragma unroll
              for (int j = 0; j < kPer; j += 4)
                *reinterpret_cast<f32x4*>(to + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
              if ((tid & 15) == 0) {
                a.rec_ml[((long long)rec * kRows + row) * 2] = top;
                a.rec_ml[((long long)rec * kRows + row) * 2 + 1] = l;
              }
            }
          }
        }
        __syncthreads();
      }
    }
    if (!whole && tile1 == tiles && tid == 0) {
      // The task ends here and began in an earlier run: that run, and which of its
      // two records holds it (the first segment's, or the last's).
      const long long began = before + (long long)task * tiles;
      int w0 = (int)(began * run.runs / run.total);
      while (run_start(run.total, run.runs, w0) > began) --w0;
      while (run_start(run.total, run.runs, w0 + 1) <= began) ++w0;
      a.joins[wg] = int4{b, task, w0, run_start(run.total, run.runs, w0) == began ? 0 : 1};
    }
    first = false;
    at += tile1 - tile0;
  }

  // Requests without a token: zeros.
  const int step = split ? grid : 1;
  for (int e = split ? wg : wg / per; e < a.B; e += step) {
    if (clamped_len(a, e) == 0) {
      const int lo = split ? 0 : wg % per, hi = split ? per : lo + 1;
      for (int task = lo; task < hi; ++task) {
        const int head = task / a.row_blocks, row0 = (task % a.row_blocks) * kRows;
        const int rows = min(kRows, a.rows - row0);
        for (int i = tid; i < rows * (D / 8); i += kThreads) {
          const int R = row0 + i / (D / 8), t = R / a.G, h = head * a.G + R - t * a.G;
          *reinterpret_cast<u32x4*>(a.out + 2 * (e * a.out_s[0] + t * a.out_s[1] + h * a.out_s[2] + 8 * (i % (D / 8)))) =
              u32x4{0u, 0u, 0u, 0u};
          if (a.lse && i % (D / 8) == 0) a.lse[((long long)e * a.q_len + t) * a.Hq + h] = -__builtin_inff();
        }
      }
    }
    if (!split) break;
  }
}

// Joins the records of a task that several runs hold: rows of O and (m, l), summed in
// the order of the runs. Launched for every run; one that ends no such task
// returns. PER_ROW waves share a row's records.
template <int D, int NT, int PER_ROW>
__global__ __launch_bounds__(kThreads) void gqa_join_kernel(const DecodeArgs a) {
  constexpr int kRows = 16 * NT, kPer = D / 64;
  __shared__ float sh[PER_ROW > 1 ? PER_ROW : 1][D];
  const int wg = blockIdx.x;
  const int4 j = a.joins[wg];
  if (j.x < 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int head = j.y / a.row_blocks, row0 = (j.y % a.row_blocks) * kRows;
  const int row = blockIdx.y * (kWaves / PER_ROW) + wave / PER_ROW;
  if (row >= min(kRows, a.rows - row0)) return;
  const int n = wg - j.z + 1;
  const auto record = [&](int i) { return ((long long)(2 * (j.z + i) + (i == 0 ? j.w : 0)) * kRows + row); };
  float top = kNegFltMax;
  for (int i = lane; i < n; i += 64) top = fmaxf(top, a.rec_ml[record(i) * 2]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  float l = 0.f;
  for (int i = lane; i < n; i += 64)
    l += a.rec_ml[record(i) * 2 + 1] * __builtin_amdgcn_exp2f(a.rec_ml[record(i) * 2] - top);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
  float o[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int i = wave % PER_ROW; i < n; i += PER_ROW) {
    const long long r = record(i);
    const float f = __builtin_amdgcn_exp2f(a.rec_ml[r * 2] - top);
    const float* from = a.rec_o + r * D + lane * kPer;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] += f * from[e];
  }
  if constexpr (PER_ROW > 1) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) sh[wave][lane * kPer + e] = o[e];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      o[e] = 0.f;
#pragma unroll
      for (int i = 0; i < PER_ROW; ++i) o[e] += sh[i][lane * kPer + e];
    }
  }
  const int R = row0 + row, t = R / a.G, h = head * a.G + R - t * a.G;
  const float inv = 1.f / l;
  uint16_t* to = reinterpret_cast<uint16_t*>(a.out) + j.x * a.out_s[0] + t * a.out_s[1] + h * a.out_s[2] + lane * kPer;
  if constexpr (kPer == 1) {
    *to = (uint16_t)pack2_bf16_canon<kRTNE>(o[0] * inv, 0.f);
  } else {
#pragma unroll
    for (int e = 0; e < kPer; e += 2)
      *reinterpret_cast<uint32_t*>(to + e) = pack2_bf16_canon<kRTNE>(o[e] * inv, o[e + 1] * inv);
  }
  if (a.lse && lane == 0) a.lse[((long long)j.x * a.q_len + t) * a.Hq + h] = kLn2 * (top + __builtin_amdgcn_logf(l));
}

// How a call is laid out: query rows of a task, tasks, workgroups, and whether they
// share the tiles out evenly (with a join) or take a whole task each.
struct Plan {
  int nt, row_blocks, grid, split;
  long long tasks;
};
constexpr int kCus = 256;
// Up to this many tiles in the longest request a call runs a workgroup for each
// task, without the plan's reads and the second launch.
constexpr int kShortTiles = 4;

inline bool plan_call(int B, int q_len, int Hq, int Hkv, int D, int page, int width, Plan* p) {
  const long long rows = (long long)(Hq / Hkv) * q_len;
  p->nt = rows <= 16 ? 1 : (rows <= 32 || D == 256) ? 2 : 4;
  p->row_blocks = (int)((rows + 16 * p->nt - 1) / (16 * p->nt));
  p->tasks = (long long)B * Hkv * p->row_blocks;
  const long long tiles = ((long long)page * width + kTile - 1) / kTile;
  const long long slots = kCus * (D * p->nt <= 128 ? 2 : 1);
  p->split = tiles > kShortTiles;
  const long long grid = p->split ? (p->tasks >= slots ? slots : (p->tasks * tiles < slots ? p->tasks * tiles : slots)) : p->tasks;
  if (grid > INT_MAX) return false;
  p->grid = (int)grid;
  return true;
}
inline size_t record_bytes(const Plan& p, int D) { return (size_t)2 * p.grid * 16 * p.nt * (D + 2) * 4; }

template <int D, bool FP8, int NT>
int launch(DecodeArgs& a, const Plan& p, hipStream_t stream) {
  hipLaunchKernelGGL((gqa_decode_kernel<D, FP8, NT>), dim3(p.grid), dim3(kThreads), 0, stream, a, p.split);
  if (p.split) {
    const int rows = a.rows < 16 * NT ? a.rows : 16 * NT;
    if (p.tasks * 8 >= p.grid)
      hipLaunchKernelGGL((gqa_join_kernel<D, NT, 1>), dim3(p.grid, (rows + 3) / 4), dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((gqa_join_kernel<D, NT, 4>), dim3(p.grid, rows), dim3(kThreads), 0, stream, a);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}

template <bool FP8>
int dispatch(DecodeArgs& a, const Plan& p, int D, hipStream_t st) {
  if (D == 64) return p.nt == 1 ? launch<64, FP8, 1>(a, p, st) : p.nt == 2 ? launch<64, FP8, 2>(a, p, st) : launch<64, FP8, 4>(a, p, st);
  if (D == 128) return p.nt == 1 ? launch<128, FP8, 1>(a, p, st) : p.nt == 2 ? launch<128, FP8, 2>(a, p, st) : launch<128, FP8, 4>(a, p, st);
  return p.nt == 1 ? launch<256, FP8, 1>(a, p, st) : launch<256, FP8, 2>(a, p, st);
}

// -2 head_dim, -3 heads, -4 sizes, -5 page; 0 where the call can be planned.
inline int check_sizes(int B, int q_len, int Hq, int Hkv, int D, int page, int width) {
  if (D != 64 && D != 128 && D != 256) return -2;
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv != 0) return -3;
  if (B < 0 || q_len < 1 || q_len > kMaxQLen) return -4;
  if (page < 16 || (page & (page - 1)) != 0) return -5;
  if (width < 1) return -11;
  return 0;
}

}  // namespace gqa
}  // namespace mm

extern "C" {

size_t moonmath_gqa_decode_workspace(int B, int q_len, int Hq, int Hkv, int head_dim, int page, int max_blocks) {
  using namespace mm::gqa;
  Plan p;
  if (B == 0 || check_sizes(B, q_len, Hq, Hkv, head_dim, page, max_blocks) != 0) return 0;
  if (!plan_call(B, q_len, Hq, Hkv, head_dim, page, max_blocks, &p) || !p.split) return 0;
  return record_bytes(p, head_dim) + (size_t)p.grid * sizeof(int4);
}

int launch_gqa_decode_paged(const void* q, const void* k_cache, const void* v_cache, const void* k_scale,
                            const void* v_scale, void* out, void* lse, const void* seq_lens, const void* block_table,
                            int B, int q_len, int Hq, int Hkv, int head_dim, int num_blocks, int page, int max_blocks,
                            const long long* strides, float scale, void* workspace, void* stream) {
  using namespace mm::gqa;
  const int rc = check_sizes(B, q_len, Hq, Hkv, head_dim, page, max_blocks);
  if (rc != 0) return rc;
  if (num_blocks < 1) return -11;
  if (B == 0) return 0;
  if (!q || !k_cache || !v_cache || !out || !seq_lens || !block_table || !strides || !k_scale != !v_scale) return -6;
  Plan p;
  if (!plan_call(B, q_len, Hq, Hkv, head_dim, page, max_blocks, &p)) return -8;
  if (p.split && !workspace) return -6;
  DecodeArgs a{};
  a.q = (const char*)q;
  a.k = make_cache(k_cache, k_scale, strides + 6);
  a.v = make_cache(v_cache, v_scale, strides + 11);
  a.out = (char*)out;
  a.lse = (float*)lse;
  a.seq_lens = (const int*)seq_lens;
  a.table = (const int*)block_table;
  for (int i = 0; i < 3; ++i) {
    a.q_s[i] = strides[i];
    a.out_s[i] = strides[3 + i];
  }
  a.table_s = strides[16];
  // A lane adds up to 15 rows to a page's address in 32 bits.
  const long long widest = 1LL << 26;
  if (a.k.row_s < 0 || a.v.row_s < 0 || a.k.row_s > widest || a.v.row_s > widest) return -9;
  a.rec_o = (float*)workspace;
  a.rec_ml = a.rec_o + (size_t)2 * p.grid * 16 * p.nt * head_dim;
  a.joins = (int4*)(a.rec_ml + (size_t)2 * p.grid * 16 * p.nt * 2);
  a.B = B;
  a.q_len = q_len;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.rows = a.G * q_len;
  a.row_blocks = p.row_blocks;
  a.num_blocks = num_blocks;
  a.width = max_blocks;
  a.page_shift = __builtin_ctz(page);
  a.scale2 = scale * kLog2e;
  return k_scale ? dispatch<true>(a, p, head_dim, (hipStream_t)stream) : dispatch<false>(a, p, head_dim, (hipStream_t)stream);
}

}  // extern "C"
