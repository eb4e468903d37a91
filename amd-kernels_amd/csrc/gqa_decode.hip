// Decode attention of grouped query heads over a paged K/V cache (MI355X, gfx950).
//
// For each request b of S cached tokens, query position t of q_len and query head
// h (kv head h / G, G = Hq / Hkv):
//   o = sum_j softmax_j(scale * q . k_j) v_j   over the tokens j < S - q_len + t + 1,
// zeros where that leaves no token, with lse = ln sum_j exp(scale * q . k_j).
//
// A task is one request and RW "row sets" of 16 * NT query rows (row t * G + g of a kv
// head): those of one kv head, or of neighbouring ones. The tasks' steps of 32 tokens, in
// order, are cut into equal runs, one for each workgroup; a task that a cut divides
// leaves fp32 records (O, m, l) that a second kernel joins. So the work is even whatever
// the lengths are, they are read on the device, and the workspace depends on neither.
//
// Within a workgroup RW waves take a row set each and the same tokens, and WAVES / RW
// such groups of waves take the steps in turn, each with its own running
// maximum and sum (one pass over the data); they are joined in LDS at the task's end.
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

constexpr int kStep = 32;  // tokens of a wave's step
constexpr int kMaxQLen = 8;
constexpr int kMaxHeads = 1 << 16;
constexpr long long kMaxTokens = (1LL << 31) - 4096;  // of a request's table
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DecodeArgs {
  const char* q;         // [B, q_len, Hq, D] bf16 by strides
  Cache k, v;
  char* out;             // [B, q_len, Hq, D] bf16 by strides
  float* lse;            // [B, q_len, Hq] contiguous, or null
  const int* seq_lens;   // [B]
  const int* table;      // [B, width] by table_s
  float* rec_o;          // [2 * grid][16 * NT * RW][D]
  float* rec_ml;         // [2 * grid][16 * NT * RW][2]
  int4* joins;           // by task, or by run where there are more tasks than runs: what is to be joined
  long long q_s[3], out_s[3];  // batch, position, head; elements
  long long table_s;
  int B, q_len, Hq, G, rows;   // rows = q_len * G
  int sets;                    // row sets of one kv head that a task holds: RW, RW / 2 or RW / 4
  int row_blocks, per;         // tasks of a kv head's rows, and of a request
  int joins_by_task;
  int num_blocks, width, page_shift;
  float scale2;          // softmax scale * log2(e)
  float inv_g;           // 1 / G
  double per_run;        // 1 / grid
};

// Workgroups of a CU: two where a 16-row tile of up to 128 dims, or two of 64, fits two
// waves a SIMD with room, else one. Three leave more records and more starts: one request
// of 65537 tokens fp8 30.4 us, 31.5; 64 of 1K..8K, 8 kv heads of 64, fp8, token-major
// 76, 84; 8 of 128, bf16 195, 199. Two of a 32-row tile of 128 dims: 32 requests of
// windows of 4, 16 rows a position, 4 kv heads 86 us, one 79.
constexpr int per_cu(int D, int nt) { return D * nt <= 128 ? 2 : 1; }

// What a task's start and end cost a workgroup, as steps: about 4 us, in which one of
// two on a CU streams some 48 KB (half and three times as much counted for it measured
// alike), and half a step of each group of waves that has none.
constexpr int lead_steps(int D, bool fp8, int rw) { return 4 / rw / 2 + 512 / (fp8 ? D : 2 * D); }

// Waves of a workgroup that takes a task whole.
constexpr int whole_waves(int D, int nt) { return D * nt <= 128 ? 8 : 4; }

// The kernel's shape: NT tiles of 16 rows for each wave, RW row sets; CACHED: V is loaded
// through the caches, as several waves read it.
template <int D_, bool FP8_, int NT_, int RW_, bool CACHED_, bool SPLIT_>
struct Shape {
  static constexpr int D = D_, NT = NT_, RW = RW_;
  static constexpr bool FP8 = FP8_, SPLIT = SPLIT_;
  static constexpr int kWaves = SPLIT ? 4 : whole_waves(D, NT), kThreads = 64 * kWaves;
  static constexpr int kGroups = kWaves / RW;           // of waves, by tokens
  static constexpr int kRow = FP8 ? D : 2 * D;          // bytes of a cached row
  static constexpr int kRows = 16 * NT * RW;            // of a task
  static constexpr int kPerCu = SPLIT ? per_cu(D, NT) : 2;
  static constexpr bool kOnce = !CACHED_ && SPLIT;      // V is streamed past the caches
  static constexpr int kKLoads = kRow / 64;             // 16-byte loads of K per lane and 16 tokens
  static constexpr int kVWords = kRow / 64;             // dwords of V per lane and token
  static constexpr int kLead = SPLIT ? lead_steps(D, FP8, RW) : 0;
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

__device__ __forceinline__ int clamped(const DecodeArgs& a, int n) {
  const long long most = (long long)a.width << a.page_shift;
  return n < 0 ? 0 : (n > most ? (int)most : n);
}
__device__ __forceinline__ int len_of(const DecodeArgs& a, int b) { return clamped(a, ((ConstInts)(uintptr_t)a.seq_lens)[b]); }
__host__ __device__ __forceinline__ int steps_of(int len) { return (len >> 5) + ((len & 31) != 0); }

__device__ __forceinline__ long long uniform(long long x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (long long)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// What one step of a wave reads, in halves of 16 tokens, each within a page.
template <class C>
struct Step {
  u32x4 k[2][C::kKLoads];
  uint32_t v[8][C::kVWords];
  f32x4 ks[2], vs[2];
};

// The pages of a step's halves.
template <class C>
struct Pages {
  int id[2];
};
template <class C>
__device__ __forceinline__ Pages<C> step_pages(const DecodeArgs& a, ConstInts row, int tok) {
  Pages<C> p;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int id = row[min((tok + 16 * i) >> a.page_shift, a.width - 1)];
    p.id[i] = min(max(id, 0), a.num_blocks - 1);
  }
  return p;
}

// V's rows are read whole by one load each, and once. K goes through the caches: a load
// takes 64 bytes of each of 16 rows, the next one the other half of their lines (64
// requests of 1K..8K tokens, 8 kv heads of 128, bf16: both through the caches 209 us,
// both past them 192, K past them 206, V alone 181; fp8: 118, 111, 121 and 105).
template <class T, bool ONCE>
__device__ __forceinline__ T stream(const char* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
  return *reinterpret_cast<const T*>(p);
}

template <class C>
__device__ __forceinline__ void load_k(const DecodeArgs& a, Step<C>& s, const Pages<C>& pg, int tok, int head, int lane,
                                       uint32_t mask = ~0u) {
  constexpr int kElem = C::FP8 ? 1 : 2;
  const uint32_t off = ((uint32_t)(lane & 15) * (uint32_t)(a.k.row_s * kElem) + 16u * (lane >> 4)) & mask;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = (tok + 16 * i) & ((1 << a.page_shift) - 1);
    const char* kb = a.k.base + (pg.id[i] * a.k.block_s + head * a.k.head_s + row * a.k.row_s) * kElem;
#pragma unroll
    for (int c = 0; c < C::kKLoads; ++c) s.k[i][c] = *reinterpret_cast<const u32x4*>(kb + off + 64 * c);
    if constexpr (C::FP8)
      s.ks[i] = *reinterpret_cast<const f32x4*>(a.k.scale + pg.id[i] * a.k.sblock_s + head * a.k.shead_s + row +
                                                4 * (lane >> 4));
  }
}

template <class C>
__device__ __forceinline__ void load_v(const DecodeArgs& a, Step<C>& s, const Pages<C>& pg, int tok, int head, int lane,
                                       uint32_t mask = ~0u) {
  constexpr int kElem = C::FP8 ? 1 : 2;
  const uint32_t off = (4u * (lane >> 4) * (uint32_t)(a.v.row_s * kElem) + (uint32_t)(C::kVWords * 4 * (lane & 15))) & mask;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = (tok + 16 * i) & ((1 << a.page_shift) - 1);
    const char* vb = a.v.base + (pg.id[i] * a.v.block_s + head * a.v.head_s + row * a.v.row_s) * kElem;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const char* p = vb + r * (a.v.row_s * kElem) + off;
      uint32_t* to = s.v[4 * i + r];
      if constexpr (C::kVWords == 1) {
        to[0] = stream<uint32_t, C::kOnce>(p);
      } else if constexpr (C::kVWords == 2) {
        const u32x2 x = stream<u32x2, C::kOnce>(p);
        to[0] = x[0];
        to[1] = x[1];
      } else {
#pragma unroll
        for (int c = 0; c < C::kVWords / 4; ++c) {
          const u32x4 x = stream<u32x4, C::kOnce>(p + 16 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) to[4 * c + e] = x[e];
        }
      }
    }
    if constexpr (C::FP8)
      s.vs[i] = *reinterpret_cast<const f32x4*>(a.v.scale + pg.id[i] * a.v.sblock_s + head * a.v.shead_s + row +
                                                4 * (lane >> 4));
  }
}

// A wave's query rows and what it has summed for them.
template <class C>
struct Rows {
  bf16x8 q[C::NT][C::D / 32];
  f32x4 o[C::NT][C::D / 16];     // o[nt][j][r]: row lane % 16, dim (D / 16) * (4 g + r) + j
  float m[C::NT], l[C::NT];      // log2 domain; l over this lane's tokens only
  int pos[C::NT];                // the row's query position
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

// Whether V is finite in every token of [from, to) that the wave holds.
template <class C>
__device__ __forceinline__ bool finite_tail(const Step<C>& s, int tok0, int from, int to) {
  constexpr uint32_t kOnes = C::FP8 ? 0x7F7F7F7Fu : 0x7F807F80u, kUnit = C::FP8 ? 0x01010101u : 0x00800080u,
                     kTop = C::FP8 ? 0x80808080u : 0x80008000u;
  uint32_t bad = 0;  // a field of ones carries into its top bit
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int t = tok0 + (e & 3) + 16 * (e >> 2);
    uint32_t any = 0;
#pragma unroll
    for (int c = 0; c < C::kVWords; ++c) any |= (s.v[e][c] & kOnes) + kUnit;
    bad |= t >= from && t < to ? any & kTop : 0u;
  }
  return !__any(bad != 0);
}

// O^T += V^T P^T for the step's 32 tokens. TAIL: tokens of `end` and above are hidden from
// query position `only` (-1: from all of them) and must not reach it even as 0 * NaN.
template <class C, bool TAIL>
__device__ __forceinline__ void add_pv(Rows<C>& w, const Step<C>& s, const bf16x8 (&hi)[C::NT],
                                       const bf16x8 (&lo)[C::NT], int tok0, int end, int only) {
  constexpr int kPerWord = C::FP8 ? 4 : 2;  // elements of one dword of V
#pragma unroll
  for (int c = 0; c < C::kVWords; ++c) {
    if (c % (8 / kPerWord) == 0) sched_fence();
    uint32_t x[8][kPerWord / 2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t word = s.v[e][c];
      if constexpr (TAIL) word = tok0 + (e & 3) + 16 * (e >> 2) < end ? word : 0u;
      if constexpr (C::FP8) {
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
      for (int nt = 0; nt < C::NT; ++nt) {
        f32x4 acc = mfma16(vf, hi[nt], w.o[nt][j]);
        acc = mfma16(vf, lo[nt], acc);
        if constexpr (TAIL) {
#pragma unroll
          for (int r = 0; r < 4; ++r) w.o[nt][j][r] = only < 0 || w.pos[nt] == only ? acc[r] : w.o[nt][j][r];
        } else {
          w.o[nt][j] = acc;
        }
      }
    }
  }
}

// One step. Without TAIL every query position sees all its tokens, and each operand's
// registers take the next step's loads as soon as the products have read them, so
// about a step (16 KB) is in flight for each wave at any time.
template <class C, bool TAIL>
__device__ __forceinline__ void compute_step(const DecodeArgs& a, Rows<C>& w, Step<C>& s, int tok, int len,
                                             const Pages<C>& pg, int next, uint32_t mask, int head, int lane) {
  const int tok0 = tok + 4 * (lane >> 4);  // this lane's tokens: tok0 + 16 i + r
  f32x4 sc[C::NT][2];
#pragma unroll
  for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) sc[nt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (C::FP8) sched_fence();
#pragma unroll
    for (int c = 0; c < C::kKLoads; ++c) {
      if constexpr (C::FP8) {
        // 16 dims of a load feed two MFMAs: Q is laid out to match.
        bf16x8 kf[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x2 x = fp8x4_to_bf16(s.k[i][c][2 * h]), y = fp8x4_to_bf16(s.k[i][c][2 * h + 1]);
          kf[h] = __builtin_bit_cast(bf16x8, u32x4{x[0], x[1], y[0], y[1]});
        }
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          sc[nt][i] = mfma16(kf[0], w.q[nt][2 * c], sc[nt][i]);
          sc[nt][i] = mfma16(kf[1], w.q[nt][2 * c + 1], sc[nt][i]);
        }
      } else {
        const bf16x8 kf = __builtin_bit_cast(bf16x8, s.k[i][c]);
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) sc[nt][i] = mfma16(kf, w.q[nt][c], sc[nt][i]);
      }
    }
  }
  f32x4 ks[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) ks[i] = s.ks[i];
  if constexpr (!TAIL) {
    sched_fence();
    load_k<C>(a, s, pg, next, head, lane, mask);
    sched_fence();
  }
#pragma unroll
  for (int nt = 0; nt < C::NT; ++nt) {
    const int end = len - a.q_len + w.pos[nt] + 1;  // the row sees the tokens before it
    float mx = w.m[nt];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = sc[nt][i][r] * a.scale2;
        if constexpr (C::FP8) x *= ks[i][r];
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
      for (int j = 0; j < C::D / 16; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) w.o[nt][j][r] *= f;
      w.m[nt] = mx;
    }
  }
  bool apiece = false;  // query positions see different numbers of these tokens, and not all V is finite
  if constexpr (TAIL) apiece = !finite_tail<C>(s, tok0, len - a.q_len + 1, len);
  sched_fence();
  bf16x8 hi[C::NT], lo[C::NT];
#pragma unroll
  for (int nt = 0; nt < C::NT; ++nt) {
    const int end = len - a.q_len + w.pos[nt] + 1;
    float p[8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = __builtin_amdgcn_exp2f(sc[nt][i][r] - w.m[nt]);
        sum += x;
        if constexpr (C::FP8) x *= s.vs[i][r];
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
  if constexpr (!TAIL) {
    add_pv<C, false>(w, s, hi, lo, tok0, 0, 0);
  } else {  // a hidden token weighs 0, which suffices where V is finite; one past the end is taken as 0
    for (int t = apiece ? 0 : a.q_len - 1; t < a.q_len; ++t)
      add_pv<C, true>(w, s, hi, lo, tok0, len - a.q_len + t + 1, apiece ? t : -1);
  }
  if constexpr (!TAIL) load_v<C>(a, s, pg, next, head, lane, mask);
}

// x / d of whole numbers below 2^52 (inv: 1 / d, rounded): the rounded product is at
// most one off. A 64-bit division takes some 150 instructions, at a point that
// everything waits for.
__host__ __device__ __forceinline__ long long quotient(long long x, long long d, double inv) {
  long long q = (long long)((double)x * inv);
  const long long r = x - q * d;
  q += r >= d ? 1 : 0;
  q -= r < 0 ? 1 : 0;
  return q;
}

// The runs: the tasks lie one behind the other, each as long as its steps and `lead`
// places more in front for its own cost; run w has the places from start(w) = floor(w *
// total / runs) up to start(w + 1). Where there are not steps enough for all workgroups,
// a task is as long as its steps in whole rounds of the groups of waves, and a run a round.
struct Run {
  long long total;
  int runs;               // the grid's workgroups, or as many as give each group of waves a step
  int lead, pad, snap;
  double per_run;         // 1 / runs
  long long start, end;   // this workgroup's run
  long long before;       // places before request b, in which it starts
  int b, len;             // and that request's length
  __host__ __device__ __forceinline__ long long start_of(int w) const { return quotient(w * total, runs, per_run); }
  __host__ __device__ __forceinline__ void by_rounds(int groups) {
    lead = 0;
    pad = groups - 1;  // groups: a power of two
  }
  __host__ __device__ __forceinline__ void by_cost(int steps) {
    lead = steps;
    pad = 0;
  }
  __host__ __device__ __forceinline__ int places_of(int steps) const { return (steps + lead + pad) & ~pad; }
  __host__ __device__ __forceinline__ void lay_out(long long places, int grid, double per_grid, int groups) {
    total = places;
    const long long most = (total + groups - 1) / groups;
    runs = grid < most ? grid : (int)most;
    per_run = runs == grid ? per_grid : 1.0 / (double)runs;
    snap = pad ? 0 : total >= 2LL * groups * runs ? groups : (int)(total / 2) / runs;
  }
  // The steps of a task of `steps` that lie before its place v: a run's border near the
  // task's start or end is moved there, so that it costs no segment of its own.
  __host__ __device__ __forceinline__ int cut(long long v, int steps) const {
    const long long r = v - lead;
    const int late = snap < steps >> 1 ? snap : steps >> 1;
    return r < least_cut(steps) ? 0 : r >= steps - late ? steps : (int)r;
  }
  __host__ __device__ __forceinline__ int least_cut(int steps) const {
    const int soon = snap < (steps + 1) >> 1 ? snap : (steps + 1) >> 1;
    return soon > 1 ? soon : 1;
  }
  // The run that holds the beginning of a task that starts at place `at` and has been
  // cut: the last whose start is not yet cut into the task. `guess`: a later one.
  __host__ __device__ __forceinline__ int holder(long long at, int steps, int guess) const {
    const long long first = at + lead + least_cut(steps);
    int w = (int)((double)first / (double)total * runs);
    w = w < guess ? w : guess - 1;
    while (start_of(w) >= first) --w;
    while (start_of(w + 1) < first) ++w;
    return w;
  }
};
// Every thread calls it. Requests are taken THREADS at a time, one for each thread, and
// a prefix sum finds the one that holds the run's first place.
template <int THREADS, int GROUPS, int LEAD>
__device__ Run find_run(const DecodeArgs& a, int wg, int grid) {
  constexpr int kWaves = THREADS / 64;
  __shared__ int sh_sum[2][kWaves];
  __shared__ long long sh_found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // A wave's 64 requests have fewer than 2^32 places; sums over waves are 64 bits.
  Run run{};
  const auto group = [&](int b0, int turn, int& len, int& n, int& incl, long long& ahead, long long& sum) {
    len = b0 + tid < a.B ? clamped(a, a.seq_lens[b0 + tid]) : 0;
    n = len > 0 ? run.places_of(steps_of(len)) : 0;
    incl = wave_incl_scan(n);
    if (lane == 63) sh_sum[turn][wave] = incl;
    __syncthreads();
    ahead = sum = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) ahead += (uint32_t)sh_sum[turn][i];
      sum += (uint32_t)sh_sum[turn][i];
    }
  };
  int len, n, incl;
  long long ahead, sum, total;
  if constexpr (GROUPS > 1)
    run.by_rounds(GROUPS);
  else
    run.by_cost(LEAD);
  while (true) {
    total = 0;
    for (int b0 = 0, turn = 0; b0 < a.B; b0 += THREADS, turn ^= 1) {
      group(b0, turn, len, n, incl, ahead, sum);
      total += sum;
    }
    total = uniform(total * a.per);
    if (run.pad == 0 || total <= (long long)grid * GROUPS) break;
    run.by_cost(LEAD);
    __syncthreads();
  }
  run.lay_out(total, grid, a.per_run, GROUPS);
  run.b = a.B;
  if (wg >= run.runs) return run;
  run.start = uniform(run.start_of(wg));
  run.end = uniform(run.start_of(wg + 1));
  long long base = 0;
  for (int b0 = 0, turn = 0; b0 < a.B; b0 += THREADS, turn ^= 1) {
    if (a.B > THREADS) {
      __syncthreads();
      group(b0, turn, len, n, incl, ahead, sum);
    }
    const long long before = (base + ahead + (uint32_t)incl - (uint32_t)n) * a.per;
    if (run.start >= before && run.start < before + (long long)n * a.per) {
      sh_found[0] = b0 + tid;
      sh_found[1] = before;
      sh_found[2] = len;
    }
    base += sum;
    if (run.start < base * a.per) break;
  }
  __syncthreads();
  run.b = uniform((int)sh_found[0]);
  run.before = uniform(sh_found[1]);
  run.len = uniform((int)sh_found[2]);
  return run;
}

// Row `row` of a task: kv head, and row of that head's q_len * G (it may be past them).
template <int NT>
__device__ __forceinline__ void row_of(const DecodeArgs& a, int head0, int block, int row, int& head, int& r) {
  const int set = row / (16 * NT), in_head = a.sets == 1 ? set : a.sets == 2 ? set >> 1 : set >> 2;
  head = head0 + in_head;
  r = (block * a.sets + (set & (a.sets - 1))) * 16 * NT + row % (16 * NT);
}
// r / G for r below q_len * G: exact, as (r + 1/2) / G lies 1 / (2 G) from a whole number.
__device__ __forceinline__ int position(const DecodeArgs& a, int r) { return (int)(((float)r + 0.5f) * a.inv_g); }

// The part of a task that a workgroup takes, all of it wave-uniform.
struct Segment {
  long long before, start;    // places before request b, and before the task
  int b, task, len, steps;    // the request's length and a task's steps
  int step0, step1;           // its part: steps [step0, step1)
  int head0, block;           // the task's first kv head and block of its rows
};
template <class C>
__device__ __forceinline__ void place(const DecodeArgs& a, Segment& x) {
  const int group = a.row_blocks == 1 ? x.task : x.task / a.row_blocks;
  x.block = a.row_blocks == 1 ? 0 : x.task - group * a.row_blocks;
  x.head0 = a.sets == C::RW ? group : a.sets * 2 == C::RW ? group * 2 : group * 4;
}

// The next task's part in the run; false where it has none.
template <class C>
__device__ __forceinline__ bool next_task(const DecodeArgs& a, const Run& run, Segment& x) {
  x.start += run.places_of(x.steps);
  if (x.start >= run.end) return false;
  if (++x.task == a.per) {
    x.task = 0;
    x.before = x.start;
    do {
      if (++x.b >= a.B) return false;
      x.len = len_of(a, x.b);
    } while (x.len == 0);
    x.steps = steps_of(x.len);
  }
  x.step0 = 0;
  x.step1 = uniform(run.cut(run.end - x.start, x.steps));
  return x.step1 > 0;
}

// A wave's first loads for a segment: its query rows and its first step.
template <class C>
__device__ __forceinline__ void begin(const DecodeArgs& a, const Segment& x, Rows<C>& w, Step<C>& s, int rw, int tg,
                                      int lane) {
  constexpr int NT = C::NT;
  const int st = x.step0 + tg, n = lane & 15, g = lane >> 4;
  const ConstInts table = (ConstInts)(uintptr_t)(a.table + (long long)x.b * a.table_s);
  const Pages<C> pg = step_pages<C>(a, table, st * kStep);
  int head, row0;
  row_of<NT>(a, x.head0, x.block, rw * 16 * NT, head, row0);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = row0 + 16 * nt + n;
    const bool live = r < a.rows;
    const int t = live ? position(a, r) : a.q_len - 1;
    w.pos[nt] = t;
    const char* qr = a.q + 2 * (x.b * a.q_s[0] + t * a.q_s[1] + (head * a.G + (live ? r - t * a.G : 0)) * a.q_s[2]);
#pragma unroll
    for (int c = 0; c < C::D / 32; ++c) {
      // dims of MFMA c for lane group g, as K's loads have them
      const int d = C::FP8 ? 64 * (c / 2) + 16 * g + 8 * (c & 1) : 32 * c + 8 * g;
      u32x4 y = *reinterpret_cast<const u32x4*>(qr + 2 * d);
      if (!live) y = u32x4{0u, 0u, 0u, 0u};
      w.q[nt][c] = __builtin_bit_cast(bf16x8, y);
    }
  }
  // K before V here as in the loop: the compiler's wait for K there counts the loads
  // that may have been issued since on every way into it.
  sched_fence();
  load_k<C>(a, s, pg, st * kStep, head, lane);
  sched_fence();
  load_v<C>(a, s, pg, st * kStep, head, lane);
  sched_fence();
}

// SPLIT: the workgroup takes its run of all tasks' steps. Otherwise a whole task:
// nothing is planned, and the first step is loaded before the request's length is there.
template <class C>
__global__ __launch_bounds__(C::kThreads, C::kPerCu) void gqa_decode_kernel(const DecodeArgs a) {
  constexpr int D = C::D, NT = C::NT, kWaves = C::kWaves, kThreads = C::kThreads;
  constexpr bool SPLIT = C::SPLIT;
  constexpr int kPitch = D + 4;  // floats: rows of the join start on different banks
  __shared__ float sh_o[kWaves][16][kPitch];
  __shared__ float sh_ml[C::kGroups][C::kRows][2];

  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = uniform(tid >> 6), rw = wave % C::RW, tg = wave / C::RW;

  int wg = 0, grid = 0;
  Run run{};
  Segment x{};
  bool more = true;
  if constexpr (SPLIT) {
    grid = gridDim.x;
    wg = xcd_remap(blockIdx.x, grid);
    run = find_run<kThreads, C::kGroups, C::kLead>(a, wg, grid);
    if (!a.joins_by_task && tid == 0) a.joins[wg] = int4{-1, 0, 0, 0};
    more = run.start < run.end;
    if (more) {
      x.b = run.b;
      x.before = run.before;
      x.len = run.len;
      x.steps = steps_of(x.len);
      const long long in = run.start - x.before;
      const int places = run.places_of(x.steps);
      x.task = uniform(in >> 32 ? (int)(in / places) : (int)((uint32_t)in / (uint32_t)places));
      x.start = x.before + (long long)x.task * places;
      x.step0 = uniform(run.cut(run.start - x.start, x.steps));
      x.step1 = uniform(run.cut(run.end - x.start, x.steps));
      more = x.step0 < x.step1 || (x.step0 == x.steps && next_task<C>(a, run, x));
    }
  } else {
    x.b = blockIdx.x;
    x.task = blockIdx.y;
  }
  while (more) {
    place<C>(a, x);
    Rows<C> w;
    Step<C> s;
    begin<C>(a, x, w, s, rw, tg, lane);
    if constexpr (!SPLIT) {
      x.len = len_of(a, x.b);
      x.step1 = x.steps = steps_of(x.len);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      w.m[nt] = kNegFltMax;
      w.l[nt] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) w.o[nt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // A wave's steps are every kGroups-th one. Those from s_full on hold tokens that
    // some position does not see: a step's worth and q_len - 1, in two steps at most.
    // Loads past the last step read its first row of each 16 or 4 over again (mask 0):
    // a load under a branch would make the compiler wait for all of them, and the whole
    // step again was 4% of the bytes read.
    {
      const ConstInts table = (ConstInts)(uintptr_t)(a.table + (long long)x.b * a.table_s);
      int head, row0;
      row_of<NT>(a, x.head0, x.block, rw * 16 * NT, head, row0);
      int st = x.step0 + tg;
      const int s_end = x.step1;
      if (st < s_end && row0 < a.rows) {
        const int s_last = st + (s_end - 1 - st) / C::kGroups * C::kGroups;
        const int seen = x.len - a.q_len + 1;
        const int s_full = seen > 0 ? seen / kStep : 0;
        int next = min(st + C::kGroups, s_last);
        Pages<C> pg = step_pages<C>(a, table, next * kStep);
        for (; st <= s_last && st < s_full; st += C::kGroups) {
          const int after = min(next + C::kGroups, s_last);
          const Pages<C> pa = step_pages<C>(a, table, after * kStep);
          compute_step<C, false>(a, w, s, st * kStep, x.len, pg, next * kStep, st < s_last ? ~0u : 0u, head, lane);
          pg = pa;
          next = after;
        }
        while (st <= s_last) {
          compute_step<C, true>(a, w, s, st * kStep, x.len, pg, 0, 0u, head, lane);
          st += C::kGroups;
          if (C::kGroups > 1 || st > s_last) break;  // a wave of several has one such step
          pg = step_pages<C>(a, table, st * kStep);
          load_k<C>(a, s, pg, st * kStep, head, lane);
          load_v<C>(a, s, pg, st * kStep, head, lane);
        }
      }
    }

    // Join the waves. The barriers wait for LDS alone.
    const bool whole = !SPLIT || (x.step0 == 0 && x.step1 == x.steps);
    const int rec = 2 * wg + (x.step0 == 0 ? 1 : 0);  // a run has one part that begins a task, and one that does not
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      w.l[nt] = xor32_sum(xor16_sum(w.l[nt]));
      if (g == 0) {
        sh_ml[tg][(rw * NT + nt) * 16 + n][0] = w.m[nt];
        sh_ml[tg][(rw * NT + nt) * 16 + n][1] = w.l[nt];
      }
    }
    lds_reads_done_barrier();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      {
        const int row = (rw * NT + nt) * 16 + n;
        float top = sh_ml[0][row][0];
#pragma unroll
        for (int i = 1; i < C::kGroups; ++i) top = fmaxf(top, sh_ml[i][row][0]);
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
      lds_reads_done_barrier();
      {
        // The row sets' tiles nt: kAcross threads for each of 16 * RW rows, kPer dims each.
        constexpr int kAcross = kThreads / (16 * C::RW), kPer = D / kAcross;
        const int set = tid / (16 * kAcross), in = tid / kAcross % 16, d0 = tid % kAcross * kPer;
        const int row = (set * NT + nt) * 16 + in;
        int h, R;
        row_of<NT>(a, x.head0, x.block, row, h, R);
        if (R < a.rows) {
          float top = sh_ml[0][row][0];
#pragma unroll
          for (int i = 1; i < C::kGroups; ++i) top = fmaxf(top, sh_ml[i][row][0]);
          float l = 0.f;
#pragma unroll
          for (int i = 0; i < C::kGroups; ++i) l += sh_ml[i][row][1] * __builtin_amdgcn_exp2f(sh_ml[i][row][0] - top);
          float o[kPer];
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            o[j] = 0.f;
#pragma unroll
            for (int i = 0; i < C::kGroups; ++i) o[j] += sh_o[i * C::RW + set][in][d0 + j];
          }
          if (whole) {
            const int t = position(a, R), hq = h * a.G + R - t * a.G;
            const bool none = x.len - a.q_len + t + 1 <= 0;  // the row sees no token
            const float inv = 1.f / l;
            char* to = a.out + 2 * (x.b * a.out_s[0] + t * a.out_s[1] + hq * a.out_s[2] + d0);
#pragma unroll
            for (int j = 0; j < kPer; j += 2)
              *reinterpret_cast<uint32_t*>(to + 2 * j) =
                  none ? 0u : pack2_bf16_canon<kRTNE>(o[j] * inv, o[j + 1] * inv);
            if (a.lse && d0 == 0)
              a.lse[((long long)x.b * a.q_len + t) * a.Hq + hq] =
                  none ? -__builtin_inff() : kLn2 * (top + __builtin_amdgcn_logf(l));
          } else {
            float* to = a.rec_o + ((long long)rec * C::kRows + row) * D + d0;
#pragma unroll
            for (int j = 0; j < kPer; ++j) to[j] = o[j];
            if (d0 == 0) {
              a.rec_ml[((long long)rec * C::kRows + row) * 2] = top;
              a.rec_ml[((long long)rec * C::kRows + row) * 2 + 1] = l;
            }
          }
        }
      }
      lds_reads_done_barrier();
    }
    if constexpr (!SPLIT) return;
    if (x.step1 == x.steps && tid == 0) {
      // The task ends in this run: which others hold it.
      int4 join{-1, 0, 0, 0};
      if (!whole) join = int4{x.b, x.task, run.holder(x.start, x.steps, wg), wg};
      if (a.joins_by_task)
        a.joins[x.b * a.per + x.task] = join;
      else if (!whole)
        a.joins[wg] = join;  // of the first segment only: one for each run
    }
    more = x.step1 == x.steps && next_task<C>(a, run, x);
  }

  // Requests without a token: zeros.
  for (int e = wg; SPLIT && e < a.B; e += grid) {
    if (len_of(a, e) != 0) continue;
    for (int i = tid; i < a.q_len * a.Hq * (D / 8); i += kThreads) {
      const int th = i / (D / 8), t = th / a.Hq, h = th - t * a.Hq;
      *reinterpret_cast<u32x4*>(a.out + 2 * (e * a.out_s[0] + t * a.out_s[1] + h * a.out_s[2] + 8 * (i % (D / 8)))) =
          u32x4{0u, 0u, 0u, 0u};
      if (a.lse && i % (D / 8) == 0) a.lse[(long long)e * a.q_len * a.Hq + th] = -__builtin_inff();
    }
    if (a.joins_by_task)
      for (int i = tid; i < a.per; i += kThreads) a.joins[e * a.per + i] = int4{-1, 0, 0, 0};
  }
}

// Joins the records of a task that several runs hold: rows of O and (m, l), in an order
// that the call's shape and lengths alone decide. D / 4 lanes hold a row (16 bytes
// each); PER_ROW such groups share a row's records, each with a running maximum over
// its own, four loaded at once.
constexpr int kJoinThreads = 512;
template <int D, int NT, int RW, int PER_ROW>
__global__ __launch_bounds__(kJoinThreads) void gqa_join_kernel(const DecodeArgs a) {
  constexpr int kRows = 16 * NT * RW, kLanes = D / 4, kGroups = kJoinThreads / kLanes;
  __shared__ f32x4 sh_o[PER_ROW > 1 ? kGroups : 1][kLanes];
  __shared__ float sh_ml[kGroups][2];
  const int4 j = a.joins[blockIdx.x];
  if (j.x < 0) return;
  const int lane = threadIdx.x % kLanes, mine = threadIdx.x / kLanes, sub = mine % PER_ROW;
  const int group = j.y / a.row_blocks, block = j.y % a.row_blocks;
  const int row = blockIdx.y * (kGroups / PER_ROW) + mine / PER_ROW;
  int head, R;
  row_of<NT>(a, group * (RW / a.sets), block, row, head, R);
  const bool live = row < kRows && R < a.rows;  // what other rows join is not stored
  const int n = j.w - j.z + 1;
  float m = kNegFltMax, l = 0.f;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  for (int i0 = sub; live && i0 < n; i0 += 4 * PER_ROW) {
    float pm[4], pl[4];
    f32x4 po[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = min(i0 + u * PER_ROW, n - 1);
      const long long r = (long long)(2 * (j.z + i) + (i == 0 ? 1 : 0)) * kRows + row;
      pm[u] = a.rec_ml[2 * r];
      pl[u] = a.rec_ml[2 * r + 1];
      po[u] = *reinterpret_cast<const f32x4*>(a.rec_o + r * D + lane * 4);
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < 4; ++u) top = fmaxf(top, pm[u]);
    float f = __builtin_amdgcn_exp2f(m - top);
    l *= f;
    o *= f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i0 + u * PER_ROW >= n) continue;
      f = __builtin_amdgcn_exp2f(pm[u] - top);
      l += f * pl[u];
      o += f * po[u];
    }
    m = top;
  }
  if constexpr (PER_ROW > 1) {
    sh_o[mine][lane] = o;
    if (lane == 0) {
      sh_ml[mine][0] = m;
      sh_ml[mine][1] = l;
    }
    __syncthreads();
    if (sub != 0) return;
    float top = m;
#pragma unroll
    for (int i = 1; i < PER_ROW; ++i) top = fmaxf(top, sh_ml[mine + i][0]);
    l = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < PER_ROW; ++i) {
      const float f = __builtin_amdgcn_exp2f(sh_ml[mine + i][0] - top);
      l += f * sh_ml[mine + i][1];
      o += f * sh_o[mine + i][lane];
    }
    m = top;
  }
  if (!live) return;
  const int t = position(a, R), h = head * a.G + R - t * a.G;
  o *= 1.f / l;
  u32x2 y;
  y[0] = pack2_bf16_canon<kRTNE>(o[0], o[1]);
  y[1] = pack2_bf16_canon<kRTNE>(o[2], o[3]);
  *reinterpret_cast<u32x2*>(a.out + 2 * (j.x * a.out_s[0] + t * a.out_s[1] + h * a.out_s[2] + lane * 4)) = y;
  if (a.lse && lane == 0) a.lse[((long long)j.x * a.q_len + t) * a.Hq + h] = kLn2 * (m + __builtin_amdgcn_logf(l));
}

// How a call is laid out.
struct Plan {
  int nt, rw, sets;          // 16-row tiles of a wave, row sets of a task, and of those one kv head's
  int row_blocks, per;       // tasks of a kv head's rows, and of a request
  int cached;                // whether V goes through the caches
  int grid, split;           // workgroups; whether they share the steps evenly or take a task each
  long long tasks;
};
constexpr int kCus = 256;
// Whether a workgroup takes each task whole, without the plan's reads and the second
// launch: where the longest request is two steps of each wave, or four where there are
// tasks enough for a quarter of the CUs; but not where there are more tasks than two for
// each CU (eight, of rows of 128 bytes and less), as most waves of a short one have
// nothing to do. 8 kv heads of 128: one request of 200 tokens (bf16) 6.7 us, shared out
// 9.6; of 1000 13.1 and 9.8; 64 of up to 500 18 and 24; 128 of up to 500 39 and 35 (fp8
// 22 and 30); 256 of up to 60 36 and 27 (fp8 22 and 28).
inline bool short_call(long long most, long long tasks, int D, int nt, bool fp8) {
  if (tasks > ((fp8 ? D : 2 * D) >= 256 ? 2 : 8) * kCus) return false;
  return most <= (tasks >= kCus / 4 ? 4 : 2) * 32 * whole_waves(D, nt);
}

// A K cache whose tokens hold their heads side by side (strides: as the launcher's).
inline bool token_major(const long long* strides) { return strides[8] > strides[7]; }
inline bool plan_call(int B, int q_len, int Hq, int Hkv, int D, int page, int width, bool fp8, bool by_token,
                      Plan* p) {
  const long long rows = (long long)(Hq / Hkv) * q_len, most = (long long)page * width;
  const long long steps = (most + kStep - 1) / kStep, all = (long long)B * Hkv;
  if (all * ((rows + 15) / 16) > INT_MAX) return false;
  // Few steps for many rows: 16 rows a task, each reading K and V for itself, rather than
  // more runs for a task and the records of all its rows (28 requests of 702 tokens, 96
  // rows of 128 dims: 12 us, 22.8 in tasks of 128 rows; 8 of 2000, 48 rows: 14.9 and 13.9).
  // Rows of 256 dims leave records twice as large (2 of 8917, 64 rows: 18.4 us, 28.1 in
  // one task; two tasks read as much more as that saves: 8 of 4000, 32 rows: 26.6, 24.2).
  const bool few = all * ((rows + 15) / 16) * steps <= (D < 256 ? 18LL : rows > 32 ? 24LL : 6LL) * kCus;
  p->nt = rows <= 16 || D == 256 || few ? 1 : 2;
  const long long sets = (rows + 16 * p->nt - 1) / (16 * p->nt), slots = per_cu(D, p->nt) * kCus;
  p->sets = sets == 1 || few ? 1 : sets == 2 ? 2 : 4;
  p->rw = p->sets;
  const long long blocks = (sets + p->sets - 1) / p->sets;
  p->split = p->sets > 1 || !short_call(most, all * blocks, D, p->nt, fp8);
  // Rows of neighbouring heads: waves that read them together read whole lines and
  // neighbouring ones (64 requests of 1K..8K tokens, fp8, 8 heads of 64: 76 us, 100
  // apart; of 128 112 and 117). Their records are as many times larger: only where a run
  // then has steps enough (one request of 20000, windows of 4: 28 us, 23 apart).
  if (p->split && by_token)
    while (p->rw < 4 && p->nt == 1 && blocks == 1 && Hkv % (p->rw / p->sets * 2) == 0 &&
           all / (p->rw / p->sets * 2) * steps >= 24 * slots)
      p->rw *= 2;
  p->cached = p->sets > 1;
  p->row_blocks = (int)blocks;
  const long long per = (long long)(Hkv / (p->rw / p->sets)) * p->row_blocks;
  if (per > 65535) return false;
  p->per = (int)per;
  p->tasks = B * per;
  const long long places = steps + lead_steps(D, fp8, p->rw);
  const long long runs = (p->tasks * places * p->rw + 3) / 4;  // of a step for each group of waves
  p->grid = (int)(runs < slots ? runs : slots);
  return p->tasks * places < 1LL << 42;  // quotient()'s range
}
inline size_t record_bytes(const Plan& p, int D) { return (size_t)2 * p.grid * 16 * p.nt * p.rw * (D + 2) * 4; }
// One entry for each task or run, whichever are fewer.
inline long long join_count(const Plan& p) { return p.tasks < p.grid ? p.tasks : p.grid; }

template <int D, bool FP8, int NT, int RW, bool CACHED>
int launch(const DecodeArgs& a, const Plan& p, hipStream_t stream) {
  if (!p.split) {
    if constexpr (RW == 1) {
      using C = Shape<D, FP8, NT, 1, false, false>;
      hipLaunchKernelGGL((gqa_decode_kernel<C>), dim3(a.B, p.per), dim3(C::kThreads), 0, stream, a);
    }
  } else {
    using C = Shape<D, FP8, NT, RW, CACHED, true>;
    hipLaunchKernelGGL((gqa_decode_kernel<C>), dim3(p.grid), dim3(C::kThreads), 0, stream, a);
    // Records of a row: as many as runs share a task, or two ends of a run. A group of
    // lanes takes four at once.
    constexpr int kMost = D == 256 ? 8 : 16, kGroups = kJoinThreads / (D / 4);
    const long long n = p.grid / p.tasks + 2, count = join_count(p);
    const int rows = p.row_blocks > 1 || p.rw > p.sets ? C::kRows : a.rows;
    const auto blocks = [&](int per_row) { return dim3((unsigned)count, (rows * per_row + kGroups - 1) / kGroups); };
    if (n <= 4)
      hipLaunchKernelGGL((gqa_join_kernel<D, NT, RW, 1>), blocks(1), dim3(kJoinThreads), 0, stream, a);
    else if (n <= 16)
      hipLaunchKernelGGL((gqa_join_kernel<D, NT, RW, 4>), blocks(4), dim3(kJoinThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((gqa_join_kernel<D, NT, RW, kMost>), blocks(kMost), dim3(kJoinThreads), 0, stream, a);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : (int)e;
}

// The shapes that plan_call() chooses: row sets of one kv head are of two tiles, or of 256
// dims, and heads are grouped in single tiles.
template <int D, bool FP8, int NT>
int with_rw(const DecodeArgs& a, const Plan& p, hipStream_t st) {
  if (p.rw == 1) return launch<D, FP8, NT, 1, false>(a, p, st);
  if constexpr (NT > 1 || D == 256)
    if (p.cached) return p.rw == 2 ? launch<D, FP8, NT, 2, true>(a, p, st) : launch<D, FP8, NT, 4, true>(a, p, st);
  if constexpr (NT == 1)
    if (!p.cached) return p.rw == 2 ? launch<D, FP8, NT, 2, false>(a, p, st) : launch<D, FP8, NT, 4, false>(a, p, st);
  return -8;
}
template <bool FP8>
int dispatch(const DecodeArgs& a, const Plan& p, int D, hipStream_t st) {
  if (D == 256) return with_rw<256, FP8, 1>(a, p, st);
  if (D == 64) return p.nt == 1 ? with_rw<64, FP8, 1>(a, p, st) : with_rw<64, FP8, 2>(a, p, st);
  return p.nt == 1 ? with_rw<128, FP8, 1>(a, p, st) : with_rw<128, FP8, 2>(a, p, st);
}

// -2 head_dim, -3 heads, -4 sizes, -5 page; 0 where the call can be planned.
inline int check_sizes(int B, int q_len, int Hq, int Hkv, int D, int page, int width) {
  if (D != 64 && D != 128 && D != 256) return -2;
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv != 0 || Hq > kMaxHeads) return -3;
  if (B < 0 || q_len < 1 || q_len > kMaxQLen) return -4;
  if (page < 16 || (page & (page - 1)) != 0) return -5;
  if (width < 1 || (long long)page * width > kMaxTokens) return -11;
  return 0;
}

}  // namespace gqa
}  // namespace mm

extern "C" {

size_t moonmath_gqa_decode_workspace(int B, int q_len, int Hq, int Hkv, int head_dim, int page, int max_blocks,
                                     int fp8, const long long* strides) {
  using namespace mm::gqa;
  Plan p;
  if (B == 0 || !strides || check_sizes(B, q_len, Hq, Hkv, head_dim, page, max_blocks) != 0) return 0;
  if (!plan_call(B, q_len, Hq, Hkv, head_dim, page, max_blocks, fp8 != 0, token_major(strides), &p) || !p.split) return 0;
  return record_bytes(p, head_dim) + (size_t)join_count(p) * sizeof(int4);
}

int moonmath_gqa_decode_split(int B, const int* lens, int q_len, int Hq, int Hkv, int head_dim, int page,
                              int max_blocks, int fp8, const long long* strides, int* segments, int max_segments) {
  using namespace mm::gqa;
  const int rc = check_sizes(B, q_len, Hq, Hkv, head_dim, page, max_blocks);
  if (rc != 0) return rc;
  if (!lens || !strides || (!segments && max_segments > 0)) return -6;
  Plan p;
  if (B == 0) return 0;
  if (!plan_call(B, q_len, Hq, Hkv, head_dim, page, max_blocks, fp8 != 0, token_major(strides), &p)) return -8;
  if (!p.split) return 0;
  const int lead = lead_steps(head_dim, fp8 != 0, p.rw);
  Run run{};
  const auto places = [&] {
    long long sum = 0;
    for (int b = 0; b < B; ++b) sum += lens[b] > 0 ? run.places_of(steps_of(lens[b])) : 0;
    return sum * p.per;
  };
  const int groups = 4 / p.rw;
  run.by_rounds(groups);
  if (groups == 1 || places() > (long long)p.grid * groups) run.by_cost(lead);
  run.lay_out(places(), p.grid, 1.0 / p.grid, groups);
  long long n = 0;
  long long before = 0;
  for (int b = 0; b < B; ++b) {
    if (lens[b] <= 0) continue;
    const int steps = steps_of(lens[b]), length = run.places_of(steps);
    for (int task = 0; task < p.per; ++task, before += length) {
      // The runs that start within the task's places, and the one before them.
      int w = (int)((double)before / (double)run.total * run.runs);
      while (w > 0 && run.start_of(w) > before) --w;
      while (w + 1 < run.runs && run.start_of(w + 1) <= before) ++w;
      for (; w < run.runs && run.start_of(w) < before + length; ++w) {
        const int s0 = run.cut(run.start_of(w) - before, steps), s1 = run.cut(run.start_of(w + 1) - before, steps);
        if (s0 >= s1) continue;
        const int part[8] = {w, b, task, s0, s1, s0 == 0 && s1 == steps ? -1 : 2 * w + (s0 == 0 ? 1 : 0),
                             s0 > 0 && s1 == steps ? run.holder(before, steps, w) : -1, steps};
        for (int i = 0; i < 8; ++i)
          if (n < max_segments) segments[8 * n + i] = part[i];
        ++n;
      }
    }
  }
  return n > INT_MAX ? -8 : (int)n;
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
  DecodeArgs a{};
  a.k = make_cache(k_cache, k_scale, strides + 6);
  a.v = make_cache(v_cache, v_scale, strides + 11);
  // A lane adds up to 15 rows to a page's address in 32 bits.
  const long long widest = 1LL << 26;
  if (a.k.row_s < 0 || a.v.row_s < 0 || a.k.row_s > widest || a.v.row_s > widest) return -9;
  Plan p;
  if (!plan_call(B, q_len, Hq, Hkv, head_dim, page, max_blocks, k_scale != nullptr, token_major(strides), &p)) return -8;
  if (p.split && !workspace) return -6;
  a.q = (const char*)q;
  a.out = (char*)out;
  a.lse = (float*)lse;
  a.seq_lens = (const int*)seq_lens;
  a.table = (const int*)block_table;
  for (int i = 0; i < 3; ++i) {
    a.q_s[i] = strides[i];
    a.out_s[i] = strides[3 + i];
  }
  a.table_s = strides[16];
  a.rec_o = (float*)workspace;
  a.rec_ml = a.rec_o + (size_t)2 * p.grid * 16 * p.nt * p.rw * head_dim;
  a.joins = (int4*)(a.rec_ml + (size_t)2 * p.grid * 16 * p.nt * p.rw * 2);
  a.B = B;
  a.q_len = q_len;
  a.Hq = Hq;
  a.G = Hq / Hkv;
  a.rows = a.G * q_len;
  a.sets = p.sets;
  a.row_blocks = p.row_blocks;
  a.per = p.per;
  a.joins_by_task = p.tasks <= p.grid;
  a.num_blocks = num_blocks;
  a.width = max_blocks;
  a.page_shift = __builtin_ctz(page);
  a.scale2 = scale * kLog2e;
  a.inv_g = 1.f / (float)a.G;
  a.per_run = 1.0 / (double)p.grid;
  return k_scale ? dispatch<true>(a, p, head_dim, (hipStream_t)stream) : dispatch<false>(a, p, head_dim, (hipStream_t)stream);
}

}  // extern "C"
