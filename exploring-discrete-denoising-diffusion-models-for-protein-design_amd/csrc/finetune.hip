// Fine-tuning objectives at the logits of a denoiser or a language model: token log-probabilities, distillation from
// a teacher's top logits, the preference loss of paired sequences and the clipped policy loss with its KL term, with
// the gradient at the logits.
//
// Every one of them is a function of the rows' softmax, p = exp((z - m) / tau) / S with m the row's maximum and
// S = sum_v exp((z_v - m) / tau), and its gradient at a row is
//     dz_v = c (target_v - Q p_v)
// with one coefficient c of the row, target the token's indicator (Q = 1) or the teacher's distribution over its kept
// entries (Q = 1, or 0 where none is kept).  The distillation and the policy loss know c as soon as the row's m and S
// are known, so one pass over a row held in registers gives loss and gradient (k_rows); the preference loss needs the
// sums of two whole sequences first and the log-probabilities' backward an upstream gradient per row: those write m, S
// and c per row and a second kernel makes the gradient from them (k_token_grad).
//
// A row with its gradient is read once and written once, and takes 14 vector instructions per 16-bit logit (statistics
// alone: 9; one of them per sweep an exponential, at a quarter of the rate).  The memory system bounds it: 8192 x 131072
// bf16 with the gradient 811 us, 5.3 TB/s, vector units busy 0.59 of the time (a copy of that size: 4.8 TB/s); statistics
// of 8192 x 65536 bf16 180 us, 6.0 TB/s, vector units busy 0.83.
#include "d3pm_device.h"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

namespace d3pm {
namespace ft {

constexpr int MAX_K = 256;              // entries of a teacher's list
constexpr int MAX_PARTIALS = 8192;      // workgroups of a loss launch: one partial sum each

enum Head { HEAD_LOGPROB = 0, HEAD_PREFERENCE = 1, HEAD_POLICY = 2 };

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// ------------------------------------------------------------------------------------------------ element types
// A 16-byte piece of a row as it lies in memory (rows of odd widths start anywhere: the vector accesses ask for the
// element's alignment only, which the hardware's global accesses take), its E values as float, and back (one
// rounding to nearest).
typedef uint32_t raw_f32 __attribute__((ext_vector_type(4), aligned(4), may_alias));
typedef uint32_t raw_16 __attribute__((ext_vector_type(4), aligned(2), may_alias));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct F32 {
  static constexpr int E = 4, SIZE = 4;
  static constexpr uint32_t NEG_INF = 0xFF800000u;       // as often as it fits a dword
  typedef raw_f32 Raw;
  typedef float __attribute__((may_alias)) Elem;
  static __device__ __forceinline__ void unpack(u32x4 r, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __builtin_bit_cast(float, (uint32_t)r[i]);
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, f[i]);
    return r;
  }
  static __device__ __forceinline__ float get(const void* p, long i) { return ((const Elem*)p)[i]; }
  static __device__ __forceinline__ void put(void* p, long i, float v) { ((Elem*)p)[i] = v; }
};

struct F16 {
  static constexpr int E = 8, SIZE = 2;
  static constexpr uint32_t NEG_INF = 0xFC00FC00u;
  typedef raw_16 Raw;
  typedef _Float16 __attribute__((may_alias)) Elem;
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ void unpack(u32x4 r, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const h2 h = __builtin_bit_cast(h2, (uint32_t)r[i]);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, (h2){(_Float16)f[2 * i], (_Float16)f[2 * i + 1]});
    return r;
  }
  static __device__ __forceinline__ float get(const void* p, long i) { return (float)((const Elem*)p)[i]; }
  static __device__ __forceinline__ void put(void* p, long i, float v) { ((Elem*)p)[i] = (_Float16)v; }
};

struct BF16 {
  static constexpr int E = 8, SIZE = 2;
  static constexpr uint32_t NEG_INF = 0xFF80FF80u;
  typedef raw_16 Raw;
  typedef __bf16 __attribute__((may_alias)) Elem;
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ void unpack(u32x4 r, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __builtin_bit_cast(float, (uint32_t)(r[i] << 16));
      f[2 * i + 1] = __builtin_bit_cast(float, (uint32_t)(r[i] & 0xFFFF0000u));
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float* f) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){f[2 * i], f[2 * i + 1]}, b2));
    return r;
  }
  static __device__ __forceinline__ float get(const void* p, long i) { return (float)((const Elem*)p)[i]; }
  static __device__ __forceinline__ void put(void* p, long i, float v) { ((Elem*)p)[i] = (__bf16)v; }
};

__device__ __forceinline__ float get_any(const void* p, int dtype, long i) {
  return dtype == D3PM_F32 ? F32::get(p, i) : dtype == D3PM_F16 ? F16::get(p, i) : BF16::get(p, i);
}
// an int32 or int64 index: -1 for any negative one, else at most INT_MAX
__device__ __forceinline__ int get_int(const void* p, int bytes, long i) {
  const long v = bytes == 4 ? (long)((const int*)p)[i] : ((const long*)p)[i];
  return v < 0 ? -1 : v > INT_MAX ? INT_MAX : (int)v;
}

// A piece of a gradient row: nothing in the launch reads it again, and the caches are better kept for the logits
// (2 % of a launch at 32 k classes and more).
template <typename T, bool NT = true>
__device__ __forceinline__ void store_piece(char* p, u32x4 v) {
  if constexpr (NT) __builtin_nontemporal_store((typename T::Raw)v, (typename T::Raw*)p);
  else *(typename T::Raw*)p = (typename T::Raw)v;
}

// ------------------------------------------------------------------------------------------------------ arguments
struct RowArgs {
  const void* z; long sb, sl; int L, V, N; int dense;         // dense: row n lies at n * sl
  const void* tokens; int tok_bytes; const uint8_t* mask;
  float c_hi, c_lo, inv_tau, inv_tau_lo;                      // log2(e) / tau and 1 / tau, each in two floats
  float d_min;                                                // z - m from which on exp((z - m) / tau) is 0
  int head;
  const float* old_lp; const float* ref_lp; const float* adv; int adv_per_seq; float clip_lo, clip_hi, kl_coeff;
  const void* t_logits; int t_dtype; const void* t_index; int t_index_bytes; int k;
  float weight;                                               // of a counted row: out_scale (x tau or / tau) ...
  int* count; int count_here; float inv_count;                // ... over *count, which the launch finds itself with
                                                              // count_here (NULL: inv_count, every row counts)
  const float* upstream; int only_if_rescaled;                // gradient only: times *upstream; nothing to do at 1
  float4* stats;                                              // m, S, c, the token's logit; S = -1: not counted
  float* per_row; double* partial; void* dz;
  float* loss; float out_scale;                               // a loss of one workgroup is written by it
};
__device__ __forceinline__ float4 not_counted() { return make_float4(0.0f, -1.0f, 0.0f, 0.0f); }
// The sum of one workgroup's rows: a partial sum, or the loss.
__device__ __forceinline__ void put_sum(const RowArgs& a, double s) {
  if (gridDim.x > 1) a.partial[blockIdx.x] = s;
  else *a.loss = (float)(s * (double)a.out_scale * (a.count ? 1.0 / (double)max(*a.count, 1) : 1.0 / (double)a.N));
}

__device__ __forceinline__ const char* row_ptr(const RowArgs& a, int n, int size) {
  long at;
  if (a.dense) at = (long)n * a.sl;
  else {
    const unsigned b = (unsigned)n / (unsigned)a.L;
    at = (long)b * a.sb + (long)((unsigned)n - b * (unsigned)a.L) * a.sl;
  }
  return (const char*)a.z + at * size;
}

// exp((z - m) / tau) of d = z - m <= 0, the constant in two floats: its rounding alone would shift every S the same
// way (1e-7 at d = -10), which the sum over a sequence of a preference loss would gather up.
__device__ __forceinline__ float exp_d(float d, float c_hi, float c_lo) { return exp2_hw(fmaf(d, c_hi, d * c_lo)); }

__device__ __forceinline__ float rcp_acc(float x) {      // v_rcp_f32 and one step of Newton's: 1 ulp
  const float r = __builtin_amdgcn_rcpf(x);
  return fmaf(fmaf(-x, r, 1.0f), r, r);
}
// exp(x): log2(e) in two floats (the second above 0: an infinite x stays what it is)
__device__ __forceinline__ float exp_any(float x) { return exp2_hw(fmaf(x, 1.44269502f, x * 1.92596299e-8f)); }
// exp(x) - 1 - x: near 0 its series (up to 0.35 the next term is 9e-8 of it), where the difference would cancel
__device__ __forceinline__ float exp_rest(float x) {
  float q = fmaf(x, 1.0f / 5040.0f, 1.0f / 720.0f);
  q = fmaf(x, q, 1.0f / 120.0f);
  q = fmaf(x, q, 1.0f / 24.0f);
  q = fmaf(x, q, 1.0f / 6.0f);
  q = fmaf(x, q, 0.5f);
  return fabsf(x) < 0.35f ? x * x * q : exp_any(x) - 1.0f - x;
}

// (z - m) / tau - log S as hi + lo, to about 4e-8 whatever its size (of -8, float32 keeps 2.4e-7): 1 / tau is there in two
// floats (of one, -60 would be 2e-6 off at tau = 1.7, in every row the same way), with S = 2^e f, e ln 2 is taken off in
// one exact step and a second for its rest, and what rounds there is kept.
struct LogProb { float hi, lo; };
__device__ __forceinline__ LogProb log_prob(float zy_m, float inv_tau, float inv_tau_lo, float S) {
#pragma clang fp contract(off)
  const float e = (float)__builtin_amdgcn_frexp_expf(S);
  const float K = e * 0.693145752f;                                      // ln 2 to 16 bits: exact
  const float k = fmaf(e, 1.42860677e-6f, logf(__builtin_amdgcn_frexp_mantf(S)));
  const float p = zy_m * inv_tau, p_lo = fmaf(zy_m, inv_tau_lo, fmaf(zy_m, inv_tau, -p));
  const float s = p - K, b = s - p;
  const float s_lo = (p - (s - b)) - (K + b);
  return LogProb{s, fabsf(s) < INFINITY ? s_lo + p_lo - k : -k};         // (a token ruled out: -inf)
}

// What a row's token gives once m and S are known: its log-probability, its share of the loss and the coefficient
// c of its gradient (without the weight).  Comparisons are written so that a NaN stays one.  Every lane of the row
// computes this: at 32 classes its instructions are most of the launch, hence the short forms above.  Differences of
// log-probabilities are taken from both parts: a mean over advantages of both signs is small against its terms, and an
// error of 2.4e-7 in each of them showed in it.
struct TokenOut { float lp, loss, c; };
__device__ __forceinline__ TokenOut token_head(const RowArgs& a, int n, float zy_m, float S) {
  TokenOut o;
  const LogProb lp = log_prob(zy_m, a.inv_tau, a.inv_tau_lo, S);
  o.lp = lp.hi + lp.lo;
  o.loss = 0.0f;
  o.c = 1.0f;
  if (a.head == HEAD_POLICY) {
    const float A = a.adv[a.adv_per_seq ? (unsigned)n / (unsigned)a.L : (unsigned)n];
    const float r = exp_any((lp.hi - a.old_lp[n]) + lp.lo);
    const float held_r = r < a.clip_lo ? a.clip_lo : r > a.clip_hi ? a.clip_hi : r;
    const float free_s = r * A, held_s = held_r * A;
    const bool clipped = free_s > held_s;
    o.loss = clipped ? -held_s : -free_s;
    o.c = clipped ? 0.0f : -free_s;
    if (a.ref_lp) {
      const float x = (a.ref_lp[n] - lp.hi) - lp.lo, q = exp_rest(x);
      o.loss = fmaf(a.kl_coeff, q, o.loss);
      o.c = fmaf(-a.kl_coeff, x + q, o.c);
    }
  }
  return o;
}
// c (1 - p) of the token: S less its own exponential is exact where that is the row's largest
__device__ __forceinline__ float token_grad(float c, float zy_m, float S, float c_hi, float c_lo) {
  return c * ((S - exp_d(zy_m, c_hi, c_lo)) / S);
}

// ------------------------------------------------------------------------------------- one pass, rows in registers
// A row is held by a group of G lanes, NV 16-byte pieces each (lane g: pieces g, g + G, ...), and one element of the
// end of the row that fills no piece.  Up to 64 lanes a group is a part of a wave and a workgroup of 256 has 256 / G
// rows; beyond, a group is a workgroup.
template <int G>
struct Shape {
  static constexpr int WG = G <= 64 ? 256 : G;
  static constexpr int ROWS = WG / G;
  static constexpr int GL = G < 64 ? G : 64;        // lanes that a teacher's list is spread over
};

// The pieces of a row as a buffer resource, for the shapes whose row is the same for a whole wave: an access beyond the
// last piece reads 0 or writes nothing, so neither loads nor stores need a branch.  (The whole offset goes into the lane
// offset: the range check compares that with the size less the scalar offset, which must not pass the size.)
// Its base is a multiple of 4: of the logits' pieces always (of 16, by PEEL), of the gradient's where `in_dwords` says so.
// The gradient's rows begin elsewhere than the logits' where these are strided, in 16-bit rows of odd widths at any
// multiple of 2: those take global stores, each behind a branch (policy loss of 2048 rows of 32003 bf16 classes: 57 us
// where they are cut out of rows of 32004, 56 where they are dense).
typedef __amdgpu_buffer_rsrc_t Rsrc;
template <typename T>
__device__ __forceinline__ bool in_dwords(const char* p) { return T::SIZE == 4 || ((uintptr_t)p & 3) == 0; }
__device__ __forceinline__ Rsrc pieces_of(const void* body, int full) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)body, 0, full * 16, 0x00027000);
}
// A lane's byte offset in the first pieces.  It is made again for every sweep: kept over the loop of the rows, the offsets
// of 16 pieces would take 16 registers.
__device__ __forceinline__ int lane_offset(int g) {
  int at = g * 16;
  asm volatile("" : "+v"(at));
  return at;
}
template <bool NT>
__device__ __forceinline__ u32x4 load_piece(Rsrc r, int lane16, int j, int G) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, lane16 + j * (G * 16), 0, NT ? 2 /* non-temporal */ : 0);
}
template <bool NT>
__device__ __forceinline__ void store_piece(Rsrc r, int lane16, int j, int G, u32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(v, r, lane16 + j * (G * 16), 0, NT ? 2 /* non-temporal */ : 0);
}

// Counted positions of a mask, by a whole workgroup of up to 1024: every thread gets the sum.
__device__ __forceinline__ int count_mask(const uint8_t* mask, int N, int* lds) {
  int c = 0;
  const int words = ((uintptr_t)mask & 15) ? 0 : N / 16;
  for (int i = threadIdx.x; i < words; i += blockDim.x) {
    const u32x4 v = ((const u32x4*)mask)[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t x = v[j] | ((v[j] >> 4) & 0x0F0F0F0Fu);  // any bit of a byte into its lowest
      x |= (x >> 2) & 0x3F3F3F3Fu;
      x |= (x >> 1) & 0x7F7F7F7Fu;
      c += __popc(x & 0x01010101u);
    }
  }
  for (int i = words * 16 + threadIdx.x; i < N; i += blockDim.x) c += mask[i] != 0;
  c = group_sum<64>(c);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = c;
  __syncthreads();
  c = 0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) c += lds[i];
  return c;
}
// The weight of a counted row.  A mask of few positions is counted by every workgroup that needs it (COUNT_HERE: 16 KB
// from the L2 each), which saves a launch ahead of this one: 4.5 us on the device, 2 on the host.
constexpr int COUNT_HERE = 16384;
__device__ __forceinline__ float row_weight(const RowArgs& a, int* lds) {
  float w = a.weight;
  if (a.count) {
    int c;
    if (a.count_here) {
      c = count_mask(a.mask, a.N, lds);
      if (blockIdx.x == 0 && threadIdx.x == 0) *a.count = c;
    } else c = *a.count;
    w *= 1.0f / (float)max(c, 1);
  } else w *= a.inv_count;
  return a.upstream ? w * *a.upstream : w;
}

// How a row falls into 16-byte pieces and the elements at its ends that fill none.  Rows of odd widths start anywhere;
// with PEEL their pieces begin at the first 16-byte boundary (a piece across two cache lines costs two accesses).
// Lane g of the row has the end element `edge(g)`, if there is one.
template <typename T, bool PEEL>
struct Cut {
  int head, full, rest, V;
  __device__ __forceinline__ Cut(const char* row, int V_) : V(V_) {
    head = PEEL ? min((int)((-(uintptr_t)row & 15) / T::SIZE), V) : 0;
    full = (V - head) / T::E;
    rest = V - head - full * T::E;
  }
  __device__ __forceinline__ bool has_edge(int g) const { return g < head + rest; }
  __device__ __forceinline__ int edge(int g) const { return g < head ? g : g + full * T::E; }
  // the lane of G that holds class y
  __device__ __forceinline__ int lane_of(int y, int G) const {
    const int in = y - head;
    return in < 0 ? y : in < full * T::E ? (in / T::E) % G : y - full * T::E;
  }
};

// Keeps the compiler from carrying the unpacked values of one sweep over a row into the next: they take twice the
// registers of the 16-bit pieces that they are unpacked from (220 instead of 64 + 36 at 16 pieces a lane).  WAY: of two
// sweeps in the two ways of a branch each has a text of its own, or their unpacking would be moved up before the branch.
template <int NV, bool WAY = false>
__device__ __forceinline__ void fresh(u32x4 (&v)[NV]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if constexpr (WAY) asm volatile("; sweep" : "+v"(v[j]));
    else asm volatile("" : "+v"(v[j]));
  }
}

// Whether the j-th pieces of a row's lanes may hold any of its `full` pieces: those of rows of several waves, where the
// answer is one branch, are passed over if not (a row fills at least half of its shape's pieces).  12288 rows of 70001
// bf16 classes: distillation 866 -> 709 us, policy loss 820 -> 655; 8192 of 100003: 671 -> 647 and 640 -> 641.  (Rows of
// one wave have no registers left for it: 99 -> 106 us at 2000 classes.)
template <int G, int NV>
__device__ __forceinline__ bool holds(int j, int full) { return G <= 64 || j < NV / 2 || j * G < full; }

// The places of v that hold no piece of the row hold -inf.
template <typename T, int G, int NV>
__device__ __forceinline__ void mask_pieces(u32x4 (&v)[NV], int full, int g) {
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if ((j + 1) * G > full) {
      const bool in = j * G + g < full;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j][i] = in ? v[j][i] : T::NEG_INF;
    }
}

// m and S of the group's row from its lanes' values, in two steps: of the wave (a wave takes its exponentials against its
// own maximum, so a row of several waves needs one exchange, not two; the reference is kept off -inf, for a wave that
// has only padding), and of the row.  KEEP: the pieces are needed again, for the gradient.
// EXACT: S in 64 bits, as hi + lo, from the elements on in a row of up to one wave, else from the lanes' float32 sums of two
// chains each on.  A preference loss sums a sequence's log-ratios, which may nearly cancel, and a policy
// loss means over advantages of both signs.  With EXACT in a row of up to one wave the rounding of each exponent x is kept
// as x_lo, and exp2(x + x_lo) = exp2(x) (1 + ln 2 x_lo); over the many terms of longer rows it averages out.
struct RowSum { float m, hi, lo; };
constexpr double LN2 = 0.69314718055994530942;
// v_exp_f32 is low by 3.4e-9 of its value on average (over 6 M arguments in [-24, 0]; exact at 0, where the largest logit
// is): nothing to one row, but a sequence's sum gathers it up (1537 tokens: 7e-6 of log-probability).
constexpr double EXP2_LOW = 3.4e-9;
__device__ __forceinline__ float exp_parts(float d, const RowArgs& a, float& low) {
  d = __builtin_elementwise_maximum(d, a.d_min);     // (of a class ruled out, x_lo is no number; a NaN stays one)
  const float x = d * a.c_hi, e = exp2_hw(x);
  low = fmaf(e, fmaf(d, a.c_lo, fmaf(d, a.c_hi, -x)), low);
  return e;
}
__device__ __forceinline__ RowSum in_parts(float m, double S) {
  const float hi = (float)S;
  return RowSum{m, hi, (float)(S - (double)hi)};
}
template <typename T, int G, int NV>
__device__ __forceinline__ float wave_max(const u32x4 (&v)[NV], float edge, int full) {
  float f[T::E];
  float mx = edge;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (!holds<G, NV>(j, full)) break;
    T::unpack(v[j], f);
#pragma unroll
    for (int e = 0; e < T::E; ++e) mx = fmaxf(mx, f[e]);
  }
  return fmaxf(group_max<(G < 64 ? G : 64)>(mx), -FLT_MAX);
}
template <typename T, int G, int NV, bool KEEP, bool EXACT>
__device__ __forceinline__ RowSum wave_sum(u32x4 (&v)[NV], float edge, float mx, int full, const RowArgs& a) {
  constexpr int GL = G < 64 ? G : 64;
  float f[T::E];
  fresh<NV, EXACT>(v);
  if constexpr (EXACT && G <= 64) {
    float low = 0.0f;
    double s = (double)exp_parts(edge - mx, a, low);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!holds<G, NV>(j, full)) break;
      T::unpack(v[j], f);
#pragma unroll
      for (int e = 0; e < T::E; ++e) s += (double)exp_parts(f[e] - mx, a, low);
    }
    if constexpr (KEEP) fresh<NV>(v);
    return in_parts(mx, group_sum<GL>(fma((double)low, LN2, s)));
  } else {
    float s0 = exp_d(edge - mx, a.c_hi, a.c_lo), s1 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!holds<G, NV>(j, full)) break;
      T::unpack(v[j], f);
#pragma unroll
      for (int e = 0; e < T::E; e += 2) {
        s0 += exp_d(f[e] - mx, a.c_hi, a.c_lo);
        s1 += exp_d(f[e + 1] - mx, a.c_hi, a.c_lo);
      }
    }
    if constexpr (KEEP) fresh<NV>(v);
    if constexpr (EXACT) return in_parts(mx, group_sum<GL>((double)s0 + (double)s1));
    return RowSum{mx, group_sum<GL>(s0 + s1), 0.0f};
  }
}
// What a sum taken against a maximum counts for against one that is higher by -d.  (EXP2_LOW: of this exponential; at
// d = 0 there is none)
__device__ __forceinline__ double share_of(float d, const RowArgs& a) {
  float low = 0.0f;
  const float e = exp_parts(d, a, low);
  return e == 1.0f ? 1.0 : fma((double)low, LN2, (double)e) * (1.0 + EXP2_LOW);
}
// (Lane l of a wave takes the entry of wave l % WAVES, and the lanes add up among themselves.)
template <int WAVES, bool EXACT>
__device__ __forceinline__ RowSum join_stats(const float2* red, const float* red_lo, const RowArgs& a) {
  const int w = threadIdx.x % WAVES;
  const float2 r = red[w];
  const float m = fmaxf(group_max<WAVES>(r.x), -FLT_MAX);
  if constexpr (!EXACT) return in_parts(m, group_sum<WAVES>((double)(r.y * exp_d(r.x - m, a.c_hi, a.c_lo))));
  return in_parts(m, group_sum<WAVES>(((double)r.y + (double)red_lo[w]) * share_of(r.x - m, a)));
}

template <typename T, int G, int NV, bool KEEP, bool EXACT>
__device__ __forceinline__ RowSum row_sum(u32x4 (&v)[NV], float edge, float mx, int full, const RowArgs& a, float2* red,
                                          float* red_lo) {
  const RowSum st = wave_sum<T, G, NV, KEEP, EXACT>(v, edge, mx, full, a);
  if constexpr (G <= 64) return st;
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = make_float2(st.m, st.hi);
    if (EXACT) red_lo[threadIdx.x >> 6] = st.lo;
  }
  __syncthreads();
  return join_stats<G / 64, EXACT>(red, red_lo, a);
}

// The teacher's list of a row, spread over GL lanes of one wave: the kept entries' classes (-1: not kept), exponentials
// and student logits go to LDS, padded to whole fours, the sums stay with the lanes.
//
// A class may be listed twice.  Every kept entry writes its number to its class' place in a table of bytes and looks what
// is there afterwards: its own number everywhere means that no class is.  (In a table smaller than the alphabet two
// classes may share a place; that costs the search of list_grad, no more.)  65536 rows of 100 float32 classes with 64
// entries: 43 us, 82 with the search for every entry.  Rows of 16 pieces a lane search (8192 rows of 131072 bf16 classes:
// 813 us without the table, 835 with it).
constexpr int TAGS = 16384;             // bytes of a workgroup's tables: every class of a row of up to 64 lanes has a place
struct List {
  int* idx; float* e; float* z; uint8_t* tag; int tag_mask;
  float St, A; int kept, twice;
};
__host__ __device__ constexpr int list_pad(int k) { return (k + 3) & ~3; }
constexpr size_t list_bytes(int rows, int k, bool tagged) { return (tagged ? TAGS : 0) + (size_t)rows * list_pad(k) * 12; }
template <bool TAGGED>
__device__ __forceinline__ List list_place(char* lds, int rows, int slot, int k) {
  const int pad = list_pad(k);
  float* at = (float*)(lds + (TAGGED ? TAGS : 0));
  return List{(int*)at + slot * pad, at + (rows + slot) * pad, at + (2 * rows + slot) * pad,
              (uint8_t*)lds + slot * (TAGS / rows), TAGS / rows - 1, 0.0f, 0.0f, 0, TAGGED ? 0 : 1};
}
template <int GL, bool TAGGED>
__device__ __forceinline__ void list_load(const RowArgs& a, int n, int g, List& l) {
  const long at = (long)n * a.k;
  float mt = -INFINITY;
  int kept = 0;
  for (int i = g; i < list_pad(a.k); i += GL) {
    float t = -INFINITY;
    int c = -1;
    if (i < a.k) {
      t = get_any(a.t_logits, a.t_dtype, at + i);
      c = get_int(a.t_index, a.t_index_bytes, at + i);
    }
    if (c < 0 || t == -INFINITY) c = -1;
    else {
      c = min(c, a.V - 1);
      mt = fmaxf(mt, t);
      kept = 1;
    }
    l.idx[i] = c;
    l.e[i] = t;
    if (TAGGED && c >= 0) l.tag[c & l.tag_mask] = (uint8_t)i;
  }
  if constexpr (TAGGED) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  mt = fmaxf(group_max<GL>(mt), -FLT_MAX);          // a NaN entry alone leaves -inf here: its exponential is NaN
  l.kept = (int)group_max<GL>((float)kept);
  float St = 0.0f, A = 0.0f;
  int twice = 0;
  for (int i = g; i < list_pad(a.k); i += GL) {
    const float d = l.e[i] - mt;
    const int c = l.idx[i];
    const float e = c < 0 ? 0.0f : exp_d(d, a.c_hi, a.c_lo);
    if (TAGGED && c >= 0 && l.tag[c & l.tag_mask] != i) twice = 1;
    St += e;
    if (e != 0.0f) A = fmaf(e, d * a.inv_tau, A);
    l.e[i] = e;
  }
  l.St = group_sum<GL>(St);
  l.A = group_sum<GL>(A);
  if constexpr (TAGGED) l.twice = (int)group_max<GL>((float)twice);
}
// tau^2 KL(teacher || student) of the row
template <typename T, int GL>
__device__ __forceinline__ float list_loss(const RowArgs& a, const char* row, int g, const List& l, float m, float S) {
  float Bs = 0.0f;
  for (int i = g; i < a.k; i += GL) {
    const float e = l.e[i], z = T::get(row, max(l.idx[i], 0));
    l.z[i] = z;
    if (e != 0.0f) Bs = fmaf(e, (z - m) * a.inv_tau, Bs);
  }
  Bs = group_sum<GL>(Bs);
  const float tau = 1.0f / a.inv_tau;
  return l.kept ? tau * tau * ((l.A - Bs) / l.St - logf(l.St) + logf(S)) : 0.0f;
}
// Gradient elements of the kept classes, c (q - p), over the -c p that the row's pieces hold there.  A class listed twice
// gets the sum of its entries, in the list's order, from each of them.
template <typename T, int GL, bool TAGGED>
__device__ __forceinline__ void list_grad(const RowArgs& a, char* out, int g, const List& l, float m, float inv_S, float c) {
  const float inv_St = rcp_acc(l.St);
  for (int i = g; i < a.k; i += GL) {
    const int cls = l.idx[i];
    if (cls < 0) continue;
    float q = TAGGED ? l.e[i] : 0.0f;
    if (!TAGGED || l.twice) {
      q = 0.0f;
#pragma unroll (TAGGED ? 1 : 4)
      for (int j = 0; j < list_pad(a.k); j += 4) {
        const int4 x = *(const int4*)(l.idx + j);
        const float4 e = *(const float4*)(l.e + j);
        q += x.x == cls ? e.x : 0.0f;
        q += x.y == cls ? e.y : 0.0f;
        q += x.z == cls ? e.z : 0.0f;
        q += x.w == cls ? e.w : 0.0f;
      }
    }
    const float p = exp_d(l.z[i] - m, a.c_hi, a.c_lo) * inv_S;
    T::put(out, cls, c * (q * inv_St - p));
  }
}

// the gradient row of a position that is not counted
template <typename T, bool PEEL>
__device__ __forceinline__ void zero_row(char* out, int V, int g, int G) {
  const Cut<T, PEEL> cut(out, V);
  const u32x4 zero = {0, 0, 0, 0};
  char* body = out + cut.head * T::SIZE;
  for (int j = g; j < cut.full; j += G) *(typename T::Raw*)(body + (uint32_t)j * 16u) = zero;
  if (cut.has_edge(g)) T::put(out, cut.edge(g), 0.0f);
}

// scale exp((z - m) / tau) of a piece.  For the 16-bit types the scale goes into the exponent and the constant is one
// float: 1e-6 of the value, against the 2^-12 and 2^-9 of their rounding, for 7.5 instructions instead of 9.5.
struct Scale {
  float scale, log2_abs;
  uint32_t sign;                       // of both halves of a dword
  __device__ __forceinline__ explicit Scale(float s)
      : scale(s), log2_abs(__builtin_amdgcn_logf(fabsf(s))), sign(s < 0.0f ? 0x80008000u : 0u) {}
};
template <typename T, typename Args>
__device__ __forceinline__ u32x4 grad_piece(u32x4 v, const Args& a, float m, const Scale& sc) {
  float f[T::E];
  T::unpack(v, f);
  if constexpr (T::SIZE == 4) {
#pragma unroll
    for (int e = 0; e < T::E; ++e) f[e] = sc.scale * exp_d(f[e] - m, a.c_hi, a.c_lo);
    return T::pack(f);
  } else {
#pragma unroll
    for (int e = 0; e < T::E; ++e) f[e] = exp2_hw(fmaf(f[e] - m, a.c_hi, sc.log2_abs));
    return T::pack(f) ^ sc.sign;
  }
}
// The gradient pieces of a row from the pieces of its logits, and its end elements.
template <typename T, int G, int NV, bool NT, bool PEEL>
__device__ __forceinline__ void grad_pieces(u32x4 (&v)[NV], float edge, const RowArgs& a, const Cut<T, PEEL>& cut,
                                            char* out, int g, float m, float scale) {
  char* body = out + cut.head * T::SIZE;
  const Scale sc(scale);
  if (G >= 64 && in_dwords<T>(body)) {
    const Rsrc to = pieces_of(body, cut.full);
    const int at = lane_offset(g);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!holds<G, NV>(j, cut.full)) break;
      store_piece<NT>(to, at, j, G, grad_piece<T>(v[j], a, m, sc));
    }
  } else if (G < 64 || T::SIZE < 4) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * G + g < cut.full) store_piece<T, NT>(body + j * (G * 16) + (uint32_t)g * 16u, grad_piece<T>(v[j], a, m, sc));
  }
  if (cut.has_edge(g)) T::put(out, cut.edge(g), scale * exp_d(edge - m, a.c_hi, a.c_lo));
}

// Waves of a SIMD that the registers are to leave room for: with 8 the small rows take 54 us instead of 57 (32 x 32 images,
// 256 classes), the 8-piece ones gain 3 % with 6; the lists' registers would spill there (107 us with 4, 113 with 6).
template <int G, int NV, bool DISTILL>
constexpr int WAVES_PER_SIMD = G <= 64 ? (DISTILL ? 6 : 8) : NV == 8 && !DISTILL ? 6 : 4;
template <typename T, int G, int NV, bool DISTILL, bool GRAD>
__global__ __launch_bounds__(Shape<G>::WG)
__attribute__((amdgpu_waves_per_eu(WAVES_PER_SIMD<G, NV, DISTILL>))) void k_rows(RowArgs a) {
  typedef Shape<G> Sh;
  constexpr bool PEEL = G >= 2 * T::E; // (a row of fewer lanes has no lane for every end element)
  constexpr bool TAGGED = NV < 16;
  // Logits that are read once, for the gradient too, pass the caches by: 3 to 10 % of 268 MB of them at 4096 classes and
  // more.  (A statistics launch leaves them there for the gradient launch: 588 us against 606 for 4 pairs of 1537 x 49999
  // float16; and walking workgroups of 1024 lose 3 %: 821 us against 844 at 8192 x 131072 bf16.)
  constexpr bool NT_LOADS = GRAD && G < 1024;
  // A list's gradient goes over elements of pieces just written: in rows of up to four pieces a lane it hits much of them,
  // which have to be in the caches still (64 entries: 65536 rows of 2000 bf16 classes 186 -> 150 us, 32768 of 8000 322 ->
  // 272; at 4000 rows of 32003 103 -> 110).  So does a token's element in short float32 rows (2 M rows of 32 classes 159 ->
  // 147; of 1 M rows of 24 bf16 classes 80 -> 84).
  constexpr bool NT_STORES = DISTILL ? NV > 4 : G > 8 || T::SIZE == 2;
  __shared__ float2 red[2][G > 64 ? G / 64 : 1];
  __shared__ float red_lo[2][G > 64 ? G / 64 : 1];
  __shared__ int kept_flag[2];
  __shared__ float list_sums[3];
  __shared__ double wg_sum[Sh::ROWS];
  __shared__ int counts[16];
  extern __shared__ __align__(16) char lists[];
  if (a.only_if_rescaled && *a.upstream == 1.0f) return;

  const int g = threadIdx.x % G, slot = Sh::ROWS == 1 ? 0 : threadIdx.x / G, wave = threadIdx.x >> 6;
  const float w = row_weight(a, counts);
  double acc = 0.0;
  int phase = 0;

  for (int n0 = blockIdx.x * Sh::ROWS; n0 < a.N; n0 += gridDim.x * Sh::ROWS) {
    int n = n0 + slot;
    if (Sh::ROWS > 1 && n >= a.N) break;
    if constexpr (G == 64) n = __builtin_amdgcn_readfirstlane(n);        // the row of a whole wave: scalar addresses
    char* out = GRAD ? (char*)a.dz + (long)n * a.V * T::SIZE : nullptr;
    if (a.mask && !a.mask[n]) {                      // not counted: nothing of its row is read
      if constexpr (GRAD) zero_row<T, PEEL>(out, a.V, g, G);
      if (g == 0) {
        if (a.per_row) a.per_row[n] = 0.0f;
        if (a.stats) a.stats[n] = not_counted();
      }
      continue;
    }
    const char* row = row_ptr(a, n, T::SIZE);
    const Cut<T, PEEL> cut(row, a.V);
    const char* body = row + cut.head * T::SIZE;
    u32x4 v[NV];
    if constexpr (G >= 64) {
      const Rsrc from = pieces_of(body, cut.full);
      const int at = lane_offset(g);
#pragma unroll
      for (int j = 0; j < NV; ++j) v[j] = load_piece<NT_LOADS>(from, at, j, G);
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        v[j] = (u32x4){T::NEG_INF, T::NEG_INF, T::NEG_INF, T::NEG_INF};
        if (j * G + g < cut.full) v[j] = *(const typename T::Raw*)(body + j * (G * 16) + (uint32_t)g * 16u);
      }
    }
    const float edge = cut.has_edge(g) ? T::get(row, cut.edge(g)) : -INFINITY;
    // what the row's own arithmetic needs is on its way too
    int y = 0;
    float zy = 0.0f;
    List l = list_place<TAGGED>(lists, Sh::ROWS, slot, a.k);
    const bool lister = G <= 64 || wave == 0;        // a row of several waves: the first has the list
    if constexpr (!DISTILL) {
      y = min(max(get_int(a.tokens, a.tok_bytes, n), 0), a.V - 1);
      zy = T::get(row, y);
    } else if (lister) {
      list_load<Sh::GL, TAGGED>(a, n, g, l);
      if (G > 64 && g == 0) {
        kept_flag[phase] = l.kept;
        list_sums[0] = l.St;                          // (not carried in registers over the sweeps)
        list_sums[1] = l.A;
        if (TAGGED) list_sums[2] = (float)l.twice;
      }
    }
    if constexpr (G >= 64) mask_pieces<T, G, NV>(v, cut.full, g);
    const float mx = wave_max<T, G, NV>(v, edge, cut.full);
    RowSum st;
    if constexpr (DISTILL || GRAD)
      st = row_sum<T, G, NV, GRAD, !DISTILL>(v, edge, mx, cut.full, a, red[phase], red_lo[phase]);
    else if (a.head != HEAD_LOGPROB)
      st = row_sum<T, G, NV, false, true>(v, edge, mx, cut.full, a, red[phase], red_lo[phase]);
    else st = row_sum<T, G, NV, false, false>(v, edge, mx, cut.full, a, red[phase], red_lo[phase]);
    const float m = st.m, S = st.hi;

    if constexpr (!DISTILL) {
      const TokenOut o = token_head(a, n, zy - m, S);
      if (g == 0) {
        if (a.per_row) a.per_row[n] = o.lp;
        if (a.stats) a.stats[n] = make_float4(m, S, a.head == HEAD_LOGPROB ? a.inv_tau : st.lo, zy);
        acc += (double)o.loss;
      }
      if constexpr (GRAD) {
        const float c = w * o.c, inv_S = rcp_acc(S);
        grad_pieces<T, G, NV, NT_STORES>(v, edge, a, cut, out, g, m, -c * inv_S);
        // the token's own element, c (1 - p), by the lane that wrote its place above
        if (g == cut.lane_of(y, G)) T::put(out, y, token_grad(c, zy - m, S, a.c_hi, a.c_lo));
      }
    } else {
      const int kept = G > 64 ? kept_flag[phase] : l.kept;
      if (lister) {
        if constexpr (G > 64) {
          l.St = list_sums[0];
          l.A = list_sums[1];
          l.kept = kept;
        }
        const float loss = list_loss<T, Sh::GL>(a, row, g, l, m, S);
        if (g == 0) {
          if (a.per_row) a.per_row[n] = loss;
          acc += (double)loss;
        }
      }
      if constexpr (GRAD) {
        const float inv_S = rcp_acc(S);
        grad_pieces<T, G, NV, NT_STORES>(v, edge, a, cut, out, g, m, kept ? w * inv_S : 0.0f);
        if constexpr (G > 64) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (lister && kept) {
          if constexpr (G > 64) {
            l.St = list_sums[0];
            if (TAGGED) l.twice = list_sums[2] != 0.0f;
          }
          list_grad<T, Sh::GL, TAGGED>(a, out, g, l, m, inv_S, -w);
        }
      }
    }
    phase ^= 1;
  }
  if (a.partial) {
    if (g == 0) wg_sum[slot] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
      double s = 0.0;
      for (int i = 0; i < Sh::ROWS; ++i) s += wg_sum[i];
      put_sum(a, s);
    }
  }
}

// -------------------------------------------------------------------------- rows wider than the registers: two reads
constexpr int WIDE = 1024;
template <typename T, bool DISTILL>
__global__ __launch_bounds__(WIDE) void k_rows_wide(RowArgs a) {
  constexpr int E = T::E;
  __shared__ float2 red[2][WIDE / 64];
  __shared__ float red_lo[2][WIDE / 64];
  __shared__ int kept_flag[2];
  extern __shared__ __align__(16) char lists[];
  if (a.only_if_rescaled && *a.upstream == 1.0f) return;
  const int g = threadIdx.x, wave = threadIdx.x >> 6;
  __shared__ int counts[16];
  const float w = row_weight(a, counts);
  double acc = 0.0;
  int phase = 0;
  for (int n = blockIdx.x; n < a.N; n += gridDim.x) {
    char* out = a.dz ? (char*)a.dz + (long)n * a.V * T::SIZE : nullptr;
    if (a.mask && !a.mask[n]) {
      if (out) zero_row<T, true>(out, a.V, g, WIDE);
      if (g == 0) {
        if (a.per_row) a.per_row[n] = 0.0f;
        if (a.stats) a.stats[n] = not_counted();
      }
      continue;
    }
    const char* row = row_ptr(a, n, T::SIZE);
    const Cut<T, true> cut(row, a.V);
    const char* body = row + cut.head * T::SIZE;
    char* obody = out + cut.head * T::SIZE;
    const float edge = cut.has_edge(g) ? T::get(row, cut.edge(g)) : -INFINITY;
    // The lane's running maximum and sum.  The sum is held in 64 bits: a lane of the widest rows adds 131072 terms, and
    // what a float32 addition of equal terms rounds away is the same every time (6e-5 of S at 4 M classes).  Two chains
    // of at most 16 additions stay in float32.
    float mx = fmaxf(edge, -FLT_MAX);
    double s = (double)exp_d(edge - mx, a.c_hi, a.c_lo);
    float f[E];
    for (int j = g; j < cut.full; j += 4 * WIDE) {       // four pieces on their way at a time
      u32x4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        v[u] = (u32x4){T::NEG_INF, T::NEG_INF, T::NEG_INF, T::NEG_INF};
        if (j + u * WIDE < cut.full) v[u] = *(const typename T::Raw*)(body + u * (WIDE * 16) + (uint32_t)j * 16u);
      }
      float top = mx;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        T::unpack(v[u], f);
#pragma unroll
        for (int e = 0; e < E; ++e) top = fmaxf(top, f[e]);
      }
      if (top > mx) s *= share_of(mx - top, a);
      mx = top;
      float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        T::unpack(v[u], f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          s0 += exp_d(f[e] - mx, a.c_hi, a.c_lo);
          s1 += exp_d(f[e + 1] - mx, a.c_hi, a.c_lo);
        }
      }
      s += (double)s0 + (double)s1;
    }
    int y = 0;
    float zy = 0.0f;
    List l = list_place<false>(lists, 1, 0, a.k);
    if constexpr (!DISTILL) {
      y = min(max(get_int(a.tokens, a.tok_bytes, n), 0), a.V - 1);
      zy = T::get(row, y);
    } else {
      if (wave == 0) {
        list_load<64, false>(a, n, g, l);
        if (g == 0) kept_flag[phase] = l.kept;
      }
    }
    const float mw = group_max<64>(mx);
    const RowSum part = in_parts(mw, group_sum<64>(s * share_of(mx - mw, a)));
    if ((g & 63) == 0) {
      red[phase][wave] = make_float2(mw, part.hi);
      red_lo[phase][wave] = part.lo;
    }
    __syncthreads();
    const RowSum st = join_stats<WIDE / 64, true>(red[phase], red_lo[phase], a);
    const float m = st.m, S = st.hi;

    float c, scale;
    const float inv_S = rcp_acc(S);
    int kept = 1;
    if constexpr (!DISTILL) {
      const TokenOut o = token_head(a, n, zy - m, S);
      if (g == 0) {
        if (a.per_row) a.per_row[n] = o.lp;
        if (a.stats) a.stats[n] = make_float4(m, S, a.head == HEAD_LOGPROB ? a.inv_tau : st.lo, zy);
        acc += (double)o.loss;
      }
      c = w * o.c;
      scale = -c * inv_S;
    } else {
      kept = kept_flag[phase];
      if (wave == 0) {
        const float loss = list_loss<T, 64>(a, row, g, l, m, S);
        if (g == 0) {
          if (a.per_row) a.per_row[n] = loss;
          acc += (double)loss;
        }
      }
      c = kept ? -w : 0.0f;
      scale = kept ? w * inv_S : 0.0f;
    }
    if (out) {
      const Scale sc(scale);
#pragma unroll 4
      for (int j = g; j < cut.full; j += WIDE)
        store_piece<T>(obody + (uint32_t)j * 16u, grad_piece<T>(*(const typename T::Raw*)(body + (uint32_t)j * 16u), a, m, sc));
      if (cut.has_edge(g)) T::put(out, cut.edge(g), scale * exp_d(edge - m, a.c_hi, a.c_lo));
      if constexpr (!DISTILL) {
        if (g == cut.lane_of(y, WIDE)) T::put(out, y, token_grad(c, zy - m, S, a.c_hi, a.c_lo));
      } else {
        __syncthreads();
        if (wave == 0 && kept) list_grad<T, 64, false>(a, out, g, l, m, inv_S, c);
      }
    }
    phase ^= 1;
  }
  if (a.partial && g == 0) put_sum(a, acc);
}

// ------------------------------------------------------------------------------- gradient from the rows' statistics
// dz = c u (1[v = y] - p): m, S, c and the token's logit from stats, u the upstream gradient of the row (u_stride 1) or
// of the whole (0).  A group of `lanes` takes a row of up to GRAD_PIECES pieces a lane; of a longer one (SPLIT) a
// workgroup takes SPLIT_PIECES a lane, so that few long rows fill the chip too.  All pieces are asked for before the
// first is used, and the logits are not looked at again: non-temporal loads too.  8 x 1024 x 65536 bf16
// log-probabilities, forward and backward: 500 us; 503 with 4 pieces a lane, 510 with 8, 538 with cached loads, 563 with
// 8 pieces a lane in a loop of 4096 workgroups.
constexpr int GRAD_WG = 256, GRAD_PIECES = 4, SPLIT_PIECES = 2;
struct GradArgs {
  RowArgs r;                          // logits, tokens, stats, dz
  const float* upstream; int u_stride; int only_if_rescaled;
  int lanes, chunks;                  // chunks of a row
};
template <typename T, bool SPLIT>
__global__ __launch_bounds__(GRAD_WG) void k_token_grad(GradArgs a) {
  constexpr int E = T::E, NV = SPLIT ? SPLIT_PIECES : GRAD_PIECES;
  constexpr bool PEEL = SPLIT;
  if (a.only_if_rescaled && *a.upstream == 1.0f) return;
  const int lanes = SPLIT ? GRAD_WG : a.lanes;
  const int g = threadIdx.x & (lanes - 1), slot = SPLIT ? 0 : threadIdx.x / lanes, groups = SPLIT ? 1 : GRAD_WG / lanes;
  const unsigned jobs = (unsigned)a.r.N * (unsigned)a.chunks;
  for (unsigned job = blockIdx.x * groups + slot; job < jobs; job += gridDim.x * groups) {
    const int n = SPLIT ? (int)(job / (unsigned)a.chunks) : (int)job;
    const int part = SPLIT ? (int)(job - (unsigned)n * (unsigned)a.chunks) : 0, lo = part * (NV * GRAD_WG);
    const bool last = !SPLIT || part == a.chunks - 1;
    const float4 st = a.r.stats[n];
    // A row that is not counted, whatever its upstream gradient (a NaN or inf there is common: 0 times it is none), or
    // one whose coefficient is 0: its logits are not read.
    const float u = a.upstream ? a.upstream[(long)n * a.u_stride] : 1.0f;      // (asked for with the statistics)
    const float c = st.y < 0.0f ? 0.0f : st.z * u;
    char* out = (char*)a.r.dz + (long)n * a.r.V * T::SIZE;
    const bool zero = c == 0.0f;
    const char* row = zero ? out : row_ptr(a.r, n, T::SIZE);
    const Cut<T, PEEL> cut(row, a.r.V);
    const char* body = row + cut.head * T::SIZE;
    char* obody = out + cut.head * T::SIZE;
    const float m = st.x, scale = zero ? 0.0f : -c * rcp_acc(st.y);
    const Scale sc(scale);
    u32x4 v[NV];
    if constexpr (SPLIT) {
      const int some = max(0, min(cut.full - lo, NV * GRAD_WG));
      const Rsrc from = pieces_of(body + (long)lo * 16, zero ? 0 : some);
      char* to = obody + (long)lo * 16;
#pragma unroll
      for (int j = 0; j < NV; ++j) v[j] = load_piece<true>(from, g * 16, j, GRAD_WG);
      auto piece = [&](int j) { return zero ? (u32x4){0, 0, 0, 0} : grad_piece<T>(v[j], a.r, m, sc); };
      if (in_dwords<T>(to)) {
#pragma unroll
        for (int j = 0; j < NV; ++j) store_piece<true>(pieces_of(to, some), g * 16, j, GRAD_WG, piece(j));
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (j * GRAD_WG + g < some) store_piece<T>(to + (uint32_t)(j * GRAD_WG + g) * 16u, piece(j));
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        v[j] = (u32x4){0, 0, 0, 0};
        if (!zero && j * lanes + g < cut.full)
          v[j] = __builtin_nontemporal_load((const typename T::Raw*)(body + (uint32_t)(j * lanes + g) * 16u));
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * lanes + g < cut.full)
          store_piece<T>(obody + (uint32_t)(j * lanes + g) * 16u, zero ? (u32x4){0, 0, 0, 0} : grad_piece<T>(v[j], a.r, m, sc));
    }
    if (last && cut.has_edge(g)) {
      const int i = cut.edge(g);
      T::put(out, i, zero ? 0.0f : scale * exp_d(T::get(row, i) - m, a.r.c_hi, a.r.c_lo));
    }
    if (zero) continue;
    // the token's own element, c (1 - p), by the lane that wrote its place above
    const int y = min(max(get_int(a.r.tokens, a.r.tok_bytes, n), 0), a.r.V - 1), in = y - cut.head;
    const bool piece = in >= 0 && in < cut.full * E;
    if (piece ? in / E >= lo && in / E < lo + NV * lanes && ((in / E - lo) & (lanes - 1)) == g : last && cut.lane_of(y, 1) == g)
      T::put(out, y, token_grad(c, st.w - m, st.y, a.r.c_hi, a.r.c_lo));
  }
}

// ------------------------------------------------------------------------------------------------- small kernels
constexpr int SUM_WG = 1024;
__device__ __forceinline__ double block_sum(double v, double* lds) {
  v = group_sum<64>(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += lds[i];
  __syncthreads();
  return s;
}
__global__ __launch_bounds__(SUM_WG) void k_count(const uint8_t* mask, int N, int* count) {
  __shared__ int lds[SUM_WG / 64];
  const int c = count_mask(mask, N, lds);
  if (threadIdx.x == 0) *count = c;
}
// loss = scale / count * sum of the partial sums, in a fixed order
__global__ __launch_bounds__(SUM_WG) void k_finish(const double* partial, int n, const int* count, double inv_count,
                                                   float scale, float* loss) {
  __shared__ double lds[SUM_WG / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += SUM_WG) s += partial[i];
  s = block_sum(s, lds);
  if (threadIdx.x == 0) *loss = (float)(s * (double)scale * (count ? 1.0 / (double)max(*count, 1) : inv_count));
}

// ----------------------------------------------------------------------------------------------- preference pairs
struct PairArgs {
  RowArgs r;                                                  // logits, tokens, mask, stats, dz
  const float* ref;
  int P; float beta, smooth; int average; float out_scale;
  float* rewards; double* pair_loss; float* loss;             // loss: of a single pair, written here
};
constexpr int PAIR_WG = 1024;
// A row's log-ratio in 64 bits: a sequence's is a long sum of small differences of large terms.  (S = y + z: the place of
// c holds the rest of S until the pair's sums are known.)
__device__ __forceinline__ double row_ratio(const PairArgs& a, float4 st, long n) {
  const double S = (double)st.y + (double)st.z;
  return (double)st.w - (double)st.x - (log(S) + EXP2_LOW * (1.0 - 1.0 / S)) - (double)(a.ref ? a.ref[n] : 0.0f);
}
// Sums and counts of a pair's two sequences over the workgroup; then, by the first wave alone (every wave with its share
// of double-precision functions took 4 us of the workgroup), the pair's loss, its rewards, and c of its sequences' rows.
struct PairShared { double D[2][PAIR_WG / 64]; int n[2][PAIR_WG / 64]; float2 c; };
__device__ __forceinline__ float2 pair_finish(const PairArgs& a, int p, double D0, double D1, int n0, int n1,
                                              PairShared& sh) {
  constexpr int W = PAIR_WG / 64;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  D0 = group_sum<64>(D0);
  D1 = group_sum<64>(D1);
  n0 = group_sum<64>(n0);
  n1 = group_sum<64>(n1);
  if (lane == 0) {
    sh.D[0][wave] = D0;
    sh.D[1][wave] = D1;
    sh.n[0][wave] = n0;
    sh.n[1][wave] = n1;
  }
  __syncthreads();
  if (wave == 0) {
    D0 = group_sum<W>(sh.D[0][lane % W]);
    D1 = group_sum<W>(sh.D[1][lane % W]);
    const double c0 = (double)max(group_sum<W>(sh.n[0][lane % W]), 1), c1 = (double)max(group_sum<W>(sh.n[1][lane % W]), 1);
    if (a.average) {
      D0 /= c0;
      D1 /= c1;
    }
    const double margin = (double)a.beta * (D0 - D1), e = (double)a.smooth;
    const double z = exp(-fabs(margin)), soft = log1p(z), top = 1.0 / (1.0 + z);
    const double sig = margin >= 0.0 ? top : z * top, gis = margin >= 0.0 ? z * top : top;  // sigma(margin), sigma(-margin)
    const double neg = margin < 0.0 ? -margin : 0.0, pos = margin > 0.0 ? margin : 0.0;
    // a term of weight 0 is not there (a token that the model rules out makes the other one infinite)
    const double loss = (e < 1.0 ? (1.0 - e) * (soft + neg) : 0.0) + (e > 0.0 ? e * (soft + pos) : 0.0);
    const double slope = -(double)a.out_scale * (double)a.beta / (double)a.P * ((1.0 - e) * gis - e * sig);
    if (lane == 0) {
      a.rewards[p] = (float)((double)a.beta * D0);
      a.rewards[p + a.P] = (float)((double)a.beta * D1);
      if (a.loss) *a.loss = (float)(loss * (double)a.out_scale);
      else a.pair_loss[p] = loss;
      sh.c = make_float2((float)(slope / (a.average ? c0 : 1.0)), (float)(-slope / (a.average ? c1 : 1.0)));
    }
  }
  __syncthreads();
  return sh.c;
}

// From the rows' statistics, one workgroup a pair.
__global__ __launch_bounds__(PAIR_WG) void k_pair(PairArgs a) {
  __shared__ PairShared sh;
  const int p = blockIdx.x, L = a.r.L;
  const uint8_t* mask = a.r.mask;
  float4* stats = a.r.stats;
  double D[2] = {0.0, 0.0};
  int cnt[2] = {0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long n0 = (long)(p + h * a.P) * L;
    for (int l = threadIdx.x; l < L; l += PAIR_WG) {
      if (mask && !mask[n0 + l]) continue;
      D[h] += row_ratio(a, stats[n0 + l], n0 + l);
      ++cnt[h];
    }
  }
  const float2 c = pair_finish(a, p, D[0], D[1], cnt[0], cnt[1], sh);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long n0 = (long)(p + h * a.P) * L;
    for (int l = threadIdx.x; l < L; l += PAIR_WG)
      if (!mask || mask[n0 + l]) stats[n0 + l].z = h ? c.y : c.x;
  }
}

// Pairs of few rows in one launch: a workgroup reads its pair's rows, sums, and makes the gradient from a second look at
// them, which the caches still hold.  Rows' statistics wait in LDS (2 L float4) and go to memory for the backward.
// One launch against three, on the device: 128 pairs of 263 x 24 float32 (four and a bit sweeps of the workgroup over its
// rows) 16.7 / 19.7 us, of 320 (five) 18.4 / 20.9, of 400 21.3 / 22.8, of 600 27.8 / 28.8, 1024 pairs of 263 46 / 65; a pair
// alone, with three launches that spread it over the chip, 6.5 / 9.8 at 30 rows a sequence, 9.5 / 10.7 at 160, 13.7 / 11.2
// at 320, 21.1 / 12.1 at 600.  Up to five sweeps, and rows that a wave holds: beyond, many pairs gain 4 to 7 % and few lose
// half.
constexpr int PAIR_SWEEPS = 5;
constexpr long PAIR_BYTES = 128 << 10;
constexpr int pair_lanes(int full) { return full <= 32 ? 8 : full <= 64 ? 16 : full <= 128 ? 32 : 64; }
template <typename T, int G, int NV>
__global__ __launch_bounds__(PAIR_WG) void k_pair_rows(PairArgs a) {
  constexpr int ROWS = PAIR_WG / G;
  __shared__ PairShared sh;
  extern __shared__ __align__(16) char stats_lds[];
  float4* stats = (float4*)stats_lds;
  const int p = blockIdx.x, L = a.r.L, g = threadIdx.x % G, slot = threadIdx.x / G;
  auto row_of = [&](int i) { return i < L ? (long)p * L + i : (long)(p + a.P) * L + (i - L); };
  for (int i = slot; i < 2 * L; i += ROWS) {
    const int n = (int)row_of(i);
    if (a.r.mask && !a.r.mask[n]) {
      if (g == 0) stats[i] = not_counted();
      continue;
    }
    const char* row = row_ptr(a.r, n, T::SIZE);
    const Cut<T, false> cut(row, a.r.V);
    u32x4 v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      v[j] = (u32x4){T::NEG_INF, T::NEG_INF, T::NEG_INF, T::NEG_INF};
      if (j * G + g < cut.full) v[j] = *(const typename T::Raw*)(row + j * (G * 16) + (uint32_t)g * 16u);
    }
    const float edge = cut.has_edge(g) ? T::get(row, cut.edge(g)) : -INFINITY;
    const int y = min(max(get_int(a.r.tokens, a.r.tok_bytes, n), 0), a.r.V - 1);
    const float zy = T::get(row, y);
    const RowSum st = wave_sum<T, G, NV, false, true>(v, edge, wave_max<T, G, NV>(v, edge, NV * G), NV * G, a.r);
    if (g == 0) stats[i] = make_float4(st.m, st.hi, st.lo, zy);
  }
  __syncthreads();
  double D[2] = {0.0, 0.0};
  int cnt[2] = {0, 0};
  for (int i = threadIdx.x; i < 2 * L; i += PAIR_WG) {
    const float4 st = stats[i];
    if (st.y < 0.0f) continue;
    const double r = row_ratio(a, st, row_of(i));
    D[0] += i < L ? r : 0.0;
    D[1] += i < L ? 0.0 : r;
    cnt[0] += i < L;
    cnt[1] += i >= L;
  }
  const float2 c = pair_finish(a, p, D[0], D[1], cnt[0], cnt[1], sh);
  for (int i = threadIdx.x; i < 2 * L; i += PAIR_WG) {
    float4 st = stats[i];
    if (!(st.y < 0.0f)) st.z = i < L ? c.x : c.y;
    stats[i] = st;
    a.r.stats[row_of(i)] = st;
  }
  if (!a.r.dz) return;
  __syncthreads();
  for (int i = slot; i < 2 * L; i += ROWS) {
    const int n = (int)row_of(i);
    const float4 st = stats[i];
    char* out = (char*)a.r.dz + (long)n * a.r.V * T::SIZE;
    if (st.z == 0.0f) {                  // (of a row that is not counted too)
      zero_row<T, false>(out, a.r.V, g, G);
      continue;
    }
    const char* row = row_ptr(a.r, n, T::SIZE);
    const Cut<T, false> cut(row, a.r.V);
    const float m = st.x, scale = -st.z * rcp_acc(st.y);
    const Scale sc(scale);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * G + g < cut.full) {
        const uint32_t at = j * (G * 16) + (uint32_t)g * 16u;
        store_piece<T>(out + at, grad_piece<T>(*(const typename T::Raw*)(row + at), a.r, m, sc));
      }
    if (cut.has_edge(g)) {
      const int k = cut.edge(g);
      T::put(out, k, scale * exp_d(T::get(row, k) - m, a.r.c_hi, a.r.c_lo));
    }
    const int y = min(max(get_int(a.r.tokens, a.r.tok_bytes, n), 0), a.r.V - 1);
    if (g == cut.lane_of(y, G)) T::put(out, y, token_grad(st.z, st.w - m, st.y, a.r.c_hi, a.r.c_lo));
  }
}

// ----------------------------------------------------------------------------------------------------- host side
static int check_logits(const d3pm_logits* z, const char* who) {
  D3PM_CHECK_ARG(z != nullptr, "%s: null logits descriptor", who);
  D3PM_CHECK_ARG(z->dtype >= D3PM_F32 && z->dtype <= D3PM_BF16, "%s: logits dtype %d", who, z->dtype);
  D3PM_CHECK_ARG(z->V >= 1 && z->V <= (1 << 27), "%s: V = %d classes, need 1 .. 2^27", who, z->V);
  D3PM_CHECK_ARG(z->B >= 0 && z->L >= 0 && (z->B == 0 || z->L <= (long)(INT_MAX - 65536) / z->B),
                 "%s: B = %ld x L = %ld positions, need fewer than 2^31 - 65536", who, z->B, z->L);
  D3PM_CHECK_ARG(z->stride_b >= 0 && z->stride_l >= 0, "%s: negative strides", who);
  D3PM_CHECK_ARG(z->data != nullptr || z->B * z->L == 0, "%s: null logits", who);
  return D3PM_OK;
}
static int check_temperature(float t, const char* who) {
  D3PM_CHECK_ARG(t >= 1e-6f && t <= 1e6f, "%s: temperature %g, need 1e-6 .. 1e6", who, (double)t);
  return D3PM_OK;
}
static int check_int_bytes(int b, const char* what, const char* who) {
  D3PM_CHECK_ARG(b == 4 || b == 8, "%s: %s of %d bytes, need int32 or int64", who, what, b);
  return D3PM_OK;
}

// log2(e) / tau and 1 / tau, each in two floats.  The second of log2(e) / tau is above 0: a class ruled out with -inf
// stays -inf in both products of exp_d.
static void set_temperature(float tau, float* c_hi, float* c_lo, float* inv_tau, float* inv_tau_lo) {
  const double c = 1.44269504088896340736 / (double)tau;
  *c_hi = (float)c;
  if ((double)*c_hi >= c) *c_hi = std::nextafterf(*c_hi, 0.0f);
  *c_lo = (float)(c - (double)*c_hi);
  *inv_tau = (float)(1.0 / (double)tau);
  *inv_tau_lo = (float)(1.0 / (double)tau - (double)*inv_tau);
}
static bool is_dense(const d3pm_logits* z) { return z->B <= 1 || z->stride_b == z->L * z->stride_l; }

static RowArgs row_args(const d3pm_logits* z, float tau) {
  RowArgs a{};
  a.z = z->data; a.sb = z->stride_b; a.sl = z->stride_l;
  a.L = (int)z->L; a.V = z->V; a.N = (int)(z->B * z->L); a.dense = is_dense(z) ? 1 : 0;
  set_temperature(tau, &a.c_hi, &a.c_lo, &a.inv_tau, &a.inv_tau_lo);
  a.d_min = -200.0f * tau;                                    // (exp2 of -288)
  a.inv_count = 1.0f;
  return a;
}

// Launches the shape that holds a row in the fewest lanes of up to four pieces each, beyond 512 lanes in more pieces:
// few lanes a row share the row's own arithmetic and short reductions among more rows of a wave (32 x 32 images of 256
// float32 classes: 57 us at 16 lanes of 4 pieces, 70 at 32 of 2, 100 at 64 of 1; 32 k bf16 classes: 103 us at 512 x 8,
// 111 at 256 x 16, 142 at 1024 x 4).  *grid: the workgroups it took (as many partial sums).
template <typename T, int G, int NV, bool DISTILL>
static int launch_rows(const RowArgs& a, int* grid, hipStream_t s) {
  typedef Shape<G> Sh;
  const int want = (a.N - 1) / Sh::ROWS + 1;
  // Parts of a wave: as many workgroups as the 256 compute units hold, which walk over the rows.  A row to a workgroup:
  // one each, as they come (5 to 10 % less than with walking ones), up to 1024 lanes, where a compute unit holds one
  // and the next would wait for its last store (walking against as they come, distillation and policy loss: 648 / 678 and
  // 641 / 675 us at 8192 rows of 100003 bf16 classes, 709 / 731 and 655 / 704 at 12288 of 70001, 808 / 812 and 806 / 814 at
  // 8192 of 131072; float32 alone prefers the other: 432 / 425 and 417 / 415 at 4096 of 65528).
  *grid = std::min(want, G <= 64 ? 2048 : G < 1024 ? MAX_PARTIALS : 256);
  const size_t lds = DISTILL ? list_bytes(Sh::ROWS, a.k, NV < 16) : 0;
  if (a.dz) hipLaunchKernelGGL((k_rows<T, G, NV, DISTILL, true>), dim3(*grid), dim3(Sh::WG), lds, s, a);
  else hipLaunchKernelGGL((k_rows<T, G, NV, DISTILL, false>), dim3(*grid), dim3(Sh::WG), lds, s, a);
  D3PM_LAUNCH_CHECK("k_rows");
  return D3PM_OK;
}
template <typename T, bool DISTILL>
static int dispatch_rows(const RowArgs& a, int* grid, hipStream_t s) {
  const int full = a.V / T::E;
  if (full <= 8) return launch_rows<T, 8, 1, DISTILL>(a, grid, s);
  if (full <= 16) return launch_rows<T, 8, 2, DISTILL>(a, grid, s);
  if (full <= 32) return launch_rows<T, 8, 4, DISTILL>(a, grid, s);
  if (full <= 64) return launch_rows<T, 16, 4, DISTILL>(a, grid, s);
  if (full <= 128) return launch_rows<T, 32, 4, DISTILL>(a, grid, s);
  if (full <= 256) return launch_rows<T, 64, 4, DISTILL>(a, grid, s);
  if (full <= 512) return launch_rows<T, 128, 4, DISTILL>(a, grid, s);
  if (full <= 1024) return launch_rows<T, 256, 4, DISTILL>(a, grid, s);
  if (full <= 2048) return launch_rows<T, 512, 4, DISTILL>(a, grid, s);
  if (full <= 4096) return launch_rows<T, 512, 8, DISTILL>(a, grid, s);
  if (full <= 8192) return launch_rows<T, 512, 16, DISTILL>(a, grid, s);
  if (full <= 16384) return launch_rows<T, 1024, 16, DISTILL>(a, grid, s);
  *grid = std::min(a.N, MAX_PARTIALS);
  hipLaunchKernelGGL((k_rows_wide<T, DISTILL>), dim3(*grid), dim3(WIDE), DISTILL ? list_bytes(1, a.k, false) : 0, s, a);
  D3PM_LAUNCH_CHECK("k_rows_wide");
  return D3PM_OK;
}
template <bool DISTILL>
static int run_rows(const RowArgs& a, int dtype, int* grid, hipStream_t s) {
  return dtype == D3PM_F32 ? dispatch_rows<F32, DISTILL>(a, grid, s)
       : dtype == D3PM_F16 ? dispatch_rows<F16, DISTILL>(a, grid, s) : dispatch_rows<BF16, DISTILL>(a, grid, s);
}

template <typename T, int G, int NV>
static int launch_pairs(const PairArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((k_pair_rows<T, G, NV>), dim3(a.P), dim3(PAIR_WG), (size_t)2 * a.r.L * sizeof(float4), s, a);
  D3PM_LAUNCH_CHECK("k_pair_rows");
  return D3PM_OK;
}
template <typename T>
static int dispatch_pairs(const PairArgs& a, hipStream_t s) {
  const int full = a.r.V / T::E;                     // at most 256 pieces
  if (full <= 8) return launch_pairs<T, 8, 1>(a, s);
  if (full <= 16) return launch_pairs<T, 8, 2>(a, s);
  switch (pair_lanes(full)) {
    case 8: return launch_pairs<T, 8, 4>(a, s);
    case 16: return launch_pairs<T, 16, 4>(a, s);
    case 32: return launch_pairs<T, 32, 4>(a, s);
    default: return launch_pairs<T, 64, 4>(a, s);
  }
}
template <typename T>
static int launch_grad(GradArgs& a, hipStream_t s) {
  const int full = a.r.V / T::E;
  a.lanes = 8;
  while (a.lanes < 64 && a.lanes * GRAD_PIECES < full) a.lanes <<= 1;
  const bool split = a.lanes * GRAD_PIECES < full;
  a.chunks = split ? (full + GRAD_WG * SPLIT_PIECES - 1) / (GRAD_WG * SPLIT_PIECES) : 1;
  const long jobs = (long)a.r.N * a.chunks, per = split ? 1 : GRAD_WG / a.lanes;
  D3PM_CHECK_ARG(jobs < INT_MAX, "token gradient: %d rows of %d classes", a.r.N, a.r.V);
  // (the call that mostly finds nothing to do is not to cost the dispatch of all that would do it)
  const int grid = (int)std::min<long>((jobs + per - 1) / per, a.only_if_rescaled ? 2048 : 1 << 20);
  if (split) hipLaunchKernelGGL((k_token_grad<T, true>), dim3(grid), dim3(GRAD_WG), 0, s, a);
  else hipLaunchKernelGGL((k_token_grad<T, false>), dim3(grid), dim3(GRAD_WG), 0, s, a);
  D3PM_LAUNCH_CHECK("k_token_grad");
  return D3PM_OK;
}
static int run_grad(const d3pm_logits* z, const void* tokens, int tok_bytes, float tau, const float* stats,
                    const float* upstream, int per_row, int only_if_rescaled, void* dz, hipStream_t s) {
  GradArgs a{};
  a.r = row_args(z, tau);
  a.r.tokens = tokens; a.r.tok_bytes = tok_bytes;
  a.r.stats = (float4*)stats; a.r.dz = dz;
  a.upstream = upstream; a.u_stride = per_row; a.only_if_rescaled = only_if_rescaled;
  return z->dtype == D3PM_F32 ? launch_grad<F32>(a, s) : z->dtype == D3PM_F16 ? launch_grad<F16>(a, s) : launch_grad<BF16>(a, s);
}

// The count of the mask (first 8 bytes of the workspace, where a later call for the gradient alone finds it) and the
// partial sums behind it.
struct Scratch { int* count; double* partial; };
static int scratch(void* ws, size_t have, long partials, Scratch* out) {
  D3PM_CHECK_WORKSPACE(ws, have, 8 + 8 * (size_t)partials);
  out->count = (int*)ws;
  out->partial = (double*)ws + 1;
  return D3PM_OK;
}
static int run_count(const uint8_t* mask, int N, int* count, hipStream_t s) {
  hipLaunchKernelGGL(k_count, dim3(1), dim3(SUM_WG), 0, s, mask, N, count);
  D3PM_LAUNCH_CHECK("k_count");
  return D3PM_OK;
}
static int run_finish(const double* partial, int n, const int* count, double inv_count, float scale, float* loss,
                      hipStream_t s) {
  hipLaunchKernelGGL(k_finish, dim3(1), dim3(SUM_WG), 0, s, partial, n, count, inv_count, scale, loss);
  D3PM_LAUNCH_CHECK("k_finish");
  return D3PM_OK;
}

// the part that the distillation and the policy loss share: count, pass over the rows, loss
template <bool DISTILL>
static int run_mean_loss(RowArgs& a, int dtype, float out_scale, float* loss, const float* upstream,
                         int only_if_rescaled, void* ws, size_t ws_bytes, hipStream_t s) {
  Scratch sc;
  if (int rc = scratch(ws, ws_bytes, MAX_PARTIALS, &sc)) return rc;
  const double inv = 1.0 / (double)std::max(a.N, 1);
  a.inv_count = (float)inv;
  a.upstream = upstream;
  a.only_if_rescaled = upstream ? only_if_rescaled : 0;
  int grid = 0;
  if (a.N > 0) {
    if (a.mask) {
      a.count = sc.count;                              // a gradient alone finds it as the loss call left it
      a.count_here = loss && a.N <= COUNT_HERE;
      if (loss && !a.count_here)
        if (int rc = run_count(a.mask, a.N, sc.count, s)) return rc;
    }
    a.partial = loss ? sc.partial : nullptr;
    a.loss = loss;
    a.out_scale = out_scale;
    if (int rc = run_rows<DISTILL>(a, dtype, &grid, s)) return rc;
  }
  if (!loss || grid == 1) return D3PM_OK;
  return run_finish(sc.partial, grid, a.count, inv, out_scale, loss, s);
}

}  // namespace ft
}  // namespace d3pm

using namespace d3pm;
using namespace d3pm::ft;

extern "C" size_t d3pm_objective_workspace(long B, long L) {
  (void)L;
  return 8 + 8 * (size_t)std::max<long>(MAX_PARTIALS, B);
}

extern "C" int d3pm_token_logprobs(const d3pm_logits* z, const void* tokens, int tok_bytes, const uint8_t* mask,
                                   float temperature, float* logprobs, float* row_stats, void* stream) {
  const char* who = "d3pm_token_logprobs";
  if (int rc = check_logits(z, who)) return rc;
  if (int rc = check_temperature(temperature, who)) return rc;
  if (int rc = check_int_bytes(tok_bytes, "tokens", who)) return rc;
  if (z->B * z->L == 0) return D3PM_OK;
  D3PM_CHECK_ARG(tokens && logprobs, "%s: null pointer", who);
  RowArgs a = row_args(z, temperature);
  a.head = HEAD_LOGPROB;
  a.tokens = tokens; a.tok_bytes = tok_bytes; a.mask = mask;
  a.per_row = logprobs; a.stats = (float4*)row_stats;
  int grid;
  return run_rows<false>(a, z->dtype, &grid, (hipStream_t)stream);
}

extern "C" int d3pm_token_grad(const d3pm_logits* z, const void* tokens, int tok_bytes, float temperature,
                               const float* row_stats, const float* upstream, int upstream_per_row,
                               int only_if_rescaled, void* dlogits, void* stream) {
  const char* who = "d3pm_token_grad";
  if (int rc = check_logits(z, who)) return rc;
  if (int rc = check_temperature(temperature, who)) return rc;
  if (int rc = check_int_bytes(tok_bytes, "tokens", who)) return rc;
  D3PM_CHECK_ARG(!only_if_rescaled || (upstream && !upstream_per_row), "%s: only_if_rescaled needs one upstream gradient", who);
  if (z->B * z->L == 0) return D3PM_OK;
  D3PM_CHECK_ARG(tokens && row_stats && dlogits, "%s: null pointer", who);
  return run_grad(z, tokens, tok_bytes, temperature, row_stats, upstream, upstream_per_row ? 1 : 0, only_if_rescaled,
                  dlogits, (hipStream_t)stream);
}

extern "C" int d3pm_topk_distill_loss(const d3pm_logits* z, const void* teacher_logits, int teacher_dtype,
                                      const void* teacher_index, int index_bytes, int k, const uint8_t* mask,
                                      float temperature, float out_scale, const float* upstream, int only_if_rescaled,
                                      float* loss, float* per_token, void* dlogits, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const char* who = "d3pm_topk_distill_loss";
  if (int rc = check_logits(z, who)) return rc;
  if (int rc = check_temperature(temperature, who)) return rc;
  if (int rc = check_int_bytes(index_bytes, "teacher_index", who)) return rc;
  D3PM_CHECK_ARG(teacher_dtype >= D3PM_F32 && teacher_dtype <= D3PM_BF16, "%s: teacher dtype %d", who, teacher_dtype);
  D3PM_CHECK_ARG(k >= 1 && k <= MAX_K, "%s: k = %d entries, need 1 .. %d", who, k, MAX_K);
  D3PM_CHECK_ARG(z->B * z->L == 0 || (teacher_logits && teacher_index), "%s: null teacher", who);
  D3PM_CHECK_ARG(std::isfinite(out_scale), "%s: out_scale is not finite", who);
  RowArgs a = row_args(z, temperature);
  a.mask = mask;
  a.t_logits = teacher_logits; a.t_dtype = teacher_dtype;
  a.t_index = teacher_index; a.t_index_bytes = index_bytes; a.k = k;
  a.weight = out_scale * temperature;
  a.per_row = per_token; a.dz = dlogits;
  return run_mean_loss<true>(a, z->dtype, out_scale, loss, upstream, only_if_rescaled, workspace, workspace_bytes,
                             (hipStream_t)stream);
}

extern "C" int d3pm_policy_loss(const d3pm_logits* z, const void* tokens, int tok_bytes, const float* old_logprobs,
                                const float* advantages, int advantages_per_sequence, const float* ref_logprobs,
                                const uint8_t* mask, float temperature, float clip_low, float clip_high,
                                float kl_coeff, float out_scale, const float* upstream, int only_if_rescaled,
                                float* loss, float* logprobs, void* dlogits, void* workspace, size_t workspace_bytes,
                                void* stream) {
  const char* who = "d3pm_policy_loss";
  if (int rc = check_logits(z, who)) return rc;
  if (int rc = check_temperature(temperature, who)) return rc;
  if (int rc = check_int_bytes(tok_bytes, "tokens", who)) return rc;
  D3PM_CHECK_ARG(clip_low >= 0.0f && clip_low <= 1.0f && clip_high >= 0.0f, "%s: clip range [1 - %g, 1 + %g]", who,
                 (double)clip_low, (double)clip_high);
  D3PM_CHECK_ARG(std::isfinite(kl_coeff) && std::isfinite(out_scale), "%s: kl_coeff or out_scale is not finite", who);
  D3PM_CHECK_ARG(z->B * z->L == 0 || (tokens && old_logprobs && advantages), "%s: null pointer", who);
  D3PM_CHECK_ARG(kl_coeff == 0.0f || ref_logprobs || z->B * z->L == 0, "%s: kl_coeff without ref_logprobs", who);
  RowArgs a = row_args(z, temperature);
  a.head = HEAD_POLICY;
  a.tokens = tokens; a.tok_bytes = tok_bytes; a.mask = mask;
  a.old_lp = old_logprobs; a.adv = advantages; a.adv_per_seq = advantages_per_sequence ? 1 : 0;
  a.ref_lp = kl_coeff == 0.0f ? nullptr : ref_logprobs;
  a.clip_lo = 1.0f - clip_low; a.clip_hi = 1.0f + clip_high; a.kl_coeff = kl_coeff;
  a.weight = out_scale / temperature;
  a.per_row = logprobs; a.dz = dlogits;
  return run_mean_loss<false>(a, z->dtype, out_scale, loss, upstream, only_if_rescaled, workspace, workspace_bytes,
                              (hipStream_t)stream);
}

extern "C" int d3pm_preference_loss(const d3pm_logits* z, const void* tokens, int tok_bytes, const float* ref_logprobs,
                                    const uint8_t* mask, float beta, float label_smoothing, int average,
                                    float out_scale, float* loss, float* rewards, float* row_stats, void* dlogits,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "d3pm_preference_loss";
  if (int rc = check_logits(z, who)) return rc;
  if (int rc = check_int_bytes(tok_bytes, "tokens", who)) return rc;
  D3PM_CHECK_ARG(z->B >= 2 && z->B % 2 == 0, "%s: B = %ld sequences, need pairs", who, z->B);
  D3PM_CHECK_ARG(std::isfinite(beta) && std::isfinite(out_scale), "%s: beta or out_scale is not finite", who);
  D3PM_CHECK_ARG(label_smoothing >= 0.0f && label_smoothing <= 1.0f, "%s: label_smoothing %g", who, (double)label_smoothing);
  D3PM_CHECK_ARG(loss && rewards, "%s: null output", who);
  D3PM_CHECK_ARG(z->L == 0 || (tokens && row_stats), "%s: null pointer", who);
  const int P = (int)(z->B / 2);
  Scratch sc;
  if (int rc = scratch(workspace, workspace_bytes, P, &sc)) return rc;
  hipStream_t s = (hipStream_t)stream;
  PairArgs a{};
  a.r = row_args(z, 1.0f);
  a.r.head = HEAD_PREFERENCE;
  a.r.tokens = tokens; a.r.tok_bytes = tok_bytes; a.r.mask = mask;
  a.r.stats = (float4*)row_stats;
  a.ref = ref_logprobs;
  a.P = P; a.beta = beta; a.smooth = label_smoothing; a.average = average; a.out_scale = out_scale;
  a.rewards = rewards; a.pair_loss = sc.partial; a.loss = P == 1 ? loss : nullptr;
  const int size = z->dtype == D3PM_F32 ? 4 : 2;
  const long width = (long)a.r.V * size;
  const bool one = width <= 4096 && 2 * z->L <= PAIR_SWEEPS * (PAIR_WG / pair_lanes((int)width / 16)) &&
                   2 * z->L * width <= PAIR_BYTES;
  if (one) {
    a.r.dz = dlogits;
    const int rc = z->dtype == D3PM_F32 ? dispatch_pairs<F32>(a, s)
                 : z->dtype == D3PM_F16 ? dispatch_pairs<F16>(a, s) : dispatch_pairs<BF16>(a, s);
    if (rc) return rc;
  } else {
    if (a.r.N > 0) {
      int grid;
      if (int rc = run_rows<false>(a.r, z->dtype, &grid, s)) return rc;
    }
    hipLaunchKernelGGL(k_pair, dim3(P), dim3(PAIR_WG), 0, s, a);
    D3PM_LAUNCH_CHECK("k_pair");
  }
  if (P > 1)
    if (int rc = run_finish(sc.partial, P, nullptr, 1.0 / (double)P, out_scale, loss, s)) return rc;
  if (one || !dlogits || a.r.N == 0) return D3PM_OK;
  return run_grad(z, tokens, tok_bytes, 1.0f, row_stats, nullptr, 0, 0, dlogits, s);
}
