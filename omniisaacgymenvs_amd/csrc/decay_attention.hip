// Linear attention with one decay per head, for gfx950 (MI355X): whole sequences (forward, backward) and single steps.
//
//   S_t = a_t S_{t-1} + k_t v_t^T     a_t = decay_h, 0 where a reset flags token t        S: dk x dv, fp32
//   o_t = scale S_t^T q_t
// backward, with G_t the gradient of S_t:
//   dq_t = scale S_t do_t        G_t = scale q_t do_t^T + a_{t+1} G_{t+1}  (+ the final state's gradient at the last token)
//   dk_t = G_t v_t               dv_t = G_t^T k_t                            dS_0 = a_0 G_0
// so the backward pass is the forward recurrence with exchanged roles: dq reads (do, v, k) over S^T, dv reads (k, q, do) over G and
// dk reads (v, do, q) over G^T, the last two from the last token to the first.  One kernel serves all four.
//
// A wave owns one sequence, one head and 16 NV columns of the state, which it keeps in registers as the accumulator tiles of
// v_mfma_f32_16x16x4_f32 while it walks the tokens in blocks of 16:
//   P  = (Q K^T) o decay^(i-j)                  16 x 16, only j <= i with no reset in (j, i]
//   O  = P V + decay^(i+1) Q S
//   S <- decay^16 S + (decay^(15-j) K)^T V
// Every product is a 32-bit matrix instruction on operands widened from the tensors' type, so no intermediate is rounded to
// fewer bits.  The transposed forms are taken (P^T = K Q^T, O^T = V^T P^T + S^T Q^T): P^T and S then come out of one product in the very
// register layout the next one takes them in, and nothing goes through LDS.  The order of the dk (dv) columns over tiles is
// the kernel's own: tile s, row m holds dk = NK m + s, so that every lane's operand elements are neighbours in memory.
#include "oige_elem.hpp"

namespace oige {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int DA_TOKENS = 16;   // tokens per block
constexpr int DA_MAX_DIM = 128; // head sizes
constexpr int DA_WAVES = 4;     // waves per workgroup: neighbouring heads or column slices, whose rows are neighbours in memory

// One operand: rows of a (N, T, heads, d) tensor, in elements; `group` query heads share one of its heads.
struct DaRows {
  const void* p;
  int64_t sn, st, sh;
  int group;
};

struct DaCore {
  DaRows q, k, v;  // q, k: rows of dk elements; v: rows of dv elements
  void* o;         // rows of dv elements, per query head
  int64_t on, ot, oh;
  const float* s_in;   // NULL: zero
  float* s_out;        // NULL: not wanted
  float* seg_states;   // states between time segments, in register order
  float* seg_factors;  // (N, H, nseg): what a segment multiplies the state with, -1: it drops it
  const float* decay;
  const void* resets;
  const void* lengths;
  int64_t rsn, rst;  // element strides of resets
  int64_t n, t, seg_len;
  float out_scale, kv_scale;
  int h, dk, dv, slices, nseg;
  int resets_bytes, lengths_bytes;
  int reverse;     // walk from the last token to the first; the first one taken in is not preceded by a decay, the state is multiplied once more at the end
  int transposed;  // the states in memory are (N, H, dv, dk)
  int o_float;     // o is fp32 whatever T is
};

__device__ __forceinline__ int64_t da_length(const DaCore& c, int64_t n) {
  if (!c.lengths) return c.t;
  const int64_t l = c.lengths_bytes == 8 ? static_cast<const int64_t*>(c.lengths)[n] : static_cast<const int32_t*>(c.lengths)[n];
  return l < 0 ? 0 : (l > c.t ? c.t : l);
}

__device__ __forceinline__ bool da_reset(const DaCore& c, int64_t n, int64_t t) {
  const int64_t i = n * c.rsn + t * c.rst;
  return c.resets_bytes == 8 ? static_cast<const int64_t*>(c.resets)[i] != 0 : static_cast<const uint8_t*>(c.resets)[i] != 0;
}

// decay^n.  Products of squares in 64 bits: exact where the result is used in 32, also for decays of 0 and above 1.
__device__ __forceinline__ double da_power(double decay, int64_t n) {
  double r = 1.0, sq = decay;
  for (; n > 0; n >>= 1) {
    if (n & 1) r *= sq;
    sq *= sq;
  }
  return r;
}
struct DaPowers {  // decay^n for n in 0 .. 16 without a loop, within 4 roundings
  float p1, p2, p4, p8, p16;
  __device__ __forceinline__ explicit DaPowers(double d) : p1((float)d), p2((float)(d * d)) {
    const double d4 = (d * d) * (d * d);
    p4 = (float)d4;
    p8 = (float)(d4 * d4);
    p16 = (float)((d4 * d4) * (d4 * d4));
  }
  __device__ __forceinline__ float operator()(int n) const {
    float r = (n & 1) ? p1 : 1.f;
    r *= (n & 2) ? p2 : 1.f;
    r *= (n & 4) ? p4 : 1.f;
    r *= (n & 8) ? p8 : 1.f;
    return (n & 16) ? p16 : r;
  }
};

// This wave's piece of a state matrix in memory: tile (s, sv), register r, lane (c, g) holds dk = NK (4 g + r) + s,
// dv = dv0 + NV c + sv.
template <int NK, int NV, int MODE>
__device__ __forceinline__ void da_load_state(f32x4 (&S)[NK][NV], const float* p, const DaCore& a, int dv0, int c, int g) {
  if (a.transposed) {
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) {
      const int d = dv0 + NV * c + sv;
      float x[4 * NK];
      load_run<float, 4 * NK, MODE>(x, p + (int64_t)(d < a.dv ? d : 0) * a.dk, 4 * NK * g, d < a.dv ? a.dk : 0);
#pragma unroll
      for (int s = 0; s < NK; ++s) S[s][sv] = f32x4{x[s], x[NK + s], x[2 * NK + s], x[3 * NK + s]};
    }
    asm volatile("" ::: "memory");  // keeps the two branches' ends apart: merged, they address S's tiles, which then leave the registers
  } else {
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      float x[4][NV];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = NK * (4 * g + r) + s;
        load_run<float, NV, MODE>(x[r], p + (int64_t)(d < a.dk ? d : 0) * a.dv, dv0 + NV * c, d < a.dk ? a.dv : 0);
      }
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) S[s][sv] = f32x4{x[0][sv], x[1][sv], x[2][sv], x[3][sv]};
    }
  }
}

template <int NK, int NV, int MODE>
__device__ __forceinline__ void da_store_state(const f32x4 (&S)[NK][NV], float* p, const DaCore& a, int dv0, int c, int g) {
  if (a.transposed) {
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) {
      const int d = dv0 + NV * c + sv;
      float x[4 * NK];
#pragma unroll
      for (int s = 0; s < NK; ++s) {
        x[s] = S[s][sv].x;
        x[NK + s] = S[s][sv].y;
        x[2 * NK + s] = S[s][sv].z;
        x[3 * NK + s] = S[s][sv].w;
      }
      if (d < a.dv) store_run<float, 4 * NK, MODE>(x, p + (int64_t)d * a.dk, 4 * NK * g, a.dk);
    }
  } else {
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      float x[4][NV];
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) {
        x[0][sv] = S[s][sv].x;
        x[1][sv] = S[s][sv].y;
        x[2][sv] = S[s][sv].z;
        x[3][sv] = S[s][sv].w;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = NK * (4 * g + r) + s;
        if (d < a.dk) store_run<float, NV, MODE>(x[r], p + (int64_t)d * a.dv, dv0 + NV * c, a.dv);
      }
    }
  }
}

// O^T's part from the state in front of the block: S^T Q^T, weighted; nothing where a reset lies between.
template <int NK, int NV>
__device__ __forceinline__ void da_state_part(f32x4 (&acc)[NV], const f32x4 (&S)[NK][NV], const float (&Q)[4 * NK], bool from_state, float head_w) {
#pragma unroll
  for (int sv = 0; sv < NV; ++sv) acc[sv] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < NK; ++s) {
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) acc[sv] = __builtin_amdgcn_mfma_f32_16x16x4f32(S[s][sv].x, Q[s], acc[sv], 0, 0, 0);
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) acc[sv] = __builtin_amdgcn_mfma_f32_16x16x4f32(S[s][sv].y, Q[NK + s], acc[sv], 0, 0, 0);
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) acc[sv] = __builtin_amdgcn_mfma_f32_16x16x4f32(S[s][sv].z, Q[2 * NK + s], acc[sv], 0, 0, 0);
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) acc[sv] = __builtin_amdgcn_mfma_f32_16x16x4f32(S[s][sv].w, Q[3 * NK + s], acc[sv], 0, 0, 0);
  }
  const f32x4 zero{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int sv = 0; sv < NV; ++sv) acc[sv] = from_state ? acc[sv] * head_w : zero;
}

// No conditional block stands between a matrix instruction and the first ordinary one that reads its result: with one, the
// compiler has counted the wait states of the longer way only, and the shorter way read the registers too early.
// da_settle() stands where the state's tiles leave the loop.
__device__ __forceinline__ void da_settle() { asm volatile("s_nop 15" ::: "memory"); }

// One block's rows of the operands.  Rows behind the block's L tokens re-read its last one; `low` is the earliest of its tokens
// in memory, and in reverse the block's first token is the latest.
struct DaBlock {
  int64_t low;
  int L, reverse;
  __device__ __forceinline__ int row(int i) const {
    const int r = i < L ? i : L - 1;
    return reverse ? L - 1 - r : r;
  }
  template <typename T>
  __device__ __forceinline__ const T* at(const T* head, int64_t st, int i) const {  // row * stride in 32 x 32 bits: checked on the host
    return head + low * st + (uint64_t)(uint32_t)row(i) * (uint32_t)st;
  }
};
__device__ __forceinline__ DaBlock da_block(const DaCore& a, int64_t p0, int64_t end, int64_t len) {
  DaBlock b;
  b.L = end - p0 < DA_TOKENS ? (int)(end - p0) : DA_TOKENS;
  b.reverse = a.reverse;
  b.low = a.reverse ? len - p0 - b.L : p0;
  return b;
}

// STATES: only the states at the segments' ends (no q, no o), for sequences cut over time.
//
// The next block's rows are asked for as soon as the registers of this block's are free: q and the first copy of k behind the
// products that read them, the other copy and v at the end, so that their way from memory runs beside the matrix instructions.
template <typename T, int NK, int NV, int MODE, bool STATES>
__global__ __launch_bounds__(DA_WAVES* WAVE, 2) void decay_attention_kernel(const DaCore a) {
  const int lane = lane_id(), c = lane & 15, g = lane >> 4;
  const int64_t u = (int64_t)blockIdx.x * DA_WAVES + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int64_t units = a.n * a.h * a.slices;
  if (u >= units) return;
  const int seg = blockIdx.y;
  const int slice = (int)(u % a.slices);
  const int64_t nh = u / a.slices;
  const int h = (int)(nh % a.h);
  const int64_t n = nh / a.h;
  const int dv0 = slice * 16 * NV;
  const int64_t len = da_length(a, n);
  const int64_t begin = (int64_t)seg * a.seg_len;
  int64_t end = begin + a.seg_len;
  if (end > len) end = len;

  const T* qh = static_cast<const T*>(a.q.p) + n * a.q.sn + (int64_t)(h / a.q.group) * a.q.sh;
  const T* kh = static_cast<const T*>(a.k.p) + n * a.k.sn + (int64_t)(h / a.k.group) * a.k.sh;
  const T* vh = static_cast<const T*>(a.v.p) + n * a.v.sn + (int64_t)(h / a.v.group) * a.v.sh;

  Run<T, 4 * NK, MODE> q_run, k1_run;
  Run<T, NK, MODE> k2_run[4];
  Run<T, NV, MODE> v_run[4];
  bool flag = false;
  auto issue_rows = [&](const DaBlock& b) {
    if (!STATES) {
      q_run.issue(b.at(qh, a.q.st, c), 4 * NK * g, a.dk);
      k1_run.issue(b.at(kh, a.k.st, c), 4 * NK * g, a.dk);
    }
  };
  auto issue_columns = [&](const DaBlock& b, bool not_first) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v_run[r].issue(b.at(vh, a.v.st, 4 * g + r), dv0 + NV * c, a.dv);
      k2_run[r].issue(b.at(kh, a.k.st, 4 * g + r), NK * c, a.dk);
    }
    if (a.resets) flag = (not_first || !b.reverse || c > 0) && c < b.L && da_reset(a, n, b.low + b.row(c) + b.reverse);
  };

  DaBlock blk = da_block(a, begin, end, len);
  if (begin < end) {
    issue_rows(blk);
    issue_columns(blk, begin > 0);
  }

  f32x4 S[NK][NV];
  const f32x4 zero{0.f, 0.f, 0.f, 0.f};
  constexpr int UNIT = NK * NV * 4 * WAVE;  // floats of a wave's state
  float* seg_slot = a.seg_states + ((nh * a.nseg + seg) * a.slices + slice) * (int64_t)UNIT;
  if (seg > 0 && !STATES) {
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) S[s][sv] = *reinterpret_cast<const f32x4*>(seg_slot + ((s * NV + sv) * WAVE + lane) * 4);
  } else if (seg == 0 && a.s_in) {
    da_load_state<NK, NV, MODE>(S, a.s_in + nh * a.dk * a.dv, a, dv0, c, g);
  } else {
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) S[s][sv] = zero;
  }

  const double decay = (double)a.decay[h];
  const DaPowers pw(decay);
  bool dropped = false;  // a reset inside the segment
  float head_w = 0.f, pair_w[4], tail_w[4], keep_hi = 0.f, keep_lo = 0.f;
  const uint32_t upto = (2u << c) - 1u;  // bits 0 .. i

  for (int64_t p0 = begin; p0 < end; p0 += DA_TOKENS) {
    const int L = blk.L;
    if (p0 == begin || p0 == DA_TOKENS || L < DA_TOKENS) {
      const int first = a.reverse && p0 == 0 ? 1 : 0;  // the first token in reverse: nothing decays in front of it
      const double keep = da_power(decay, L - first);
      keep_hi = (float)keep;
      keep_lo = (float)(keep - (double)keep_hi);  // the rounding of decay^16 would pile up over a long memory
      head_w = pw(c + 1 - first);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * g + r;
        pair_w[r] = j <= c ? pw(c - j) * a.kv_scale : 0.f;
        tail_w[r] = j < L ? pw(L - 1 - j) * a.kv_scale : 0.f;
      }
    }
    const uint32_t m = (uint32_t)(__ballot(flag) & 0xFFFFull);  // bit i: a reset in front of the block's token i
    const bool more = p0 + DA_TOKENS < end;
    const DaBlock next = da_block(a, more ? p0 + DA_TOKENS : p0, end, len);  // behind the last block: the same rows once more

    float P[4];
    f32x4 acc[NV];
    float Q[4 * NK];
    const bool from_state = !(m & upto);
    if (!STATES) {
      float K1[4 * NK];
      q_run.take(Q, 4 * NK * g, a.dk);
      k1_run.take(K1, 4 * NK * g, a.dk);
      f32x4 pt = zero;
#pragma unroll
      for (int e = 0; e < 4 * NK; ++e) pt = __builtin_amdgcn_mfma_f32_16x16x4f32(K1[e], Q[e], pt, 0, 0, 0);
      const float p4[4] = {pt.x, pt.y, pt.z, pt.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * g + r;
        const bool sees = j <= c && !(m & upto & ~((2u << j) - 1u));
        P[r] = sees ? p4[r] * pair_w[r] : 0.f;  // a masked product may be infinite or NaN: selected away, not multiplied
      }
      da_state_part<NK, NV>(acc, S, Q, from_state, head_w);
    }
    float V[4][NV], K2[4][NK];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v_run[r].take(V[r], dv0 + NV * c, a.dv);
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) V[r][sv] = 4 * g + r < L ? V[r][sv] : 0.f;
    }
    if (!STATES) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) acc[sv] = __builtin_amdgcn_mfma_f32_16x16x4f32(V[r][sv], P[r], acc[sv], 0, 0, 0);
      // An infinite or NaN value in a row that some tokens must not see has met their zero weights in the product.  Such blocks
      // (any output not finite) are summed again pair by pair.
      f32x4 z = zero;
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) z += acc[sv] * 0.f;
      const float z1 = (z.x + z.y) + (z.z + z.w);
      if (__any(c < L && z1 != z1)) {
        da_state_part<NK, NV>(acc, S, Q, from_state, head_w);
#pragma unroll 1
        for (int gj = 0; gj < 4; ++gj) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 4 * gj + r, at = gj * 16 + 4 * g;
            const float w = __shfl(P[r], gj * 16 + c, WAVE);
            const bool sees = j <= c && !(m & upto & ~((2u << j) - 1u));
#pragma unroll
            for (int sv = 0; sv < NV; ++sv) {
              const f32x4 v{__shfl(V[r][sv], at, WAVE), __shfl(V[r][sv], at + 1, WAVE), __shfl(V[r][sv], at + 2, WAVE), __shfl(V[r][sv], at + 3, WAVE)};
              acc[sv] = sees ? acc[sv] + v * w : acc[sv];
            }
          }
        }
      }
      issue_rows(next);
      if (c < L) {
        float out[4 * NV];
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) {
          out[sv] = acc[sv].x * a.out_scale;
          out[NV + sv] = acc[sv].y * a.out_scale;
          out[2 * NV + sv] = acc[sv].z * a.out_scale;
          out[3 * NV + sv] = acc[sv].w * a.out_scale;
        }
        const int64_t row = n * a.on + (blk.low + blk.row(c)) * a.ot + (int64_t)h * a.oh;
        if (a.o_float) store_run<float, 4 * NV, MODE>(out, static_cast<float*>(a.o) + row, dv0 + 4 * NV * g, a.dv);
        else store_run<T, 4 * NV, MODE>(out, static_cast<T*>(a.o) + row, dv0 + 4 * NV * g, a.dv);
      }
    }

    // the state behind the block: rows in front of its last reset, and behind the end, stay out of the sum altogether
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool in = 4 * g + r < L && !(m & ~((2u << (4 * g + r)) - 1u));
      k2_run[r].take(K2[r], NK * c, a.dk);
#pragma unroll
      for (int s = 0; s < NK; ++s) K2[r][s] = in ? K2[r][s] : 0.f;
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) V[r][sv] = in ? V[r][sv] * tail_w[r] : 0.f;
    }
    dropped |= m != 0;
    issue_columns(next, true);
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) {
        S[s][sv] = m ? zero : __builtin_elementwise_fma(S[s][sv], f32x4(keep_hi), S[s][sv] * keep_lo);
#pragma unroll
        for (int r = 0; r < 4; ++r) S[s][sv] = __builtin_amdgcn_mfma_f32_16x16x4f32(K2[r][s], V[r][sv], S[s][sv], 0, 0, 0);
      }
    da_settle();
    blk = next;
  }

  if (STATES) {
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) *reinterpret_cast<f32x4*>(seg_slot + ((s * NV + sv) * WAVE + lane) * 4) = S[s][sv];
    if (slice == 0 && lane == 0) {
      const int64_t count = (end > begin ? end - begin : 0) - (a.reverse && seg == 0 && end > 0 ? 1 : 0);
      a.seg_factors[nh * a.nseg + seg] = dropped ? -1.f : (float)da_power(decay, count);
    }
    return;
  }
  // rows behind the sequence's end inside this segment's stretch of the tensor
  const int64_t stop = begin + a.seg_len < a.t ? begin + a.seg_len : a.t;
  for (int64_t t = (begin > len ? begin : len) + c; t < stop; t += 16) {
    const int64_t row = n * a.on + t * a.ot + (int64_t)h * a.oh;
    const float none[4 * NV] = {};
    if (a.o_float) store_run<float, 4 * NV, MODE>(none, static_cast<float*>(a.o) + row, dv0 + 4 * NV * g, a.dv);
    else store_run<T, 4 * NV, MODE>(none, static_cast<T*>(a.o) + row, dv0 + 4 * NV * g, a.dv);
  }
  if (a.s_out && seg == a.nseg - 1) {
    if (a.reverse && len > 0) {  // dS_0 = a_0 G_0
      const bool drop = a.resets && da_reset(a, n, 0);
#pragma unroll
      for (int s = 0; s < NK; ++s)
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) S[s][sv] = drop ? zero : S[s][sv] * (float)decay;
    }
    da_store_state<NK, NV, MODE>(S, a.s_out + nh * a.dk * a.dv, a, dv0, c, g);
  }
}

// The states in front of every segment from those at the segments' ends (in place, register order): carry = factor carry + end.
// Segment 0's end already holds the initial state.  A thread owns four floats of one (sequence, head) over all segments.
__global__ __launch_bounds__(256) void decay_attention_join_kernel(float* __restrict__ states, const float* __restrict__ factors,
                                                                   int64_t quads, int64_t per_head, int nseg) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  const int64_t nh = i / per_head, e = i % per_head;
  f32x4* s = reinterpret_cast<f32x4*>(states) + nh * nseg * per_head + e;
  f32x4 carry = s[0];
  constexpr int U = 8;  // ends in flight (they do not depend on the carry, but lie where it goes)
  for (int seg0 = 1; seg0 < nseg; seg0 += U) {
    f32x4 end[U];
    float f[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int seg = seg0 + i < nseg - 1 ? seg0 + i : nseg - 2;  // (the last segment's own end is nobody's start)
      end[i] = s[seg * per_head];
      f[i] = factors[nh * nseg + seg];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (seg0 + i >= nseg) break;
      s[(seg0 + i) * per_head] = carry;
      carry = f[i] < 0.f ? end[i] : __builtin_elementwise_fma(carry, f32x4(f[i]), end[i]);
    }
  }
}

// Gradients of shared key / value heads: the sum over the query heads that share one, from fp32 rows (N, T, H, d) -> T.
template <typename T>
__global__ __launch_bounds__(256) void decay_attention_share_kernel(const float* __restrict__ in, T* __restrict__ out, int64_t n, int64_t t,
                                                                    int hk, int group, int d, int64_t on, int64_t ot, int64_t oh) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * t * hk * d) return;
  const int e = (int)(i % d);
  const int64_t r = i / d;  // (n, t, hk)
  const int head = (int)(r % hk);
  const int64_t nt = r / hk;
  float v = 0.f;
  for (int k = 0; k < group; ++k) v += in[((r * group) + k) * d + e];
  out[(nt / t) * on + (nt % t) * ot + head * oh + e] = (T)v;
}

// ---------------------------------------------------------------- one token per sequence, the state updated in place
// Bound by the state's one read and one write (8 bytes per entry).  A wave (or a workgroup of four, for states of more than
// 8 KiB) owns one (sequence, head): lanes take 16-byte pieces of the state's rows, update them where they are and add
// q's product up over the rows they hold, then over the lanes and waves that share a column.
struct DaStep {
  const void *q, *k, *v;
  void* o;
  float* state;
  const float* decay;
  const void* resets;
  int64_t n, rsn;
  int64_t qn, qh, kn, kh, vn, vh;
  float scale;
  int h, group, dk, dv, resets_bytes;
  int lanes;  // lanes per state row
};

template <typename T, int VEC, int WAVES>
__global__ __launch_bounds__(256) void decay_attention_step_kernel(const DaStep a) {
  constexpr int UNITS = 4 / WAVES, THREADS = WAVES * WAVE;
  __shared__ float rows[UNITS][3][DA_MAX_DIM];
  __shared__ float part[UNITS][WAVES][DA_MAX_DIM];
  const int unit = threadIdx.x / THREADS, tid = threadIdx.x % THREADS;
  const int64_t nh_raw = (int64_t)blockIdx.x * UNITS + unit;
  const bool live = nh_raw < a.n * a.h;
  const int64_t nh = live ? nh_raw : a.n * a.h - 1;
  const int h = (int)(nh % a.h);
  const int64_t n = nh / a.h;
  bool reset = false;
  if (a.resets) reset = a.resets_bytes == 8 ? static_cast<const int64_t*>(a.resets)[n * a.rsn] != 0 : static_cast<const uint8_t*>(a.resets)[n * a.rsn] != 0;
  const float decay = a.decay[h];
  const T* q = static_cast<const T*>(a.q) + n * a.qn + h * a.qh;
  const T* k = static_cast<const T*>(a.k) + n * a.kn + (int64_t)(h / a.group) * a.kh;
  const T* v = static_cast<const T*>(a.v) + n * a.vn + (int64_t)(h / a.group) * a.vh;
  for (int i = tid; i < a.dk; i += THREADS) {
    rows[unit][0][i] = (float)q[i] * a.scale;
    rows[unit][1][i] = (float)k[i];
  }
  for (int i = tid; i < a.dv; i += THREADS) rows[unit][2][i] = (float)v[i];
  __syncthreads();
  float* state = a.state + nh * a.dk * a.dv;
  const int rl = tid & (a.lanes - 1), r0 = tid / a.lanes, step = THREADS / a.lanes;
  for (int col0 = 0; col0 < a.dv; col0 += a.lanes * VEC) {
    const int col = col0 + rl * VEC;
    const bool in = col < a.dv;
    float vv[VEC], acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      vv[e] = in ? rows[unit][2][col + e] : 0.f;
      acc[e] = 0.f;
    }
    if (in && live) {
      constexpr int U = 4;  // rows in flight
      for (int r = r0; r < a.dk; r += U * step) {
        Pack<float, VEC> s[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int row = r + i * step;
          s[i] = *reinterpret_cast<const Pack<float, VEC>*>(state + (row < a.dk ? row : r) * a.dv + col);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int row = r + i * step;
          if (row < a.dk) {
            const float kk = rows[unit][1][row], qq = rows[unit][0][row];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              s[i].v[e] = fmaf(kk, vv[e], reset ? 0.f : decay * s[i].v[e]);
              acc[e] = fmaf(qq, s[i].v[e], acc[e]);
            }
            *reinterpret_cast<Pack<float, VEC>*>(state + row * a.dv + col) = s[i];
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      for (int off = a.lanes; off < WAVE; off <<= 1) acc[e] += __shfl_xor(acc[e], off, WAVE);
      if (in && lane_id() < a.lanes) part[unit][tid >> 6][col + e] = acc[e];
    }
  }
  __syncthreads();
  if (!live) return;
  T* o = static_cast<T*>(a.o) + nh * a.dv;
  for (int i = tid; i < a.dv; i += THREADS) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += part[unit][w][i];
    o[i] = (T)s;
  }
}

// ---------------------------------------------------------------- host side
struct DaPlan {
  int nk, nv, slices, nseg;
  int64_t seg_len, seg_floats;  // scratch: states between segments and the segments' factors
};

// Tiles per wave: 16 NK rows cover dk, 16 NV columns are a slice of dv; at most 16 tiles (64 registers) of state.
// A call with fewer waves than the chip has SIMDs is cut over time, into pieces of 64 tokens at least: the pieces' end states first,
// joined by one small launch, then every piece by itself.
constexpr int64_t DA_FEW_WAVES = 1024, DA_WANT_WAVES = 2048, DA_MIN_SEGMENT = 64;

static DaPlan decay_attention_plan(int64_t n, int64_t t, int h, int dk, int dv) {
  DaPlan p;
  p.nk = dk <= 16 ? 1 : dk <= 32 ? 2 : dk <= 64 ? 4 : 8;
  p.nv = dv <= 16 ? 1 : (dv <= 32 || p.nk == 8) ? 2 : 4;
  p.slices = (dv + 16 * p.nv - 1) / (16 * p.nv);
  const int64_t waves = n * h * p.slices;
  p.nseg = 1;
  p.seg_len = t > 0 ? t : 1;
  if (waves < DA_FEW_WAVES && t >= 2 * DA_MIN_SEGMENT) {
    int64_t want = (DA_WANT_WAVES + waves - 1) / waves;
    if (want > t / DA_MIN_SEGMENT) want = t / DA_MIN_SEGMENT;
    p.seg_len = (t + want - 1) / want;
    p.seg_len = (p.seg_len + DA_TOKENS - 1) / DA_TOKENS * DA_TOKENS;
    p.nseg = (int)((t + p.seg_len - 1) / p.seg_len);
  }
  p.seg_floats = p.nseg > 1 ? n * h * p.nseg * (p.slices * (int64_t)(p.nk * p.nv * 4 * WAVE) + 4) : 0;
  return p;
}

template <typename T, int NK, int NV, int MODE>
static int decay_attention_run(DaCore c, const DaPlan& p, float* workspace, hipStream_t stream) {
  c.slices = p.slices;
  c.nseg = p.nseg;
  c.seg_len = p.seg_len;
  const int64_t units = c.n * c.h * p.slices, blocks = (units + DA_WAVES - 1) / DA_WAVES;
  const int64_t per_head = (int64_t)p.slices * NK * NV * WAVE;  // in 16-byte quads
  OIGE_REQUIRE(blocks < ((int64_t)1 << 31), "decay_attention: %lld sequences x heads are too many for one launch", (long long)(c.n * c.h));
  if (p.nseg > 1) {
    c.seg_states = workspace;
    c.seg_factors = workspace + c.n * c.h * p.nseg * per_head * 4;
    hipLaunchKernelGGL((decay_attention_kernel<T, NK, NV, MODE, true>), dim3((unsigned)blocks, (unsigned)(p.nseg - 1)), dim3(DA_WAVES * WAVE), 0,
                       stream, c);
    int rc = check_launch("decay_attention_kernel (states)");
    if (rc) return rc;
    const int64_t quads = c.n * c.h * per_head;
    hipLaunchKernelGGL(decay_attention_join_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, stream, c.seg_states, c.seg_factors,
                       quads, per_head, p.nseg);
    rc = check_launch("decay_attention_join_kernel");
    if (rc) return rc;
  }
  hipLaunchKernelGGL((decay_attention_kernel<T, NK, NV, MODE, false>), dim3((unsigned)blocks, (unsigned)p.nseg), dim3(DA_WAVES * WAVE), 0, stream, c);
  return check_launch("decay_attention_kernel");
}

template <typename T, int MODE>
static int decay_attention_tiles(const DaCore& c, const DaPlan& p, float* ws, hipStream_t s) {
  switch (p.nk * 8 + p.nv) {
    case 8 + 1: return decay_attention_run<T, 1, 1, MODE>(c, p, ws, s);
    case 8 + 2: return decay_attention_run<T, 1, 2, MODE>(c, p, ws, s);
    case 8 + 4: return decay_attention_run<T, 1, 4, MODE>(c, p, ws, s);
    case 16 + 1: return decay_attention_run<T, 2, 1, MODE>(c, p, ws, s);
    case 16 + 2: return decay_attention_run<T, 2, 2, MODE>(c, p, ws, s);
    case 16 + 4: return decay_attention_run<T, 2, 4, MODE>(c, p, ws, s);
    case 32 + 1: return decay_attention_run<T, 4, 1, MODE>(c, p, ws, s);
    case 32 + 2: return decay_attention_run<T, 4, 2, MODE>(c, p, ws, s);
    case 32 + 4: return decay_attention_run<T, 4, 4, MODE>(c, p, ws, s);
    case 64 + 1: return decay_attention_run<T, 8, 1, MODE>(c, p, ws, s);
    case 64 + 2: return decay_attention_run<T, 8, 2, MODE>(c, p, ws, s);
  }
  return fail(OIGE_EINVAL, "decay_attention: no variant for %d x %d tiles", p.nk, p.nv);
}

// 16-byte accesses: head sizes and strides in whole vectors, every pointer on a boundary.
static bool da_wide_rows(const DaRows& r, int bytes) {
  const int v = 16 / bytes;
  return aligned16(r.p) && r.sn % v == 0 && r.st % v == 0 && r.sh % v == 0;
}
static bool da_wide(const DaCore& c, int bytes) {
  const int v = 16 / bytes;
  return c.dk % v == 0 && c.dv % v == 0 && da_wide_rows(c.q, bytes) && da_wide_rows(c.k, bytes) && da_wide_rows(c.v, bytes) && aligned16(c.o) &&
         c.on % v == 0 && c.ot % v == 0 && c.oh % v == 0 && aligned16(c.s_in) && aligned16(c.s_out);
}

template <typename T>
static int decay_attention_typed(const DaCore& c, const DaPlan& p, float* ws, hipStream_t s) {
  if (!da_wide(c, sizeof(T))) return decay_attention_tiles<T, ELEMS_SINGLE>(c, p, ws, s);
  if (c.dk == 16 * p.nk && c.dv == 16 * p.nv * p.slices) return decay_attention_tiles<T, ELEMS_FULL>(c, p, ws, s);
  return decay_attention_tiles<T, ELEMS_WIDE>(c, p, ws, s);
}

static int decay_attention_core(const DaCore& c, int dtype, float* ws, hipStream_t s) {
  const int64_t most = (int64_t)1 << 32;
  OIGE_REQUIRE(c.q.st >= 0 && c.q.st < most && c.k.st >= 0 && c.k.st < most && c.v.st >= 0 && c.v.st < most,
               "decay_attention: token strides must be below 2^32 elements and not negative");
  const DaPlan p = decay_attention_plan(c.n, c.t, c.h, c.dk, c.dv);
  if (dtype == OIGE_F32) return decay_attention_typed<float>(c, p, ws, s);
  if (dtype == OIGE_F16) return decay_attention_typed<_Float16>(c, p, ws, s);
  return decay_attention_typed<__bf16>(c, p, ws, s);
}

static int decay_attention_share(const float* in, void* out, const oige_decay_attention_io& io, int d, const int64_t* stride, hipStream_t s) {
  const int64_t total = io.num_envs * io.num_tokens * io.kv_heads * d, blocks = (total + 255) / 256;
  OIGE_REQUIRE(blocks < ((int64_t)1 << 31), "decay_attention_backward: too many key / value rows for one launch");
  const int group = io.heads / io.kv_heads;
#define OIGE_SHARE(T)                                                                                                                        \
  hipLaunchKernelGGL((decay_attention_share_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, in, static_cast<T*>(out), io.num_envs,       \
                     io.num_tokens, (int)io.kv_heads, group, d, stride[0], stride[1], stride[2])
  if (io.dtype == OIGE_F32) OIGE_SHARE(float);
  else if (io.dtype == OIGE_F16) OIGE_SHARE(_Float16);
  else OIGE_SHARE(__bf16);
#undef OIGE_SHARE
  return check_launch("decay_attention_share_kernel");
}

static int decay_attention_check(const oige_decay_attention_io* io, const char* what) {
  OIGE_REQUIRE(io != nullptr, "%s: null io", what);
  OIGE_REQUIRE(elem_bytes(io->dtype), "%s: dtype must be OIGE_F32, OIGE_F16 or OIGE_BF16", what);
  OIGE_REQUIRE(io->num_envs >= 0 && io->num_tokens >= 0 && io->num_tokens < ((int64_t)1 << 31), "%s: %lld sequences of %lld tokens", what,
               (long long)io->num_envs, (long long)io->num_tokens);
  OIGE_REQUIRE(io->heads >= 1 && io->kv_heads >= 1 && io->heads % io->kv_heads == 0, "%s: %d heads over %d key / value heads", what, io->heads,
               io->kv_heads);
  OIGE_REQUIRE(io->key_dim >= 1 && io->key_dim <= DA_MAX_DIM && io->value_dim >= 1 && io->value_dim <= DA_MAX_DIM,
               "%s: head sizes %d and %d (1 .. %d)", what, io->key_dim, io->value_dim, DA_MAX_DIM);
  OIGE_REQUIRE(io->decay, "%s: null decay", what);
  OIGE_REQUIRE(!io->resets || io->resets_bytes == 1 || io->resets_bytes == 8, "%s: resets are bytes or int64", what);
  OIGE_REQUIRE(!io->lengths || io->lengths_bytes == 4 || io->lengths_bytes == 8, "%s: lengths are int32 or int64", what);
  return OIGE_OK;
}

static int64_t da_workspace(const oige_decay_attention_io& io, bool backward) {
  const int64_t n = io.num_envs, t = io.num_tokens;
  if (!backward) return decay_attention_plan(n, t, io.heads, io.key_dim, io.value_dim).seg_floats;
  const int64_t a = decay_attention_plan(n, t, io.heads, io.value_dim, io.key_dim).seg_floats;
  const int64_t b = decay_attention_plan(n, t, io.heads, io.key_dim, io.value_dim).seg_floats;
  int64_t most = (a > b ? a : b);
  most = (most + 3) / 4 * 4;
  const int64_t d = io.key_dim > io.value_dim ? io.key_dim : io.value_dim;
  return most + (io.heads != io.kv_heads ? n * t * io.heads * d : 0);  // per query head, dv and then dk
}

static DaCore da_core(const oige_decay_attention_io& io) {
  DaCore c{};
  c.decay = io.decay;
  c.resets = io.resets;
  c.lengths = io.lengths;
  c.rsn = io.resets_stride[0];
  c.rst = io.resets_stride[1];
  c.n = io.num_envs;
  c.t = io.num_tokens;
  c.h = io.heads;
  c.resets_bytes = io.resets_bytes;
  c.lengths_bytes = io.lengths_bytes;
  c.out_scale = c.kv_scale = 1.f;
  return c;
}
static DaRows da_rows(const void* p, const int64_t* s, int group) { return DaRows{p, s[0], s[1], s[2], group}; }
static void da_out(DaCore& c, void* p, const int64_t* s) {
  c.o = p;
  c.on = s[0];
  c.ot = s[1];
  c.oh = s[2];
}

}  // namespace oige

using namespace oige;

extern "C" {

int64_t oige_decay_attention_workspace_floats(const oige_decay_attention_io* io, int32_t backward) {
  const int rc = decay_attention_check(io, "decay_attention_workspace");
  return rc ? rc : da_workspace(*io, backward != 0);
}

int oige_decay_attention_forward(const oige_decay_attention_io* io, oige_stream_t stream) {
  const int rc = decay_attention_check(io, "decay_attention_forward");
  if (rc) return rc;
  if (io->num_envs == 0) return OIGE_OK;
  OIGE_REQUIRE(io->num_tokens == 0 || (io->q && io->k && io->v && io->o), "decay_attention_forward: null q, k, v or o");
  OIGE_REQUIRE(io->num_tokens > 0 || io->state_out, "decay_attention_forward: no tokens and no final state asked for");
  const int64_t need = da_workspace(*io, false);
  OIGE_REQUIRE(need == 0 || (io->workspace && aligned16(io->workspace) && io->workspace_floats >= need),
               "decay_attention_forward: needs a 16-byte aligned workspace of %lld floats", (long long)need);
  const int group = io->heads / io->kv_heads;
  DaCore c = da_core(*io);
  c.q = da_rows(io->q, io->q_stride, 1);
  c.k = da_rows(io->k, io->k_stride, group);
  c.v = da_rows(io->v, io->v_stride, group);
  da_out(c, io->o, io->o_stride);
  c.s_in = io->state_in;
  c.s_out = io->state_out;
  c.out_scale = io->scale;
  c.dk = io->key_dim;
  c.dv = io->value_dim;
  return decay_attention_core(c, io->dtype, io->workspace, (hipStream_t)stream);
}

int oige_decay_attention_backward(const oige_decay_attention_io* io, oige_stream_t stream) {
  int rc = decay_attention_check(io, "decay_attention_backward");
  if (rc) return rc;
  if (io->num_envs == 0) return OIGE_OK;
  OIGE_REQUIRE(io->num_tokens == 0 || (io->q && io->k && io->v && io->d_o && io->dq && io->dk && io->dv),
               "decay_attention_backward: null q, k, v, d_o, dq, dk or dv");
  OIGE_REQUIRE(io->num_tokens > 0 || io->d_state_in, "decay_attention_backward: no tokens and no initial state's gradient asked for");
  const int64_t need = da_workspace(*io, true);
  OIGE_REQUIRE(need == 0 || (io->workspace && aligned16(io->workspace) && io->workspace_floats >= need),
               "decay_attention_backward: needs a 16-byte aligned workspace of %lld floats", (long long)need);
  hipStream_t s = (hipStream_t)stream;
  const int group = io->heads / io->kv_heads;
  const DaRows q = da_rows(io->q, io->q_stride, 1), k = da_rows(io->k, io->k_stride, group), v = da_rows(io->v, io->v_stride, group),
               d_o = da_rows(io->d_o, io->d_o_stride, 1);
  DaCore c = da_core(*io);
  if (io->num_tokens > 0) {  // dq_t = scale S_t do_t
    c.q = d_o;
    c.k = v;
    c.v = k;
    da_out(c, io->dq, io->dq_stride);
    c.s_in = io->state_in;
    c.transposed = 1;
    c.out_scale = io->scale;
    c.dk = io->value_dim;
    c.dv = io->key_dim;
    rc = decay_attention_core(c, io->dtype, io->workspace, s);
    if (rc) return rc;
  }
  c = da_core(*io);
  c.reverse = 1;
  c.s_in = io->d_state_out;
  c.kv_scale = io->scale;
  // shared heads: rows per query head in fp32 behind the segments' scratch, then their sums
  const int64_t t = io->num_tokens, h = io->heads;
  float* wide = nullptr;
  if (group > 1) {
    const int64_t d = io->key_dim > io->value_dim ? io->key_dim : io->value_dim;
    wide = io->workspace + (need - io->num_envs * t * h * d);
    c.o_float = 1;
  }
  {  // dv_t = G_t^T k_t, and the initial state's gradient
    DaCore b = c;
    b.q = k;
    b.k = q;
    b.v = d_o;
    const int64_t rows[3] = {t * h * io->value_dim, h * io->value_dim, io->value_dim};
    da_out(b, wide ? wide : io->dv, wide ? rows : io->dv_stride);
    b.s_out = io->d_state_in;
    b.dk = io->key_dim;
    b.dv = io->value_dim;
    rc = decay_attention_core(b, io->dtype, io->workspace, s);
    if (rc) return rc;
    if (wide && t > 0) rc = decay_attention_share(wide, io->dv, *io, io->value_dim, io->dv_stride, s);
    if (rc) return rc;
  }
  if (t > 0) {  // dk_t = G_t v_t
    DaCore b = c;
    b.q = v;
    b.k = d_o;
    b.v = q;
    const int64_t rows[3] = {t * h * io->key_dim, h * io->key_dim, io->key_dim};
    da_out(b, wide ? wide : io->dk, wide ? rows : io->dk_stride);
    b.transposed = 1;
    b.dk = io->value_dim;
    b.dv = io->key_dim;
    rc = decay_attention_core(b, io->dtype, io->workspace, s);
    if (rc) return rc;
    if (wide) rc = decay_attention_share(wide, io->dk, *io, io->key_dim, io->dk_stride, s);
  }
  return rc;
}

int oige_decay_attention_step(const oige_decay_attention_step_io* io, oige_stream_t stream) {
  OIGE_REQUIRE(io != nullptr, "decay_attention_step: null io");
  OIGE_REQUIRE(elem_bytes(io->dtype), "decay_attention_step: dtype must be OIGE_F32, OIGE_F16 or OIGE_BF16");
  OIGE_REQUIRE(io->num_envs >= 0, "decay_attention_step: %lld sequences", (long long)io->num_envs);
  OIGE_REQUIRE(io->heads >= 1 && io->kv_heads >= 1 && io->heads % io->kv_heads == 0, "decay_attention_step: %d heads over %d key / value heads",
               io->heads, io->kv_heads);
  OIGE_REQUIRE(io->key_dim >= 1 && io->key_dim <= DA_MAX_DIM && io->value_dim >= 1 && io->value_dim <= DA_MAX_DIM,
               "decay_attention_step: head sizes %d and %d (1 .. %d)", io->key_dim, io->value_dim, DA_MAX_DIM);
  OIGE_REQUIRE(!io->resets || io->resets_bytes == 1 || io->resets_bytes == 8, "decay_attention_step: resets are bytes or int64");
  OIGE_REQUIRE(io->decay, "decay_attention_step: null decay");
  if (io->num_envs == 0) return OIGE_OK;
  OIGE_REQUIRE(io->q && io->k && io->v && io->o && io->state, "decay_attention_step: null q, k, v, o or state");
  DaStep a{};
  a.q = io->q;
  a.k = io->k;
  a.v = io->v;
  a.o = io->o;
  a.state = io->state;
  a.decay = io->decay;
  a.resets = io->resets;
  a.n = io->num_envs;
  a.rsn = io->resets_stride;
  a.qn = io->q_stride[0];
  a.qh = io->q_stride[1];
  a.kn = io->k_stride[0];
  a.kh = io->k_stride[1];
  a.vn = io->v_stride[0];
  a.vh = io->v_stride[1];
  a.scale = io->scale;
  a.h = io->heads;
  a.group = io->heads / io->kv_heads;
  a.dk = io->key_dim;
  a.dv = io->value_dim;
  a.resets_bytes = io->resets_bytes;
  const bool wide = io->value_dim % 4 == 0 && aligned16(io->state);
  const int pieces = wide ? io->value_dim / 4 : io->value_dim;
  a.lanes = 1;
  while (a.lanes < pieces && a.lanes < WAVE) a.lanes *= 2;
  const bool big = io->key_dim * io->value_dim > 2048;
  const int64_t units = a.n * a.h, blocks = big ? units : (units + 3) / 4;
  OIGE_REQUIRE(blocks < ((int64_t)1 << 31), "decay_attention_step: %lld sequences x heads are too many for one launch", (long long)units);
  hipStream_t s = (hipStream_t)stream;
#define OIGE_STEP(T)                                                                                                                       \
  do {                                                                                                                                     \
    if (big && wide) hipLaunchKernelGGL((decay_attention_step_kernel<T, 4, 4>), dim3((unsigned)blocks), dim3(256), 0, s, a);               \
    else if (big) hipLaunchKernelGGL((decay_attention_step_kernel<T, 1, 4>), dim3((unsigned)blocks), dim3(256), 0, s, a);                  \
    else if (wide) hipLaunchKernelGGL((decay_attention_step_kernel<T, 4, 1>), dim3((unsigned)blocks), dim3(256), 0, s, a);                 \
    else hipLaunchKernelGGL((decay_attention_step_kernel<T, 1, 1>), dim3((unsigned)blocks), dim3(256), 0, s, a);                           \
  } while (0)
  if (io->dtype == OIGE_F32) OIGE_STEP(float);
  else if (io->dtype == OIGE_F16) OIGE_STEP(_Float16);
  else OIGE_STEP(__bf16);
#undef OIGE_STEP
  return check_launch("decay_attention_step_kernel");
}

}  // extern "C"
