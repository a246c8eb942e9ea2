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
// A wave owns one sequence, one head and 16 NV columns of the state, which it keeps in registers as the accumulator tiles of the
// matrix instructions while it walks the tokens in blocks of B = 16 (fp32, fp16) or 32 (bf16):
//   P  = (Q K^T) o decay^(i-j)                  B x B, only j <= i with no reset in (j, i]
//   O  = P V + decay^(i+1) Q S
//   S <- decay^B S + (decay^(B-1-j) K)^T V
// The transposed forms are taken (P^T = K Q^T, O^T = V^T P^T + S^T Q^T): P^T and S then come out of one product in the very register
// layout the next one takes them in.  The order of the dk (dv) columns over tiles is the kernel's own: tile s, row m holds
// dk = NK m + s, so that every lane's operand elements are neighbours in memory.  Only rows go through LDS: they come in and leave as
// 16 lanes read and write them side by side, and turn there into a token to a lane (64 tokens of 4096 time-major rollouts, whose
// rows lie 4 MiB apart: 338 us, 2032 us with every lane reading a row of its own).
//
// Two kernels: v_mfma_f32_16x16x4_f32 on operands widened to fp32, which rounds nothing to fewer bits, and for bf16 tensors
// v_mfma_f32_16x16x32_bf16 with the 32-bit factors split into bf16 numbers.  What bounds them:
//   short sequences: HBM, for q, k, v, o and the states.  4096 environments x 4 heads x 16 tokens, 64 x 64, fp32: forward 175 us
//     (805 MB, 4.6 TB/s; a large streaming copy reaches 6.4), backward 355 us (1.27 GB once, 3.6 TB/s): counted, every input comes from HBM
//     once, and the three roles ask the L2 for 2.4 GB.  Of the 28 thousand cycles of a backward wave 17 pass until its first rows and its
//     state are there.
//   long ones: the chain of a wave's blocks.  A bf16 block of 32 tokens with 64 x 64 of state is 126 matrix and about 1050 vector
//     instructions; two waves are all that a SIMD's registers hold, and take 7.7 us a block together (4096 heads x 512 tokens: 243 us).
//     2 sequences x 16 heads x 4096 tokens: forward 53 us (states 16, join 9.5, main 27), backward 94 (27, 11.5, 55).
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
  float2* seg_factors; // (N, H, nseg): what a segment multiplies the state with, and what its rounding left; {-1, 0}: it drops the state.  (Those
                       // that are read are powers of 32 m tokens, of segments between the first and the last: never negative.)
  const float* decay;
  const void* resets;
  const void* lengths;
  int64_t rsn, rst;  // element strides of resets
  int64_t n;
  float out_scale, kv_scale;
  int t, seg_len;  // tokens: below 2^30
  int h, dk, dv, slices, nseg;
  int resets_bytes, lengths_bytes;
  int reverse;     // walk from the last token to the first; the first one taken in is not preceded by a decay, the state is multiplied once more at the end
  int transposed;  // the states in memory are (N, H, dv, dk)
  int o_float;     // o is fp32 whatever T is
};

// Up to three recurrences of one shape over the same sequences in one launch (the backward pass).  A role's workgroups follow each
// other on the same XCD (workgroup b runs on XCD b mod 8): the rows that the roles share are read from HBM once.
constexpr int DA_XCDS = 8;
struct DaRoles {
  DaCore c[3];
  int roles;
};

__device__ __forceinline__ int da_length(const DaCore& c, int64_t n) {
  if (!c.lengths) return c.t;
  const int64_t l = c.lengths_bytes == 8 ? static_cast<const int64_t*>(c.lengths)[n] : static_cast<const int32_t*>(c.lengths)[n];
  return l < 0 ? 0 : (l > c.t ? c.t : (int)l);
}

__device__ __forceinline__ int64_t da_flag(const DaCore& c, int64_t n, int t) {  // not zero: a reset
  const int64_t i = n * c.rsn + t * c.rst;
  return c.resets_bytes == 8 ? static_cast<const int64_t*>(c.resets)[i] : (int64_t)static_cast<const uint8_t*>(c.resets)[i];
}

// decay^n.  Products of squares in 64 bits: exact where the result is used in 32, also for decays of 0 and above 1.
__device__ __forceinline__ double da_power(double decay, int64_t n) {
  double r = 1.0, sq = decay;
#pragma unroll 1
  for (; n > 0; n >>= 1) {
    if (n & 1) r *= sq;
    sq *= sq;
  }
  return r;
}
// decay^n for n in 0 .. 32, a wave's table in LDS: products in 64 bits, rounded once.
constexpr int DA_POWERS = 33;
__device__ __forceinline__ void da_powers(float* table, double decay, int lane) {
  const double d2 = decay * decay, d4 = d2 * d2, d8 = d4 * d4, d16 = d8 * d8;
  double r = (lane & 1) ? decay : 1.0;
  r *= (lane & 2) ? d2 : 1.0;
  r *= (lane & 4) ? d4 : 1.0;
  r *= (lane & 8) ? d8 : 1.0;
  r *= (lane & 16) ? d16 : 1.0;
  if (lane < DA_POWERS) table[lane] = (float)(lane == 32 ? d16 * d16 : r);
  wave_lds_fence();
}
__device__ __forceinline__ float da_weight(const float* table, int n, float scale) { return n >= 0 ? table[n > 0 ? n : 0] * scale : 0.f; }

// This wave's piece of a state matrix in memory: tile (s, sv), register r, lane (c, g) holds dk = NK (4 g + r) + s,
// dv = dv0 + NV c + sv.
//
// ELEMS_LOOSE: rows that start on no boundary, or head sizes of no whole vectors.  A group of NK (NV) neighbouring columns that
// reaches across the end is moved forward to end with the row.  What a state's row or column holds twice by that is
// computed twice, to the same bits, and stored twice; only q's doubles are cleared, so that sums over dk count every column once.
// (484 sequences x 75 tokens x 3 heads of 128 x 109, bf16, forward and backward: 295 us; 781 element by element.)
// Row `row + lane_row` of a matrix of `width` columns from column `col` on.  Whole tiles: the scalar unit takes the row's part that
// all lanes share, a lane adds 32 bits.  Else row 0 stands in for rows behind the end.
template <int MODE>
__device__ __forceinline__ const float* da_state_row(const float* p, int row, int lane_row, int height, int width) {
  if (MODE == ELEMS_FULL)
    return reinterpret_cast<const float*>(reinterpret_cast<const char*>(p + row * width) + (uint32_t)(lane_row * width) * 4u);
  const int d = row + lane_row;
  return p + (d < height ? d : 0) * width;
}

template <int NK, int NV, int MODE>
__device__ __forceinline__ void da_load_state(f32x4 (&S)[NK][NV], const float* p, const DaCore& a, int dv0, int c, int g) {
  if (MODE == ELEMS_LOOSE) {
    const int v0 = run_start<NV, MODE>(dv0 + NV * c, a.dv);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k0 = run_start<NK, MODE>(NK * (4 * g + r), a.dk);
      if (a.transposed) {
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) {
          float x[NK];
          load_run<float, NK, MODE>(x, p + (v0 + sv) * a.dk, k0, a.dk);
#pragma unroll
          for (int s = 0; s < NK; ++s) S[s][sv][r] = x[s];
        }
        asm volatile("" ::: "memory");
      } else {
#pragma unroll
        for (int s = 0; s < NK; ++s) {
          float x[NV];
          load_run<float, NV, MODE>(x, p + (k0 + s) * a.dv, v0, a.dv);
#pragma unroll
          for (int sv = 0; sv < NV; ++sv) S[s][sv][r] = x[sv];
        }
      }
    }
    return;
  }
  if (a.transposed) {
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) {
      const bool in = MODE == ELEMS_FULL || dv0 + NV * c + sv < a.dv;
      float x[4 * NK];
      load_run<float, 4 * NK, MODE>(x, da_state_row<MODE>(p, dv0 + sv, NV * c, a.dv, a.dk), 4 * NK * g, in ? a.dk : 0);
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
        const bool in = MODE == ELEMS_FULL || NK * (4 * g + r) + s < a.dk;
        load_run<float, NV, MODE>(x[r], da_state_row<MODE>(p, NK * r + s, NK * 4 * g, a.dk, a.dv), dv0 + NV * c, in ? a.dv : 0);
      }
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) S[s][sv] = f32x4{x[0][sv], x[1][sv], x[2][sv], x[3][sv]};
    }
  }
}

template <int NK, int NV, int MODE>
__device__ __forceinline__ void da_store_state(const f32x4 (&S)[NK][NV], float* p, const DaCore& a, int dv0, int c, int g) {
  if (MODE == ELEMS_LOOSE) {
    const int v0 = run_start<NV, MODE>(dv0 + NV * c, a.dv);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k0 = run_start<NK, MODE>(NK * (4 * g + r), a.dk);
      if (a.transposed) {
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) {
          float x[NK];
#pragma unroll
          for (int s = 0; s < NK; ++s) x[s] = S[s][sv][r];
          store_run<float, NK, MODE>(x, p + (v0 + sv) * a.dk, k0, a.dk);
        }
      } else {
#pragma unroll
        for (int s = 0; s < NK; ++s) {
          float x[NV];
#pragma unroll
          for (int sv = 0; sv < NV; ++sv) x[sv] = S[s][sv][r];
          store_run<float, NV, MODE>(x, p + (k0 + s) * a.dv, v0, a.dv);
        }
      }
    }
    return;
  }
  if (a.transposed) {
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) {
      float x[4 * NK];
#pragma unroll
      for (int s = 0; s < NK; ++s) {
        x[s] = S[s][sv].x;
        x[NK + s] = S[s][sv].y;
        x[2 * NK + s] = S[s][sv].z;
        x[3 * NK + s] = S[s][sv].w;
      }
      if (MODE == ELEMS_FULL || dv0 + NV * c + sv < a.dv)
        store_run<float, 4 * NK, MODE>(x, const_cast<float*>(da_state_row<MODE>(p, dv0 + sv, NV * c, a.dv, a.dk)), 4 * NK * g, a.dk);
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
      for (int r = 0; r < 4; ++r)
        if (MODE == ELEMS_FULL || NK * (4 * g + r) + s < a.dk)
          store_run<float, NV, MODE>(x[r], const_cast<float*>(da_state_row<MODE>(p, NK * r + s, NK * 4 * g, a.dk, a.dv)), dv0 + NV * c, a.dv);
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
// compiler has counted the wait states of the longer way only, and the shorter way read the registers too early.  Where branches
// follow (the stores, the loop's end) the tiles pass through da_settle: the products come in front of its wait and whatever reads
// them behind it, since both sides of the wait claim to change them.
template <int A, int B>
__device__ __forceinline__ void da_settle(f32x4 (&x)[A][B]) {
#pragma unroll
  for (int a = 0; a < A; ++a)
#pragma unroll
    for (int b = 0; b < B; ++b) asm volatile("" : "+v"(x[a][b]));
  asm volatile("s_nop 15" ::: "memory");
#pragma unroll
  for (int a = 0; a < A; ++a)
#pragma unroll
    for (int b = 0; b < B; ++b) asm volatile("" : "+v"(x[a][b]));
}

template <int B>
__device__ __forceinline__ void da_settle(f32x4 (&x)[B]) {
  da_settle(reinterpret_cast<f32x4(&)[1][B]>(x));
}

// One block's rows of the operands.  Rows behind the block's L tokens re-read its last one; `low` is the earliest of its tokens
// in memory, and in reverse the block's first token is the latest.
struct DaBlock {
  int low, L, reverse;
  __device__ __forceinline__ int row(int i) const {
    const int r = i < L ? i : L - 1;
    return reverse ? L - 1 - r : r;
  }
  template <typename T>
  __device__ __forceinline__ const T* at(const T* head, int64_t st, int i) const {  // row * stride in 32 x 32 bits: checked on the host
    return head + (int64_t)low * st + (uint64_t)(uint32_t)row(i) * (uint32_t)st;
  }
};
// The flag that stands between token i of the block and the token taken in before it: its own, or in reverse the next one's (there
// is none behind the last token: what is read then is not used).
__device__ __forceinline__ int64_t da_block_flag(const DaCore& a, const DaBlock& b, int64_t n, int i) {
  const int t = b.low + b.row(i) + b.reverse;
  return da_flag(a, n, t < a.t ? t : a.t - 1);
}
template <int TOKENS>
__device__ __forceinline__ DaBlock da_block(const DaCore& a, int p0, int end, int len) {
  DaBlock b;
  b.L = end - p0 < TOKENS ? end - p0 : TOKENS;
  b.reverse = a.reverse;
  b.low = a.reverse ? len - p0 - b.L : p0;
  return b;
}

// The lane's coordinates once more, computed where they are used: blocks that few rounds of the loop enter would otherwise have
// their masks and weights hoisted out of it, into registers that the loop needs.
__device__ __forceinline__ int da_here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

__device__ __forceinline__ bool da_finite(float x) { return (__builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu) < 0x7F800000u; }
__device__ __forceinline__ f32x4 da_poison(f32x4 x, f32x4 hit) {
  const float nan = __builtin_nanf("");
  return f32x4{hit.x > 0.f ? nan : x.x, hit.y > 0.f ? nan : x.y, hit.z > 0.f ? nan : x.z, hit.w > 0.f ? nan : x.w};
}

// What a wave works on: a slice of the state's columns of one head of one sequence, over one segment of its tokens.
struct DaWave {
  int64_t n, nh;
  int len, begin, end, h, seg, last, slice, dv0;  // last: the segment that the sequence ends in; those behind it only clear their rows
  bool live;
};
// A sequence's tokens are cut evenly over all segments where the lengths differ, into pieces of DA_MIN_SEGMENT at least.
constexpr int DA_MIN_SEGMENT = 64;
__device__ __forceinline__ int da_segment(const DaCore& a, int len) {
  if (!a.lengths || a.nseg == 1) return a.seg_len;
  const int each = (int)(((uint32_t)(len + a.nseg - 1) / (uint32_t)a.nseg + 31u) & ~31u);
  return each > DA_MIN_SEGMENT ? each : DA_MIN_SEGMENT;
}
__device__ __forceinline__ int da_last_segment(const DaCore& a, int len) { return len > 0 ? (int)((uint32_t)(len - 1) / (uint32_t)da_segment(a, len)) : 0; }
__device__ __forceinline__ int da_role(const DaRoles& r) { return (int)(blockIdx.x / DA_XCDS % r.roles); }
// The role's fields once more, read behind the loop: what only its end needs stays out of the scalar registers until then.
__device__ __forceinline__ const DaCore& da_again(const DaRoles& r) {
  int role = da_role(r);
  asm volatile("" : "+s"(role));
  return r.c[role];
}
template <int NV>
__device__ __forceinline__ DaWave da_wave(const DaCore& a, int roles) {
  DaWave w{};
  const uint32_t block = blockIdx.x / DA_XCDS / (uint32_t)roles * DA_XCDS + blockIdx.x % DA_XCDS;
  const uint32_t u = block * DA_WAVES + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));  // below 2^31: checked on the host
  const uint32_t nh = u / (uint32_t)a.slices, n = nh / (uint32_t)a.h;
  w.live = n < (uint32_t)a.n;
  if (!w.live) return w;
  w.seg = blockIdx.y;
  w.slice = (int)(u - nh * (uint32_t)a.slices);
  w.nh = nh;
  w.h = (int)(nh - n * (uint32_t)a.h);
  w.n = n;
  w.dv0 = w.slice * 16 * NV;
  w.len = da_length(a, w.n);
  const int each = da_segment(a, w.len);
  w.last = w.len > 0 ? (int)((uint32_t)(w.len - 1) / (uint32_t)each) : 0;
  w.begin = w.seg * each;
  w.end = w.begin + each < w.len ? w.begin + each : w.len;
  return w;
}

// Four neighbouring groups of NV columns of a result's row, from `off` on.
template <typename T, int NV, int MODE>
__device__ __forceinline__ void da_store_groups(const float (&x)[4 * NV], T* row, int off, int limit) {
  if (MODE != ELEMS_LOOSE) {
    store_run<T, 4 * NV, MODE>(x, row, off, limit);
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float y[NV];
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) y[sv] = x[NV * r + sv];
    store_run<T, NV, MODE>(y, row, off + NV * r, limit);
  }
}

// The state in front of the segment's first token ...
template <int NK, int NV, int MODE, bool STATES>
__device__ __forceinline__ void da_open(f32x4 (&S)[NK][NV], const DaCore& a, const DaWave& w, int lane) {
  if (w.seg > 0 && w.seg <= w.last && !STATES) {
    const float* slot = a.seg_states + ((w.nh * a.nseg + w.seg) * a.slices + w.slice) * (int64_t)(NK * NV * 4 * WAVE);
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) S[s][sv] = *reinterpret_cast<const f32x4*>(slot + ((s * NV + sv) * WAVE + lane) * 4);
  } else if (w.seg == 0 && a.s_in) {
    da_load_state<NK, NV, MODE>(S, a.s_in + w.nh * a.dk * a.dv, a, w.dv0, lane & 15, lane >> 4);
  } else {
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) S[s][sv] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// ... and what becomes of the one behind its last; of the rows behind the sequence's end this segment's share (of all rows) is cleared.
template <typename T, int NK, int NV, int MODE, bool STATES>
__device__ __forceinline__ void da_close(f32x4 (&S)[NK][NV], const DaCore& a, const DaWave& w, int lane, double decay, bool dropped) {
  const int c = lane & 15, g = lane >> 4;
  if (STATES) {
    float* slot = a.seg_states + ((w.nh * a.nseg + w.seg) * a.slices + w.slice) * (int64_t)(NK * NV * 4 * WAVE);
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) *reinterpret_cast<f32x4*>(slot + ((s * NV + sv) * WAVE + lane) * 4) = S[s][sv];
    if (w.slice == 0 && lane == 0) {
      const int count = (w.end > w.begin ? w.end - w.begin : 0) - (a.reverse && w.seg == 0 && w.end > 0 ? 1 : 0);
      const double factor = da_power(decay, count);
      const float hi = (float)factor;
      a.seg_factors[w.nh * a.nseg + w.seg] = dropped ? make_float2(-1.f, 0.f) : make_float2(hi, da_finite(hi) ? (float)(factor - (double)hi) : 0.f);
    }
    return;
  }
  const int start = w.seg * a.seg_len, stop = start + a.seg_len < a.t ? start + a.seg_len : a.t;
  for (int t = (start > w.len ? start : w.len) + c; t < stop; t += 16) {
    const int64_t row = w.n * a.on + (int64_t)t * a.ot + (int64_t)w.h * a.oh;
    const float none[4 * NV] = {};
    if (a.o_float) da_store_groups<float, NV, MODE>(none, static_cast<float*>(a.o) + row, w.dv0 + 4 * NV * g, a.dv);
    else da_store_groups<T, NV, MODE>(none, static_cast<T*>(a.o) + row, w.dv0 + 4 * NV * g, a.dv);
  }
  if (a.s_out && w.seg == w.last) {
    if (a.reverse && w.len > 0) {  // dS_0 = a_0 G_0
      const bool drop = a.resets && da_flag(a, w.n, 0) != 0;
#pragma unroll
      for (int s = 0; s < NK; ++s)
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) S[s][sv] = drop ? f32x4{0.f, 0.f, 0.f, 0.f} : S[s][sv] * (float)decay;
    }
    da_store_state<NK, NV, MODE>(S, a.s_out + w.nh * a.dk * a.dv, a, w.dv0, c, g);
  }
}

// O^T's tiles hold a token's columns in one lane; they leave through LDS, so that 16 lanes store one row side by side.
template <typename T, int NV, int MODE, int LD>
__device__ __forceinline__ void da_store_out(float* lds, const f32x4 (&acc)[NV], const DaCore& a, const DaBlock& b, int64_t head, int dv0, int c, int g) {
  float* mine = lds + c * LD + 4 * NV * g;
#pragma unroll
  for (int sv = 0; sv < NV; ++sv) {
    mine[sv] = acc[sv].x;
    mine[NV + sv] = acc[sv].y;
    mine[2 * NV + sv] = acc[sv].z;
    mine[3 * NV + sv] = acc[sv].w;
  }
  wave_lds_fence();
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float out[NV];
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) out[sv] = lds[(4 * g + r) * LD + NV * c + sv];
    if (4 * g + r < b.L) {
      const int64_t row = head + (int64_t)(b.low + b.row(4 * g + r)) * a.ot;
      if (a.o_float) store_run<float, NV, MODE>(out, static_cast<float*>(a.o) + row, dv0 + NV * c, a.dv);
      else store_run<T, NV, MODE>(out, static_cast<T*>(a.o) + row, dv0 + NV * c, a.dv);
    }
  }
  wave_lds_fence();
}

// STATES: only the states at the segments' ends (no q, no o), for sequences cut over time.
//
// Rollouts of 16 tokens as above: 169 us forward and 352 backward with two waves per SIMD and 64 columns; 182 and 369 with three waves
// and nothing asked for ahead; 228 and 244 us forward with 32 and 16 columns.
//
// The next block's rows are asked for as soon as the registers of this block's are free: q and the first copy of k behind the
// products that read them, the other copy and v at the end, so that their way from memory runs beside the matrix instructions.
template <typename T, int NK, int NV, int MODE, bool STATES>
__global__ __launch_bounds__(DA_WAVES* WAVE, 2) void decay_attention_kernel(const DaRoles roles) {
  const DaCore a = roles.c[da_role(roles)];  // by value: loaded in a few wide reads, not field by field
  const int lane = lane_id(), c = lane & 15, g = lane >> 4;
  const DaWave w = da_wave<NV>(a, roles.roles);
  if (!w.live || (STATES && w.seg >= w.last)) return;
  const int64_t n = w.n;
  const int len = w.len, begin = w.begin, end = w.end;
  const int h = w.h, dv0 = w.dv0;

  const T* qh = static_cast<const T*>(a.q.p) + n * a.q.sn + (int64_t)(h / a.q.group) * a.q.sh;
  const T* kh = static_cast<const T*>(a.k.p) + n * a.k.sn + (int64_t)(h / a.k.group) * a.k.sh;
  const T* vh = static_cast<const T*>(a.v.p) + n * a.v.sn + (int64_t)(h / a.v.group) * a.v.sh;

  // Rows come in as 16 lanes read them side by side, 16 or less bytes each: lane (c, g) holds columns NK c .. of tokens 4 g .. 4 g + 3.
  // That is how the state's product takes k and v; the others take q and k with a token to a lane, by way of LDS.
  constexpr int LD = 16 * (NK > NV ? NK : NV) + 4;
  __shared__ __align__(16) float lds_rows[DA_WAVES][DA_TOKENS * LD];
  float* lds = lds_rows[threadIdx.x >> 6];
  Run<T, NK, MODE> q_run[4], k_run[4];
  Run<T, NV, MODE> v_run[4];
  int64_t flag = 0;
  const auto issue_q = [&](const DaBlock& b) {
    if (STATES) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) q_run[r].issue(b.at(qh, a.q.st, 4 * g + r), NK * c, a.dk);
  };
  const auto issue_k = [&](const DaBlock& b) {
#pragma unroll
    for (int r = 0; r < 4; ++r) k_run[r].issue(b.at(kh, a.k.st, 4 * g + r), NK * c, a.dk);
    if (a.resets) flag = da_block_flag(a, b, n, c);
  };
  const auto issue_v = [&](const DaBlock& b) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v_run[r].issue(b.at(vh, a.v.st, 4 * g + r), dv0 + NV * c, a.dv);
  };
  const auto forget = [&](auto& run) {
#pragma unroll
    for (auto& x : run) x.forget();
  };
  const auto put_rows = [&](const Run<T, NK, MODE> (&run)[4], bool once) {  // once: columns held twice are cleared the second time
    uint32_t in[NK];
    if (MODE == ELEMS_LOOSE) {
      const int off = NK * (da_here(lane) & 15), twice = off - run_start<NK, MODE>(off, a.dk);
#pragma unroll
      for (int s = 0; s < NK; ++s) in[s] = bits_if(s >= twice);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x[NK];
      run[r].take(x, NK * c, a.dk);
#pragma unroll
      for (int s = 0; s < NK; ++s) lds[(4 * g + r) * LD + NK * c + s] = MODE == ELEMS_LOOSE && once ? and_bits(x[s], in[s]) : x[s];
    }
    wave_lds_fence();
  };
  const auto get_token = [&](float (&x)[4 * NK]) {
#pragma unroll
    for (int e = 0; e < 4 * NK; ++e) x[e] = lds[c * LD + 4 * NK * g + e];
    wave_lds_fence();
  };

  DaBlock blk = da_block<DA_TOKENS>(a, begin, end, len);
  if (begin < end) {
    issue_q(blk);
    issue_k(blk);
    issue_v(blk);
  }

  f32x4 S[NK][NV];
  const f32x4 zero{0.f, 0.f, 0.f, 0.f};
  da_open<NK, NV, MODE, STATES>(S, a, w, lane);

  const double decay = (double)a.decay[h];
  __shared__ float lds_powers[DA_WAVES][DA_POWERS];
  float* powers = lds_powers[threadIdx.x >> 6];
  da_powers(powers, decay, lane);
  bool dropped = false;  // a reset inside the segment
  float head_w = 0.f, pair_w[4], tail_w[4], keep_hi = 0.f, keep_lo = 0.f, keep_off = 0.f;
  const uint32_t upto = (2u << c) - 1u;  // bits 0 .. i

  for (int p0 = begin; p0 < end; p0 += DA_TOKENS) {
    const int L = blk.L;
    if (p0 == begin || (a.reverse && p0 == DA_TOKENS) || L < DA_TOKENS) {
      const int first = a.reverse && p0 == 0 ? 1 : 0;  // the first token in reverse: nothing decays in front of it
      const int c = da_here(lane) & 15, g = da_here(lane) >> 4;
      const double keep = da_power(decay, L - first);
      const float pair_scale = a.kv_scale * a.out_scale;  // (one of them is 1)
      keep_hi = (float)keep;
      keep_lo = (float)(keep - (double)keep_hi);
      head_w = da_weight(powers, c + 1 - first, a.out_scale);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * g + r;
        pair_w[r] = da_weight(powers, c - j, pair_scale);
        tail_w[r] = da_weight(powers, L - 1 - j, a.kv_scale);
      }
    }
    // bit i: a reset in front of the block's token i
    const uint32_t m = a.resets ? (uint32_t)(__ballot(flag != 0 && c < L && !(a.reverse && p0 == 0 && c == 0)) & 0xFFFFull) : 0u;
    const bool more = p0 + DA_TOKENS < end;
    const DaBlock next = da_block<DA_TOKENS>(a, more ? p0 + DA_TOKENS : p0, end, len);

    f32x4 acc[NV];
    float V[4][NV], K2[4][NK];
    if (!STATES) {
      float Q[4 * NK], K1[4 * NK];
      put_rows(q_run, true);
      get_token(Q);
      if (more) issue_q(next);
      else forget(q_run);
      put_rows(k_run, false);
      get_token(K1);
      if (more) issue_k(next);
      else forget(k_run);
      f32x4 pt = zero;
#pragma unroll
      for (int e = 0; e < 4 * NK; ++e) pt = __builtin_amdgcn_mfma_f32_16x16x4f32(K1[e], Q[e], pt, 0, 0, 0);
      da_state_part<NK, NV>(acc, S, Q, !(m & upto), head_w);
      // a masked product may be infinite or NaN: selected away, not multiplied
      float P[4] = {pt.x, pt.y, pt.z, pt.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) P[r] = 4 * g + r <= c ? P[r] * pair_w[r] : 0.f;
      if (m) {
        const int g = da_here(lane) >> 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) P[r] = m & upto & ~((2u << (4 * g + r)) - 1u) ? 0.f : P[r];
      }
      uint32_t top = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v_run[r].take(V[r], dv0 + NV * c, a.dv);
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) top = max(top, __builtin_bit_cast(uint32_t, V[r][sv]) & 0x7FFFFFFFu);
      }
      if (__any(top >= 0x7F800000u)) {
        // An infinite or NaN value: where a token sees it the result is NaN, everywhere else (its weight is zero) it is left out.
        const int g = da_here(lane) >> 4;
        f32x4 hit[NV];
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) hit[sv] = zero;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float seen = 4 * g + r <= c && !(m & upto & ~((2u << (4 * g + r)) - 1u)) ? 1.f : 0.f;
#pragma unroll
          for (int sv = 0; sv < NV; ++sv) hit[sv] = __builtin_amdgcn_mfma_f32_16x16x4f32(da_finite(V[r][sv]) ? 0.f : 1.f, seen, hit[sv], 0, 0, 0);
        }
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) acc[sv] = da_poison(acc[sv], hit[sv]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int sv = 0; sv < NV; ++sv)
            acc[sv] = __builtin_amdgcn_mfma_f32_16x16x4f32(da_finite(V[r][sv]) ? V[r][sv] : 0.f, P[r], acc[sv], 0, 0, 0);
        da_settle(acc);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int sv = 0; sv < NV; ++sv) acc[sv] = __builtin_amdgcn_mfma_f32_16x16x4f32(V[r][sv], P[r], acc[sv], 0, 0, 0);
        da_settle(acc);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int s = 0; s < NK; ++s) K2[r][s] = lds[(4 * g + r) * LD + NK * c + s];
      wave_lds_fence();
      da_store_out<T, NV, MODE, LD>(lds, acc, a, blk, n * a.on + (int64_t)h * a.oh, dv0, c, g);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v_run[r].take(V[r], dv0 + NV * c, a.dv);
        k_run[r].take(K2[r], NK * c, a.dk);
      }
    }

    // rows in front of the block's last reset, and behind the end, stay out of the state's sum altogether
    if (m || L < DA_TOKENS) {
      const int g = da_here(lane) >> 4;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool in = 4 * g + r < L && !(m & ~((2u << (4 * g + r)) - 1u));
#pragma unroll
        for (int s = 0; s < NK; ++s) K2[r][s] = in ? K2[r][s] : 0.f;
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) V[r][sv] = in ? V[r][sv] : 0.f;
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) V[r][sv] *= tail_w[r];
    // decay^tokens in 32 bits; what its rounding leaves is carried along, or it would pile up over a long memory
    keep_off += keep_lo;
    const float kept = keep_hi + keep_off;
    keep_off -= kept - keep_hi;
    if (m) {  // (a state that is not finite is dropped too: cleared, not multiplied)
      dropped = true;
#pragma unroll
      for (int s = 0; s < NK; ++s)
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) S[s][sv] = zero;
    }
    if (STATES) {
      if (more) issue_k(next);
      else forget(k_run);
    }
    if (more) issue_v(next);
    else forget(v_run);
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) {
        S[s][sv] *= kept;
#pragma unroll
        for (int r = 0; r < 4; ++r) S[s][sv] = __builtin_amdgcn_mfma_f32_16x16x4f32(K2[r][s], V[r][sv], S[s][sv], 0, 0, 0);
      }
    da_settle(S);
    blk = next;
  }
  da_close<T, NK, NV, MODE, STATES>(S, da_again(roles), w, lane, decay, dropped);
}

// ---------------------------------------------------------------- the same for bf16 tensors
// bf16 operands go into v_mfma_f32_16x16x32_bf16, 16 times the rate of the 32-bit instruction, in blocks of 32 tokens:
//   K Q^T        both operands as they are: exact products, 32-bit sums
//   S Q, P V, K^T (w V)   the 32-bit factor as the sum of three bf16 numbers that it is, three products: every result is a 32-bit
//                sum of exact terms.  (Two numbers leave out 2^-18 of S and P, 64 fp32 roundings, which a cancelling sum shows; they take
//                3 to 14 % less: 4 prompts of 8192 tokens, 16 heads, 128 x 128: forward 274 us instead of 290, backward 799 of 912.)
// The operand that a product sums over lies packed along registers, eight to a lane: for tokens, lane group g holds 4 g + {0..3} and
// 16 + 4 g + {0..3}, as K Q^T leaves them; for dk, the four rows of two neighbouring tiles side by side, as q's words hold them.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
constexpr int DB_TOKENS = 32;

__device__ __forceinline__ f32x4 db_mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t db_pack(float x, float y) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2)); }
__device__ __forceinline__ float db_low(uint32_t p) { return __builtin_bit_cast(float, p << 16); }
__device__ __forceinline__ float db_high(uint32_t p) { return __builtin_bit_cast(float, p & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t db_lows(uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x05040100); }   // {x.low, y.low}
__device__ __forceinline__ uint32_t db_highs(uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x07060302); }  // {x.high, y.high}
// x, y = hi + mid + lo, cut after 8 bits each: 24 in all, nothing is left out (and, cut not rounded, nothing becomes infinite)
__device__ __forceinline__ void db_split(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  uint32_t a = __builtin_bit_cast(uint32_t, x), b = __builtin_bit_cast(uint32_t, y);
  hi = db_highs(a, b);
  x -= db_high(a);
  y -= db_high(b);
  a = __builtin_bit_cast(uint32_t, x), b = __builtin_bit_cast(uint32_t, y);
  mid = db_highs(a, b);
  lo = db_highs(__builtin_bit_cast(uint32_t, x - db_high(a)), __builtin_bit_cast(uint32_t, y - db_high(b)));
}

// CNT bf16 elements of a row, two to a register (one, where CNT is 1); elements behind the limit are 0.
template <int CNT, int MODE>
struct Bits {
  static constexpr int REGS = CNT == 1 ? 1 : CNT / 2;
  Run<uint16_t, CNT, MODE> run;
  // `base` is the same for the whole wave, `row` this lane's row in elements behind it
  __device__ __forceinline__ void issue(const __bf16* base, uint32_t row, int off, int limit) {
    constexpr int W = Run<uint16_t, CNT, MODE>::W;
#pragma unroll
    for (int b = 0; b < CNT / W; ++b) {
      if (MODE == ELEMS_LOOSE) {
        const uint32_t at = 2u * (row + (uint32_t)(run_start<CNT, MODE>(off, limit) + b * W));
        run.x[b] = __builtin_bit_cast(Pack<uint16_t, W>, *reinterpret_cast<const Loose<uint16_t, W>*>(reinterpret_cast<const char*>(base) + at));
      } else {
        const uint32_t at = 2u * (row + (uint32_t)(MODE == ELEMS_FULL || off + b * W < limit ? off + b * W : 0));
        run.x[b] = *reinterpret_cast<const Pack<uint16_t, W>*>(reinterpret_cast<const char*>(base) + at);
      }
    }
  }
  __device__ __forceinline__ void take(uint32_t (&out)[REGS], int off, int limit) const {
    constexpr int W = Run<uint16_t, CNT, MODE>::W;
#pragma unroll
    for (int i = 0; i < REGS; ++i) {
      const int e = CNT == 1 ? 0 : 2 * i;
      const uint32_t lo = run.x[e / W].v[e % W], hi = CNT == 1 ? 0u : (uint32_t)run.x[(e + 1) / W].v[(e + 1) % W];
      out[i] = lo | hi << 16;
      if (MODE == ELEMS_WIDE) out[i] &= bits_if(off + e / W * W < limit);  // (a pair lies in one piece)
    }
  }
};

// The scalar part of the addresses of a whole block's rows: lane group 0's in the order 0 .. 3, 16 .. 19, or in reverse, where
// token i lies 31 - i rows behind the block's earliest, 19 .. 16, 3 .. 0.  CHAIN: each from the one before, where eight addresses
// per tensor computed ahead of the loop are more than the scalar registers hold (52 of them went to vector registers; the kernel
// that only makes states has room: 42 us against 50 with the chain, 64 sequences of 8192 tokens at most, 128 x 128).
template <bool CHAIN>
struct DbWalk {
  const char* p;
  int step;  // bytes; 16 of them are below 2^31: checked on the host
  __device__ __forceinline__ DbWalk(const char* base, int64_t st, int reverse)
      : p(base + (reverse ? 19 * 2 * st : 0)), step(reverse ? -2 * (int)st : 2 * (int)st) {}
  __device__ __forceinline__ const char* at(int e) {  // e: 0, 1, .. 7
    if (!CHAIN) return p + (e < 4 ? e : 12 + e) * (int64_t)step;
    if (e > 0) p += e == 4 ? 13 * (int64_t)step : (int64_t)step;
    asm volatile("" : "+s"(p));
    return p;
  }
};

// O^T's part from the state: for both halves of the block's tokens, the state's three parts against q.
template <int NK, int NV>
__device__ __forceinline__ void db_state_part(f32x4 (&acc)[2][NV], const f32x4 (&S)[NK][NV], const uint32_t (&Q)[2][2 * NK],
                                              const bool (&from_state)[2], const float (&head_w)[2]) {
  const f32x4 zero{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int it = 0; it < 2; ++it)
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) acc[it][sv] = zero;
#pragma unroll
  for (int p = 0; p < NK / 2; ++p) {
    u32x4 q[2];
#pragma unroll
    for (int it = 0; it < 2; ++it)
      q[it] = u32x4{Q[it][p], Q[it][NK / 2 + p], Q[it][NK + p], Q[it][3 * NK / 2 + p]};
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) {
      const f32x4 s0 = S[2 * p][sv], s1 = S[2 * p + 1][sv];
      uint32_t hi[4], mid[4], lo[4];
      db_split(s0.x, s1.x, hi[0], mid[0], lo[0]);
      db_split(s0.y, s1.y, hi[1], mid[1], lo[1]);
      db_split(s0.z, s1.z, hi[2], mid[2], lo[2]);
      db_split(s0.w, s1.w, hi[3], mid[3], lo[3]);
      const u32x4 h{hi[0], hi[1], hi[2], hi[3]}, m{mid[0], mid[1], mid[2], mid[3]}, l{lo[0], lo[1], lo[2], lo[3]};
#pragma unroll
      for (int it = 0; it < 2; ++it) acc[it][sv] = db_mfma(l, q[it], acc[it][sv]);
#pragma unroll
      for (int it = 0; it < 2; ++it) acc[it][sv] = db_mfma(m, q[it], acc[it][sv]);
#pragma unroll
      for (int it = 0; it < 2; ++it) acc[it][sv] = db_mfma(h, q[it], acc[it][sv]);
    }
  }
#pragma unroll
  for (int it = 0; it < 2; ++it)
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) acc[it][sv] = from_state[it] ? acc[it][sv] * head_w[it] : zero;
}

// The result's way out, as above; two bf16 to a word.  Rows per query head of shared ones (fp32) go straight from the registers.
template <int NV, int MODE, int LD>
__device__ __forceinline__ void db_store_out(uint32_t* lds, const f32x4 (&acc)[2][NV], const DaCore& a, const DaBlock& b, int64_t head, int dv0, int c,
                                             int g) {
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    float out[4 * NV];
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) {
      out[sv] = acc[it][sv].x;
      out[NV + sv] = acc[it][sv].y;
      out[2 * NV + sv] = acc[it][sv].z;
      out[3 * NV + sv] = acc[it][sv].w;
    }
    const int i = 16 * it + c;
    if (a.o_float) {
      if (i < b.L) da_store_groups<float, NV, MODE>(out, static_cast<float*>(a.o) + head + (int64_t)(b.low + b.row(i)) * a.ot, dv0 + 4 * NV * g, a.dv);
    } else {
#pragma unroll
      for (int e = 0; e < 2 * NV; ++e) lds[i * LD + 2 * NV * g + e] = db_pack(out[2 * e], out[2 * e + 1]);
    }
  }
  if (a.o_float) return;
  wave_lds_fence();
  // what lane (c, g) stores of token e: NV elements, two words, one or half of one
  const auto put = [&](uint16_t* at, int e) {
    const int i = (e < 4 ? 0 : 12) + 4 * g + e;
    if (MODE == ELEMS_LOOSE && NV > 1) *reinterpret_cast<Loose<uint16_t, NV>*>(at) = *reinterpret_cast<const Loose<uint16_t, NV>*>(lds + i * LD + NV / 2 * c);
    else if (NV == 4) *reinterpret_cast<Pack<uint32_t, 2>*>(at) = *reinterpret_cast<const Pack<uint32_t, 2>*>(lds + i * LD + 2 * c);
    else if (NV == 2) *reinterpret_cast<uint32_t*>(at) = lds[i * LD + c];
    else *at = reinterpret_cast<const uint16_t*>(lds + i * LD)[c];
  };
  const int col = run_start<NV, MODE>(dv0 + NV * c, a.dv);
  const bool in = MODE != ELEMS_WIDE || col < a.dv;
  uint16_t* first = static_cast<uint16_t*>(a.o) + head + (int64_t)b.low * a.ot;
  if (b.L == DB_TOKENS) {  // as with the loads: 32 bits from the lane, the rest from the scalar unit
    const uint32_t off = 2u * ((uint32_t)(b.reverse ? 12 - 4 * g : 4 * g) * (uint32_t)a.ot + (uint32_t)col);
    DbWalk<true> walk(reinterpret_cast<const char*>(first), a.ot, b.reverse);
    if (in) {
#pragma unroll
      for (int e = 0; e < 8; ++e) put(reinterpret_cast<uint16_t*>(const_cast<char*>(walk.at(e)) + off), e);
    }
    asm volatile("" ::: "memory");  // (keeps the branches' ends apart)
  } else {
    const int g0 = da_here(lane_id()) >> 4;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = (e < 4 ? 0 : 12) + 4 * g0 + e;
      if (in && i < b.L) put(first + (int64_t)b.row(i) * a.ot + col, e);
    }
  }
  wave_lds_fence();
}

// Offset of token `i` of a block of L from its earliest one, in elements of less than 32 bits: `step` = the token stride times i.
__device__ __forceinline__ uint32_t db_offset(const DaBlock& b, uint32_t step, uint32_t st) {
  const uint32_t last = (uint32_t)(b.L - 1) * st;
  const uint32_t off = step < last ? step : last;
  return b.reverse ? last - off : off;
}

template <int NK, int NV, int MODE, bool STATES>
__global__ __launch_bounds__(DA_WAVES* WAVE, 2) void decay_attention_bf16_kernel(const DaRoles roles) {
  const DaCore a = roles.c[da_role(roles)];  // by value: loaded in a few wide reads, not field by field
  const int lane = lane_id(), c = lane & 15, g = lane >> 4;
  const DaWave w = da_wave<NV>(a, roles.roles);
  if (!w.live || (STATES && w.seg >= w.last)) return;
  const int64_t n = w.n;
  const int len = w.len, begin = w.begin, end = w.end;
  const int h = w.h, dv0 = w.dv0;
  __shared__ f32x4 lds_weights[DA_WAVES][4][WAVE];
  const __bf16* qh = static_cast<const __bf16*>(a.q.p) + n * a.q.sn + (int64_t)(h / a.q.group) * a.q.sh;
  const __bf16* kh = static_cast<const __bf16*>(a.k.p) + n * a.k.sn + (int64_t)(h / a.k.group) * a.k.sh;
  const __bf16* vh = static_cast<const __bf16*>(a.v.p) + n * a.v.sn + (int64_t)(h / a.v.group) * a.v.sh;

  // As in the kernel above: lane (c, g) holds columns NK c .. of tokens 4 g + {0..3} and 16 + 4 g + {0..3}, q and the first use of k
  // take whole tokens by way of LDS.
  constexpr int LD = 8 * NK + 4;  // in registers' words
  __shared__ __align__(16) uint32_t lds_rows[DA_WAVES][DB_TOKENS * LD];
  constexpr int LD_OUT = 8 * NV + 4;
  __shared__ __align__(16) uint32_t lds_out[DA_WAVES][DB_TOKENS * LD_OUT];
  uint32_t *lds = lds_rows[threadIdx.x >> 6], *out = lds_out[threadIdx.x >> 6];
  Bits<NK, MODE> q_run[8], k_run[8];
  Bits<NV, MODE> v_run[8];
  int64_t flag = 0;
  const uint32_t qst = (uint32_t)a.q.st, kst = (uint32_t)a.k.st, vst = (uint32_t)a.v.st;
  // whole blocks: a lane's offset is the same in each, rows differ by a multiple of the token stride that the scalar base takes
  const int rev = a.reverse;
  const uint32_t group = rev ? 12 - 4 * g : 4 * g;
  const uint32_t q_group = group * qst, k_group = group * kst, v_group = group * vst;
  const auto issue = [&](auto& run, const __bf16* head, int64_t st, uint32_t lane_off, const DaBlock& b, int off, int limit) {
    const __bf16* base = head + (int64_t)b.low * st;
    if (b.L == DB_TOKENS) {
      DbWalk<!STATES> walk(reinterpret_cast<const char*>(base), st, rev);
#pragma unroll
      for (int e = 0; e < 8; ++e) run[e].issue(reinterpret_cast<const __bf16*>(walk.at(e)), lane_off, off, limit);
    } else {
      const int g = da_here(lane) >> 4;
#pragma unroll
      for (int e = 0; e < 8; ++e) run[e].issue(base, db_offset(b, (uint32_t)(4 * g + (e < 4 ? e : 12 + e)) * (uint32_t)st, (uint32_t)st), off, limit);
      asm volatile("" ::: "memory");  // as above: merged, both branches' loads would go through addresses in vector registers
    }
  };
  const auto issue_q = [&](const DaBlock& b) {
    if (!STATES) issue(q_run, qh, a.q.st, q_group, b, NK * c, a.dk);
  };
  const auto issue_k = [&](const DaBlock& b) {
    issue(k_run, kh, a.k.st, k_group, b, NK * c, a.dk);
    if (a.resets) flag = da_block_flag(a, b, n, da_here(lane) & 31);
  };
  const auto issue_v = [&](const DaBlock& b) { issue(v_run, vh, a.v.st, v_group, b, dv0 + NV * c, a.dv); };
  const auto forget = [&](auto& run) {
#pragma unroll
    for (auto& x : run) x.run.forget();
  };
  const auto lds_row = [&](int e) { return lds + ((e < 4 ? 0 : 12) + 4 * g + e) * LD; };
  const auto put_rows = [&](const Bits<NK, MODE> (&run)[8], bool once) {  // once: columns held twice are cleared the second time
    uint32_t in[NK / 2];
    if (MODE == ELEMS_LOOSE) {
      const int off = NK * (da_here(lane) & 15), twice = off - run_start<NK, MODE>(off, a.dk);
#pragma unroll
      for (int i = 0; i < NK / 2; ++i) in[i] = twice <= 2 * i ? 0xFFFFFFFFu : twice == 2 * i + 1 ? 0xFFFF0000u : 0u;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t x[NK / 2];
      run[e].take(x, NK * c, a.dk);
#pragma unroll
      for (int i = 0; i < NK / 2; ++i) lds_row(e)[NK / 2 * c + i] = MODE == ELEMS_LOOSE && once ? x[i] & in[i] : x[i];
    }
    wave_lds_fence();
  };
  const auto get_tokens = [&](uint32_t (&x)[2][2 * NK]) {
#pragma unroll
    for (int it = 0; it < 2; ++it)
#pragma unroll
      for (int i = 0; i < 2 * NK; ++i) x[it][i] = lds[(16 * it + c) * LD + 2 * NK * g + i];
    wave_lds_fence();
  };

  DaBlock blk = da_block<DB_TOKENS>(a, begin, end, len);
  if (begin < end) {
    issue_q(blk);
    issue_k(blk);
    issue_v(blk);
  }
  f32x4 S[NK][NV];
  const f32x4 zero{0.f, 0.f, 0.f, 0.f};
  da_open<NK, NV, MODE, STATES>(S, a, w, lane);

  const double decay = (double)a.decay[h];
  __shared__ float lds_powers[DA_WAVES][DA_POWERS];
  float* powers = lds_powers[threadIdx.x >> 6];
  da_powers(powers, decay, lane);
  bool dropped = false;
  float head_w[2] = {0.f, 0.f}, keep_hi = 0.f, keep_lo = 0.f, keep_off = 0.f;
  // this lane's weights: within 16 tokens, from the first 16 to the last, and the two halves' up to the block's end
  f32x4* weights = &lds_weights[(threadIdx.x >> 6)][0][lane];

  for (int p0 = begin; p0 < end; p0 += DB_TOKENS) {
    const int L = blk.L;
    if (p0 == begin || (rev && p0 == DB_TOKENS) || L < DB_TOKENS) {
      const int first = a.reverse && p0 == 0 ? 1 : 0;  // the first token in reverse: nothing decays in front of it
      const int c = da_here(lane) & 15, g = da_here(lane) >> 4;
      const double keep = da_power(decay, L - first);
      const float pair_scale = a.kv_scale * a.out_scale;  // (one of them is 1)
      keep_hi = (float)keep;
      keep_lo = (float)(keep - (double)keep_hi);
      head_w[0] = da_weight(powers, c + 1 - first, a.out_scale);
      head_w[1] = da_weight(powers, c + 17 - first, a.out_scale);
      float x[16];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 4 * g + r;
        x[r] = da_weight(powers, c - j, pair_scale);
        x[4 + r] = da_weight(powers, 16 + c - j, pair_scale);
        x[8 + r] = da_weight(powers, L - 1 - j, a.kv_scale);
        x[12 + r] = da_weight(powers, L - 17 - j, a.kv_scale);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) weights[i * WAVE] = f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
      wave_lds_fence();
    }
    // bit i: a reset in front of the block's token i
    const uint32_t m = a.resets ? (uint32_t)__ballot(flag != 0 && (lane & 31) < L && !(rev && p0 == 0 && (lane & 31) == 0)) : 0u;
    const bool more = p0 + DB_TOKENS < end;
    const DaBlock next = da_block<DB_TOKENS>(a, more ? p0 + DB_TOKENS : p0, end, len);
    const uint32_t upto[2] = {(2u << c) - 1u, (0x20000u << c) - 1u};  // bits 0 .. i for token i = c, 16 + c

    uint32_t V[8][Bits<NV, MODE>::REGS], K2[STATES ? 8 : 1][NK / 2];  // k stays in LDS where it went there
    if (!STATES) {
      f32x4 acc[2][NV];
      uint32_t Q[2][2 * NK], K1[2][2 * NK];
      put_rows(q_run, true);
      get_tokens(Q);
      put_rows(k_run, false);
      get_tokens(K1);
      f32x4 pt[3] = {zero, zero, zero};  // P^T: tokens 0-15 for 0-15, 0-15 for 16-31, 16-31 for 16-31
#pragma unroll
      for (int p = 0; p < NK / 2; ++p) {
        u32x4 q[2], k[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          q[i] = u32x4{Q[i][4 * p], Q[i][4 * p + 1], Q[i][4 * p + 2], Q[i][4 * p + 3]};
          k[i] = u32x4{K1[i][4 * p], K1[i][4 * p + 1], K1[i][4 * p + 2], K1[i][4 * p + 3]};
        }
        pt[0] = db_mfma(k[0], q[0], pt[0]);
        pt[1] = db_mfma(k[0], q[1], pt[1]);
        pt[2] = db_mfma(k[1], q[1], pt[2]);
      }
      if (more) issue_k(next);
      else forget(k_run);
      const bool from_state[2] = {!(m & upto[0]), !(m & upto[1])};
      db_state_part<NK, NV>(acc, S, Q, from_state, head_w);
      // a masked product may be infinite or NaN: selected away, not multiplied
      const f32x4 w0 = weights[0], w1 = weights[WAVE];
      const float pair_w[4] = {w0.x, w0.y, w0.z, w0.w}, cross_w[4] = {w1.x, w1.y, w1.z, w1.w};
      float P[3][4] = {{pt[0].x, pt[0].y, pt[0].z, pt[0].w}, {pt[1].x, pt[1].y, pt[1].z, pt[1].w}, {pt[2].x, pt[2].y, pt[2].z, pt[2].w}};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        P[0][r] = 4 * g + r <= c ? P[0][r] * pair_w[r] : 0.f;
        P[1][r] *= cross_w[r];
        P[2][r] = 4 * g + r <= c ? P[2][r] * pair_w[r] : 0.f;
      }
      if (m) {
        const int g = da_here(lane) >> 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t behind = ~((2u << (4 * g + r)) - 1u);  // bits j + 1 ..
          P[0][r] = m & upto[0] & behind ? 0.f : P[0][r];
          P[1][r] = m & upto[1] & behind ? 0.f : P[1][r];
          P[2][r] = m & upto[1] & (behind << 16) ? 0.f : P[2][r];
        }
      }
      u32x4 parts[3][2];  // of P, the smallest first
      {
        uint32_t x[3][6];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          db_split(P[i][0], P[i][1], x[2][2 * i], x[1][2 * i], x[0][2 * i]);
          db_split(P[i][2], P[i][3], x[2][2 * i + 1], x[1][2 * i + 1], x[0][2 * i + 1]);
        }
#pragma unroll
        for (int part = 0; part < 3; ++part) {
          parts[part][0] = u32x4{x[part][0], x[part][1], 0u, 0u};
          parts[part][1] = u32x4{x[part][2], x[part][3], x[part][4], x[part][5]};
        }
      }
      u16x2 top = {0, 0};  // the largest magnitudes' bits
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v_run[e].take(V[e], dv0 + NV * c, a.dv);
#pragma unroll
        for (int i = 0; i < Bits<NV, MODE>::REGS; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, V[e][i] & 0x7FFF7FFFu));
      }
      const bool odd = top.x >= 0x7F80 || top.y >= 0x7F80;  // infinite or NaN
      if (__any(odd)) {
        // An infinite or NaN value: where a token sees it the result is NaN, everywhere else (its weight is zero) it is left out.
        const int c = da_here(lane) & 15, g = da_here(lane) >> 4;
        u32x4 seen[2];
#pragma unroll
        for (int it = 0; it < 2; ++it) {
          uint32_t x[4];
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const int j = (p < 2 ? 0 : 12) + 4 * g + 2 * p;
            const bool s0 = j <= 16 * it + c && !(m & upto[it] & ~((2u << j) - 1u)), s1 = j + 1 <= 16 * it + c && !(m & upto[it] & ~((4u << j) - 1u));
            x[p] = (s0 ? 0x3F80u : 0u) | (s1 ? 0x3F800000u : 0u);
          }
          seen[it] = u32x4{x[0], x[1], x[2], x[3]};
        }
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) {
          uint32_t kept[4], bad[4];
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const uint32_t x = sv & 1 ? db_highs(V[2 * p][sv / 2], V[2 * p + 1][sv / 2]) : db_lows(V[2 * p][sv / 2], V[2 * p + 1][sv / 2]);
            const bool b0 = (x & 0x7F80u) == 0x7F80u, b1 = (x & 0x7F800000u) == 0x7F800000u;
            bad[p] = (b0 ? 0x3F80u : 0u) | (b1 ? 0x3F800000u : 0u);
            kept[p] = x & ((b0 ? 0u : 0xFFFFu) | (b1 ? 0u : 0xFFFF0000u));
          }
          const u32x4 v{kept[0], kept[1], kept[2], kept[3]}, b{bad[0], bad[1], bad[2], bad[3]};
#pragma unroll
          for (int it = 0; it < 2; ++it) {
            acc[it][sv] = da_poison(acc[it][sv], db_mfma(b, seen[it], zero));
#pragma unroll
            for (int part = 0; part < 3; ++part) acc[it][sv] = db_mfma(v, parts[part][it], acc[it][sv]);
          }
        }
        da_settle(acc);
      } else {
        u32x4 v[NV];
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) {
          const int i = sv / 2;
          v[sv] = sv & 1 ? u32x4{db_highs(V[0][i], V[1][i]), db_highs(V[2][i], V[3][i]), db_highs(V[4][i], V[5][i]), db_highs(V[6][i], V[7][i])}
                         : u32x4{db_lows(V[0][i], V[1][i]), db_lows(V[2][i], V[3][i]), db_lows(V[4][i], V[5][i]), db_lows(V[6][i], V[7][i])};
        }
#pragma unroll
        for (int part = 0; part < 3; ++part)  // (no product waits for the one just in front of it)
#pragma unroll
          for (int sv = 0; sv < NV; ++sv)
#pragma unroll
            for (int it = 0; it < 2; ++it) acc[it][sv] = db_mfma(v[sv], parts[part][it], acc[it][sv]);
        da_settle(acc);
      }
      if (more) issue_q(next);
      else forget(q_run);
      db_store_out<NV, MODE, LD_OUT>(out, acc, a, blk, n * a.on + (int64_t)h * a.oh, dv0, c, g);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v_run[e].take(V[e], dv0 + NV * c, a.dv);
        if constexpr (STATES) k_run[e].take(K2[e], NK * c, a.dk);
      }
    }

    // rows in front of the block's last reset, and behind the end, stay out of the state's sum altogether
    if (m || L < DB_TOKENS) {
      const int g = da_here(lane) >> 4;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = (e < 4 ? 0 : 12) + 4 * g + e;
        const bool in = j < L && !(m & ~((2u << j) - 1u));
        if constexpr (STATES) {
#pragma unroll
          for (int i = 0; i < NK / 2; ++i) K2[e][i] = in ? K2[e][i] : 0u;
        } else if (!in) {
#pragma unroll
          for (int i = 0; i < NK / 2; ++i) lds_row(e)[NK / 2 * c + i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < Bits<NV, MODE>::REGS; ++i) V[e][i] = in ? V[e][i] : 0u;
      }
      wave_lds_fence();
    }
    u32x4 vh3[NV], vm3[NV], vl3[NV];
    const f32x4 w2 = weights[2 * WAVE], w3 = weights[3 * WAVE];
    const float tail_w[8] = {w2.x, w2.y, w2.z, w2.w, w3.x, w3.y, w3.z, w3.w};
#pragma unroll
    for (int sv = 0; sv < NV; ++sv) {
      uint32_t hi[4], mid[4], lo[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t b0 = V[2 * p][sv / 2], b1 = V[2 * p + 1][sv / 2];
        db_split((sv & 1 ? db_high(b0) : db_low(b0)) * tail_w[2 * p], (sv & 1 ? db_high(b1) : db_low(b1)) * tail_w[2 * p + 1], hi[p], mid[p], lo[p]);
      }
      vh3[sv] = u32x4{hi[0], hi[1], hi[2], hi[3]};
      vm3[sv] = u32x4{mid[0], mid[1], mid[2], mid[3]};
      vl3[sv] = u32x4{lo[0], lo[1], lo[2], lo[3]};
    }
    // decay^tokens in 32 bits; what its rounding leaves is carried along, or it would pile up over a long memory
    keep_off += keep_lo;
    const float kept = keep_hi + keep_off;
    keep_off -= kept - keep_hi;
    if (m) {  // (a state that is not finite is dropped too: cleared, not multiplied)
      dropped = true;
#pragma unroll
      for (int s = 0; s < NK; ++s)
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) S[s][sv] = zero;
    }
    if (STATES) {
      if (more) issue_k(next);
      else forget(k_run);
    }
    if (more) issue_v(next);
    else forget(v_run);
    uint32_t kk[8];
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      const int i = s / 2;
      if (!(s & 1)) {
        if constexpr (NK == 8 && !STATES) __builtin_amdgcn_sched_barrier(0);  // or all of k is read at once, into registers there are not
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (STATES) kk[e] = K2[e][i];
          else kk[e] = lds_row(e)[NK / 2 * c + i];
        }
      }
      const u32x4 k = s & 1 ? u32x4{db_highs(kk[0], kk[1]), db_highs(kk[2], kk[3]), db_highs(kk[4], kk[5]), db_highs(kk[6], kk[7])}
                            : u32x4{db_lows(kk[0], kk[1]), db_lows(kk[2], kk[3]), db_lows(kk[4], kk[5]), db_lows(kk[6], kk[7])};
#pragma unroll
      for (int sv = 0; sv < NV; ++sv) S[s][sv] *= kept;
#pragma unroll
      for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int sv = 0; sv < NV; ++sv) S[s][sv] = db_mfma(k, part == 0 ? vl3[sv] : part == 1 ? vm3[sv] : vh3[sv], S[s][sv]);
    }
    wave_lds_fence();
    da_settle(S);
    blk = next;
  }
  da_close<__bf16, NK, NV, MODE, STATES>(S, da_again(roles), w, lane, decay, dropped);
}

// The states in front of every segment from those at the segments' ends (in place, register order): carry = factor carry + end.
// Segment 0's end already holds the initial state.  A thread owns four floats of one (sequence, head) over all segments, eight of
// them in flight.  It moves the states once each way (64 heads' 128 x 128 over 8 segments, 2 x 34 MB: 12 us; 32 heads' 64 x 64
// over 32 segments, 2 x 17 MB: 9.5 us), mostly from and to the caches; 16 in flight are no faster.
__global__ __launch_bounds__(256) void decay_attention_join_kernel(const DaRoles roles, int64_t quads, int64_t per_head, int nseg) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  const DaCore& a = roles.c[blockIdx.y];
  const float2* factors = a.seg_factors;
  const int64_t nh = i / per_head, e = i % per_head;
  const int last = da_last_segment(a, da_length(a, nh / a.h));
  if (last == 0) return;
  f32x4* s = reinterpret_cast<f32x4*>(a.seg_states) + nh * nseg * per_head + e;
  f32x4 carry = s[0];
  constexpr int U = 8;  // ends in flight (they do not depend on the carry, but lie where it goes)
  for (int seg0 = 1; seg0 <= last; seg0 += U) {
    f32x4 end[U];
    float2 f[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int seg = seg0 + i < last ? seg0 + i : last - 1;  // (the last segment's own end is nobody's start)
      end[i] = s[seg * per_head];
      f[i] = factors[nh * nseg + seg];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (seg0 + i > last) break;
      s[(seg0 + i) * per_head] = carry;
      const f32x4 part = {da_finite(carry.x) ? carry.x : 0.f, da_finite(carry.y) ? carry.y : 0.f, da_finite(carry.z) ? carry.z : 0.f,
                          da_finite(carry.w) ? carry.w : 0.f};  // (what is infinite stays so: no part of it of the other sign)
      const f32x4 left = __builtin_elementwise_fma(part, f32x4(f[i].y), end[i]);
      carry = f[i].x < 0.f ? end[i] : __builtin_elementwise_fma(carry, f32x4(f[i].x), left);
    }
  }
}

// Gradients of shared key / value heads: the sum over the query heads that share one, from fp32 rows (N, T, H, d) -> T, of k's and
// v's heads in one launch.  Bound by the fp32 rows' read (mostly from the caches that they were just written through).  A thread
// adds up VEC columns; the 64-bit divisions that find its row are the workgroup's, once: with one element and its own divisions
// to a thread, 64 x 512 tokens of 8 heads over 2, 64 x 64 in bf16, took 2 x 23 us; now 23 us, 6.4 TB/s.
struct DaShare {
  const float* in;
  void* out;
  int64_t on, ot, oh;
  int d;
};
template <typename T, int VEC>
__global__ __launch_bounds__(256) void decay_attention_share_kernel(const DaShare of_k, const DaShare of_v, int64_t rows, int t, int hk, int group) {
  const DaShare a = blockIdx.y ? of_v : of_k;
  const int per = a.d / VEC, each = 256 / per, mine = (int)threadIdx.x / per, e = ((int)threadIdx.x - mine * per) * VEC;
  const int64_t first = (int64_t)blockIdx.x * each;  // rows (n, t, hk)
  if (mine >= each || first + mine >= rows) return;
  const int64_t first_nt = first / hk, first_n = first_nt / t;
  const int head_raw = (int)(first - first_nt * hk) + mine, t_raw = (int)(first_nt - first_n * t) + head_raw / hk;
  const int head = head_raw % hk, n_more = t_raw / t;
  const float* in = a.in + ((first + mine) * group) * a.d + e;
  float v[VEC] = {};
#pragma unroll 4
  for (int k = 0; k < group; ++k) {
    const Pack<float, VEC> x = *reinterpret_cast<const Pack<float, VEC>*>(in + k * a.d);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] += x.v[i];
  }
  Pack<T, VEC> y;
#pragma unroll
  for (int i = 0; i < VEC; ++i) y.v[i] = (T)v[i];
  *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.out) + (first_n + n_more) * a.on + (int64_t)(t_raw - n_more * t) * a.ot + head * a.oh + e) = y;
}

// ---------------------------------------------------------------- one token per sequence, the state updated in place
// Bound by the state's one read and one write (8 bytes per entry).  A wave (or a workgroup of four, for states of more than
// 8 KiB) owns one (sequence, head): lanes take 16-byte pieces of the state's rows, update them where they are and add
// q's product up over the rows they hold, then over the lanes and waves that share a column.  4096 environments x 4 heads, 64 x 64: 100 us,
// 5.3 TB/s; 1024 x 16 heads, 128 x 128: 413 us, 5.2 TB/s; one environment: 4 us, a launch's latency.
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
  // All pieces of a row are one access of one wave.  A piece across the row's end starts earlier instead: what it shares with the one
  // before both lanes read, update and store, to the same bits.
  const int rl = tid & (a.lanes - 1), r0 = tid / a.lanes, step = THREADS / a.lanes;
  const bool in = rl * VEC < a.dv;
  const int col = in ? run_start<VEC, ELEMS_LOOSE>(rl * VEC, a.dv) : 0;
  float vv[VEC], acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    vv[e] = rows[unit][2][col + e];
    acc[e] = 0.f;
  }
  if (in && live) {
    constexpr int U = 4;  // rows in flight
    for (int r = r0; r < a.dk; r += U * step) {
      Loose<float, VEC> s[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int row = r + i * step;
        s[i] = *reinterpret_cast<const Loose<float, VEC>*>(state + (row < a.dk ? row : r) * a.dv + col);
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
          *reinterpret_cast<Loose<float, VEC>*>(state + row * a.dv + col) = s[i];
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    for (int off = a.lanes; off < WAVE; off <<= 1) acc[e] += __shfl_xor(acc[e], off, WAVE);
    if (in && lane_id() < a.lanes) part[unit][tid >> 6][col + e] = acc[e];
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
constexpr int64_t DA_MAX_BLOCKS = ((int64_t)1 << 24) - 1;  // workgroups of 256: a launch's threads are counted in 32 bits

struct DaPlan {
  int nk, nv, slices, nseg;
  int64_t seg_len, seg_floats;  // scratch: states between segments and the segments' factors
};

// Tiles per wave: 16 NK rows cover dk, 16 NV columns are a slice of dv; at most 16 tiles (64 registers) of state.  Wider slices share
// q, k and their product among more columns (bf16, 64 x 64, 512 tokens of 4096 heads: 243 us with four tiles, 309 with two), narrower
// ones leave fewer columns empty behind dv: the width with the least matrix instructions over all slices is taken.  Calls that
// neither fill the chip nor have many tokens to a wave take narrower ones: the chain of one wave's blocks is what lasts (fp32,
// 64 x 64, 128 tokens of 256 heads: 38 us with four tiles, 31 with two, 22 with one; with 2048 tokens four are the best).
//
// A call with fewer waves than the chip has SIMDs is cut over time, into pieces of 64 tokens at least: the pieces' end states first,
// joined by one small launch, then every piece by itself.  Two launches more cost about 10 us: below 192 tokens (256 in bf16) the
// call stays whole (64 heads of 64 x 64, bf16: 128 tokens 18 us cut and 14 whole, 256 tokens 21 cut and 24 whole; fp32: 128 tokens
// 21 and 20, 192 tokens 23 and 28).  The aim is two waves per SIMD, and not one more, which would run alone behind the others.
// Where lengths differ every sequence's own tokens are cut evenly (bf16 prompts between a quarter and all of 8192 tokens, 4 x 16 heads
// of 128 x 128, mean of eight draws: 231 us; 252 with pieces of the same length in all, 247 with twice as many of them).
constexpr int64_t DA_FEW_WAVES = 1024, DA_WANT_WAVES = 2048, DA_WIDE_TOKENS = 12288;

static DaPlan decay_attention_plan(int64_t n, int64_t t, int h, int dk, int dv, bool bf16, int roles) {
  DaPlan p;
  p.nk = dk <= 16 && !bf16 ? 1 : dk <= 32 ? 2 : dk <= 64 ? 4 : 8;
  p.nv = 1;
  int64_t least = 0;
  for (int nv = 1; nv <= (p.nk == 8 ? 2 : 4); nv *= 2) {
    const int64_t slices = (dv + 16 * nv - 1) / (16 * nv), cost = slices * (4 * p.nk + 4 * nv + 8 * p.nk * nv);
    const int64_t waves = n * h * slices * roles;  // (n and h are in the products the launch checks; t is below 2^30)
    if (nv > 1 && waves < DA_FEW_WAVES && waves * t < DA_WIDE_TOKENS * nv * nv) break;
    if (nv == 1 || cost <= least) {
      least = cost;
      p.nv = nv;
    }
  }
  p.slices = (dv + 16 * p.nv - 1) / (16 * p.nv);
  const int64_t waves = n * h * p.slices * roles;
  p.nseg = 1;
  p.seg_len = t > 0 ? t : 1;
  if (waves < DA_FEW_WAVES && t >= (bf16 ? 4 : 3) * DA_MIN_SEGMENT) {
    int64_t want = DA_WANT_WAVES / waves;
    if (want > t / DA_MIN_SEGMENT) want = t / DA_MIN_SEGMENT;
    p.seg_len = (t + want - 1) / want;
    p.seg_len = (p.seg_len + DB_TOKENS - 1) / DB_TOKENS * DB_TOKENS;
    p.nseg = (int)((t + p.seg_len - 1) / p.seg_len);
  }
  p.seg_floats = p.nseg > 1 ? n * h * p.nseg * (p.slices * (int64_t)(p.nk * p.nv * 4 * WAVE) + 4) : 0;
  return p;
}

template <typename T, int NK, int NV, int MODE, bool BF16>
static int decay_attention_run(const DaRoles& in, const DaPlan& p, float* workspace, hipStream_t stream) {
  DaRoles r = in;
  const int64_t heads = r.c[0].n * r.c[0].h, units = heads * p.slices, groups = ((units + DA_WAVES - 1) / DA_WAVES + DA_XCDS - 1) / DA_XCDS;
  const int64_t blocks = groups * DA_XCDS * r.roles, per_head = (int64_t)p.slices * NK * NV * WAVE;  // the last in 16-byte quads
  OIGE_REQUIRE(blocks <= DA_MAX_BLOCKS,
               "decay_attention: %lld sequences x heads are too many for one launch", (long long)heads);
  for (int i = 0; i < r.roles; ++i) {
    DaCore& c = r.c[i];
    c.slices = p.slices;
    c.nseg = p.nseg;
    c.seg_len = (int)p.seg_len;
    if (p.nseg > 1) {
      c.seg_states = workspace + i * p.seg_floats;
      c.seg_factors = reinterpret_cast<float2*>(c.seg_states + heads * p.nseg * per_head * 4);
    }
  }
  void (*states)(DaRoles);
  void (*main)(DaRoles);
  if constexpr (BF16) {
    states = decay_attention_bf16_kernel<NK, NV, MODE, true>;
    main = decay_attention_bf16_kernel<NK, NV, MODE, false>;
  } else {
    states = decay_attention_kernel<T, NK, NV, MODE, true>;
    main = decay_attention_kernel<T, NK, NV, MODE, false>;
  }
  if (p.nseg > 1) {
    hipLaunchKernelGGL(states, dim3((unsigned)blocks, (unsigned)(p.nseg - 1)), dim3(DA_WAVES * WAVE), 0, stream, r);
    int rc = check_launch("decay_attention_kernel (states)");
    if (rc) return rc;
    const int64_t quads = heads * per_head;
    hipLaunchKernelGGL(decay_attention_join_kernel, dim3((unsigned)((quads + 255) / 256), (unsigned)r.roles), dim3(256), 0, stream, r, quads,
                       per_head, p.nseg);
    rc = check_launch("decay_attention_join_kernel");
    if (rc) return rc;
  }
  hipLaunchKernelGGL(main, dim3((unsigned)blocks, (unsigned)p.nseg), dim3(DA_WAVES * WAVE), 0, stream, r);
  return check_launch("decay_attention_kernel");
}

template <typename T, int MODE>
static int decay_attention_tiles(const DaRoles& c, const DaPlan& p, float* ws, hipStream_t s) {
  switch (p.nk * 8 + p.nv) {
    case 8 + 1: return decay_attention_run<T, 1, 1, MODE, false>(c, p, ws, s);
    case 8 + 2: return decay_attention_run<T, 1, 2, MODE, false>(c, p, ws, s);
    case 8 + 4: return decay_attention_run<T, 1, 4, MODE, false>(c, p, ws, s);
    case 16 + 1: return decay_attention_run<T, 2, 1, MODE, false>(c, p, ws, s);
    case 16 + 2: return decay_attention_run<T, 2, 2, MODE, false>(c, p, ws, s);
    case 16 + 4: return decay_attention_run<T, 2, 4, MODE, false>(c, p, ws, s);
    case 32 + 1: return decay_attention_run<T, 4, 1, MODE, false>(c, p, ws, s);
    case 32 + 2: return decay_attention_run<T, 4, 2, MODE, false>(c, p, ws, s);
    case 32 + 4: return decay_attention_run<T, 4, 4, MODE, false>(c, p, ws, s);
    case 64 + 1: return decay_attention_run<T, 8, 1, MODE, false>(c, p, ws, s);
    case 64 + 2: return decay_attention_run<T, 8, 2, MODE, false>(c, p, ws, s);
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

template <int MODE>
static int decay_attention_bf16_tiles(const DaRoles& c, const DaPlan& p, float* ws, hipStream_t s) {
  switch (p.nk * 8 + p.nv) {
    case 16 + 1: return decay_attention_run<__bf16, 2, 1, MODE, true>(c, p, ws, s);
    case 16 + 2: return decay_attention_run<__bf16, 2, 2, MODE, true>(c, p, ws, s);
    case 16 + 4: return decay_attention_run<__bf16, 2, 4, MODE, true>(c, p, ws, s);
    case 32 + 1: return decay_attention_run<__bf16, 4, 1, MODE, true>(c, p, ws, s);
    case 32 + 2: return decay_attention_run<__bf16, 4, 2, MODE, true>(c, p, ws, s);
    case 32 + 4: return decay_attention_run<__bf16, 4, 4, MODE, true>(c, p, ws, s);
    case 64 + 1: return decay_attention_run<__bf16, 8, 1, MODE, true>(c, p, ws, s);
    case 64 + 2: return decay_attention_run<__bf16, 8, 2, MODE, true>(c, p, ws, s);
  }
  return fail(OIGE_EINVAL, "decay_attention: no variant for %d x %d tiles", p.nk, p.nv);
}

// The kernel and the accesses that suit all of the roles, whose head sizes ask for the same tiles.  bf16 tensors have a kernel of
// their own, for heads of two columns at least (two to a register) and where a block of tokens spans less than 2^32 bytes.
static int decay_attention_core(const DaRoles& r, int dtype, float* ws, hipStream_t s) {
  const int64_t most = (int64_t)1 << 32, most_bf16 = (most - 1024) / (2 * DB_TOKENS);
  const int bytes = elem_bytes(dtype);
  bool wide = true, bf16 = dtype == OIGE_BF16;
  for (int i = 0; i < r.roles; ++i) {
    const DaCore& c = r.c[i];
    OIGE_REQUIRE(c.q.st >= 0 && c.q.st < most && c.k.st >= 0 && c.k.st < most && c.v.st >= 0 && c.v.st < most,
                 "decay_attention: token strides must be below 2^32 elements and not negative");
    wide = wide && da_wide(c, bytes);
    bf16 = bf16 && c.dk > 1 && c.q.st <= most_bf16 && c.k.st <= most_bf16 && c.v.st <= most_bf16 && c.ot <= most_bf16;
  }
  const DaCore& c = r.c[0];
  const DaPlan p = decay_attention_plan(c.n, c.t, c.h, c.dk, c.dv, bf16, r.roles);
  bool full = wide;
  for (int i = 0; i < r.roles; ++i) full = full && r.c[i].dk == 16 * p.nk && r.c[i].dv == 16 * p.nv * p.slices;
  if (bf16)
    return full ? decay_attention_bf16_tiles<ELEMS_FULL>(r, p, ws, s)
                : wide ? decay_attention_bf16_tiles<ELEMS_WIDE>(r, p, ws, s) : decay_attention_bf16_tiles<ELEMS_LOOSE>(r, p, ws, s);
  if (dtype == OIGE_BF16) return decay_attention_tiles<__bf16, ELEMS_LOOSE>(r, p, ws, s);
  if (dtype == OIGE_F16)
    return full ? decay_attention_tiles<_Float16, ELEMS_FULL>(r, p, ws, s)
                : wide ? decay_attention_tiles<_Float16, ELEMS_WIDE>(r, p, ws, s) : decay_attention_tiles<_Float16, ELEMS_LOOSE>(r, p, ws, s);
  return full ? decay_attention_tiles<float, ELEMS_FULL>(r, p, ws, s)
              : wide ? decay_attention_tiles<float, ELEMS_WIDE>(r, p, ws, s) : decay_attention_tiles<float, ELEMS_LOOSE>(r, p, ws, s);
}

// The share kernel's accesses and workgroups, checked in front of the pass's first launch.
struct DaSharePlan {
  DaShare k, v;
  bool wide;  // four columns to a thread
  int64_t rows, blocks;
};
static DaSharePlan decay_attention_share_plan(const float* in_k, const float* in_v, const oige_decay_attention_io& io) {
  const int64_t *sk = io.dk_stride, *sv = io.dv_stride;
  DaSharePlan p{{in_k, io.dk, sk[0], sk[1], sk[2], io.key_dim}, {in_v, io.dv, sv[0], sv[1], sv[2], io.value_dim}, true, 0, 0};
  for (const DaShare& x : {p.k, p.v})
    p.wide = p.wide && x.d % 4 == 0 && x.on % 4 == 0 && x.ot % 4 == 0 && x.oh % 4 == 0 && aligned16(x.in) && aligned16(x.out);
  p.rows = io.num_envs * io.num_tokens * io.kv_heads;
  const int d = io.key_dim > io.value_dim ? io.key_dim : io.value_dim, each = 256 / (p.wide ? d / 4 : d);
  p.blocks = (p.rows + each - 1) / each;
  return p;
}
static int decay_attention_share(const DaSharePlan& p, const oige_decay_attention_io& io, hipStream_t s) {
  const dim3 grid((unsigned)p.blocks, 2);
  const int t = (int)io.num_tokens, hk = (int)io.kv_heads, group = io.heads / io.kv_heads;
#define OIGE_SHARE(T)                                                                                                                    \
  do {                                                                                                                                   \
    if (p.wide) hipLaunchKernelGGL((decay_attention_share_kernel<T, 4>), grid, dim3(256), 0, s, p.k, p.v, p.rows, t, hk, group);         \
    else hipLaunchKernelGGL((decay_attention_share_kernel<T, 1>), grid, dim3(256), 0, s, p.k, p.v, p.rows, t, hk, group);                \
  } while (0)
  if (io.dtype == OIGE_F32) OIGE_SHARE(float);
  else if (io.dtype == OIGE_F16) OIGE_SHARE(_Float16);
  else OIGE_SHARE(__bf16);
#undef OIGE_SHARE
  return check_launch("decay_attention_share_kernel");
}

static int decay_attention_check(const oige_decay_attention_io* io, const char* what) {
  OIGE_REQUIRE(io != nullptr, "%s: null io", what);
  OIGE_REQUIRE(elem_bytes(io->dtype), "%s: dtype must be OIGE_F32, OIGE_F16 or OIGE_BF16", what);
  OIGE_REQUIRE(io->num_envs >= 0 && io->num_tokens >= 0 && io->num_tokens < ((int64_t)1 << 30), "%s: %lld sequences of %lld tokens", what,
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

// Head sizes that ask for the same tiles in either order: the backward pass is one launch of three roles.
static bool da_square(const oige_decay_attention_io& io) {
  bool same = true;
  for (int bf16 = 0; bf16 < 2; ++bf16) {
    const DaPlan a = decay_attention_plan(io.num_envs, io.num_tokens, io.heads, io.key_dim, io.value_dim, bf16, 3);
    const DaPlan b = decay_attention_plan(io.num_envs, io.num_tokens, io.heads, io.value_dim, io.key_dim, bf16, 3);
    same = same && a.nk == b.nk && a.nv == b.nv && a.slices == b.slices;
  }
  return same;
}
static int64_t da_seg_floats(const oige_decay_attention_io& io, int dk, int dv, int roles) {
  const int64_t f = decay_attention_plan(io.num_envs, io.num_tokens, io.heads, dk, dv, false, roles).seg_floats;
  const int64_t b = decay_attention_plan(io.num_envs, io.num_tokens, io.heads, dk, dv, true, roles).seg_floats;
  return ((f > b && io.dtype == OIGE_BF16) || io.dtype != OIGE_BF16 ? f : b) * roles;
}
static int64_t da_workspace(const oige_decay_attention_io& io, bool backward) {
  if (!backward) return da_seg_floats(io, io.key_dim, io.value_dim, 1);
  int64_t most = da_seg_floats(io, io.key_dim, io.value_dim, 3);
  if (!da_square(io)) {
    const int64_t a = da_seg_floats(io, io.value_dim, io.key_dim, 1), b = da_seg_floats(io, io.key_dim, io.value_dim, 1);
    most = a > b ? a : b;
  }
  most = (most + 3) / 4 * 4;
  return most + (io.heads != io.kv_heads ? io.num_envs * io.num_tokens * io.heads * (io.key_dim + io.value_dim) : 0);  // rows per query head
}

static DaCore da_core(const oige_decay_attention_io& io) {
  DaCore c{};
  c.decay = io.decay;
  c.resets = io.resets;
  c.lengths = io.lengths;
  c.rsn = io.resets_stride[0];
  c.rst = io.resets_stride[1];
  c.n = io.num_envs;
  c.t = (int)io.num_tokens;
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
  OIGE_REQUIRE(!io->state_out || io->state_out != io->state_in, "decay_attention_forward: state_out must not be state_in (other waves still read it)");
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
  DaRoles r{};
  r.c[0] = c;
  r.roles = 1;
  return decay_attention_core(r, io->dtype, io->workspace, (hipStream_t)stream);
}

int oige_decay_attention_backward(const oige_decay_attention_io* io, oige_stream_t stream) {
  int rc = decay_attention_check(io, "decay_attention_backward");
  if (rc) return rc;
  if (io->num_envs == 0) return OIGE_OK;
  OIGE_REQUIRE(io->num_tokens == 0 || (io->q && io->k && io->v && io->d_o && io->dq && io->dk && io->dv),
               "decay_attention_backward: null q, k, v, d_o, dq, dk or dv");
  OIGE_REQUIRE(io->num_tokens > 0 || io->d_state_in, "decay_attention_backward: no tokens and no initial state's gradient asked for");
  OIGE_REQUIRE(!io->d_state_in || (io->d_state_in != io->d_state_out && io->d_state_in != io->state_in),
               "decay_attention_backward: d_state_in must be neither d_state_out nor state_in (other waves still read them)");
  const int64_t need = da_workspace(*io, true);
  OIGE_REQUIRE(need == 0 || (io->workspace && aligned16(io->workspace) && io->workspace_floats >= need),
               "decay_attention_backward: needs a 16-byte aligned workspace of %lld floats", (long long)need);
  hipStream_t s = (hipStream_t)stream;
  const int group = io->heads / io->kv_heads;
  const DaRows q = da_rows(io->q, io->q_stride, 1), k = da_rows(io->k, io->k_stride, group), v = da_rows(io->v, io->v_stride, group),
               d_o = da_rows(io->d_o, io->d_o_stride, 1);
  // shared heads: dk and dv per query head in fp32 behind the segments' scratch, then their sums
  const int64_t t = io->num_tokens, h = io->heads;
  float *wide_v = nullptr, *wide_k = nullptr;
  DaSharePlan share{};
  if (group > 1) {
    wide_v = io->workspace + (need - io->num_envs * t * h * (io->key_dim + io->value_dim));
    wide_k = wide_v + io->num_envs * t * h * io->value_dim;
    share = decay_attention_share_plan(wide_k, wide_v, *io);
    OIGE_REQUIRE(share.blocks <= DA_MAX_BLOCKS, "decay_attention_backward: %lld key / value rows are too many for one launch", (long long)share.rows);
  }
  const int64_t rows_v[3] = {t * h * io->value_dim, h * io->value_dim, io->value_dim}, rows_k[3] = {t * h * io->key_dim, h * io->key_dim, io->key_dim};
  DaRoles r{};
  for (int i = 0; i < 3; ++i) {
    DaCore& c = r.c[i];
    c = da_core(*io);
    c.dk = i == 0 ? io->key_dim : io->value_dim;
    c.dv = i == 0 ? io->value_dim : io->key_dim;
    if (i < 2) {
      c.reverse = 1;
      c.s_in = io->d_state_out;
      c.kv_scale = io->scale;
      c.o_float = group > 1;
    }
  }
  // dv_t = G_t^T k_t, and the initial state's gradient
  r.c[0].q = k;
  r.c[0].k = q;
  r.c[0].v = d_o;
  da_out(r.c[0], wide_v ? wide_v : io->dv, wide_v ? rows_v : io->dv_stride);
  r.c[0].s_out = io->d_state_in;
  // dk_t = G_t v_t
  r.c[1].q = v;
  r.c[1].k = d_o;
  r.c[1].v = q;
  da_out(r.c[1], wide_k ? wide_k : io->dk, wide_k ? rows_k : io->dk_stride);
  r.c[1].transposed = 1;
  // dq_t = scale S_t do_t
  r.c[2].q = d_o;
  r.c[2].k = v;
  r.c[2].v = k;
  da_out(r.c[2], io->dq, io->dq_stride);
  r.c[2].s_in = io->state_in;
  r.c[2].transposed = 1;
  r.c[2].out_scale = io->scale;
  if (t == 0) {
    r.roles = 1;  // the state's gradient passes through
    return decay_attention_core(r, io->dtype, io->workspace, s);
  }
  if (da_square(*io)) {
    r.roles = 3;
    rc = decay_attention_core(r, io->dtype, io->workspace, s);
    if (rc) return rc;
  } else {
    for (int i = 0; i < 3; ++i) {
      DaRoles one{};
      one.c[0] = r.c[i];
      one.roles = 1;
      rc = decay_attention_core(one, io->dtype, io->workspace, s);
      if (rc) return rc;
    }
  }
  if (group == 1) return OIGE_OK;
  return decay_attention_share(share, *io, s);
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
  const bool wide = io->value_dim >= 4;  // on any boundary: 64 x 63 fp32, 4096 x 4 heads, took 117 us by single floats, 85 now
  const int pieces = wide ? (io->value_dim + 3) / 4 : io->value_dim;
  a.lanes = 1;
  while (a.lanes < pieces) a.lanes *= 2;  // 32 at most
  const bool big = io->key_dim * io->value_dim > 2048;
  const int64_t units = a.n * a.h, blocks = big ? units : (units + 3) / 4;
  OIGE_REQUIRE(blocks <= DA_MAX_BLOCKS, "decay_attention_step: %lld sequences x heads are too many for one launch", (long long)units);
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
