// Attention of serving layers: a batch's queries over keys whose number differs by sample, with shared K/V heads, and over
// a prefix that all samples share (the history of hy_nomas/model.py:199-223, stored as hy_nomas/world.py:83-90 does).
//
//   out[b, i, h, :] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[b, i, h, :] . k_j - m),  m the largest score,
//
// over the keys j that query (b, i) sees, of K/V head h / (Hq / Hkv); zeros where it sees none.
//
// Rows.  The queries that read the same keys are the rows of one matrix: the G = Hq / Hkv heads of a K/V head, all queries of
// the sample, and for a prefix those of every sample, so that up to 128 rows of all samples share a read of its keys (a short
// prefix, and one that many own rows walk anyway, is walked for each sample together with its own keys: see plan_rows).  A
// workgroup of 4 waves walks keys in tiles with a running maximum and sum: 128 rows, a wave 32, over tiles of 64 keys that
// the waves share; up to 64 rows, two waves a group of 32 rows and each half a tile's keys; up to 32 rows, every wave all rows and
// tiles of its own.  Each kind in its place in the present kernel, us: four calls (4 samples x 300 keys, 32 heads on 8; 8 samples
// over 2047 shared and 129 own keys; 64 over 32768 and 600; 16 of 4 queries over 15840 int8 keys and 260, 24 heads) take
// 10.4, 11.6, 61.3 and 62.5 with the first kind alone, 9.2, 11.9, 61.3 and 48.5 with the third, 9.2, 11.9, 60.9 and 42.7 with all
// three; 16 x 48 queries over 2000 keys 47.4 in 128-row blocks, 48.7 in half ones, 16 x 24 there 43.2, as few rows 44.3.
//
// What bounds it.  Many rows: a wave's chain of products and exponentials, of which two waves a SIMD hide a part; 4 x 2000
// queries of 32 heads on 8 over 8192 shared keys 1140 us, 1050 TFLOP/s, half the matrix cores' cycles at the clock that the
// power limit leaves.  Few rows: memory; 32 samples x 4100 keys of 16 heads of 64 dims 84 us, 5 TB/s, which is what 128-byte
// pieces 2 KB apart stream at.  Short calls: the launch and a workgroup's chain from the lengths to the last join.
//
// Products.  Scores transposed, S^T = K Q^T (keys as the A rows of the 32x32x16 product, query rows as the B columns): a lane
// holds one row and 16 keys of each 32-key block, keys 8 (r / 4) + 4 h + r % 4 in register r of lane half h.  The output
// transposed too, O^T = V^T P^T: the probabilities are the B operand straight from the score registers, and the A operand's
// keys 16 g + 4 h + 0..3 and 16 g + 8 + 4 h + 0..3 of one dim come from the V tile as it lies (keys as rows) by gfx950's
// transposing LDS reads, four keys of 16 dims a 16-lane group: no V^T is made in memory.
//
// LDS.  K rows: 16-byte chunk c of row r at c ^ (r & 15) (128 dims) or c ^ ((r >> 1) & 7) (64 dims).  V rows, whose reads take
// 64 bytes of 4 rows: c ^ (4 (r & 3) + (r & 1)) or c ^ (5 ((r >> 1) & 1)); the low bit spreads the widened int8 rows' writes.
// Every read spreads over all banks, and so do the direct loads.  (The widened int8 rows' 16-byte writes do not: 0.24 cycles of
// conflicts a cycle of LDS access for 16 x 4 queries over 15840 int8 keys, 0.006 without these writes.)  Direct-to-LDS loads one tile ahead, two buffers, one barrier a tile; the lane fetches
// the logical chunk of its physical slot.
//
// int8 keys (a history as stored) pass through registers: loaded a tile ahead, widened once a workgroup, while the score products
// of the tile before run, and written to the same LDS layout.  Codes are exact in bf16 and fp16, so the key scale
// multiplies the fp32 score and the value scale the fp32 probability, before its one rounding.  (In fp16, whose range a
// probability times a scale could leave, the reference is that of the products: scores plus the scales' logarithms.)
//
// Hidden keys.  A tile's seen keys are one 64-bit mask.  Rows that are not seen are loaded from a seen row of the tile, so that
// nothing they hold enters a product; a tile without a seen key is passed over.  Under a causal limit some rows of a tile see a
// key that others do not, and a value of it that is not finite reaches these as 0 times it: a row with a result that is not
// finite, and with keys that it does not see, is walked again by a wave over the keys that it sees (`mend_row`).
//
// Splits.  Where the rows leave compute units idle, several workgroups take ranges of the tiles and leave fp32 partials with
// their reference maximum and sum, which row_combine_kernel joins; a prefix and the samples' own keys are joined the same way.  An
// int8 prefix is always a job of its own (a workgroup's tiles are of one type), so each row of such a call leaves at least two
// partials of D + 2 floats: 2 GB for 16 x 4096 queries of 32 heads, some 0.7 of the 13 ms that they take over 8192 shared and 4096
// own keys.  Next to a short prefix it shows: 4 x 2000 queries over 64 and 2000 keys 287 us, 178 with a bf16 prefix in one pass.
//
// The reference maximum moves only when a tile's maximum exceeds it by more than 8 (base 2), so that the accumulators are
// rescaled a few times a row; the quotient is the same.
#include <type_traits>

#include "hn_common.h"

namespace hn {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int v4i_r __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;

constexpr int kRows = 128;    // rows of a workgroup of many
constexpr int kKeys = 64;     // keys of a tile
constexpr int kWaves = 4;
constexpr float kSlack = 8.0f;

// A run of keys: strides in elements, `len` keys at most, `lengths` the keys of each sample (32 or 64 bits) or null,
// `mask` one byte a key (0: hidden) or null.  With ks / vs, k and v are int8 codes and these their scales.
struct KeySource {
  const void *k, *v;
  int64_t skb, skh, skj, svb, svh, svj;
  const float *ks, *vs;
  int64_t ksh, ksj, vsh, vsj;
  int64_t len;
  const void* lengths;
  int lengths64;
  const uint8_t* mask;
  int64_t smb;
  int causal;  // the sample's last keys are its Lq queries' own: query i sees keys up to n - Lq + i
};

// Division of numbers below 2^31 by d from 1 to 2^31: with s = ceil(log2 d) and mul = floor(2^(31 + s) / d) + 1 the error
// mul d - 2^(31 + s) lies in (0, 2^s], so that n mul / 2^(31 + s) has the quotient as its whole part.  (A workgroup makes a
// dozen divisions before its first tile; numbers that are the same in a wave take two scalar instructions each.)
struct Divisor {
  uint32_t mul, shift;
  void set(int64_t d) {
    shift = 0;
    while (((int64_t)1 << shift) < d) shift++;
    mul = (uint32_t)(((uint64_t)1 << (31 + shift)) / (uint64_t)d + 1);
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)(__umulhi(2u * (uint32_t)n, mul) >> shift); }
};

enum JobKind { kFew, kHalf, kMany };  // up to 32 rows a unit, up to 64, more

// Rows that walk the same sources: `units` of them (K/V heads, or samples times K/V heads), each in `blocks` blocks of kRows
// rows (one, but for many rows) and `splits` ranges of tiles, from workgroup `wg0` on; partials from slot `slot0` on.

struct RowJob {
  JobKind kind;
  int64_t wg0;
  int rows, stacked;  // rows of a unit; they run over the samples too
  int units;
  int blocks, splits, slot0;
  int src0, nsrc;
  Divisor by_group, by_last, by_units, by_splits;  // group: the workgroups of 8 units and ranges; last: the last one's width
};

struct RowArgs {
  const uint16_t* q;
  int64_t sqb, sqh, sqi;
  uint16_t* o;
  int64_t sob, soh, soi;
  KeySource src[2];
  RowJob job[2];
  int njobs;
  int slots;          // of partials; 0: the results are final
  float* po;          // [slot][row id][D], row id (b Lq + i) Hq + h
  float2* pml;        // [slot][row id]: reference maximum (base 2) and sum
  int64_t ids;
  int64_t B, Lq;
  int Hq, Hkv, G;
  Divisor by_hkv, by_g, by_per, by_hq, by_lq;  // per: Lq G
  float scale_log2;
};

__device__ __forceinline__ int64_t sample_length(const KeySource& s, int64_t b) {
  if (s.lengths == nullptr) return s.len;
  const int64_t n = s.lengths64 ? ((const int64_t*)s.lengths)[b] : ((const int32_t*)s.lengths)[b];
  return n < 0 ? 0 : n > s.len ? s.len : n;
}

template <int DT>
__device__ __forceinline__ v16f mma(v4i_r a, v4i_r b, v16f c) {
  if constexpr (DT == HN_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// two fp32 values -> the packed pair, to nearest even by the hardware pair conversion (a NaN stays one)
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == HN_DTYPE_BF16) {
    return bf16x2_finite(a, b);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
  }
}

// four int8 codes -> four values of the type (exact)
template <int DT>
__device__ __forceinline__ uint2 widen_codes(uint32_t w) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; i++) f[i] = (float)(int)(int8_t)(w >> (8 * i));
  if constexpr (DT == HN_DTYPE_BF16)  // whole numbers up to 128: the low halves are zero
    return make_uint2(__builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u),
                      __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u));
  else
    return make_uint2(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]));
}

__device__ __forceinline__ float row_max_xor32(float x) {  // max over lanes l and l ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// this wave's loads are done, direct ones among them, and its stores, which the same counter holds
__device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // vmcnt(0)
  asm volatile("" ::: "memory");
}

// lane `from`'s pointer
template <typename P>
__device__ __forceinline__ P* of_lane(P* mine, int from) {
  const uint64_t v = reinterpret_cast<uint64_t>(mine);
  const uint32_t lo = __builtin_amdgcn_ds_bpermute(from * 4, (int)(uint32_t)v), hi = __builtin_amdgcn_ds_bpermute(from * 4, (int)(v >> 32));
  return reinterpret_cast<P*>((uint64_t)hi << 32 | lo);
}

// every load and LDS access of this wave is done, and then every wave's
__device__ __forceinline__ void tile_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // vmcnt(0)
  __builtin_amdgcn_s_waitcnt(0xc07f);                // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// the same for LDS accesses alone
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 16 bytes a lane at base + voff + soff (soff the same in the wave)
__device__ __forceinline__ v4i_r load16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_bit_cast(v4i_r, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0));
}

typedef uint32_t out8 __attribute__((ext_vector_type(4), aligned(8)));  // (an output row is 8-byte aligned)

__device__ __forceinline__ uint64_t low_bits(int k) { return k >= 64 ? ~0ull : (1ull << k) - 1; }

// Where a lane's pieces of K and V rows lie in LDS.
template <int D>
struct Rows {
  static constexpr int kRow = D * 2;  // bytes of a K or V row
  static constexpr int kChunks = kRow / 16;
  __device__ __forceinline__ static int kswz(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
  __device__ __forceinline__ static int vswz(int r) { return D == 128 ? (r & 3) << 2 | (r & 1) : ((r >> 1) & 1) * 5; }
};

// A workgroup's unit, range of tiles and row block.  Workgroups go to the eight XCDs in turn, each with an L2 of its own: the
// row blocks that walk the same tiles are put eight apart, so that one XCD reads the tiles once.
struct Share {
  int unit, split, block;
  __device__ __forceinline__ Share(const RowJob& job, int index) {
    const int group = job.by_group(index), r = index - group * 8 * job.blocks;
    const int wide = min(8, job.units * job.splits - group * 8);  // the last group may be narrower
    block = wide == 8 ? r >> 3 : job.by_last(r);
    const int at = group * 8 + r - block * wide;
    split = job.by_units(at);
    unit = at - split * job.units;
  }
};

// The sample, query and query head of a unit's row.
__device__ __forceinline__ void locate(const RowArgs& a, const RowJob& job, int unit, int row, int64_t& b, int& qi, int& h) {
  const int of = a.by_hkv(unit), sample = job.stacked ? a.by_per(row) : 0;
  const int in = row - sample * (int)a.Lq * a.G;
  b = job.stacked ? sample : of;
  qi = a.by_g(in);
  h = (unit - of * a.Hkv) * a.G + in - qi * a.G;
}

// Where range `split` of `total` begins: the first total % splits ranges are one longer.
__device__ __forceinline__ int range_start(const RowJob& job, int total, int split) {
  const int each = job.by_splits(total);
  return split * each + min(split, total - each * job.splits);
}

// A unit's and a lane's place: the query row of lane l (lanes l and l + 32 share one) and the keys it may see.
struct Place {
  int hk, qi, h;
  int64_t b_unit, b;
  int n[2];      // keys of the job's sources, up to the last one that any row up to `last_row` sees
  int row_keys;  // causal: the own keys that this lane's row sees
  bool causal;
  __device__ __forceinline__ Place(const RowArgs& a, const RowJob& job, const KeySource* src, int nsrc, int unit, int row, int last_row) {
    const int of = a.by_hkv(unit);
    hk = unit - of * a.Hkv;
    b_unit = of;  // 0 for stacked rows
    locate(a, job, unit, min(row, job.rows - 1), b, qi, h);
    int own = 0;
#pragma unroll
    for (int t = 0; t < 2; t++) {
      n[t] = 0;
      if (t < nsrc) {
        const KeySource& s = src[t];
        n[t] = (int)sample_length(s, b_unit);
        if (s.causal) {
          own = n[t];
          n[t] = max(0, min(n[t], n[t] - (int)a.Lq + a.by_g(min(last_row, job.rows - 1)) + 1));
        }
      }
    }
    causal = src[nsrc - 1].causal;
    row_keys = own - (int)a.Lq + qi + 1;
  }
};

// The running attention of a wave's 32 rows over tiles of NKB blocks of 32 keys in LDS.
// QL: the rows' fragments are read from LDS for every tile, where the registers are needed for tiles in flight.
template <int DT, int D, bool I8, int NKB, bool QL>
struct RowCore {
  static constexpr int KS = D / 16, DB = D / 32, kRow = Rows<D>::kRow;
  // fp16 codes: the reference follows the scores with the value scales' logarithms added, so that the probabilities times
  // these scales, not the probabilities, are what stays under 2^8 and next to it
  static constexpr bool kWeighted = I8 && DT == HN_DTYPE_F16;
  v4i_r qf[QL ? 1 : KS];  // the rows' B fragments
  const char* qrow;       // QL: the lane's row in LDS, laid out as K rows
  v16f oacc[DB];
  // the reference maximum m (base-2 units, -inf until a score is seen); the score products start from -m / scale_log2, so
  // that a probability is exp2(s scale_log2) (I8: the fused product with the key scale adds it)
  v16f mref;  // (I8: one register)
  float m, mref_m, lsum, scale_log2, inv_scale;
  int h2, krow, kx, voffs[DB];

  // the lane's fragments, from memory
  __device__ __forceinline__ static void load_rows(const RowArgs& a, const Place& at, int lane, v4i_r (&f)[KS]) {
    const uint16_t* qp = a.q + at.b * a.sqb + at.h * a.sqh + at.qi * a.sqi + 8 * (lane >> 5);
#pragma unroll
    for (int ks = 0; ks < KS; ks++) f[ks] = *reinterpret_cast<const v4i_r*>(qp + 16 * ks);
  }

  // `ql`: LDS for the 32 rows (QL), written by every wave alike
  __device__ __forceinline__ RowCore(const RowArgs& a, const v4i_r (&f)[KS], int lane, char* ql) : RowCore(a, lane) {
    qrow = ql + (lane & 31) * kRow;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      if constexpr (QL) *reinterpret_cast<v4i_r*>(const_cast<char*>(qrow) + (((2 * ks + h2) ^ kx) << 4)) = f[ks];
      else qf[ks] = f[ks];
    }
  }
  __device__ __forceinline__ RowCore(const RowArgs& a, int lane) {  // (the rows follow)
    h2 = lane >> 5;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
      for (int r = 0; r < 16; r++) oacc[db][r] = 0.0f;
    scale_log2 = a.scale_log2;
    inv_scale = 1.0f / a.scale_log2;
    m = -__builtin_inff();
    set_reference(0.0f);
    lsum = 0.0f;
    krow = (lane & 31) * kRow;
    kx = Rows<D>::kswz(lane & 31);
    const int rj = (lane & 15) >> 2;  // the row of its 4-key group that the lane reads for a transposing read
    const int turn = D == 128 ? rj & 1 : rj >> 1;  // the swizzle's low bit
    const int vrow = (4 * h2 + rj) * kRow + ((lane >> 4) & 1) * 32 + (((lane >> 1) & 1) ^ turn) * 16 + (lane & 1) * 8;
#pragma unroll
    for (int db = 0; db < DB; db++) voffs[db] = vrow + ((db ^ (D == 128 ? rj : rj >> 1)) << 6);
  }

  // A value scale's logarithm in units of the scores, for scales of 2^-40 to 2^60: fp16 results cannot tell smaller ones from
  // zero, and larger ones leave the type.
  __device__ __forceinline__ float scale_log(float vs) const {
    return __builtin_amdgcn_logf(__builtin_fminf(__builtin_fmaxf(__builtin_fabsf(vs), 0x1p-40f), 0x1p60f)) * inv_scale;
  }

  __device__ __forceinline__ void set_reference(float base2) {
    mref_m = base2;
    const float r = -base2 * inv_scale;
#pragma unroll
    for (int i = 0; i < (I8 ? 1 : 16); i++) mref[i] = r;
  }

  // S^T of a tile: the lane's row against keys 32 kb + 8 (r / 4) + 4 h2 + r % 4, relative to the reference
  __device__ __forceinline__ void scores(const char* kl, const float* kscale, v16f (&sc)[NKB]) {
    v16f zero;
#pragma unroll
    for (int r = 0; r < 16; r++) zero[r] = 0.0f;
    int x = (kx ^ h2) << 4;  // chunk 2 ks + h2 of the lane's row: 32 ks ^ x
    if constexpr (QL) asm volatile("" : "+v"(x));  // (the places are worked out for each tile: their registers hold tiles)
    // the fragments two steps ahead of their products (a ring of three), the order pinned
    v4i_r kf[3][NKB], q[3];
    auto read = [&](int ks) __attribute__((always_inline)) {
      const int at = (32 * ks) ^ x;
      if constexpr (QL) q[ks % 3] = *reinterpret_cast<const v4i_r*>(qrow + at);
#pragma unroll
      for (int kb = 0; kb < NKB; kb++) kf[ks % 3][kb] = *reinterpret_cast<const v4i_r*>(kl + 32 * kb * kRow + krow + at);
    };
    read(0);
    read(1);
    if constexpr (!QL) __builtin_amdgcn_sched_group_barrier(0x100, 2 * NKB, 0);
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
#pragma unroll
      for (int kb = 0; kb < NKB; kb++)
        sc[kb] = mma<DT>(kf[ks % 3][kb], QL ? q[ks % 3] : qf[QL ? 0 : ks], ks == 0 ? (I8 ? zero : mref) : sc[kb]);
      if constexpr (!QL) __builtin_amdgcn_sched_group_barrier(0x008, NKB, 0);
      if (ks + 2 < KS) {
        read(ks + 2);
        if constexpr (!QL) __builtin_amdgcn_sched_group_barrier(0x100, NKB, 0);
      }
    }
    if constexpr (I8) {
#pragma unroll
      for (int kb = 0; kb < NKB; kb++)
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++) {
          const float4 k4 = *reinterpret_cast<const float4*>(kscale + 32 * kb + 8 * q4 + 4 * h2);
          sc[kb][4 * q4] = __builtin_fmaf(sc[kb][4 * q4], k4.x, mref[0]);
          sc[kb][4 * q4 + 1] = __builtin_fmaf(sc[kb][4 * q4 + 1], k4.y, mref[0]);
          sc[kb][4 * q4 + 2] = __builtin_fmaf(sc[kb][4 * q4 + 2], k4.z, mref[0]);
          sc[kb][4 * q4 + 3] = __builtin_fmaf(sc[kb][4 * q4 + 3], k4.w, mref[0]);
        }
    }
  }

  // hides the keys whose bits are clear, and those from `lim` on in this lane's row
  __device__ __forceinline__ void hide(v16f (&sc)[NKB], uint64_t bits, bool causal, int lim) {
    if (bits != low_bits(32 * NKB)) {
      const uint64_t mine = ~bits >> (4 * h2);
      uint32_t word[2] = {(uint32_t)mine, (uint32_t)(mine >> 32)};
      asm volatile("" : "+v"(word[0]), "+v"(word[1]));  // (stays in the branch: whole tiles are the usual case)
#pragma unroll
      for (int kb = 0; kb < NKB; kb++)
#pragma unroll
        for (int r = 0; r < 16; r++)
        {  // (a bit of the hidden ones over the whole register chooses, two instructions a score)
          uint32_t gone = (uint32_t)__builtin_amdgcn_sbfe((int)word[kb], 8 * (r / 4) + r % 4, 1);
          asm("" : "+v"(gone));  // (or it becomes a test, a compare and a select with waits between)
          sc[kb][r] = __uint_as_float((gone & 0xff800000u) | (~gone & __float_as_uint(sc[kb][r])));
        }
    }
    if (causal && __builtin_amdgcn_ballot_w64(lim < 32 * NKB) != 0) {
      int mine = lim - 4 * h2;
      asm volatile("" : "+v"(mine));
#pragma unroll
      for (int kb = 0; kb < NKB; kb++)
#pragma unroll
        for (int r = 0; r < 16; r++)
          if (32 * kb + 8 * (r / 4) + r % 4 >= mine) sc[kb][r] = -__builtin_inff();
    }
  }

  // the tile's probabilities as packed pairs, the running reference and sum moved along
  __device__ __forceinline__ void softmax(v16f (&sc)[NKB], const float* vscale, const float* vlog, uint32_t (&pk)[NKB][8]) {
    float mx = -__builtin_inff();
#pragma unroll
    for (int kb = 0; kb < NKB; kb++)
#pragma unroll
      for (int q4 = 0; q4 < 4; q4++) {
        float4 l4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if constexpr (kWeighted) l4 = *reinterpret_cast<const float4*>(vlog + 32 * kb + 8 * q4 + 4 * h2);
        const float l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
        for (int i = 0; i < 4; i++) mx = __builtin_fmaxf(mx, kWeighted ? sc[kb][4 * q4 + i] + l[i] : sc[kb][4 * q4 + i]);
      }
    const float mrel = row_max_xor32(mx) * scale_log2;  // the tile's maximum, relative to the reference
    if (__builtin_amdgcn_ballot_w64(!(mrel + mref_m <= m + kSlack)) != 0) {
      const float mt = mrel + mref_m;
      const bool grow = mt > m + kSlack;
      const float mnew = grow ? mt : mref_m;
      const float alpha = grow ? __builtin_amdgcn_exp2f(m - mt) : 1.0f;  // 0 for the first scores
      m = grow ? mt : m;
      if (__builtin_amdgcn_ballot_w64(lsum != 0.0f) != 0) {  // (a wave's first scores find nothing to rescale)
        lsum *= alpha;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
          for (int r = 0; r < 16; r++) oacc[db][r] *= alpha;
      }
      const float delta = (mref_m - mnew) * inv_scale;
#pragma unroll
      for (int kb = 0; kb < NKB; kb++)
#pragma unroll
        for (int r = 0; r < 16; r++) sc[kb][r] += delta;
      set_reference(mnew);
    }
#pragma unroll
    for (int kb = 0; kb < NKB; kb++)
#pragma unroll
      for (int q4 = 0; q4 < 4; q4++) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = __builtin_amdgcn_exp2f(sc[kb][4 * q4 + i] * scale_log2);
        lsum += (e[0] + e[1]) + (e[2] + e[3]);
        if constexpr (I8) {
          const float4 v4 = *reinterpret_cast<const float4*>(vscale + 32 * kb + 8 * q4 + 4 * h2);
          e[0] *= v4.x; e[1] *= v4.y; e[2] *= v4.z; e[3] *= v4.w;
        }
        pk[kb][2 * q4] = pack2<DT>(e[0], e[1]);
        pk[kb][2 * q4 + 1] = pack2<DT>(e[2], e[3]);
      }
  }

  // O^T += V^T P^T
  __device__ __forceinline__ void values(const char* vl, const uint32_t (&pk)[NKB][8]) {
#pragma unroll
    for (int kb = 0; kb < NKB; kb++)
#pragma unroll
      for (int k2 = 0; k2 < 2; k2++) {
        const v4i_r bi = {(int)pk[kb][4 * k2], (int)pk[kb][4 * k2 + 1], (int)pk[kb][4 * k2 + 2], (int)pk[kb][4 * k2 + 3]};
        const char* vg = vl + (32 * kb + 16 * k2) * kRow;
#pragma unroll
        for (int db = 0; db < DB; db++) {
          const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(vg + voffs[db]));
          const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(vg + 8 * kRow + voffs[db]));
          typedef short v8s __attribute__((ext_vector_type(8)));
          const v8s af = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          oacc[db] = mma<DT>(__builtin_bit_cast(v4i_r, af), bi, oacc[db]);
        }
      }
  }

  __device__ __forceinline__ bool finite() const {  // the lane's results
    float x = 0.0f;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
      for (int r = 0; r < 16; r++) x = __builtin_fmaf(oacc[db][r], 0.0f, x);
    return x == 0.0f;
  }

  __device__ __forceinline__ float total() const { return lsum + __shfl_xor(lsum, 32); }
};

// 16 codes of a K or V row (16-byte piece c) to LDS, widened to the type: chunks 2 c and 2 c + 1
template <int DT>
__device__ __forceinline__ void store_codes(char* row, int swz, int c, v4i_r w) {
  const uint2 a0 = widen_codes<DT>(w[0]), a1 = widen_codes<DT>(w[1]);
  const uint2 b0 = widen_codes<DT>(w[2]), b1 = widen_codes<DT>(w[3]);
  *reinterpret_cast<uint4*>(row + (((2 * c) ^ swz) << 4)) = make_uint4(a0.x, a0.y, a1.x, a1.y);
  *reinterpret_cast<uint4*>(row + (((2 * c + 1) ^ swz) << 4)) = make_uint4(b0.x, b0.y, b1.x, b1.y);
}

// One row's attention again, by a whole wave over the keys that the row sees and no others, in fp32: 64 keys a step, D / 8 lanes a
// key and 8 dims a lane, for K and V alike.  For rows whose result is not finite under a causal limit although their scores are,
// so that what a later token's values hold stays with the rows that see it; slow beside the tiles, and rare: 4 x 2000 queries
// over 8192 and 2000 keys take 1.1 ms, with a NaN in one sample's last value 11, in the first own value of every sample (where the
// rows are walked again for nothing) 55.  A: keys of a lane whose rows are loaded together (in a kernel of many registers all
// of a step's).  CODES: a source may hold int8 codes.
template <int DT, int D, int A, bool CODES>
__device__ __forceinline__ void mend_row(int src0, int nsrc, int b, int qi, int h, int lane) {
  const RowArgs& a = *(const RowArgs*)__builtin_amdgcn_kernarg_segment_ptr();  // (as a reference handed on, the arguments are copied)
  constexpr int L = D / 8, N = L;  // lanes of a key, keys of a lane in a step
  constexpr int kAhead = A < N ? A : N;
  const int chunk = lane % L, sub = lane / L, hk = a.by_g(h);
  float q[8], o[8] = {}, m = -__builtin_inff(), l = 0.0f;
  In<DT>::widen8(*reinterpret_cast<const uint4*>(a.q + b * a.sqb + h * a.sqh + qi * a.sqi + 8 * chunk), q);
#pragma unroll
  for (int i = 0; i < 8; i++) q[i] *= a.scale_log2;
  auto walk = [&](const KeySource& s, auto coded_c) __attribute__((always_inline)) {
    constexpr bool coded = decltype(coded_c)::value;
    int n = (int)sample_length(s, b);
    if (s.causal) n = max(0, min(n, n - (int)a.Lq + qi + 1));
    constexpr int eb = coded ? 1 : 2;
    const char* const k0 = (const char*)s.k + (b * s.skb + hk * s.skh) * eb;
    const char* const v0 = (const char*)s.v + (b * s.svb + hk * s.svh) * eb;
    const uint32_t kj = (uint32_t)s.skj * eb, vj = (uint32_t)s.svj * eb;
    auto fetch = [&](__amdgpu_buffer_rsrc_t r, uint32_t at) {  // 8 values, or 8 codes in the first half
      if constexpr (coded) {
        const auto c = __builtin_amdgcn_raw_buffer_load_b64(r, at + 8 * chunk, 0, 0);
        return v4i_r{(int)c[0], (int)c[1], 0, 0};
      }
      return load16(r, at + 16 * chunk, 0);
    };
    auto widen = [&](v4i_r w, float (&f)[8]) {
      if constexpr (coded) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = (float)(int)(int8_t)((uint32_t)w[i / 4] >> (8 * (i & 3)));
      } else {
        In<DT>::widen8(__builtin_bit_cast(uint4, w), f);
      }
    };
    for (int key0 = 0; key0 < n; key0 += 64) {
      const int here = n - key0;  // the lane's keys: key0 + sub + 64 / L * i, the last one of the row for those past it
      const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(k0 + (int64_t)key0 * kj), vr = buffer_rsrc(v0 + (int64_t)key0 * vj);
      float sc[N], top = m;
#pragma unroll
      for (int i0 = 0; i0 < N; i0 += kAhead) {
        int my = sub;
        if constexpr (kAhead < N) asm volatile("" : "+v"(my)::"memory");  // (no more loads and places ahead than there are registers)
        v4i_r w[kAhead];
        float scale[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
          const int key = min(my + 64 / L * (i0 + u), here - 1);
          w[u] = fetch(kr, key * kj);
          scale[u] = coded ? s.ks[hk * s.ksh + (key0 + key) * s.ksj] : 1.0f;
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
          float f[8], x = 0.0f;
          widen(w[u], f);
#pragma unroll
          for (int i = 0; i < 8; i++) x = __builtin_fmaf(q[i], f[i], x);
          x += dpp_f<0xB1>(x);
          x += dpp_f<0x4E>(x);
          x += dpp_f<0x141>(x);
          if constexpr (L == 16) x += dpp_f<0x140>(x);
          sc[i0 + u] = sub + 64 / L * (i0 + u) < here ? x * scale[u] : -__builtin_inff();
          top = __builtin_fmaxf(top, sc[i0 + u]);
        }
      }
#pragma unroll
      for (int x = L; x < 64; x <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, x));
      const float ref = top == -__builtin_inff() ? 0.0f : top;
      const float alpha = __builtin_amdgcn_exp2f(m - ref);  // 0 for the first scores
      m = top;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < 8; i++) o[i] *= alpha;
#pragma unroll
      for (int i0 = 0; i0 < N; i0 += kAhead) {
        int my = sub;
        if constexpr (kAhead < N) asm volatile("" : "+v"(my)::"memory");  // (no more loads and places ahead than there are registers)
        v4i_r w[kAhead];
        float scale[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
          const int key = min(my + 64 / L * (i0 + u), here - 1);
          w[u] = fetch(vr, key * vj);
          scale[u] = coded ? s.vs[hk * s.vsh + (key0 + key) * s.vsj] : 1.0f;
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
          const float p = __builtin_amdgcn_exp2f(sc[i0 + u] - ref), weight = p * scale[u];
          float f[8];
          widen(w[u], f);
          l += p;
          const bool seen = sub + 64 / L * (i0 + u) < here;
#pragma unroll
          for (int i = 0; i < 8; i++) o[i] = seen ? __builtin_fmaf(weight, f[i], o[i]) : o[i];
        }
      }
    }
  };
#pragma unroll 1
  for (int t = src0; t < src0 + nsrc; t++) {
    if constexpr (CODES) {
      if (a.src[t].ks) {
        walk(a.src[t], std::true_type());
        continue;
      }
    }
    walk(a.src[t], std::false_type());
  }
#pragma unroll
  for (int x = L; x < 64; x <<= 1) {
    l += __shfl_xor(l, x);
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] += __shfl_xor(o[i], x);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (lane < L)
    *reinterpret_cast<out8*>(a.o + b * a.sob + h * a.soh + qi * a.soi + 8 * chunk) =
        out8{pack2<DT>(o[0] * inv, o[1] * inv), pack2<DT>(o[2] * inv, o[3] * inv), pack2<DT>(o[4] * inv, o[5] * inv),
             pack2<DT>(o[6] * inv, o[7] * inv)};
}

// The rows of the lanes whose bits are set, one after another.
template <int DT, int D, int A, bool CODES>
__device__ __forceinline__ void mend_rows(int src0, int nsrc, uint64_t lanes, int b, int qi, int h, int lane) {
  while (lanes != 0) {
    const int from = __builtin_ctzll(lanes);
    lanes &= lanes - 1;
    mend_row<DT, D, A, CODES>(src0, nsrc, __builtin_amdgcn_readlane(b, from), __builtin_amdgcn_readlane(qi, from), __builtin_amdgcn_readlane(h, from), lane);
  }
}

// The rows, of L lanes each, in which a lane is `bad`.
template <int DT, int D, int A, bool CODES, int L>
__device__ __forceinline__ void mend_lanes(int src0, int nsrc, bool bad, int b, int qi, int h, int lane) {
  uint64_t lanes = __builtin_amdgcn_ballot_w64(bad);
  if (__builtin_expect(lanes == 0, 1)) return;
  uint64_t rows = 0;
#pragma unroll
  for (int r = 0; r < 64; r += L) rows |= (lanes >> r & low_bits(L)) != 0 ? 1ull << r : 0;
  wait_loads();  // (these rows' results are written before they are written again)
  mend_rows<DT, D, A, CODES>(src0, nsrc, rows, b, qi, h, lane);
}

__device__ __forceinline__ bool finite4(float4 v) {  // (products with zero: 0 or NaN)
  return __builtin_fmaf(v.x, 0.0f, v.y * 0.0f) + __builtin_fmaf(v.z, 0.0f, v.w * 0.0f) == 0.0f;
}

// ---------------------------------------------------------------------------------------------
// Many rows: 128 a workgroup, tiles of 64 keys that its waves share.
template <int D>
struct Tile {
  static constexpr int kBytes = kKeys * Rows<D>::kRow;  // of the K or the V tile
  static constexpr int kStage = 2 * kBytes;
};

// Leaves or writes the results of 32 rows a group of waves holds: wave `w` those of row group w % RW, over part w / RW of the
// keys.  Each wave scales its output to the common maximum of its row group in LDS (over the tiles, which every wave is done
// with); the workgroup adds the parts.  `row0`: the workgroup's first row of the unit.  MEND: the results are final and under a
// causal limit that hides keys from some of the rows.
template <int DT, int D, int RW, bool MEND, typename Core>
__device__ __forceinline__ void join_parts(const RowArgs& a, const RowJob& job, const Core& core, int unit, int split, int row0,
                                           char* smem, float2* stats) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l32 = lane & 31, h2 = lane >> 5, group = wave % RW;
  const float ltot = core.total();
  if (h2 == 0) stats[wave * 32 + l32] = make_float2(core.m, ltot);
  lds_barrier();
  float top = -__builtin_inff();
#pragma unroll
  for (int w = 0; w < kWaves / RW; w++) top = __builtin_fmaxf(top, stats[(group + w * RW) * 32 + l32].x);
  const float mine = ltot == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(core.m - top);
  float* ol = reinterpret_cast<float*>(smem + wave * 32 * D * 4);  // [32 rows][D / 4 chunks of 16 bytes, chunk c of row r at c ^ r]
#pragma unroll
  for (int db = 0; db < D / 32; db++)
#pragma unroll
    for (int rr = 0; rr < 4; rr++) {
      const int c = (8 * db + 2 * rr + h2) ^ (l32 % (D / 4));
      const float4 o = make_float4(core.oacc[db][4 * rr] * mine, core.oacc[db][4 * rr + 1] * mine, core.oacc[db][4 * rr + 2] * mine,
                                   core.oacc[db][4 * rr + 3] * mine);
      *reinterpret_cast<float4*>(ol + l32 * D + 4 * c) = mine == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : o;
    }
  lds_barrier();
  const int rows = min(32 * RW, job.rows - row0);
  for (int item0 = wave * 64; item0 < rows * (D / 4); item0 += kWaves * 64) {  // (the whole wave stays for rows to mend)
    const bool in = item0 + lane < rows * (D / 4);
    const int item = in ? item0 + lane : item0;
    const int row = item / (D / 4), c = item % (D / 4), r32 = row % 32, g = row / 32;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f, mt = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kWaves / RW; w++) mt = __builtin_fmaxf(mt, stats[(g + w * RW) * 32 + r32].x);
#pragma unroll
    for (int w = 0; w < kWaves / RW; w++) {
      const float2 ml = stats[(g + w * RW) * 32 + r32];
      const float4 v = *reinterpret_cast<const float4*>(smem + (g + w * RW) * 32 * D * 4 + r32 * D * 4 + ((c ^ (r32 % (D / 4))) << 4));
      if (ml.y != 0.0f) l = __builtin_fmaf(ml.y, __builtin_amdgcn_exp2f(ml.x - mt), l);
      o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
    }
    int64_t b;
    int qi, h;
    locate(a, job, unit, row0 + row, b, qi, h);
    if (a.slots) {
      if (!in) continue;
      const int64_t id = (int64_t)(job.slot0 + split) * a.ids + (b * a.Lq + qi) * a.Hq + h;
      *reinterpret_cast<float4*>(a.po + id * D + 4 * c) = o;
      if (c == 0) a.pml[id] = make_float2(mt, l);
    } else {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
      if (in)
        *reinterpret_cast<uint2*>(a.o + b * a.sob + h * a.soh + qi * a.soi + 4 * c) =
            make_uint2(pack2<DT>(o.x * inv, o.y * inv), pack2<DT>(o.z * inv, o.w * inv));
      if constexpr (MEND) mend_lanes<DT, D, 16, false, D / 4>(job.src0, job.nsrc, in && qi < a.Lq - 1 && !finite4(o) && l == l, (int)b, qi, h, lane);
    }
  }
}

// One workgroup's rows and tiles.  I8: the job's one source holds int8 codes.  RW: row groups of 32; with 2, two waves share
// a group and take a tile's first and second 32 keys.
template <int DT, int D, bool I8, int RW, bool MEND>
__device__ __forceinline__ void attend_rows(const RowArgs& a, const RowJob& job, const KeySource* src, int nsrc, int index, char* smem, float2* stats, float* scale_lds) {
  using T = Tile<D>;
  using R = Rows<D>;
  constexpr int NKB = RW / 2;          // 32-key blocks of a wave in a tile
  constexpr int U = T::kBytes / 4096;  // 1 KB direct loads of a wave for the K tile, and for the V tile
  constexpr int RPL = 1024 / R::kRow;  // rows of one
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = wave / RW;  // of the tile's keys
  const Share sh(job, index);
  const int block = sh.block, split = sh.split, unit = sh.unit;
  const int row0 = block * 32 * RW, r0 = row0 + wave % RW * 32;
  const bool live = r0 < job.rows;  // any row of the wave
  const Place at(a, job, src, nsrc, unit, r0 + (lane & 31), row0 + 32 * RW - 1);
  using Core = RowCore<DT, D, I8, NKB, false>;
  // The wave's query rows go through the second stage's LDS, a piece of its own: whole rows are loaded side by side, where
  // the fragments' own addresses are 32 bytes of 32 rows an instruction.  With the 16-byte stores at the end, 46.7 to 41.7 us at
  // 2 x 3520 queries of 24 heads over 333 keys, 137 to 129 at 26400 of 16 over 512.
  char* const own_rows = smem + T::kStage + wave * 32 * R::kRow;
  Core core(a, lane);
  auto load_rows = [&]() __attribute__((always_inline)) {
    const uint16_t* mine = a.q + at.b * a.sqb + at.h * a.sqh + at.qi * a.sqi;
#pragma unroll
    for (int p = 0; p < 32 / RPL; p++) {
      const int r = lane / R::kChunks + p * RPL;
      const char* from = reinterpret_cast<const char*>(of_lane(mine, r));
      g2lds16(from + ((lane % R::kChunks ^ R::kswz(r)) << 4), own_rows + p * 1024);
    }
  };
  auto read_rows = [&]() __attribute__((always_inline)) {  // (before the barrier after which the stage is refilled)
    wait_loads();
#pragma unroll
    for (int ks = 0; ks < Core::KS; ks++)
      core.qf[ks] = *reinterpret_cast<const v4i_r*>(own_rows + core.krow + (((2 * ks + core.h2) ^ core.kx) << 4));
  };
  const int nt0 = (at.n[0] + kKeys - 1) / kKeys, total = nt0 + (at.n[1] + kKeys - 1) / kKeys;
  const int t0 = range_start(job, total, split), t1 = range_start(job, total, split + 1);
  const int own_tile = nsrc == 1 ? 0 : nt0;  // causal: the first tile of own keys

  int cur = -1;  // the source of the tile being loaded
  uint32_t koff[I8 ? 1 : U], voff[I8 ? 1 : U], kstride = 0, vstride = 0;
  const char *kbase = nullptr, *vbase = nullptr;
  const float *ksbase = nullptr, *vsbase = nullptr;  // int8: the head's scales
  int64_t ksstride = 0, vsstride = 0;
  auto enter = [&](int which) {
    cur = which;
    const KeySource& s = src[which];
    constexpr int eb = I8 ? 1 : 2;
    kbase = (const char*)s.k + (at.b_unit * s.skb + at.hk * s.skh) * eb;
    vbase = (const char*)s.v + (at.b_unit * s.svb + at.hk * s.svh) * eb;
    kstride = (uint32_t)(s.skj * eb);
    vstride = (uint32_t)(s.svj * eb);
    if constexpr (I8) {
      ksbase = s.ks + at.hk * s.ksh;
      vsbase = s.vs + at.hk * s.vsh;
      ksstride = s.ksj;
      vsstride = s.vsj;
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int r = (wave + 4 * u) * RPL + lane / R::kChunks, c = lane % R::kChunks;
        koff[u] = (uint32_t)r * kstride + (uint32_t)((c ^ R::kswz(r)) << 4);
        voff[u] = (uint32_t)r * vstride + (uint32_t)((c ^ R::vswz(r)) << 4);
      }
    }
  };
  // a tile's products and softmax; `between` runs while the score products do
  auto compute = [&](int t, auto buf_c, uint64_t bits, const char* stage, auto between) __attribute__((always_inline)) {
    constexpr int buf = decltype(buf_c)::value;
    const char* kl = stage + part * 32 * R::kRow;
    const float* scales = scale_lds + buf * 3 * kKeys + part * 32;
    v16f sc[NKB];
    uint32_t pk[NKB][8];
    core.scores(kl, scales, sc);
    between();
    core.hide(sc, RW == 4 ? bits : (uint32_t)(bits >> (32 * part)), at.causal && t >= own_tile,
              at.row_keys - (t - own_tile) * kKeys - 32 * part);
    core.softmax(sc, scales + kKeys, scales + 2 * kKeys, pk);
    core.values(kl + T::kBytes, pk);
  };

  if constexpr (I8) {
    constexpr int P = T::kBytes / 2 / 16 / 256;  // 16-byte pieces of a thread for the K codes, and for the V codes
    v4i_r raw_k[P], raw_v[P];
    float raw_scale = 0.0f;
    enter(0);
    constexpr int C = D / 16;  // pieces of a row
    const uint32_t koff8 = tid / C * kstride + tid % C * 16, voff8 = tid / C * vstride + tid % C * 16;
    auto load = [&](int t) __attribute__((always_inline)) {
      const int key0 = t * kKeys, here = min(kKeys, at.n[0] - key0);
      const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(kbase + (int64_t)key0 * kstride), vr = buffer_rsrc(vbase + (int64_t)key0 * vstride);
      if (here == kKeys) {
#pragma unroll
        for (int p = 0; p < P; p++) {
          raw_k[p] = load16(kr, koff8, p * (256 / C) * kstride);
          raw_v[p] = load16(vr, voff8, p * (256 / C) * vstride);
        }
      } else {  // rows past the last key repeat it
#pragma unroll
        for (int p = 0; p < P; p++) {
          const uint32_t r = min(tid / C + p * (256 / C), here - 1);
          raw_k[p] = load16(kr, r * kstride + tid % C * 16, 0);
          raw_v[p] = load16(vr, r * vstride + tid % C * 16, 0);
        }
      }
      if (tid < 2 * kKeys) {
        const int64_t key = key0 + min(tid % kKeys, here - 1);
        raw_scale = tid < kKeys ? ksbase[key * ksstride] : vsbase[key * vsstride];
      }
    };
    auto widen = [&](int buf) __attribute__((always_inline)) {
      char* kl = smem + buf * T::kStage;
      if (tid < 2 * kKeys) scale_lds[buf * 3 * kKeys + tid] = raw_scale;
      if (Core::kWeighted && tid >= kKeys && tid < 2 * kKeys) scale_lds[buf * 3 * kKeys + kKeys + tid] = core.scale_log(raw_scale);
#pragma unroll
      for (int p = 0; p < P; p++) {
        const int idx = tid + 256 * p, r = idx / (D / 16), c = idx % (D / 16);
        store_codes<DT>(kl + r * R::kRow, R::kswz(r), c, raw_k[p]);
        store_codes<DT>(kl + T::kBytes + r * R::kRow, R::vswz(r), c, raw_v[p]);
      }
    };
    if (t0 < t1) {
      load_rows();
      load(t0);
      read_rows();
      widen(0);
      if (t0 + 1 < t1) load(t0 + 1);
      auto tile = [&](int t, auto buf_c) __attribute__((always_inline)) {
        lds_barrier();  // tile t is in LDS, and every wave is done with the other buffer
        auto next = [&]() __attribute__((always_inline)) {
          if (t + 1 < t1) {
            widen(decltype(buf_c)::value ^ 1);
            if (t + 2 < t1) load(t + 2);
          }
        };
        if (live) compute(t, buf_c, low_bits(at.n[0] - t * kKeys), smem + decltype(buf_c)::value * T::kStage, next);
        else next();
      };
      for (int t = t0; t < t1; t += 2) {
        tile(t, std::integral_constant<int, 0>());
        if (t + 1 < t1) tile(t + 1, std::integral_constant<int, 1>());
      }
    }
  } else {
    // the seen keys of the next tile to load, from its mask bytes (one a lane, read a tile earlier than they are needed)
    uint32_t mask_byte = 1;
    const uint8_t* const mbase = src[0].mask ? src[0].mask + at.b_unit * src[0].smb : nullptr;
    auto read_mask = [&](int t) {  // (only a job of one source has a mask)
      if (mbase && t < t1) mask_byte = mbase[min(t * kKeys + lane, at.n[0] - 1)];
    };
    // starts loading tile t; returns its seen keys
    auto load = [&](int t, char* kl) __attribute__((always_inline)) -> uint64_t {
      const int which = t < nt0 ? 0 : 1, key0 = (t - (which ? nt0 : 0)) * kKeys;
      if (which != cur) enter(which);
      uint64_t bits = low_bits(at.n[which] - key0);
      if (mbase) bits &= __builtin_amdgcn_ballot_w64(mask_byte != 0);
      char* vl = kl + T::kBytes;
      const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(kbase + (int64_t)key0 * kstride), vr = buffer_rsrc(vbase + (int64_t)key0 * vstride);
      if (bits == ~0ull) {
#pragma unroll
        for (int u = 0; u < U; u++) b2lds16(kr, koff[u], 0, kl + (wave + 4 * u) * 1024);
#pragma unroll
        for (int u = 0; u < U; u++) b2lds16(vr, voff[u], 0, vl + (wave + 4 * u) * 1024);
      } else if (bits) {
        const int first = __builtin_ctzll(bits);
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int r = (wave + 4 * u) * RPL + lane / R::kChunks, c = lane % R::kChunks;
          const uint32_t from = (bits >> r) & 1 ? r : first;
          b2lds16(kr, from * kstride + (uint32_t)((c ^ R::kswz(r)) << 4), 0, kl + (wave + 4 * u) * 1024);
          b2lds16(vr, from * vstride + (uint32_t)((c ^ R::vswz(r)) << 4), 0, vl + (wave + 4 * u) * 1024);
        }
      }
      read_mask(t + 1);
      return bits;
    };
    if (t0 < t1) {
      read_mask(t0);
      load_rows();
      uint64_t bits_next = load(t0, smem);
      read_rows();
      // (restrict: the two stages are apart, so the transposing reads of one need not wait for the loads into the other)
      auto tile = [&](int t, auto buf_c, const char* __restrict__ cur, char* __restrict__ next) __attribute__((always_inline)) {
        const uint64_t bits = bits_next;
        tile_barrier();  // tile t has landed for every wave, and every wave is done with the buffer that tile t + 1 refills
        if (t + 1 < t1) bits_next = load(t + 1, next);
        if (live && bits) compute(t, buf_c, bits, cur, []() {});
      };
      for (int t = t0; t < t1; t += 2) {
        tile(t, std::integral_constant<int, 0>(), smem, smem + T::kStage);
        if (t + 1 < t1) tile(t + 1, std::integral_constant<int, 1>(), smem + T::kStage, smem);
      }
    }
  }

  if constexpr (RW == 2) {
    lds_barrier();  // every wave is done with the tiles
    join_parts<DT, D, RW, MEND>(a, job, core, unit, split, row0, smem, stats);
  } else {
    if (!live) return;
    const float ltot = core.total();
    const int h2 = lane >> 5;
    const bool in = r0 + (lane & 31) < job.rows;
    if (a.slots) {
      if (!in) return;
      const int64_t id = (int64_t)(job.slot0 + split) * a.ids + (at.b * a.Lq + at.qi) * a.Hq + at.h;
      float* po = a.po + id * D + 4 * h2;
#pragma unroll
      for (int db = 0; db < D / 32; db++)
#pragma unroll
        for (int rr = 0; rr < 4; rr++)
          *reinterpret_cast<float4*>(po + 32 * db + 8 * rr) =
              make_float4(core.oacc[db][4 * rr], core.oacc[db][4 * rr + 1], core.oacc[db][4 * rr + 2], core.oacc[db][4 * rr + 3]);
      if (h2 == 0) a.pml[id] = make_float2(core.m, ltot);
      return;
    }
    const float inv = ltot == 0.0f ? 0.0f : 1.0f / ltot;  // no key seen: zeros
    const bool bad = MEND && in && at.qi < a.Lq - 1 && !core.finite() && ltot == ltot;  // (a NaN among a row's own scores stays)
    // (the two halves of a row trade four values, so that each lane stores eight at once)
    uint16_t* op = a.o + at.b * a.sob + at.h * a.soh + at.qi * a.soi + 8 * h2;
#pragma unroll
    for (int db = 0; db < D / 32; db++)
#pragma unroll
      for (int rr = 0; rr < 4; rr += 2) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = pack2<DT>(core.oacc[db][4 * rr + 2 * i] * inv, core.oacc[db][4 * rr + 2 * i + 1] * inv);
        const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        if (in) *reinterpret_cast<out8*>(op + 32 * db + 8 * rr) = out8{x[0], y[0], x[1], y[1]};
      }
    if constexpr (MEND) {
      const uint64_t lanes = __builtin_amdgcn_ballot_w64(bad);
      if (__builtin_expect(lanes != 0, 0)) {
        wait_loads();  // (these rows' results are written before they are written again)
        mend_rows<DT, D, 16, false>(job.src0, job.nsrc, (lanes | lanes >> 32) & low_bits(32), (int)at.b, at.qi, at.h, lane);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Few rows (up to 32): every wave of the workgroup takes all of them over tiles of its own, the four next to each other, so
// that a step of the workgroup brings in 64 KB.  A tile passes through registers, loaded while the one before is worked on, into
// the wave's own LDS: the loop has no barrier.  The waves' results are joined in LDS at the end.
constexpr int kFewRows = 32;

template <int D>
struct FewTile {
  static constexpr int kKeys = D == 128 ? 32 : 64;
  static constexpr int kBytes = kKeys * Rows<D>::kRow;  // of the K or the V tile: 8 KB
  static constexpr int kWave = 2 * kBytes;              // LDS of a wave
  static constexpr bool kQL = D == 128;                 // the query rows' fragments lie in LDS too
};

template <int DT, int D, bool I8, bool MEND>
__device__ __forceinline__ void attend_few(const RowArgs& a, const RowJob& job, const KeySource* src, int nsrc, int index, char* smem, char* q_lds, float2* stats, float* scale_lds) {
  using T = FewTile<D>;
  using R = Rows<D>;
  constexpr int KT = T::kKeys, NKB = KT / 32;
  constexpr int eb = I8 ? 1 : 2;
  constexpr int C = D * eb / 16;            // 16-byte pieces of a row in memory
  constexpr int P = KT * C / 64;            // of a lane for the K tile, and for the V tile
  constexpr bool kQL = FewTile<D>::kQL;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Share sh(job, index);
  const int split = sh.split, unit = sh.unit;
  const Place at(a, job, src, nsrc, unit, lane & 31, job.rows - 1);
  // the rows' loads go out first, then the first tile's; neither waits for the other
  using Core = RowCore<DT, D, I8, NKB, kQL>;
  v4i_r rows[Core::KS];
  Core::load_rows(a, at, lane, rows);
  const int nt0 = (at.n[0] + KT - 1) / KT, total = nt0 + (at.n[1] + KT - 1) / KT;
  // (ranges of whole steps of four tiles)
  const int steps = (total + kWaves - 1) / kWaves;
  const int t0 = range_start(job, steps, split) * kWaves;
  const int t1 = min(total, range_start(job, steps, split + 1) * kWaves);
  const int own_tile = nsrc == 1 ? 0 : nt0;

  const uint8_t* const mbase = src[0].mask ? src[0].mask + at.b_unit * src[0].smb : nullptr;
  uint32_t mask_byte = 1;
  auto read_mask = [&](int t) {
    if (mbase && t < t1) mask_byte = mbase[min(t * KT + lane, at.n[0] - 1)];
  };
  int cur = -1;  // the source of the tile being loaded
  const char *kbase = nullptr, *vbase = nullptr;
  uint32_t ksj = 0, vsj = 0, koff = 0, voff = 0;  // bytes a key; the lane's place in the first rows
  const float *ksbase = nullptr, *vsbase = nullptr;  // int8: the head's scales
  int64_t ksstride = 0, vsstride = 0;
  auto enter = [&](int which) {
    cur = which;
    const KeySource& s = src[which];
    kbase = (const char*)s.k + (at.b_unit * s.skb + at.hk * s.skh) * eb;
    vbase = (const char*)s.v + (at.b_unit * s.svb + at.hk * s.svh) * eb;
    ksj = (uint32_t)(s.skj * eb);
    vsj = (uint32_t)(s.svj * eb);
    koff = lane / C * ksj + lane % C * 16;
    voff = lane / C * vsj + lane % C * 16;
    if constexpr (I8) {
      ksbase = s.ks + at.hk * s.ksh;
      vsbase = s.vs + at.hk * s.vsh;
      ksstride = s.ksj;
      vsstride = s.vsj;
    }
  };
  v4i_r raw_k[P], raw_v[P];
  float raw_scale[NKB];
  auto load = [&](int t) __attribute__((always_inline)) -> uint64_t {
    const int which = t < nt0 ? 0 : 1, key0 = (t - (which ? nt0 : 0)) * KT;
    if (which != cur) enter(which);
    const int here = min(KT, at.n[which] - key0);
    uint64_t bits = low_bits(here);
    if (mbase) bits &= __builtin_amdgcn_ballot_w64(mask_byte != 0);
    const char* kt = kbase + (int64_t)key0 * ksj;
    const char* vt = vbase + (int64_t)key0 * vsj;
    const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(kt), vr = buffer_rsrc(vt);
    if (bits == low_bits(KT)) {  // piece p: 64 / C rows after the one before
#pragma unroll
      for (int p = 0; p < P; p++) {
        raw_k[p] = load16(kr, koff, p * (64 / C) * ksj);
        raw_v[p] = load16(vr, voff, p * (64 / C) * vsj);
      }
    } else {
      const int first = bits ? __builtin_ctzll(bits) : 0;  // (a tile without a seen key is loaded and passed over)
      int r0 = lane / C;
      asm volatile("" : "+v"(r0));  // (what follows is worked out here, not kept in registers across the loop)
#pragma unroll
      for (int p = 0; p < P; p++) {
        const int r = r0 + p * (64 / C);
        const uint32_t from = (bits >> r) & 1 ? r : first;
        raw_k[p] = load16(kr, from * ksj + lane % C * 16, 0);
        raw_v[p] = load16(vr, from * vsj + lane % C * 16, 0);
      }
    }
    if constexpr (I8) {  // key scales in the first half, value scales in the second of 2 KT places
#pragma unroll
      for (int i = 0; i < NKB; i++) {
        const int place = lane + 64 * i;
        const int64_t key = key0 + min(place % KT, here - 1);
        raw_scale[i] = place < KT ? ksbase[key * ksstride] : vsbase[key * vsstride];
      }
    }
    return bits;
  };
  int t = t0 + wave;
  uint64_t bits = 0;
  if (t < t1) {
    read_mask(t);
    bits = load(t);
    read_mask(t + kWaves);
  }
  Core core(a, rows, lane, q_lds);
  if constexpr (kQL) lds_barrier();  // (every wave has written the same q rows)
  char* kl = smem + wave * T::kWave;
  char* vl = kl + T::kBytes;
  float* scales = scale_lds + wave * 3 * KT;
  auto to_lds = [&]() __attribute__((always_inline)) {
    int first = lane;
    if constexpr (kQL) asm volatile("" : "+v"(first));
#pragma unroll
    for (int p = 0; p < P; p++) {
      const int idx = first + 64 * p, r = idx / C, c = idx % C;
      if constexpr (I8) {
        store_codes<DT>(kl + r * R::kRow, R::kswz(r), c, raw_k[p]);
        store_codes<DT>(vl + r * R::kRow, R::vswz(r), c, raw_v[p]);
      } else {
        *reinterpret_cast<v4i_r*>(kl + r * R::kRow + ((c ^ R::kswz(r)) << 4)) = raw_k[p];
        *reinterpret_cast<v4i_r*>(vl + r * R::kRow + ((c ^ R::vswz(r)) << 4)) = raw_v[p];
      }
    }
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < NKB; i++) {
        const int place = lane + 64 * i;
        scales[place] = raw_scale[i];
        if (Core::kWeighted && place >= KT) scales[KT + place] = core.scale_log(raw_scale[i]);
      }
    }
  };
  auto compute = [&](int t, uint64_t bits) __attribute__((always_inline)) {
    if (bits == 0) return;
    asm volatile("" ::: "memory");  // (a wave's LDS accesses run in their order)
    v16f sc[NKB];
    uint32_t pk[NKB][8];
    core.scores(kl, scales, sc);
    core.hide(sc, bits, at.causal && t >= own_tile, at.row_keys - (t - own_tile) * KT);
    core.softmax(sc, scales + KT, scales + 2 * KT, pk);
    core.values(vl, pk);
    asm volatile("" ::: "memory");
  };
  if (t < t1) {
    for (; t + kWaves < t1; t += kWaves) {
      to_lds();
      const uint64_t now = bits;
      bits = load(t + kWaves);
      read_mask(t + 2 * kWaves);
      compute(t, now);
    }
    to_lds();
    compute(t, bits);
  }

  lds_barrier();
  join_parts<DT, D, 1, MEND>(a, job, core, unit, split, 0, smem, stats);
}

template <int DT, int D, bool I8, bool MEND>
__device__ __forceinline__ void attend(const RowArgs& a, const RowJob& job, const KeySource* src, int nsrc, int index, char* smem, char* q_lds, float2* stats, float* scales) {
  if (job.kind == kFew) attend_few<DT, D, I8, MEND>(a, job, src, nsrc, index, smem, q_lds, stats, scales);
  else if (job.kind == kHalf) attend_rows<DT, D, I8, 2, MEND>(a, job, src, nsrc, index, smem, stats, scales);
  else attend_rows<DT, D, I8, 4, MEND>(a, job, src, nsrc, index, smem, stats, scales);
}

// All jobs of a call.  I8: the first one's keys are int8 codes (then the own keys' job, where there is one, is a second one, and its
// results are partials).  MEND: the results are final and under a causal limit with several queries (a kernel apart:
// within one, calls without a limit took 0.2 us more, 64 samples over 32768 shared keys 61.4 in place of 59.2).
template <int DT, int D, bool I8, bool MEND>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void row_attention_kernel(const RowArgs a) {
  // one array for all of it: with several, the compiler lets every LDS read wait for the direct loads in flight
  constexpr int many = 2 * Tile<D>::kStage, few = kWaves * FewTile<D>::kWave, tiles = many > few ? many : few;
  constexpr int q_bytes = FewTile<D>::kQL ? kFewRows * Rows<D>::kRow : 0, stat_bytes = kWaves * 32 * sizeof(float2);
  constexpr int few_scales = kWaves * 3 * FewTile<D>::kKeys, nscales = I8 ? (few_scales > 6 * kKeys ? few_scales : 6 * kKeys) : 0;
  __shared__ __align__(16) char lds[tiles + q_bytes + stat_bytes + nscales * 4];
  char* const smem = lds;
  char* const q_lds = lds + tiles;
  float2* const stats = reinterpret_cast<float2*>(lds + tiles + q_bytes);
  float* const scales = reinterpret_cast<float*>(lds + tiles + q_bytes + stat_bytes);
  const bool second = a.njobs > 1 && (int64_t)blockIdx.x >= a.job[1].wg0;
  if constexpr (I8) {  // (constant places in the arguments: they are read where they lie)
    if (!second) attend<DT, D, true, false>(a, a.job[0], &a.src[0], 1, (int)blockIdx.x, smem, q_lds, stats, scales);
    else attend<DT, D, false, false>(a, a.job[1], &a.src[1], 1, (int)(blockIdx.x - a.job[1].wg0), smem, q_lds, stats, scales);
  } else {
    const RowJob& job = a.job[second];
    attend<DT, D, false, MEND>(a, job, &a.src[job.src0], job.nsrc, (int)(blockIdx.x - job.wg0), smem, q_lds, stats, scales);
  }
}

// ---------------------------------------------------------------------------------------------
// Joins the partials of a row: out = sum_s w_s O_s / sum_s w_s l_s, w_s = exp2(m_s - max m).  D / 4 lanes take a row, 16 bytes
// each, GR such groups share its slots; a slot that saw no key (sum 0) is left out, and a row of such slots is zeros.
// Short (5 to 6 us, its launch 2): four slots' loads go out together, which took 0.5 us off a slot at a time.
// MEND: under a causal limit with several queries.  Seven waves a SIMD, which costs the mending a few registers in memory: at the
// five that it takes otherwise, 64 samples of 4 queries over 9000 and 200 keys took 65.0 us, now 62.7, as without it.
template <int DT, int D, int GR, bool MEND>
__global__ __launch_bounds__(256, 7) void row_combine_kernel(const RowArgs a) {
  constexpr int L = D / 4, R = 256 / L / GR;
  const int group = threadIdx.x / L, c = threadIdx.x % L;
  const int64_t id = (int64_t)blockIdx.x * R + group / GR;
  __shared__ float4 part_o[GR > 1 ? 256 : 1];
  __shared__ float2 part_ml[GR > 1 ? 256 / L : 1];
  float top = -__builtin_inff(), l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (id < a.ids) {
    constexpr int kAhead = 4;  // slots whose loads go out together
    for (int s0 = group % GR; s0 < a.slots; s0 += kAhead * GR) {
      float2 mls[kAhead];
      float4 vs[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const int64_t at = (s0 + u * GR < a.slots ? s0 + u * GR : s0) * a.ids + id;
        mls[u] = a.pml[at];
        vs[u] = *reinterpret_cast<const float4*>(a.po + at * D + 4 * c);
      }
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const float2 ml = mls[u];
        const float4 v = vs[u];
        if (s0 + u * GR >= a.slots || ml.y == 0.0f) continue;
        const float mt = __builtin_fmaxf(top, ml.x);
        const float keep = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(top - mt), w = __builtin_amdgcn_exp2f(ml.x - mt);
        l = __builtin_fmaf(w, ml.y, l * keep);
        o.x = __builtin_fmaf(w, v.x, o.x * keep);
        o.y = __builtin_fmaf(w, v.y, o.y * keep);
        o.z = __builtin_fmaf(w, v.z, o.z * keep);
        o.w = __builtin_fmaf(w, v.w, o.w * keep);
        top = mt;
      }
    }
  }
  if constexpr (GR > 1) {
    part_o[threadIdx.x] = o;
    if (c == 0) part_ml[group] = make_float2(top, l);
    __syncthreads();
    if constexpr (MEND) {  // (a row's other groups in its first one's wave work along: the wave stays whole for a row to mend)
      if ((group & -(64 / L)) % GR != 0) return;
    } else {
      if (group % GR != 0) return;
    }
    const int of = group - group % GR;
    top = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < GR; k++) top = __builtin_fmaxf(top, part_ml[of + k].x);
    l = 0.0f;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < GR; k++) {
      const float2 ml = part_ml[of + k];
      const float4 v = part_o[(of + k) * L + c];
      if (ml.y == 0.0f) continue;
      const float w = __builtin_amdgcn_exp2f(ml.x - top);
      l = __builtin_fmaf(w, ml.y, l);
      o.x = __builtin_fmaf(w, v.x, o.x);
      o.y = __builtin_fmaf(w, v.y, o.y);
      o.z = __builtin_fmaf(w, v.z, o.z);
      o.w = __builtin_fmaf(w, v.w, o.w);
    }
  }
  const bool in = id < a.ids && group % GR == 0;
  if (!MEND && !in) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int bi = a.by_hq((int)id), h = (int)id - bi * a.Hq, b = a.by_lq(bi), i = bi - b * (int)a.Lq;
  if (in)
    *reinterpret_cast<uint2*>(a.o + b * a.sob + i * a.soi + h * a.soh + 4 * c) =
        make_uint2(pack2<DT>(o.x * inv, o.y * inv), pack2<DT>(o.z * inv, o.w * inv));
  if constexpr (MEND)
    mend_lanes<DT, D, 4, true, L>(a.src[0].len > 0 ? 0 : 1, a.src[0].len > 0 ? 2 : 1, in && i < a.Lq - 1 && !finite4(o) && l == l, b, i, h, threadIdx.x & 63);
}

// How a call runs: its jobs, and how many ranges of tiles each unit's keys are split into.
struct RowPlan {
  RowJob job[2];
  int njobs, slots;
  int64_t wgs, ids;
};

// Estimates in microseconds, fitted to sweeps of the split on 256 compute units that hold two workgroups each.  A 64-key tile
// of many rows takes a workgroup 1.15 alone on its unit and 2.0 beside another, of half rows 0.85 and 1.4 (int8 keys, which it
// widens, 0.55 more), a step of few rows 1.4 and 1.9; none is faster than memory brings it (6.2 bytes a ps for the chip).  A
// round of workgroups adds 3 for its start and end, partials 4.5 and their traffic; the workgroups of a second job fill the
// places beside the first one's.  What these bring from memory is not counted there, as the samples' lengths are not known: with
// all Ls keys counted, 72 calls whose splits it changes (of some 20000 drawn, 285) took 2 % longer, 6 % with shorter lengths.
// `merged`: one pass over both sources, which repeats the prefix for every sample, in place of two jobs.
RowPlan plan_jobs(int64_t B, int64_t Hq, int64_t Hkv, int64_t Lq, int64_t Lp, int64_t Ls, int64_t D, bool i8, bool merged,
                  double* estimate) {
  RowPlan p{};
  const int64_t G = Hq / Hkv, own_rows = Lq * G, all_rows = B * own_rows;
  auto ceil = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
  auto job = [&](int64_t rows, bool stacked, int src0, int nsrc) {
    const JobKind kind = rows <= 32 ? kFew : rows <= 64 ? kHalf : kMany;
    return RowJob{kind, 0, (int)rows, stacked, 0, kind == kMany ? (int)ceil(rows, kRows) : 1, 1, 0, src0, nsrc};
  };
  int64_t units[2], keys[2];
  if (Lp == 0 || Ls == 0 || merged) {
    p.njobs = 1;
    p.job[0] = merged ? job(own_rows, false, 0, 2) : Lp == 0 ? job(own_rows, false, 1, 1) : job(all_rows, true, 0, 1);
    keys[0] = Lp + Ls;
    units[0] = (p.job[0].stacked ? 1 : B) * Hkv;
  } else {
    p.njobs = 2;
    p.job[0] = job(all_rows, true, 0, 1);
    p.job[1] = job(own_rows, false, 1, 1);
    units[0] = Hkv; units[1] = B * Hkv;
    keys[0] = Lp; keys[1] = Ls;
  }
  p.ids = B * Lq * Hq;
  const int64_t cus = cu_count(), slots = 2 * cus;
  *estimate = 0;
  double others = 0;  // what the second job's workgroups take, all together: the first one's fill the places beside them
  for (int j = p.njobs - 1; j >= 0; j--) {
    RowJob& job = p.job[j];
    job.units = (int)units[j];
    const int64_t step = job.kind == kFew ? kWaves * (D == 128 ? 32 : 64) : kKeys;  // keys of a workgroup's step
    const int64_t tiles = ceil(keys[j], step);
    const double bytes = (double)step * D * (i8 && j == 0 ? 2 : 4) / job.blocks;  // of a step and workgroup
    double least = 0, taken = 0;
    for (int64_t k = 1; k <= 128 && k <= tiles; k++) {
      const int64_t c = ceil(tiles, k);
      if (k > 1 && ceil(tiles, c) != k) continue;  // the same ranges as a smaller k
      const int64_t wgs = units[j] * job.blocks * k, full = wgs / slots, rem = wgs % slots;
      const bool i8_job = i8 && j == 0 && job.kind != kFew;
      auto work = [&](int64_t n) {
        const bool beside = n > cus;
        return (job.kind == kFew ? (beside ? 1.9 : 1.4) : job.kind == kHalf ? (beside ? 1.4 : 0.85) : (beside ? 2.0 : 1.15)) +
               (i8_job ? 0.55 : 0.0);
      };
      auto round = [&](int64_t n) {  // n workgroups at once
        const double memory = n * bytes / 6.2e6;
        return (work(n) > memory ? work(n) : memory) * c + 3.0;
      };
      const double all = wgs * (work(wgs) * c + 3.0) + others;
      double cost = full * round(slots) + (rem ? round(rem) : 0.0);
      if (cost < all / slots) cost = all / slots;
      if (p.njobs > 1 || k > 1) cost += 4.5 + k * units[j] * job.rows * D * 8 / 5e6;
      if (k == 1 || cost < least * 0.97) {
        job.splits = (int)k;
        least = cost;
        taken = all;
      }
    }
    others = taken;
    *estimate = least + (j == 0 && p.njobs > 1 ? p.job[1].splits * units[1] * p.job[1].rows * D * 8 / 5e6 : 0.0);
  }
  for (int j = 0; j < p.njobs; j++) {
    RowJob& job = p.job[j];
    const int64_t walks = units[j] * job.splits;
    job.by_group.set(8 * job.blocks);
    job.by_last.set(walks % 8 ? walks % 8 : 8);
    job.by_units.set(units[j]);
    job.by_splits.set(job.splits);
    p.job[j].slot0 = p.slots;
    p.job[j].wg0 = p.wgs;
    p.slots += p.job[j].splits;
    p.wgs += units[j] * p.job[j].blocks * p.job[j].splits;
  }
  if (p.slots == 1) p.slots = 0;
  return p;
}

// One pass over a short prefix and the own keys, where it repeats up to 22 tiles for each row block that two jobs would leave
// two partials of, or is far cheaper by the estimate.  One pass against two jobs, us: 8 samples of one query, 32 heads on 8, 129
// own keys, 64 / 192 / 256 / 512 shared ones 8.1 : 10.6, 9.5 : 10.3, 11.0 : 10.4, 13.7 : 11.1; 4 of 40 queries, 100 and 2048 / 4096
// 26.4 : 27.4, 35.4 : 31.2; 16 of 8, 64 and 512 / 1024 13.8 : 18.0, 19.2 : 20.5 (the estimate alone, without the count of tiles,
// was wrong by 15 % at 5 samples of 100 queries, 16 heads of 64 dims on 2, over 400 and 700).
RowPlan plan_rows(int64_t B, int64_t Hq, int64_t Hkv, int64_t Lq, int64_t Lp, int64_t Ls, int64_t D, bool i8) {
  const int64_t own = Lq * (Hq / Hkv), blocks = (B * own + kRows - 1) / kRows;
  const int64_t repeated = (B * ((own + kRows - 1) / kRows) - blocks) * ((Lp + kKeys - 1) / kKeys);
  double two, one;
  const bool may = !i8 && Lp > 0 && Ls > 0;
  if (may && repeated <= 22 * blocks) return plan_jobs(B, Hq, Hkv, Lq, Lp, Ls, D, i8, true, &one);
  const RowPlan p = plan_jobs(B, Hq, Hkv, Lq, Lp, Ls, D, i8, false, &two);
  if (!may || repeated > 64 * blocks) return p;
  const RowPlan m = plan_jobs(B, Hq, Hkv, Lq, Lp, Ls, D, i8, true, &one);
  return one < 0.85 * two ? m : p;
}

int64_t plan_bytes(const RowPlan& p, int64_t D) { return (p.slots * p.ids * 8 + 255) / 256 * 256 + p.slots * p.ids * D * 4; }

bool plan_shape(int64_t B, int64_t Hq, int64_t Hkv, int64_t Lq, int64_t Lp, int64_t Ls, int64_t D) {
  return B >= 0 && B <= 65535 && Hq > 0 && Hq <= 65535 && Hkv > 0 && Hq % Hkv == 0 && Lq >= 0 && Lq <= (1 << 26) &&
         B * Lq * Hq <= (1 << 30) && Lp >= 0 && Lp <= (1 << 30) && Ls >= 0 && Ls <= (1 << 30) && (D == 64 || D == 128);
}

template <int DT, int D>
int launch_rows(const RowArgs& a, int64_t wgs, bool i8, hipStream_t st) {
  const bool mend = a.src[1].causal && a.Lq > 1 && a.src[1].len > 0;  // (a single query sees all of its own keys)
  auto attention = [&](auto i8_c, auto mend_c) {
    hipLaunchKernelGGL((row_attention_kernel<DT, D, decltype(i8_c)::value, decltype(mend_c)::value>), dim3((unsigned)wgs),
                       dim3(kWaves * 64), 0, st, a);
  };
  if (i8) attention(std::true_type(), std::false_type());
  else if (mend && a.slots == 0) attention(std::false_type(), std::true_type());
  else attention(std::false_type(), std::false_type());
  const int rc = HN_LAUNCH_CHECK("row_attention_kernel");
  if (rc != HN_OK) return rc;
  if (a.slots == 0) return HN_OK;
  // as many groups of lanes on a row as its slots feed
  constexpr int most = 256 / (D / 4);
  auto combine = [&](auto gr_c) {
    constexpr int GR = decltype(gr_c)::value, R = most / GR;
    const dim3 grid((unsigned)((a.ids + R - 1) / R)), block(256);
    if (mend) hipLaunchKernelGGL((row_combine_kernel<DT, D, GR, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((row_combine_kernel<DT, D, GR, false>), grid, block, 0, st, a);
  };
  if (a.slots >= 16) combine(std::integral_constant<int, 8>());
  else if (a.slots >= 4) combine(std::integral_constant<int, 4>());
  else combine(std::integral_constant<int, 1>());
  return HN_LAUNCH_CHECK("row_combine_kernel");
}

int check_rows(const char* who, const RowArgs& a, int64_t Hq, int64_t Hkv, int64_t D, int dtype, float scale) {
  HN_REQUIRE(a.B >= 0 && a.Lq >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && a.src[0].len >= 0 && a.src[1].len >= 0,
             "%s: bad shape B=%lld Lq=%lld Hq=%lld Hkv=%lld", who, (long long)a.B, (long long)a.Lq, (long long)Hq, (long long)Hkv);
  HN_REQUIRE(D == 64 || D == 128, "%s: head dim %lld (64 or 128)", who, (long long)D);
  HN_REQUIRE(dtype == HN_DTYPE_BF16 || dtype == HN_DTYPE_F16, "%s: bf16 or fp16 expected, got dtype %d", who, dtype);
  HN_REQUIRE(scale > 1e-30f && scale < 1e30f, "%s: scale must lie between 1e-30 and 1e30", who);
  HN_REQUIRE(plan_shape(a.B, Hq, Hkv, a.Lq, a.src[0].len, a.src[1].len, D), "%s: problem too large", who);
  HN_REQUIRE(a.B * a.Lq == 0 || (a.q && a.o), "%s: null pointer", who);
  auto rows16 = [](const void* p, int64_t b, int64_t h, int64_t j, int64_t per16) {
    return ((uintptr_t)p & 15) == 0 && b % per16 == 0 && h % per16 == 0 && j % per16 == 0;
  };
  HN_REQUIRE(rows16(a.q, a.sqb, a.sqh, a.sqi, 8) && ((uintptr_t)a.o & 7) == 0 && a.sob % 4 == 0 && a.soh % 4 == 0 && a.soi % 4 == 0,
             "%s: q rows must be 16-byte and out rows 8-byte aligned", who);
  for (int t = 0; t < 2; t++) {
    const KeySource& s = a.src[t];
    HN_REQUIRE(s.len == 0 || (s.k && s.v), "%s: null keys", who);
    HN_REQUIRE((s.ks == nullptr) == (s.vs == nullptr) && ((uintptr_t)s.ks & 3) == 0 && ((uintptr_t)s.vs & 3) == 0,
               "%s: int8 keys and values both need scales", who);
    const int64_t per16 = s.ks ? 16 : 8;
    HN_REQUIRE(rows16(s.k, s.skb, s.skh, s.skj, per16) && rows16(s.v, s.svb, s.svh, s.svj, per16),
               "%s: key and value rows must be 16-byte aligned", who);
    HN_REQUIRE(s.skj >= 0 && s.skj <= (1 << 23) && s.svj >= 0 && s.svj <= (1 << 23), "%s: token strides of k and v in [0, 2^23]", who);
    HN_REQUIRE(((uintptr_t)s.lengths & (s.lengths64 ? 7 : 3)) == 0, "%s: misaligned lengths", who);
  }
  return HN_OK;
}

int run_rows(const char* who, RowArgs& a, int64_t Hq, int64_t Hkv, int64_t D, int dtype, float scale, void* workspace,
             int64_t workspace_bytes, void* stream) {
  const int rc = check_rows(who, a, Hq, Hkv, D, dtype, scale);
  if (rc != HN_OK || a.B * a.Lq == 0) return rc;
  const bool i8 = a.src[0].ks != nullptr && a.src[0].len > 0;
  const RowPlan p = plan_rows(a.B, Hq, Hkv, a.Lq, a.src[0].len, a.src[1].len, D, i8);
  const int64_t need = plan_bytes(p, D);
  HN_REQUIRE(p.wgs <= 0x7fffffff && p.ids * p.slots <= ((int64_t)1 << 40), "%s: problem too large", who);
  HN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0),
             "%s: workspace of %lld bytes (256-byte aligned), %lld needed", who, (long long)workspace_bytes, (long long)need);
  a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.by_hkv.set(Hkv); a.by_g.set(a.G); a.by_per.set(a.Lq * a.G); a.by_hq.set(Hq); a.by_lq.set(a.Lq);
  a.job[0] = p.job[0]; a.job[1] = p.job[1];
  a.njobs = p.njobs; a.slots = p.slots; a.ids = p.ids;
  a.pml = (float2*)workspace;
  a.po = (float*)((char*)workspace + (p.slots * p.ids * 8 + 255) / 256 * 256);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == HN_DTYPE_BF16)
    return D == 128 ? launch_rows<HN_DTYPE_BF16, 128>(a, p.wgs, i8, st) : launch_rows<HN_DTYPE_BF16, 64>(a, p.wgs, i8, st);
  return D == 128 ? launch_rows<HN_DTYPE_F16, 128>(a, p.wgs, i8, st) : launch_rows<HN_DTYPE_F16, 64>(a, p.wgs, i8, st);
}

}  // namespace
}  // namespace hn

extern "C" int64_t hn_cross_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Lq, int64_t Lk, int64_t D) {
  using namespace hn;
  if (!plan_shape(B, Hq, Hkv, Lq, 0, Lk, D)) return -1;
  return B * Lq ? plan_bytes(plan_rows(B, Hq, Hkv, Lq, 0, Lk, D, false), D) : 0;
}

extern "C" int hn_cross_attention(const void* q, int64_t sqb, int64_t sqh, int64_t sqi, const void* k, int64_t skb,
                                  int64_t skh, int64_t skj, const void* v, int64_t svb, int64_t svh, int64_t svj,
                                  const void* lengths, int lengths_bits, const uint8_t* mask, int64_t smb, void* out,
                                  int64_t sob, int64_t soh, int64_t soi, int64_t B, int64_t Hq, int64_t Hkv, int64_t Lq,
                                  int64_t Lk, int64_t D, int dtype, float scale, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  using namespace hn;
  HN_REQUIRE(lengths == nullptr || lengths_bits == 32 || lengths_bits == 64, "hn_cross_attention: lengths of 32 or 64 bits");
  RowArgs a{};
  a.q = (const uint16_t*)q; a.sqb = sqb; a.sqh = sqh; a.sqi = sqi;
  a.o = (uint16_t*)out; a.sob = sob; a.soh = soh; a.soi = soi;
  a.src[1] = KeySource{k, v, skb, skh, skj, svb, svh, svj, nullptr, nullptr, 0, 0, 0, 0, Lk, lengths, lengths_bits == 64, mask, smb, 0};
  a.B = B; a.Lq = Lq;
  return run_rows("hn_cross_attention", a, Hq, Hkv, D, dtype, scale, workspace, workspace_bytes, stream);
}

extern "C" int64_t hn_prefix_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Lq, int64_t Lp, int64_t Ls,
                                                       int64_t D, int int8_prefix) {
  using namespace hn;
  if (!plan_shape(B, Hq, Hkv, Lq, Lp, Ls, D)) return -1;
  return B * Lq ? plan_bytes(plan_rows(B, Hq, Hkv, Lq, Lp, Ls, D, int8_prefix && Lp > 0), D) : 0;
}

extern "C" int hn_prefix_attention(const void* q, int64_t sqb, int64_t sqh, int64_t sqi, const int64_t* prefix, int64_t Lp,
                                   const void* k, int64_t skb, int64_t skh, int64_t skj, const void* v, int64_t svb,
                                   int64_t svh, int64_t svj, const void* lengths, int lengths_bits, int causal, void* out,
                                   int64_t sob, int64_t soh, int64_t soi, int64_t B, int64_t Hq, int64_t Hkv, int64_t Lq,
                                   int64_t Ls, int64_t D, int dtype, float scale, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  using namespace hn;
  HN_REQUIRE(lengths == nullptr || lengths_bits == 32 || lengths_bits == 64, "hn_prefix_attention: lengths of 32 or 64 bits");
  HN_REQUIRE(prefix != nullptr, "hn_prefix_attention: null prefix table");
  RowArgs a{};
  a.q = (const uint16_t*)q; a.sqb = sqb; a.sqh = sqh; a.sqi = sqi;
  a.o = (uint16_t*)out; a.sob = sob; a.soh = soh; a.soi = soi;
  const int64_t* p = prefix;
  a.src[0] = KeySource{(const void*)p[0], (const void*)p[6], 0, p[1], p[2], 0, p[7], p[8], (const float*)p[3], (const float*)p[9],
                       p[4], p[5], p[10], p[11], Lp, nullptr, 0, nullptr, 0, 0};
  a.src[1] = KeySource{k, v, skb, skh, skj, svb, svh, svj, nullptr, nullptr, 0, 0, 0, 0, Ls, lengths, lengths_bits == 64, nullptr, 0,
                       causal};
  a.B = B; a.Lq = Lq;
  return run_rows("hn_prefix_attention", a, Hq, Hkv, D, dtype, scale, workspace, workspace_bytes, stream);
}
