// Shared definitions of the attention kernels over packed sequences (attention_packed.hip) and over the paged 8-bit cache
// (attention_paged.hip).
//
//   o_i = sum_j p_ij v_j,   p_ij = exp(scale q_i . k_j - m_i) / l_i      over the keys j that row i of its sequence sees:
//   j < Lk, and j <= i + Lk - Lq if causal (the last query row sees the last key).  A row that sees no key is 0.
//
// Rows: query head hq reads key head hq / G, G = Hq / Hkv.  A work item takes ONE key head and packs its G query heads into its
// rows -- row r of a sequence is token r / G, head h G + r % G -- so a K / V tile is read once for all of them.
#pragma once
#include "common.h"

namespace iggt_seq {

struct SeqAttnParams {
    const bf16_t* q;      // 16-bit [Tq][Hq][D], strides in elements
    bf16_t* o;
    const bf16_t* k;      // packed sequences: 16-bit [Tk][Hkv][D]
    const bf16_t* v;
    long q_rs, q_hs, o_rs, o_hs, k_rs, k_hs, v_rs, v_hs;
    const int* cu_q;      // [B + 1] first row of every sequence; nullptr: sequence b is row b
    const int* cu_k;      // [B + 1] packed sequences only
    // paged cache: e4m3 codes, K [pages][Hkv][page][D] and V [pages][Hkv][page / 16][D][16] (16 keys of a channel side by side:
    // the A operand of V^T P^T without a transposition); scale exponents (2^(byte - 127)) [pages][Hkv]
    const uint8_t* k8;
    const uint8_t* v8;
    const uint8_t* k_scale;
    const uint8_t* v_scale;
    const int* tables;    // [B][table_stride] page of every page / token block, in order
    const int* lens;      // [B] keys of every request
    long table_stride;
    int table_width, num_pages, page_shift;
    int B, Hq, Hkv, G, Tq, Tk, max_q, causal;
    int qtiles, splits;
    int range_blocks;     // few rows: key range of a split in blocks of 64 keys
    unsigned items;       // work items; the grid may have more (their sequence and key head exist all the same)
    float scale_log2;     // softmax scale * log2(e)
    // splits > 1: key range s of a row leaves its unnormalised sum [splits][B][max_q][Hq][D] and (maximum, row sum) here
    float* part_o;
    float* part_ml;
};

// Grid of n < 2^31 work items and the item of a workgroup.  A grid's dimension may not have 2^32 threads: rows of 2^20 workgroups where
// there are more (one long prompt among many thousand sequences).
constexpr int GRID_ROW_LOG2 = 20;
inline dim3 seq_grid(long n) {
    return n <= (1L << GRID_ROW_LOG2) ? dim3((unsigned)n) : dim3(1u << GRID_ROW_LOG2, (unsigned)(((n - 1) >> GRID_ROW_LOG2) + 1));
}
IGGT_DEVINL unsigned seq_item() { return blockIdx.x + (blockIdx.y << GRID_ROW_LOG2); }

constexpr float M_INIT = -3.0e38f;   // running maximum before the first key: finite, so that a masked score (-inf) gives 2^-inf = 0
constexpr int FOLD_MAX = 64;         // key ranges a row is folded from at most
constexpr float P_SHIFT_F16 = 8.0f;  // fp16 numerators are 2^(s - m + 8): the small ones stay normal; cancels in O / l

struct SeqSpan {
    int q0, lq, lk, k0;
    int off;              // causal: row i sees keys j <= i + off
};
// Rows and keys of sequence b.  The prefix sums and lengths are device data nobody has checked: they are clamped to the tensors.  lq is
// the number of rows to compute (max_q at most), off that of the whole sequence.
template <bool PAGED>
IGGT_DEVINL SeqSpan seq_span(const SeqAttnParams& p, int b) {
    SeqSpan s;
    int q1;
    if (p.cu_q != nullptr) {
        s.q0 = min(max(p.cu_q[b], 0), p.Tq);
        q1 = min(max(p.cu_q[b + 1], 0), p.Tq);
    } else {
        s.q0 = min(b, p.Tq);
        q1 = min(b + 1, p.Tq);
    }
    const int lq = max(q1 - s.q0, 0);
    s.lq = min(lq, p.max_q);
    if constexpr (PAGED) {
        s.k0 = 0;
        s.lk = (int)min((long)max(p.lens[b], 0), (long)p.table_width << p.page_shift);
    } else {
        s.k0 = min(max(p.cu_k[b], 0), p.Tk);
        s.lk = max(min(max(p.cu_k[b + 1], 0), p.Tk) - s.k0, 0);
    }
    s.off = s.lk - lq;
    return s;
}

// Table entry of the page of token `at` of request b (lk > 0, so the table has an entry; tokens behind its end read the last one and
// are masked by their position).  The entry is not looked at here: a check would wait for the load.
IGGT_DEVINL int page_entry(const SeqAttnParams& p, int b, int at) {
    return p.tables[(long)b * p.table_stride + min((int)((unsigned)at >> p.page_shift), p.table_width - 1)];
}
IGGT_DEVINL bool page_ok(const SeqAttnParams& p, int id) { return (unsigned)id < (unsigned)p.num_pages; }

// 16 e4m3 codes -> two fragments of 8 in the 16-bit operand type, times 2^(e - 127) (a power of two, so bf16 is exact; fp16 is
// exact down to its subnormal step).  The instruction takes the scale as a float of which it reads the exponent.
template <int FMT>
IGGT_DEVINL void cvt16(u32x4 c, float scale, bf16x8& lo, bf16x8& hi) {
    u32x4 a, b;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (FMT == FMT_F16) {
            a[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], scale, false));
            a[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], scale, true));
            b[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i + 2], scale, false));
            b[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i + 2], scale, true));
        } else {
            a[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], scale, false));
            a[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i], scale, true));
            b[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i + 2], scale, false));
            b[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[i + 2], scale, true));
        }
    }
    lo = __builtin_bit_cast(bf16x8, a);
    hi = __builtin_bit_cast(bf16x8, b);
}
// 2^(byte - 127) as a float: bytes 1 .. 254 are the float exponent as it stands, 0 and 255 (never written) are moved inside
IGGT_DEVINL float scale_of(uint32_t byte) {
    byte = byte < 1u ? 1u : (byte > 254u ? 254u : byte);
    return __builtin_bit_cast(float, byte << 23);
}

template <int FMT>
IGGT_DEVINL uint32_t nonfinite2(uint32_t w) {   // nonzero if one of the two elements is inf or NaN
    constexpr uint32_t E = FMT == FMT_F16 ? 0x7c007c00u : 0x7f807f80u, U = FMT == FMT_F16 ? 0x04000400u : 0x00800080u;
    return ((w & E) + U) & 0x80008000u;
}
template <int FMT>
IGGT_DEVINL bool nonfinite8(bf16x8 f) {
    const u32x4 w = __builtin_bit_cast(u32x4, f);
    return (nonfinite2<FMT>(w[0]) | nonfinite2<FMT>(w[1]) | nonfinite2<FMT>(w[2]) | nonfinite2<FMT>(w[3])) != 0;
}
template <int FMT>
IGGT_DEVINL bf16x8 pack8f(const float* s) {   // softmax numerators -> operand fragment
    u32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = pack_h2<FMT, false>(s[2 * j], s[2 * j + 1]);
    return __builtin_bit_cast(bf16x8, r);
}

}  // namespace iggt_seq

// attention_packed.hip: tile kernel over packed (16-bit) or paged (8-bit) keys; attention_paged.hip: fold of key ranges
int iggt_launch_seq_tiles(const iggt_seq::SeqAttnParams& p, int D, int fmt, bool paged, bool small, hipStream_t stream);
int iggt_launch_seq_fold(const iggt_seq::SeqAttnParams& p, int D, int fmt, bool paged, hipStream_t stream);
// number of key ranges and tile height (rows of a work item) for this many (sequence, key head) pairs
struct SeqPlan {
    int splits;
    bool small;   // 128-row tiles where 256-row ones exist
    int range_blocks;
};
SeqPlan iggt_seq_tile_plan(int B, long max_q, long max_k, int Hkv, int G, int D, bool paged);
