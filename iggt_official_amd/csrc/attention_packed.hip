// Flash attention over packed sequences of different lengths: causal or not, grouped heads, head dim 64 | 128, 16-bit operands,
// fp32 statistics and accumulators; the same tile kernel serves many query rows over the paged 8-bit cache.
//
// Mathematics (seq_attention.h): online softmax over 64-key tiles.  Swapped product: S^T = K Q^T puts one query row into a lane
// (columns of the 32 x 32 MFMA), so its maximum and sum need one exchange with lane ^ 32, and the numerators P^T leave the
// accumulator already in the layout of the B operand of O^T = V^T P^T: the 8 keys a lane half holds in registers 8u .. 8u + 7 of a
// score block are (r & 3) + 8 (r >> 2) + 4 half, and V^T is fetched for exactly those keys (transposing LDS reads of the row-major
// 16-bit tile; the 8-bit tile is stored transposed already).  The maximum moves only when a row exceeds it by 2^4 (numerators
// stay <= 2^4 above it, or 2^12 with fp16's shift), so the rescale of O and l is rare.
//
// Rounding: scores, maxima, sums and O are fp32; the numerators are rounded to the operand type for the second product (the row sum
// adds them before that rounding), O once on the way out (a mean of values of that type: not saturated, inf and NaN stay).
//
// What bounds it (MI355X):
//   head dim 64, 16-bit keys: one query block per wave, nothing overlapped within it but four waves on a SIMD (128 registers).  Vector
//     pipe 80 % busy, matrix pipe 48 %.  4 sequences of up to 10 992 tokens, 16 heads, full, fp16: 1 205 - 1 300 us between machines,
//     850 - 910 TFLOP/s, at a clock that this load pulls down to 1.7 GHz; of the vector work the running maximum (its tree, exchange and
//     vote) is what the trunk's kernel, which knows its shift beforehand, does without (1 080 - 1 130 TFLOP/s).  Two waves per SIMD with two query blocks each, offset against each other: the same
//     there, 8 x 1 374 causal tokens 71 -> 57, 3 x 1 374 full 55 -> 48; pipelined over the tiles: 4 x 5 496 full 619 -> 590, 16 x 1 374
//     causal 118 -> 100.  Small grids run the pipelined form (launch_fmt).
//   head dim 128: one query block, pipelined over the tiles.  Matrix and vector pipe 50 % each, 1.8 waves.  Prompts of 12 001 and 7 645
//     tokens, 16 query and 4 key heads, causal, bf16: 800 - 880 us, 940 - 1 040 TFLOP/s at 1.9 GHz (a large library matrix product here:
//     1 430 - 1 450).  Before the pipeline and the fragments read ahead 970; eight waves and 256 rows per workgroup: 5 % slower.
//   8-bit keys: the same with the conversion in front, shared by 256 rows where there are as many (head dim 64: two query blocks per
//     wave, 128: eight waves).  1 374 rows against 12 366 tokens, 2 x 16 heads of 64, fp16: 205 - 240 us with the fold (one query block:
//     + 10 %), 580 - 680 TFLOP/s; 6 x 1 374 rows against 36 343 tokens, 8 query and 2 key heads: 524 - 565 (+ 15 %).  Head dim 128, 5 x
//     1 374 rows against <= 10 175 tokens, 8 heads: 322; 10 to 31 vector registers are spilled there.
//   small grids: the chain of one wave's tiles, 0.8 us each; loads four tiles ahead instead of one change nothing.
//
// Values that are not finite: a masked score is replaced, not added to, so NaN in K costs nothing.  V does: 0 * inf = NaN in the
// matrix product.  A tile in which some row sees a key and another does not is therefore scanned (one or two of a row's many); if
// it holds inf or NaN they are added to exactly the rows that see them and the product runs on zeros in their place.
#include "seq_attention.h"
#include "../../include/iggt_hip.h"
#include <cmath>

using namespace iggt_seq;

namespace {

constexpr float DEFER_THR = 4.0f;

// 16 bytes per lane from base + off straight into LDS at lds + 16 * lane (both uniform).  Inline assembly because the compiler's own
// bookkeeping waits for every such load in flight before the next LDS read of the kernel, which is the next tile's arrival before this
// tile's work.  No register is written, so nothing but the caller's arrive() has to know when it is done.
IGGT_DEVINL void lds_load16(const void* base, uint32_t off, const char* lds) {
    const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :: "v"(off), "s"(base), "s"(at) : "memory");   // (m0 is reserved: the compiler holds no value in it here)
}
// all of this wave's LDS loads have arrived, and every wave of the workgroup has come here
IGGT_DEVINL void arrive() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Order of the work items.  Longest first, so that the last ones to start are short: under a causal mask the last query tiles, else
// the sequences by their number of keys (up to 64 of them: ranked here, one lane each).  Key heads innermost: consecutive workgroups
// go to the XCDs in turn, so one head's tiles share an L2.  Where (sequence, head) pairs are a multiple of 8 but heads are not, an
// XCD would keep one sequence for good: the pairs move on by one every 8 tiles (grouped prompts of 12 001 and 7 645 tokens, 8 pairs:
// 932 us in place, 879 moved with every tile, 850 with every fourth, 845 every eighth: moving balances, staying shares the L2).
template <bool PAGED>
IGGT_DEVINL void work_item(const SeqAttnParams& p, int lane, int& split, int& qt, int& b, int& h) {
    int w = (int)seq_item();
    if (p.causal || p.B == 1 || p.B > 64) {
        const int npairs = p.B * p.Hkv;
        int pair = w % npairs;
        w /= npairs;
        split = w % p.splits;
        const int at = w / p.splits;
        qt = p.qtiles - 1 - at;
        pair = (pair + at / min(max(p.qtiles >> 4, 1), 8)) % npairs;
        b = pair / p.Hkv;
        h = pair - b * p.Hkv;
    } else {
        h = w % p.Hkv;
        w /= p.Hkv;
        split = w % p.splits;
        w /= p.splits;
        qt = w % p.qtiles;
        const int place = min(w / p.qtiles, p.B - 1);
        const int lk = lane < p.B ? seq_span<PAGED>(p, lane).lk : -1;
        int rank = 0;
        for (int i = 0; i < p.B; ++i) {
            const int other = __builtin_amdgcn_readlane(lk, i);
            rank += (other > lk || (other == lk && i < lane)) ? 1 : 0;
        }
        const unsigned long long mine = __ballot(lane < p.B && rank == place);
        b = (int)__builtin_ctzll(mine);
    }
}

// Waves on a SIMD.  Two have 256 registers each and overlap matrix and vector work within a wave.  Head dim 64, 16-bit keys: without a
// second tile's scores a wave needs 128, so that four run and fill each other's waits -- where there are as many (launch_fmt).
template <int D, int QB, int NW, int FMT, bool PAGED, int WPS>
__global__ __launch_bounds__(64 * NW, WPS) void seq_attn_tile_kernel(const SeqAttnParams p) {
    constexpr int ROWB = D * 2, K_BYTES = 64 * ROWB, TILE = 2 * K_BYTES, NKC = D / 16, NDH = D / 32, BM = 32 * NW * QB;
    constexpr bool PIPELINED = QB == 1 && WPS == 2;   // over the tiles
    constexpr int NT = 64 * NW;   // threads
    constexpr int SLOTS = ROWB / 16;   // 16-byte slots of a K row
    __shared__ __attribute__((aligned(16))) char smem[2 * TILE];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int frow = lane & 31, fhalf = lane >> 5;

    int split, qt, b, h;
    work_item<PAGED>(p, lane, split, qt, b, h);
    const SeqSpan sp = seq_span<PAGED>(p, b);
    const long rows = (long)sp.lq * p.G;
    const long row0 = (long)qt * BM;
    if (seq_item() >= p.items || row0 >= rows) return;   // (asked late: the arguments come in one go)
    auto limit_of = [&](long row) {   // keys that row sees
        return p.causal ? max(min(sp.lk, sp.off + (int)(row / p.G) + 1), 0) : sp.lk;
    };
    const int kend = limit_of(min(row0 + BM, rows) - 1);
    const int ktiles = (kend + 63) >> 6;
    const int t0 = (int)((long)ktiles * split / p.splits), t1 = (int)((long)ktiles * (split + 1) / p.splits);

    const int wg_first = limit_of(row0);   // keys every row of the tile sees
    const long wrow = row0 + wave * (32 * QB);
    const bool live_wave = wrow < rows;
    const int w_first = live_wave ? limit_of(wrow) : 0;                                   // keys every row of the wave sees
    const int w_last = live_wave ? limit_of(min(wrow + 32 * QB, rows) - 1) : 0;           // keys its last row sees

    bf16x8 qf[QB][NKC];
    int lim[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const long r = min(wrow + qb * 32 + frow, rows - 1);
        const int i = (int)(r / p.G), hq = h * p.G + (int)(r - (long)i * p.G);
        lim[qb] = limit_of(r);
        const bf16_t* src = p.q + (long)(sp.q0 + i) * p.q_rs + (long)hq * p.q_hs + 8 * fhalf;
#pragma unroll
        for (int kc = 0; kc < NKC; ++kc) qf[qb][kc] = *reinterpret_cast<const bf16x8*>(src + 16 * kc);
    }

    // the query fragments arrive here, so that no use of them in the tile loop waits for loads in flight
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int kc = 0; kc < NKC; ++kc) {
            u32x4 w = __builtin_bit_cast(u32x4, qf[qb][kc]);
            asm volatile("" : "+v"(w));
            qf[qb][kc] = __builtin_bit_cast(bf16x8, w);
        }

    // ---- staging.  16-bit: LDS-DMA, 1 KiB per wave and instruction; the row-image swizzles are applied to the source piece, rows
    //      past the end are clamped to the last key (masked; see the file comment for values that are not finite).
    constexpr int RPC = 1024 / ROWB;            // rows of a 1 KiB chunk
    constexpr int CPW = K_BYTES / 1024 / NW;    // chunks per wave
    const bf16_t* kb_ptr = nullptr;
    const bf16_t* vb_ptr = nullptr;
    // the lane's piece of chunk i is in row wave CPW RPC + i RPC + lane / SLOTS of the tile, at the swizzled byte column kcol ^ flip(i) of
    // K and vcol of V
    const int drow = wave * (CPW * RPC) + lane / SLOTS, pos = lane % SLOTS;
    const int kcol = (D == 64 ? pos ^ ((drow >> 1) & 7) : pos ^ (drow & 15)) * 16;
    const int vcol = (D == 64 ? (((pos >> 1) ^ (drow & 2)) << 1) | (pos & 1) : (((pos >> 1) ^ ((drow & 3) << 1)) << 1) | (pos & 1)) * 16;
    static_assert(CPW <= 1 || (RPC * CPW) % 8 == 0, "a wave's rows begin where the swizzle does");
    uint32_t koff0 = 0, voff0 = 0;              // byte offset of the first chunk's piece (host: a tile spans less than 2^32)
    if constexpr (!PAGED) {
        kb_ptr = p.k + (long)sp.k0 * p.k_rs + (long)h * p.k_hs;
        vb_ptr = p.v + (long)sp.k0 * p.v_rs + (long)h * p.v_hs;
        koff0 = (uint32_t)drow * (uint32_t)(2 * p.k_rs);
        voff0 = (uint32_t)drow * (uint32_t)(2 * p.v_rs) + vcol;
    }
    auto dma = [&](bool V, int t, char* dst) {       // one 64-key tile of K or of V
        const long rs = V ? p.v_rs : p.k_rs;
        const char* src = reinterpret_cast<const char*>((V ? vb_ptr : kb_ptr) + (long)t * 64 * rs);
        const int left = sp.lk - 1 - t * 64;
#pragma unroll
        for (int i = 0; i < CPW; ++i) {
            const int col = V ? vcol : kcol ^ (D == 64 ? (i * RPC / 2) << 4 : (i * RPC) << 4);
            uint32_t at = (V ? voff0 : koff0 + col) + (uint32_t)(i * RPC) * (uint32_t)(2 * rs);
            if (left < 63) at = (uint32_t)min(drow + i * RPC, left) * (uint32_t)(2 * rs) + col;
            lds_load16(src, at, dst + (wave * CPW + i) * 1024);
        }
    };
    // 8-bit: codes go through registers (16 bytes each), are converted and written as 16-bit tiles: K rows like above, V transposed
    // [D][64 keys] with the keys of every 16 in the order 0-3, 8-11 | 4-7, 12-15 (what the two lane halves need side by side).
    // fp16 holds half of V's values (a code of a scale near fp16's range would round to 2^16; the factor 2 goes into the epilogue), and
    // K's times a power of two that takes the largest scale of the key range to 2^7 (a cache may have been written from bf16; the inverse
    // goes into the softmax scale): exact for scales down to 2^-15, 22 powers of two below the largest, and a key that is smaller yet is
    // off by 2^-42 of the largest key.
    constexpr int PIECES = 4 * D;                                       // 16-byte pieces of K in a tile, and of V
    constexpr int PPT = PIECES / NT;                                    // a thread's of each
    static_assert(!PAGED || PIECES % NT == 0, "every thread takes as many");
    constexpr float HALF = (PAGED && FMT == FMT_F16) ? 0.5f : 1.0f;
    constexpr int HELD = PPT > 0 ? PPT : 1;                             // (16-bit keys: nothing)
    u32x4 k8r[HELD], v8r[HELD];
    uint32_t kbyte[HELD], vbyte[HELD];
    uint32_t have = 0xf, have1 = 0xf, have2 = 0xf;   // which 16-key groups have a page: this tile, the next one, the one after it
    // a wave's piece i lies in one 16-key group of D pieces: one table entry (lane l: group l & 3), loaded a tile ahead, serves its K
    // and, a tile later, its V
    const int psub = __builtin_amdgcn_readfirstlane(tid / D), pin16 = tid % D;   // group (+ i NT / D) and piece within it
    int pid_v = 0, pid_k = 0;
    auto look_up = [&](int t) { return page_entry(p, b, t * 64 + (lane & 3) * 16); };
    auto groups = [&](int pid) { return (uint32_t)__ballot(page_ok(p, pid)) & 0xfu; };
    auto fetch = [&](bool V, int t, int pid, u32x4 (&code)[HELD], uint32_t (&byte)[HELD]) {
#pragma unroll
        for (int i = 0; i < PPT; ++i) {
            const int sub = psub + i * (NT / D), id = __builtin_amdgcn_readlane(pid, sub);
            const long head = (long)(page_ok(p, id) ? id : 0) * p.Hkv + h;
            const long at = ((head << p.page_shift) + ((t * 64 + sub * 16) & ((1 << p.page_shift) - 1))) * D + pin16 * 16;
            byte[i] = (V ? p.v_scale : p.k_scale)[head];
            code[i] = *reinterpret_cast<const u32x4*>((V ? p.v8 : p.k8) + at);
        }
    };
    float kf = 1.0f, c = p.scale_log2;
    if constexpr (PAGED && FMT == FMT_F16) {
        __shared__ int s_top[NW];
        int top = 7;                                 // (the factor stays a float)
        const int pages = ((min(t1 * 64, kend) - 1) >> p.page_shift) + 1;
        for (int i = ((t0 * 64) >> p.page_shift) + tid; i < pages; i += NT) {
            const int id = page_entry(p, b, i << p.page_shift);
            if (page_ok(p, id)) top = max(top, (int)p.k_scale[(long)id * p.Hkv + h]);
        }
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) top = max(top, __shfl_xor(top, x, 64));
        if (lane == 0) s_top[wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; ++w) top = max(top, s_top[w]);
        const int shift = 134 - __builtin_amdgcn_readfirstlane(min(top, 254));
        kf = __builtin_bit_cast(float, (127 + shift) << 23);
        // (neither 0 nor inf, times which a masked score or a zero would be NaN)
        c = __builtin_amdgcn_fmed3f(__builtin_amdgcn_ldexpf(c, -shift), 0x1p-149f, 3.4028235e38f);
        c = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, c)));
    }
    auto stage_k = [&](char* sK) {
#pragma unroll
        for (int i = 0; i < PPT; ++i) {
            const int key = (psub + i * (NT / D)) * 16 + pin16 / (D / 16), piece = pin16 % (D / 16), sw = D == 64 ? (key >> 1) & 7 : key & 15;
            bf16x8 lo, hi;
            cvt16<FMT>(k8r[i], scale_of(kbyte[i]) * kf, lo, hi);
            *reinterpret_cast<bf16x8*>(sK + key * ROWB + ((2 * piece) ^ sw) * 16) = lo;
            *reinterpret_cast<bf16x8*>(sK + key * ROWB + ((2 * piece + 1) ^ sw) * 16) = hi;
        }
    };
    auto stage_v = [&](char* sV) {
#pragma unroll
        for (int i = 0; i < PPT; ++i) {
            const int sub = psub + i * (NT / D);
            bf16x8 lo, hi;
            cvt16<FMT>(v8r[i], scale_of(vbyte[i]) * HALF, lo, hi);
            const u32x4 a = __builtin_bit_cast(u32x4, lo), z = __builtin_bit_cast(u32x4, hi);
            const u32x4 x = {a[0], a[1], z[0], z[1]}, y = {a[2], a[3], z[2], z[3]};
            *reinterpret_cast<u32x4*>(sV + swz_off(pin16, 2 * sub)) = x;
            *reinterpret_cast<u32x4*>(sV + swz_off(pin16, 2 * sub + 1)) = y;
        }
    };

    f32x16 o[QB][NDH];
    float m_run[QB], l_run[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        m_run[qb] = M_INIT;
        l_run[qb] = 0.f;
#pragma unroll
        for (int dh = 0; dh < NDH; ++dh)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[qb][dh][r] = 0.f;
    }

    // lane-dependent LDS offsets
    int koff[NKC], voff[NDH];
#pragma unroll
    for (int kc = 0; kc < NKC; ++kc)
        koff[kc] = frow * ROWB + (D == 64 ? (((2 * kc + fhalf) ^ (frow >> 1)) & 7) << 4 : ((2 * kc + fhalf) ^ (frow & 15)) << 4);
    const int tr_i = lane & 15, tr_g = (lane >> 4) & 1;
    {
        const int vr = 4 * fhalf + (tr_i >> 2);
#pragma unroll
        for (int dh = 0; dh < NDH; ++dh)
            voff[dh] = vr * ROWB + (D == 64 ? ((dh * 2 + tr_g) ^ (vr & 2)) << 5 : ((dh * 2 + tr_g) ^ ((vr & 3) << 1)) << 5) + 8 * (tr_i & 3);
    }
    auto v_frag = [&](const char* sV, int kvh, int cc, int dh) -> bf16x8 {
        if constexpr (PAGED) {
            return *reinterpret_cast<const bf16x8*>(sV + swz_off(dh * 32 + frow, 2 * (2 * kvh + cc) + fhalf));
        } else {
            typedef __attribute__((address_space(3))) short4v lds_s4;
            typedef short short8v __attribute__((ext_vector_type(8)));
            const char* base = sV + (kvh * 32 + 16 * cc) * ROWB + voff[dh];
            const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(base));
            const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(base + 8 * ROWB));
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    };
    auto qk = [&](const char* sK, int qb, f32x16 (&s)[2]) __attribute__((always_inline)) {
        const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kvh = 0; kvh < 2; ++kvh)
#pragma unroll
            for (int kc = 0; kc < NKC; ++kc) {
                const bf16x8 kf = *reinterpret_cast<const bf16x8*>(sK + kvh * 32 * ROWB + koff[kc]);
                s[kvh] = mfma32h<FMT>(kf, qf[qb][kc], kc == 0 ? zero : s[kvh]);
            }
    };
    // One query block per wave: the operand fragments are read a group of four matrix instructions ahead of their use.  (The LDS reads
    // and matrix instructions keep this order, other work may move between them: left alone, the compiler reads every fragment right
    // in front of its use to save registers, and the wave waits for each.)
    auto order = [&]() { __builtin_amdgcn_sched_barrier(0x0406); };
    auto qk_ahead = [&](const char* sK, f32x16 (&s)[2]) __attribute__((always_inline)) {
        const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        bf16x8 f[2][4];
        auto read = [&](int g, bf16x8 (&x)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const bf16x8*>(sK + (j & 1) * 32 * ROWB + koff[2 * g + (j >> 1)]);
        };
        read(0, f[0]);
#pragma unroll
        for (int g = 0; g < NKC / 2; ++g) {
            order();
            if (g + 1 < NKC / 2) read(g + 1, f[(g + 1) & 1]);
            order();
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j & 1] = mfma32h<FMT>(f[g & 1][j], qf[0][2 * g + (j >> 1)], g == 0 && j < 2 ? zero : s[j & 1]);
        }
        order();
    };
    auto pv_ahead = [&](const char* sV, const bf16x8 (&pf)[2][2]) __attribute__((always_inline)) {
        bf16x8 f[2][NDH];
        auto read = [&](int g, bf16x8 (&x)[NDH]) {
#pragma unroll
            for (int dh = 0; dh < NDH; ++dh) x[dh] = v_frag(sV, g >> 1, g & 1, dh);
        };
        read(0, f[0]);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            order();
            if (g < 3) read(g + 1, f[(g + 1) & 1]);
            order();
#pragma unroll
            for (int dh = 0; dh < NDH; ++dh) o[0][dh] = mfma32h<FMT>(f[g & 1][dh], pf[g >> 1][g & 1], o[0][dh]);
        }
        order();
    };
    auto mask = [&](int t, int qb, f32x16 (&s)[2], uint32_t groups_) __attribute__((always_inline)) {
        asm volatile("");                                  // (keeps the branch: as selects this would be half of every tile's work)
        const int seen = lim[qb] - t * 64 - 4 * fhalf;     // key kvh * 32 + (r & 3) + 8 (r >> 2) (+ 4 half) is seen if it is less
#pragma unroll
        for (int kvh = 0; kvh < 2; ++kvh)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (kvh * 32 + (r & 3) + 8 * (r >> 2) >= seen || (PAGED && !((groups_ >> (kvh * 2 + (r >> 3))) & 1))) s[kvh][r] = -INFINITY;
    };
    auto row_max = [&](const f32x16 (&s)[2]) __attribute__((always_inline)) {
        float mx = s[0][0];
#pragma unroll
        for (int kvh = 0; kvh < 2; ++kvh)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kvh][r]);
        const uint32_t bits = __builtin_bit_cast(uint32_t, mx);
        const auto sw = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
        return fmaxf(__builtin_bit_cast(float, (uint32_t)sw[0]), __builtin_bit_cast(float, (uint32_t)sw[1])) * c;
    };
    auto raise_max = [&](int qb, float mx) __attribute__((always_inline)) {
        if (__any(mx > m_run[qb] + DEFER_THR)) {
            const float m_new = fmaxf(m_run[qb], mx);
            const float alpha = __builtin_amdgcn_exp2f(m_run[qb] - m_new);
            m_run[qb] = m_new;
            l_run[qb] *= alpha;
#pragma unroll
            for (int dh = 0; dh < NDH; ++dh)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[qb][dh][r] *= alpha;
        }
    };
    auto exp_pack = [&](int qb, f32x16 (&s)[2], bf16x8 (&pf)[2][2]) __attribute__((always_inline)) {
        const float m = m_run[qb] - (FMT == FMT_F16 ? P_SHIFT_F16 : 0.f);
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kvh = 0; kvh < 2; ++kvh) {
            float e[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kvh][r], c, -m));
                ls[r & 3] += e[r];
            }
            pf[kvh][0] = pack8f<FMT>(e);
            pf[kvh][1] = pack8f<FMT>(e + 8);
        }
        l_run[qb] += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    };
    auto pv = [&](const char* sV, int qb, const bf16x8 (&pf)[2][2]) {
#pragma unroll
        for (int kvh = 0; kvh < 2; ++kvh)
#pragma unroll
            for (int cc = 0; cc < 2; ++cc)
#pragma unroll
                for (int dh = 0; dh < NDH; ++dh) o[qb][dh] = mfma32h<FMT>(v_frag(sV, kvh, cc, dh), pf[kvh][cc], o[qb][dh]);
    };
    // byte of V's element (key, d) in the LDS tile
    auto v_byte = [&](int key, int d) {
        if constexpr (PAGED)
            return swz_off(d, 2 * (key >> 4) + ((key >> 2) & 1)) + 2 * ((key & 3) + ((key >> 3) & 1) * 4);
        else
            return key * ROWB + (D == 64 ? ((d >> 4) ^ (key & 2)) << 5 : ((d >> 4) ^ ((key & 3) << 1)) << 5) + 2 * (d & 15);
    };
    // a tile whose V holds inf or NaN (workgroup-uniform): with the maxima raised to the tile's, so that its rescale does not meet the
    // infinities, add them to the rows that see them and leave zeros for the matrix product
    auto absorb_nonfinite = [&](char* sK, char* sV, int t) __attribute__((always_inline)) {
        if (t * 64 < w_last) {
            if constexpr (!PIPELINED) {
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) {
                    f32x16 s[2];
                    qk(sK, qb, s);
                    mask(t, qb, s, have);
                    raise_max(qb, row_max(s));
                }
            }
#pragma unroll 1
            for (int key = 0; key < 64; ++key) {
                if (PAGED && !((have >> (key >> 4)) & 1)) continue;
                int fh = fhalf;
                asm volatile("" : "+v"(fh));   // addresses are formed here, not kept in registers across the tile loop
#pragma unroll
                for (int dh = 0; dh < NDH; ++dh)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int d = dh * 32 + (r & 3) + 8 * (r >> 2) + 4 * fh;
                        const uint32_t x = *reinterpret_cast<const uint16_t*>(sV + v_byte(key, d));
                        if (nonfinite2<FMT>(x)) {
                            const float f = h2_lo<FMT>(x);
#pragma unroll
                            for (int qb = 0; qb < QB; ++qb)
                                if (t * 64 + key < lim[qb]) o[qb][dh][r] += f;
                        }
                        // (one element after the other: all at once, their masks do not fit into the scalar registers, and what takes
                        // their place is missing in the tile loop -- 5 x <= 10 175 tokens, 8 heads of 128: 390 us, so 322; 70 x 40
                        // rows against 3 000 tokens, 16 heads of 128: 570, so 345)
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }
        __syncthreads();
        for (int i = tid * 4; i < K_BYTES; i += 4 * NT) {
            uint32_t w = *reinterpret_cast<const uint32_t*>(sV + i);
            if (nonfinite2<FMT>(w & 0xffffu)) w &= 0xffff0000u;
            if (nonfinite2<FMT>(w & 0xffff0000u)) w &= 0xffffu;
            *reinterpret_cast<uint32_t*>(sV + i) = w;
        }
        __syncthreads();
    };

    // keeps packed numerators where they are formed, beside the score products in the same block of instructions
    auto pin = [&](bf16x8 (&pf)[2][2]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u32x4 w = __builtin_bit_cast(u32x4, pf[i >> 1][i & 1]);
            asm volatile("" : "+v"(w));
            pf[i >> 1][i & 1] = __builtin_bit_cast(bf16x8, w);
        }
    };

    auto tile_nonfinite = [&](const char* sV) __attribute__((always_inline)) {
        bool bad = false;
        for (int i = tid * 16; i < K_BYTES; i += 16 * NT) bad = bad || nonfinite8<FMT>(*reinterpret_cast<const bf16x8*>(sV + i));
        return __syncthreads_or(bad) != 0;
    };

    if constexpr (PIPELINED) {
        // One query block per wave, pipelined over the tiles: the score product of tile t + 1 runs beside the exponentials of tile t, the
        // maximum of t + 1 beside the second product of t (LDS holds K of t + 1 and V of t while K of t + 2 and V of t + 1 arrive).
        auto kbuf = [&](int t) { return smem + (t & 1) * K_BYTES; };
        auto vbuf = [&](int t) { return smem + (2 + (t & 1)) * K_BYTES; };
        auto step = [&](int t, f32x16 (&s)[2], f32x16 (&sn)[2], char* k_next, char* v_here, char* k_dst, char* v_dst) __attribute__((always_inline)) {
            if constexpr (PAGED) {
                // (past the last tile it is fetched again: a branch here would make every later wait one for all loads)
                const int tk = min(t + 2, t1 - 1);
                fetch(true, t + 1, pid_v, v8r, vbyte);
                fetch(false, tk, pid_k, k8r, kbyte);
                have2 = groups(pid_k);
                pid_v = pid_k;
                pid_k = look_up(min(t + 3, t1 - 1));
            } else {
                dma(true, t + 1, v_dst);
                if (t + 2 < t1) dma(false, t + 2, k_dst);
            }
            if ((t + 1) * 64 > wg_first || (PAGED && have != 0xf)) {
                if (tile_nonfinite(v_here)) absorb_nonfinite(nullptr, v_here, t);
            }
            if (t * 64 < w_last) {
                // (behind a wave's last key the score product runs on what the buffer holds and is dropped: as a branch it would take the
                // exponentials out of the block of instructions in which they run beside it)
                const bool more = (t + 1) * 64 < w_last;
                bf16x8 pf[2][2];
                qk_ahead(k_next, sn);
                exp_pack(0, s, pf);
                pin(pf);
                if (more && ((t + 2) * 64 > w_first || (PAGED && have1 != 0xf))) mask(t + 1, 0, sn, have1);
                pv_ahead(v_here, pf);
                const float mx = row_max(sn);
                raise_max(0, more ? mx : M_INIT);
            }
            if constexpr (PAGED) {
                stage_v(v_dst);
                stage_k(k_dst);
                have = have1;
                have1 = have2;
            }
            arrive();
        };
        if (t0 < t1) {
            const int t2 = min(t0 + 1, t1 - 1);
            if constexpr (PAGED) {
                const int pid = look_up(t0);
                pid_v = look_up(t2);
                pid_k = look_up(min(t0 + 2, t1 - 1));
                have = groups(pid);
                have1 = groups(pid_v);
                fetch(false, t0, pid, k8r, kbyte);
                fetch(true, t0, pid, v8r, vbyte);
                stage_k(kbuf(t0));
                stage_v(vbuf(t0));
                fetch(false, t2, pid_v, k8r, kbyte);
                if (t2 != t0) stage_k(kbuf(t2));
            } else {
                dma(false, t0, kbuf(t0));
                dma(true, t0, vbuf(t0));
                if (t2 != t0) dma(false, t2, kbuf(t2));
            }
            f32x16 sa[2], sb[2];
            arrive();
            if (t0 * 64 < w_last) {
                qk(kbuf(t0), 0, sa);
                if ((t0 + 1) * 64 > w_first || (PAGED && have != 0xf)) mask(t0, 0, sa, have);
                raise_max(0, row_max(sa));
            }
            if (t1 - t0 > (PAGED ? 1 : 2)) __syncthreads();   // (the first step loads over the tile just read)
            for (int t = t0; t + 1 < t1; t += 2) {
                step(t, sa, sb, kbuf(t + 1), vbuf(t), kbuf(t), vbuf(t + 1));
                if (t + 2 < t1) {
                    step(t + 1, sb, sa, kbuf(t), vbuf(t + 1), kbuf(t + 1), vbuf(t));
                } else {
                    sa[0] = sb[0];
                    sa[1] = sb[1];
                }
            }
            // the last tile has no score product beside it
            char* sV = vbuf(t1 - 1);
            if (t1 * 64 > wg_first || (PAGED && have != 0xf)) {
                if (tile_nonfinite(sV)) absorb_nonfinite(nullptr, sV, t1 - 1);
            }
            if ((t1 - 1) * 64 < w_last) {
                bf16x8 pf[2][2];
                exp_pack(0, sa, pf);
                pv_ahead(sV, pf);
            }
        }
    } else {
        // One tile at a time.  Two query blocks per wave are offset against each other within it: the score product of the second runs
        // beside the exponentials of the first, the second product of the first beside the exponentials of the second.  (8-bit keys: the
        // next tile's codes are in registers meanwhile, and go into the other buffer at its end.)
        auto load = [&](int t, char* dst) {
            dma(false, t, dst);
            dma(true, t, dst + K_BYTES);
        };
        auto work = [&](int t, char* sK, char* sV) __attribute__((always_inline)) {
            const bool edge = (t + 1) * 64 > w_first || (PAGED && have != 0xf);
            f32x16 s0[2];
            bf16x8 pf0[2][2];
            qk(sK, 0, s0);
            if (edge) mask(t, 0, s0, have);
            raise_max(0, row_max(s0));
            if constexpr (QB == 2) {
                f32x16 s1[2];
                bf16x8 pf1[2][2];
                qk(sK, 1, s1);
                exp_pack(0, s0, pf0);
                pin(pf0);
                if (edge) mask(t, 1, s1, have);
                raise_max(1, row_max(s1));
                pv(sV, 0, pf0);
                exp_pack(1, s1, pf1);
                pv(sV, 1, pf1);
            } else {
                exp_pack(0, s0, pf0);
                pv(sV, 0, pf0);
            }
        };
        auto step = [&](int t, char* here, char* dst) {
            if constexpr (PAGED) {
                const int tk = min(t + 1, t1 - 1);
                fetch(false, tk, pid_k, k8r, kbyte);
                fetch(true, tk, pid_k, v8r, vbyte);
                have1 = groups(pid_k);
                pid_k = look_up(min(t + 2, t1 - 1));
            } else {
                if (t + 1 < t1) load(t + 1, dst);
            }
            char* sV = here + K_BYTES;
            if ((t + 1) * 64 > wg_first || (PAGED && have != 0xf)) {
                if (tile_nonfinite(sV)) absorb_nonfinite(here, sV, t);
            }
            if (t * 64 < w_last) work(t, here, sV);
            if constexpr (PAGED) {
                stage_k(dst);
                stage_v(dst + K_BYTES);
                have = have1;
            }
            arrive();
        };
        if (t0 < t1) {
            char* first = smem + (t0 & 1) * TILE;
            if constexpr (PAGED) {
                const int pid = look_up(t0);
                pid_k = look_up(min(t0 + 1, t1 - 1));
                have = groups(pid);
                fetch(false, t0, pid, k8r, kbyte);
                fetch(true, t0, pid, v8r, vbyte);
                stage_k(first);
                stage_v(first + K_BYTES);
            } else {
                load(t0, first);
            }
            arrive();
            for (int t = t0; t < t1; ++t) step(t, smem + (t & 1) * TILE, smem + (1 - (t & 1)) * TILE);
        }
    }

#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const float l = l_run[qb] + __shfl_xor(l_run[qb], 32, 64);
        const long r = wrow + qb * 32 + frow;
        if (r >= rows) continue;
        const int i = (int)(r / p.G), hq = h * p.G + (int)(r - (long)i * p.G);
        if (p.splits > 1) {
            const long at = (((long)split * p.B + b) * p.max_q + i) * p.Hq + hq;
            if (fhalf == 0) {
                p.part_ml[2 * at] = m_run[qb];
                p.part_ml[2 * at + 1] = l;
            }
            float* dst = p.part_o + at * D + 4 * fhalf;
            if (l != 0.f) {
#pragma unroll
                for (int dh = 0; dh < NDH; ++dh)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 w = {o[qb][dh][4 * g], o[qb][dh][4 * g + 1], o[qb][dh][4 * g + 2], o[qb][dh][4 * g + 3]};
                        *reinterpret_cast<f32x4*>(dst + dh * 32 + 8 * g) = w;
                    }
            }
        } else {
            const float inv = l == 0.f ? 0.f : (1.0f / HALF) / l;   // no key seen: 0 (O is 0)
            bf16_t* dst = p.o + (long)(sp.q0 + i) * p.o_rs + (long)hq * p.o_hs + 4 * fhalf;
#pragma unroll
            for (int dh = 0; dh < NDH; ++dh)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    u32x2 w;
                    w[0] = pack_h2<FMT, false>(o[qb][dh][4 * g + 0] * inv, o[qb][dh][4 * g + 1] * inv);
                    w[1] = pack_h2<FMT, false>(o[qb][dh][4 * g + 2] * inv, o[qb][dh][4 * g + 3] * inv);
                    *reinterpret_cast<u32x2*>(dst + dh * 32 + 8 * g) = w;
                }
        }
    }
}

long items_of(const SeqAttnParams& p, int bm) { return ((long)p.max_q * p.G + bm - 1) / bm * p.splits * p.B * p.Hkv; }

template <int D, int QB, int NW, int FMT, bool PAGED, int WPS = 2>
int launch(const SeqAttnParams& p_in, hipStream_t stream) {
    SeqAttnParams p = p_in;
    constexpr int BM = 32 * NW * QB;
    p.qtiles = (int)(((long)p.max_q * p.G + BM - 1) / BM);
    const long n = items_of(p, BM);
    if (n >= (1L << 31)) return -4;
    p.items = (unsigned)n;
    hipLaunchKernelGGL((seq_attn_tile_kernel<D, QB, NW, FMT, PAGED, WPS>), seq_grid(n), dim3(64 * NW), 0, stream, p);
    IGGT_CHECK_LAUNCH();
    return 0;
}

template <int FMT, bool PAGED>
int launch_fmt(const SeqAttnParams& p, int D, bool small, hipStream_t stream) {
    if constexpr (PAGED) {
        if (small) return D == 64 ? launch<64, 1, 4, FMT, PAGED>(p, stream) : launch<128, 1, 4, FMT, PAGED>(p, stream);
        return D == 64 ? launch<64, 2, 4, FMT, PAGED>(p, stream) : launch<128, 1, 8, FMT, PAGED>(p, stream);
    } else {
        if (D == 128) return small ? launch<128, 1, 4, FMT, PAGED>(p, stream) : -1;    // (the plan has 128-row tiles for 128 channels)
        // More than two waves per SIMD come of more than 512 work items.  Measured, 16 heads, four waves / two, pipelined over the tiles, us:
        // full 700 tokens 16.4 / 14.8, 1 374 28.4 / 24.8, 2 x 1 374 (352 items) 37.7 / 36.2, 3 x 1 374 (528) 48.5 / 53.9, 4 122 (528)
        // 122 / 133, 8 192 352 / 398; causal 1 374 28.1 / 25.4, 2 748 48.5 / 43.5, 4 x 1 374 34.0 / 38.4, 8 192 187 / 222 (but 4 122 72 / 65).
        if (small) return items_of(p, 128) <= 512 ? launch<64, 1, 4, FMT, PAGED>(p, stream) : launch<64, 1, 4, FMT, PAGED, 4>(p, stream);
        return launch<64, 1, 8, FMT, PAGED, 4>(p, stream);
    }
}

}  // namespace

int iggt_launch_seq_tiles(const SeqAttnParams& p, int D, int fmt, bool paged, bool small, hipStream_t stream) {
    if (fmt == FMT_F16) return paged ? launch_fmt<FMT_F16, true>(p, D, small, stream) : launch_fmt<FMT_F16, false>(p, D, small, stream);
    return paged ? launch_fmt<FMT_BF16, true>(p, D, small, stream) : launch_fmt<FMT_BF16, false>(p, D, small, stream);
}

// Tile height and key ranges.  128-row tiles (four waves), but
//   16-bit keys, head dim 64: 256 rows (eight waves) where they fill the chip twice (4 x 2 748 tokens, 16 heads, full: 171 -> 164 us, 2 x
//   5 496 332 -> 309, but causal 8 x 1 374: 55 -> 57);
//   8-bit keys: the workgroup converts the keys it reads, half of that work per row for 256 rows.  Head dim 128 (eight waves, whose
//   coupling costs less than that: 1 374 rows against 10 175 tokens, 5 x 8 heads: 540 -> 420 us before the spills went, 322 now; with
//   16-bit keys 974 -> 1 033): more
//   than 128 rows.  Head dim 64 (two query blocks per wave: 1 374 rows, 6 x 8 heads, 36 343 tokens 590 -> 525 us; 2 x 16 heads, 12 366
//   tokens 250 -> 237; but 3 x 16 heads, 1 374 tokens, causal 33 -> 47, 4 heads, 2 748 tokens 24 -> 31): where the estimate below is lower.
// Ranges, where the grid is small: the time of all items over the CUs, where the last CU to finish has between n and ceil(n) of n per CU
// (one alone runs at 0.8 of a full CU's rate, at head dim 64 two at 0.9 of it), half of an item for start and tail, and the fold (5 us,
// and 4 D bytes per row and range written and read), in microseconds at the rates measured here (a CU does `rate` flop in one; causal
// masks, unknown here, count for 0.7).  Measured: 192 items of 256 rows, 12 366 8-bit keys of 64: 265 us in 2 ranges, 271 in 3, 233 in 4,
// 237 in 5, 245 in 6, 235 in 8; 176 items of 128 rows, 1 374 keys of 128: 37 unsplit, 42 in 2, 51 in 3; of 64: 28, 29, 29; 344 items, 2 748
// keys of 64: 64, 61, 67; 285 causal items, 2 305 keys of 64: 42, 36.
static SeqPlan ranges_of(int bm, double rate, long pairs, long rows, long max_k, int D, double& us) {
    const long items = pairs * ((rows + bm - 1) / bm), cus = 256;
    const double item_us = 4.0 * D * bm * max_k / rate, fold_us = 8.0 * D * pairs * rows / (D == 64 ? 5.3e6 : 4.0e6);
    auto cost = [&](long s) {
        const double n = (double)items * s / cus;
        const double least = D == 128 || n <= 1.0 ? 1.25 : 1.8, even = 0.5 * (n + std::ceil(n)) + 0.1, busy = even > least ? even : least;
        return item_us * (0.7 * busy + 0.5) / s + (s > 1 ? 5.0 + fold_us * s : 0.0);
    };
    SeqPlan plan = {1, bm == 128, 0};
    us = cost(1);
    if (items >= 4 * cus || max_k < 512) return plan;
    const long most = max_k / 256 < 32 ? max_k / 256 : 32;      // at least four tiles per range
    for (long s = 2; s <= most; ++s) {
        const double c = cost(s);
        if (c < us * 0.97) {
            us = c;
            plan.splits = (int)s;
        }
    }
    return plan;
}
SeqPlan iggt_seq_tile_plan(int B, long max_q, long max_k, int Hkv, int G, int D, bool paged) {
    const long rows = max_q * G, pairs = (long)B * Hkv;
    double us, us256;
    if (!paged) {
        const bool small = D == 128 || rows <= 128 || pairs * ((rows + 255) / 256) < 2 * 256;
        return ranges_of(small ? 128 : 256, 3.1e6, pairs, rows, max_k, D, us);
    }
    const SeqPlan plan = ranges_of(128, 2.2e6, pairs, rows, max_k, D, us);
    if (rows <= 128) return plan;
    const SeqPlan plan256 = ranges_of(256, D == 64 ? 2.7e6 : 2.2e6, pairs, rows, max_k, D, us256);
    return D == 128 || us256 <= 1.04 * us ? plan256 : plan;
}

static int packed_attn_h16(int fmt, const void* q, long q_rs, long q_hs, const void* k, long k_rs, long k_hs, const void* v,
                           long v_rs, long v_hs, void* o, long o_rs, long o_hs, const int* cu_q, const int* cu_k, int B, int Tq,
                           int Tk, int max_q, int max_k, int Hq, int Hkv, int D, float scale, int causal, void* ws, long ws_len,
                           void* stream) {
    if (B < 0 || Tq < 0 || Tk < 0 || max_q < 0 || max_k < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || (D != 64 && D != 128)) return -1;
    if (Tk >= 0x7fffffff - 1024 || (long)Tq * Hq >= (1L << 31)) return -1;
    if ((q_rs | q_hs | k_rs | k_hs | v_rs | v_hs) % 8 || (o_rs | o_hs) % 4) return -2;
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 || (uintptr_t)o % 8) return -2;
    if (Tk > 1 && (k_rs < 0 || v_rs < 0 || k_rs >= (1L << 24) || v_rs >= (1L << 24))) return -2;   // 64 rows in 32-bit byte offsets
    if (!(scale > 0.f && scale <= 1e38f)) return -3;
    if (B == 0 || Tq == 0 || max_q == 0) return 0;
    SeqAttnParams p = {};
    p.q = (const bf16_t*)q; p.k = (const bf16_t*)k; p.v = (const bf16_t*)v; p.o = (bf16_t*)o;
    p.q_rs = q_rs; p.q_hs = q_hs; p.k_rs = k_rs; p.k_hs = k_hs; p.v_rs = v_rs; p.v_hs = v_hs; p.o_rs = o_rs; p.o_hs = o_hs;
    p.cu_q = cu_q; p.cu_k = cu_k;
    p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.Tq = Tq; p.Tk = Tk; p.max_q = max_q; p.causal = causal != 0;
    p.scale_log2 = scale * 1.4426950408889634f;
    const SeqPlan plan = iggt_seq_tile_plan(B, max_q, max_k, Hkv, p.G, D, false);
    p.splits = plan.splits;
    if (p.splits > 1) {
        const long n = (long)p.splits * B * max_q * Hq;
        if (ws == nullptr || ws_len < n * (D + 2) * 4 || (uintptr_t)ws % 16) return -5;
        p.part_o = (float*)ws;
        p.part_ml = p.part_o + n * D;
    }
    const int rc = iggt_launch_seq_tiles(p, D, fmt, false, plan.small, (hipStream_t)stream);
    if (rc || p.splits == 1) return rc;
    return iggt_launch_seq_fold(p, D, fmt, false, (hipStream_t)stream);
}

extern "C" {
long iggt_packed_attn_ws_bytes(int B, int max_q, int max_k, int Hq, int Hkv, int D) {
    if (B <= 0 || max_q <= 0 || max_k < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || (D != 64 && D != 128)) return 0;
    const SeqPlan plan = iggt_seq_tile_plan(B, max_q, max_k, Hkv, Hq / Hkv, D, false);
    return plan.splits > 1 ? (long)plan.splits * B * max_q * Hq * (D + 2) * 4 : 0;
}
int iggt_packed_attn_bf16(const void* q, long q_rs, long q_hs, const void* k, long k_rs, long k_hs, const void* v, long v_rs,
                          long v_hs, void* o, long o_rs, long o_hs, const int* cu_q, const int* cu_k, int B, int Tq, int Tk,
                          int max_q, int max_k, int Hq, int Hkv, int D, float scale, int causal, void* ws, long ws_len,
                          void* stream) {
    return packed_attn_h16(FMT_BF16, q, q_rs, q_hs, k, k_rs, k_hs, v, v_rs, v_hs, o, o_rs, o_hs, cu_q, cu_k, B, Tq, Tk, max_q, max_k,
                           Hq, Hkv, D, scale, causal, ws, ws_len, stream);
}
int iggt_packed_attn_f16(const void* q, long q_rs, long q_hs, const void* k, long k_rs, long k_hs, const void* v, long v_rs,
                         long v_hs, void* o, long o_rs, long o_hs, const int* cu_q, const int* cu_k, int B, int Tq, int Tk,
                         int max_q, int max_k, int Hq, int Hkv, int D, float scale, int causal, void* ws, long ws_len,
                         void* stream) {
    return packed_attn_h16(FMT_F16, q, q_rs, q_hs, k, k_rs, k_hs, v, v_rs, v_hs, o, o_rs, o_hs, cu_q, cu_k, B, Tq, Tk, max_q, max_k,
                           Hq, Hkv, D, scale, causal, ws, ws_len, stream);
}
}
