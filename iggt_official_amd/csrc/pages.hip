// Paged 8-bit K/V cache: the planner (block tables and slot maps from request lengths) and the writer.
//
// Planner.  Request b holds have = lens[b] tokens and is to hold want = new_lens[b].  Free pages lie in a ring
// (ring[(head + i) % N], i < count).  With pages(n) = ceil(n / page):
//   grow_b = max(0, pages(want) - pages(have)) pages leave the head of the ring, in request order;
//   shrink_b = max(0, pages(have) - pages(want)) pages go behind its tail, in request order (usable from the next step on);
//   token t of the step (request order, places have .. want - 1) gets slot = page * page_size + place % page_size.
// All or nothing for growth: without enough free pages (or slots) the growing requests stay as they are.  Everything that other
// launches' threads read is left unwritten, so every workgroup forms the same prefix sums by itself and there is no second launch.
// Bound by latency: two loads, one scan, one search and one scattered load per slot.  8 requests 3.9 us, 512 requests of which 73 bring
// 100 000 tokens 6.9 us.
//
// Writer.  One scale 2^e per (page, key head), for K and for V: the least with amax <= 448 * 2^e (e4m3's largest value), so x / 2^e is
// exact and only e4m3 rounds (2^-4 of the value at most, 2^-10 of the scale below 2^-6 of it).  A page that holds tokens already keeps
// max(old, needed); if it grows its codes move down by the same power of two (exact until they reach e4m3's subnormals).  A run of
// tokens with consecutive slots in one page belongs to one wave, the only writer of the page's head; a run that fits into its registers
// is read once, a longer one twice (maximum, then codes).  Bound by the latency of that chain -- slots, values, scale, maximum over the
// wave, codes -- and for prompts by the waves in flight: 64 single tokens, 16 heads of 64, 4.9 us; a prompt of 10 992 tokens 17.5 us
// (67 MB, 3.9 TB/s); 13 prompts of up to 777, 4 heads of 128, 8.9 us.
#include "common.h"
#include "../../include/iggt_hip.h"

namespace {

constexpr int PLAN_MAX_REQUESTS = 8192, PLAN_THREADS = 512, PLAN_WAVES = PLAN_THREADS / 64;

struct PlanParams {
    int* tables;
    long table_stride;
    int R, M;
    int* ring;
    int N;
    const int* counters;
    const int* lens;
    const int* new_lens;
    int shift;
    int* starts;
    int* next_lens;
    int* next_counters;
    int* slots;
    int T;
};

// last index r in [0, n) with a[r] <= x (a ascending, a[0] = 0 <= x)
IGGT_DEVINL int last_le(const int* a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(PLAN_THREADS) void plan_pages_kernel(const PlanParams p) {
    extern __shared__ int lds[];
    int* s_tok = lds;                 // exclusive prefix sums over the requests: tokens,
    int* s_grow = lds + p.R;          // pages taken,
    int* s_shrink = lds + 2 * p.R;    // pages given back
    int* s_have = lds + 3 * p.R;      // tokens held
    __shared__ int s_wave[3][PLAN_WAVES];
    __shared__ long s_total[3][PLAN_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int cap = p.M << p.shift, round = (1 << p.shift) - 1;
    const int N = p.N;
    const int head = N > 0 ? (int)((unsigned)p.counters[0] % (unsigned)N) : 0;
    const int count = min(max(p.counters[1], 0), N);
    // a thread takes `per` consecutive requests
    const int per = (p.R + PLAN_THREADS - 1) / PLAN_THREADS, r0 = tid * per, r1 = min(r0 + per, p.R);
    int sum[3] = {0, 0, 0};
    long total[3] = {0, 0, 0};        // 64 bits: lengths are whatever the caller's memory holds
    for (int r = r0; r < r1; r += 4) {
        int have[4], want[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int q = min(r + j, r1 - 1);
            have[j] = p.lens[q];
            want[j] = p.new_lens[q];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (r + j >= r1) break;
            have[j] = min(max(have[j], 0), cap);
            want[j] = min(max(want[j], 0), cap);
            const int hp = (have[j] + round) >> p.shift, wp = (want[j] + round) >> p.shift;
            const int v[3] = {max(want[j] - have[j], 0), max(wp - hp, 0), max(hp - wp, 0)};
            s_tok[r + j] = sum[0];
            s_grow[r + j] = sum[1];
            s_shrink[r + j] = sum[2];
            s_have[r + j] = have[j];
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                sum[i] = (int)((unsigned)sum[i] + (unsigned)v[i]);
                total[i] += v[i];
            }
        }
    }
    int incl[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        int x = sum[i];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x, o, 64);
            if (lane >= o) x = (int)((unsigned)x + (unsigned)y);
        }
        incl[i] = x;
        long t = total[i];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
        if (lane == 63) s_wave[i][wave] = x;
        if (lane == 0) s_total[i][wave] = t;
    }
    __syncthreads();
    long all[3] = {0, 0, 0};
    unsigned base[3] = {0, 0, 0};
#pragma unroll
    for (int w = 0; w < PLAN_WAVES; ++w)
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            all[i] += s_total[i][w];
            if (w < wave) base[i] += (unsigned)s_wave[i][w];
        }
    const bool fits = all[1] <= count && all[0] <= p.T;
    for (int r = r0; r < r1; ++r) {
        s_tok[r] += (int)(base[0] + (unsigned)(incl[0] - sum[0]));
        s_grow[r] += (int)(base[1] + (unsigned)(incl[1] - sum[1]));
        s_shrink[r] += (int)(base[2] + (unsigned)(incl[2] - sum[2]));
    }
    __syncthreads();
    const int ntok = fits ? (int)all[0] : 0, ngrow = fits ? (int)all[1] : 0;
    const int nshrink = (int)min(all[2], (long)(N - count));   // (a valid state never has more pages out than that)

    if (blockIdx.x == 0) {
        for (int r = tid; r < p.R; r += PLAN_THREADS) {
            const int have = s_have[r], want = min(max(p.new_lens[r], 0), cap);
            p.starts[r] = fits ? s_tok[r] : 0;
            p.next_lens[r] = fits ? want : min(have, want);
        }
        if (tid == 0) {
            p.starts[p.R] = ntok;
            p.next_counters[0] = N > 0 ? (int)(((unsigned)head + (unsigned)ngrow) % (unsigned)N) : 0;
            p.next_counters[1] = count - ngrow + nshrink;
            p.next_counters[2] = all[0] > p.T ? -1 : (all[1] > count ? (int)min(all[1] - count, (long)0x7fffffff) : 0);
        }
    }
    const int gtid = blockIdx.x * PLAN_THREADS + tid, gsize = gridDim.x * PLAN_THREADS;
    auto wrap = [&](unsigned i) { return i >= (unsigned)N ? i - (unsigned)N : i; };    // of i < 2 N
    auto taken = [&](int i) { return p.ring[wrap((unsigned)head + (unsigned)i)]; };     // i < count <= N
    for (int t = gtid; t < p.T; t += gsize) {
        int slot = -1;
        if (t < ntok) {
            const int r = last_le(s_tok, p.R, t);
            const int have = s_have[r], place = have + (t - s_tok[r]), at = place >> p.shift, hp = (have + round) >> p.shift;
            const int id = at < hp ? p.tables[(long)r * p.table_stride + at] : taken(s_grow[r] + (at - hp));
            slot = (unsigned)id < (unsigned)N ? (id << p.shift) + (place & round) : -1;
        }
        p.slots[t] = slot;
    }
    for (int i = gtid; i < ngrow; i += gsize) {
        const int r = last_le(s_grow, p.R, i);
        p.tables[(long)r * p.table_stride + ((s_have[r] + round) >> p.shift) + (i - s_grow[r])] = taken(i);
    }
    for (int i = gtid; i < nshrink; i += gsize) {
        const int r = last_le(s_shrink, p.R, i);
        const int wp = (min(max(p.new_lens[r], 0), cap) + round) >> p.shift;
        // (head + count + i < 3 N: twice around at most)
        p.ring[wrap(wrap((unsigned)head + (unsigned)count) + (unsigned)i)] = p.tables[(long)r * p.table_stride + wp + (i - s_shrink[r])];
    }
}

// ------------------------------------------------------------------------------------------------ writer
struct AppendParams {
    const uint16_t* k;
    const uint16_t* v;
    long k_rs, k_hs, v_rs, v_hs;
    const int* slots;
    int T, Hkv, num_slots, shift;
    uint8_t* k8;
    uint8_t* v8;
    uint8_t* k_scale;
    uint8_t* v_scale;
};

constexpr float E4M3_MAX = 448.f;

// exponent byte of the least power of two 2^e with amax <= 448 * 2^e (448 = 1.75 * 2^8)
IGGT_DEVINL int scale_byte(float amax) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
    const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, 1), 254);
}
IGGT_DEVINL float pow2_byte(int byte) { return __builtin_bit_cast(float, (uint32_t)byte << 23); }

// e4m3, round to nearest even; infinities go to the largest value, NaN stays NaN
IGGT_DEVINL uint32_t code4(float a, float b, float c, float d) {
    auto sat = [](float x) { return x != x ? x : __builtin_amdgcn_fmed3f(x, -E4M3_MAX, E4M3_MAX); };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(sat(a), sat(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(sat(c), sat(d), w, true);
}
// four codes times f <= 1 (a power of two)
IGGT_DEVINL uint32_t scale4(uint32_t w, float f) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return code4(a[0] * f, a[1] * f, b[0] * f, b[1] * f);
}
template <int FMT>
IGGT_DEVINL float amax2(float m, uint32_t w) {   // maximum of the finite ones of two packed values' magnitudes
    const float a = __builtin_fabsf(h2_lo<FMT>(w)), b = __builtin_fabsf(h2_hi<FMT>(w));
    m = a < __builtin_inff() ? fmaxf(m, a) : m;
    return b < __builtin_inff() ? fmaxf(m, b) : m;
}

// One wave writes `len` tokens (rows t0 ..) of one key head at places at .. at + len - 1 of a page.
template <int D, int FMT, bool V>
IGGT_DEVINL void write_run(const AppendParams& p, int t0, int len, int page, int at, int h) {
    const int lane = threadIdx.x & 63;
    const long rs = V ? p.v_rs : p.k_rs;
    const uint16_t* src = (V ? p.v + (long)h * p.v_hs : p.k + (long)h * p.k_hs) + (long)t0 * rs;
    const long head = (long)page * p.Hkv + h;
    uint8_t* scale = (V ? p.v_scale : p.k_scale) + head;
    uint8_t* dst = (V ? p.v8 : p.k8) + ((head << p.shift) * D);
    const int old = at > 0 ? (int)*scale : 0;
    float m = 0.f;

    // Rows outside the run are read as its first or last one: the maximum is the same, and what they give is not written.  (A load under
    // a condition of its own costs more than it saves.)
    // rows: LPR lanes of 8 values each, U loads of RPI rows in flight
    constexpr int LPR = D / 8, RPI = 64 / LPR, U = D == 64 ? 8 : 4;
    const int lr = lane / LPR, lc = (lane % LPR) * 8;
    u32x4 x[U];
    auto read_rows = [&](int from) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (from + j * RPI < len) x[j] = *reinterpret_cast<const u32x4*>(src + (long)min(from + j * RPI + lr, len - 1) * rs + lc);
        }
    };
    auto max_rows = [&]() {
        for (int from = 0; from < len; from += U * RPI) {
            read_rows(from);
#pragma unroll
            for (int j = 0; j < U; ++j)
                if (from + j * RPI < len)
#pragma unroll
                    for (int q = 0; q < 4; ++q) m = amax2<FMT>(m, x[j][q]);
        }
    };
    // V columns: 16 tokens of a channel pair per lane, LPG lanes for a group of 16 places, NB groups of a lane at a time
    constexpr int LPG = D / 2, GPI = 64 / LPG, NB = D == 64 ? 2 : 1;
    const int d = (lane % LPG) * 2, g0 = at >> 4, g1 = (at + len + 15) >> 4;
    uint32_t y[NB][16];
    u32x4 c[NB][2];             // what a group that the run does not fill holds
    auto out_of = [&](int g) { return dst + ((long)g * D + d) * 16; };
    auto whole = [&](int g) { return g * 16 >= at && g * 16 + 16 <= at + len; };
    auto read_groups = [&](int from) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (from + b * GPI >= g1) continue;
            const int gb = from + b * GPI + lane / LPG, first = gb * 16 - at;
            if (gb < g1 && !whole(gb)) {
                c[b][0] = *reinterpret_cast<const u32x4*>(out_of(gb));
                c[b][1] = *reinterpret_cast<const u32x4*>(out_of(gb) + 16);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j)
                y[b][j] = *reinterpret_cast<const uint32_t*>(src + (long)min(max(first + j, 0), len - 1) * rs + d);
        }
    };

    const bool at_once = V && g1 - g0 <= NB * GPI;      // V of a run that fits into a lane's registers is read once
    if constexpr (V) {
        if (at_once) {
            read_groups(g0);
#pragma unroll
            for (int b = 0; b < NB; ++b)
                if (g0 + b * GPI < g1)
#pragma unroll
                    for (int j = 0; j < 16; ++j) m = amax2<FMT>(m, y[b][j]);
        } else {
            max_rows();
        }
    } else {
        max_rows();
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const int now = max(old, scale_byte(m));
    // 2^(127 - now): the last two exponents have a subnormal reciprocal (2^-127)
    const float inv = now >= 254 ? __builtin_bit_cast(float, 0x00400000u) : pow2_byte(254 - now);
    const bool moved = at > 0 && now > old;
    // 2^(old - now); below e4m3's whole range it is as good as 0
    const float down = moved ? (now - old > 40 ? 0.f : pow2_byte(127 - (now - old))) : 1.f;
    if (moved) {    // held codes: K rows before the run, V groups before its first (that group below)
        const int pieces = V ? g0 * D : at * (D / 16);
        for (int i = lane; i < pieces; i += 64) {
            u32x4 w = reinterpret_cast<u32x4*>(dst)[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = scale4(w[j], down);
            reinterpret_cast<u32x4*>(dst)[i] = w;
        }
    }
    if constexpr (!V) {
        for (int from = 0; from < len; from += U * RPI) {
            if (len > U * RPI) read_rows(from);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int i = from + j * RPI + lr;
                if (from + j * RPI < len && i < len) {
                    u32x2 w;
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                        w[q] = code4(h2_lo<FMT>(x[j][2 * q]) * inv, h2_hi<FMT>(x[j][2 * q]) * inv, h2_lo<FMT>(x[j][2 * q + 1]) * inv, h2_hi<FMT>(x[j][2 * q + 1]) * inv);
                    *reinterpret_cast<u32x2*>(dst + (long)(at + i) * D + lc) = w;
                }
            }
        }
    } else {
        for (int from = g0; from < g1; from += NB * GPI) {
            if (!at_once) read_groups(from);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int gb = from + b * GPI + lane / LPG, first = gb * 16 - at;
                if (gb >= g1) continue;
                const bool full = whole(gb);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t nw[2];
                    nw[0] = code4(h2_lo<FMT>(y[b][4 * q]) * inv, h2_lo<FMT>(y[b][4 * q + 1]) * inv, h2_lo<FMT>(y[b][4 * q + 2]) * inv, h2_lo<FMT>(y[b][4 * q + 3]) * inv);
                    nw[1] = code4(h2_hi<FMT>(y[b][4 * q]) * inv, h2_hi<FMT>(y[b][4 * q + 1]) * inv, h2_hi<FMT>(y[b][4 * q + 2]) * inv, h2_hi<FMT>(y[b][4 * q + 3]) * inv);
                    if (full) {
                        c[b][0][q] = nw[0];
                        c[b][1][q] = nw[1];
                    } else {
                        uint32_t fresh = 0, before = 0;   // bytes of the run, bytes of tokens held before it
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int i = first + 4 * q + j;
                            if (i >= 0 && i < len) fresh |= 0xffu << (8 * j);
                            if (i < 0) before |= 0xffu << (8 * j);
                        }
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            uint32_t w = c[b][s][q];
                            if (moved) w = (scale4(w, down) & before) | (w & ~before);
                            c[b][s][q] = (nw[s] & fresh) | (w & ~fresh);
                        }
                    }
                }
                *reinterpret_cast<u32x4*>(out_of(gb)) = c[b][0];
                *reinterpret_cast<u32x4*>(out_of(gb) + 16) = c[b][1];
            }
        }
    }
    if (lane == 0 && (now != old)) *scale = (uint8_t)now;
}

// Workgroup: GROUP consecutive tokens, two key heads (two waves each: K, V).  A wave takes the runs that begin in its group.
template <int D, int FMT>
__global__ __launch_bounds__(256) void append_pages_kernel(const AppendParams p, int group) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.y * 2 + (wave >> 1);
    if (h >= p.Hkv) return;
    const int psize = 1 << p.shift, lane = threadIdx.x & 63;
    const int a = blockIdx.x * group;
    auto slot_at = [&](int t) {
        const int s = (t >= 0 && t < p.T) ? p.slots[t] : -1;
        return (unsigned)s < (unsigned)p.num_slots ? s : -1;
    };
    // lane l looks at token a + l: does a run begin there
    const int mine = slot_at(a + lane), before = slot_at(a + lane - 1);
    unsigned long long begins = __ballot(lane < group && mine >= 0 && (before < 0 || before != mine - 1 || (mine & (psize - 1)) == 0));
    while (begins != 0) {
        const int l = __builtin_ctzll(begins), t = a + l;
        begins &= begins - 1;
        const int s = __builtin_amdgcn_readlane(mine, l), at = s & (psize - 1), most = min(psize - at, p.T - t);
        // length of the run: among the 64 slots at hand, and only if it goes on behind them 64 more at a time
        const unsigned long long goes_on = __ballot(mine == s + (lane - l)) >> l;
        int len = min(goes_on == ~0ull ? 64 : __builtin_ctzll(~goes_on), most);
        while (len >= 64 - l && len < most) {
            const int i = len + lane;
            const unsigned long long same = __ballot(i < most && p.slots[t + (i < most ? i : 0)] == s + i);
            const int run = same == ~0ull ? 64 : __builtin_ctzll(~same);
            len += run;
            if (run < 64) break;
        }
        if (wave & 1) write_run<D, FMT, true>(p, t, len, s >> p.shift, at, h);
        else write_run<D, FMT, false>(p, t, len, s >> p.shift, at, h);
    }
}

int append_h16(int fmt, const void* k, long k_rs, long k_hs, const void* v, long v_rs, long v_hs, const int* slots, int T,
               void* k_codes, void* k_scale, void* v_codes, void* v_scale, int num_pages, int page, int Hkv, int D, void* stream) {
    const int shift = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1;
    if (T < 0 || num_pages < 0 || shift < 0 || Hkv <= 0 || (D != 64 && D != 128)) return -1;
    if (((long)num_pages << shift) >= (1L << 31) || Hkv > 131070 || T >= (1 << 30)) return -1;   // (grid: T / 64 x 256 threads)
    if ((k_rs | k_hs | v_rs | v_hs) % 8 || ((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_codes | (uintptr_t)v_codes) % 16) return -2;
    if (T == 0 || num_pages == 0) return 0;
    AppendParams p = {(const uint16_t*)k, (const uint16_t*)v, k_rs, k_hs, v_rs, v_hs, slots, T, Hkv, num_pages << shift, shift,
                      (uint8_t*)k_codes, (uint8_t*)v_codes, (uint8_t*)k_scale, (uint8_t*)v_scale};
    // Single tokens of many requests are all runs of their own: a workgroup each.  A prompt has a run per page: groups as long as leave
    // about four workgroups per CU.
    const long heads2 = (Hkv + 1) / 2;
    const int group = (long)T / 64 * heads2 >= 1024 ? 64 : ((long)T / 16 * heads2 >= 256 ? 16 : 1);
    const dim3 grid((T + group - 1) / group, (Hkv + 1) / 2), block(256);
    const hipStream_t st = (hipStream_t)stream;
    if (fmt == FMT_F16) {
        if (D == 64) hipLaunchKernelGGL((append_pages_kernel<64, FMT_F16>), grid, block, 0, st, p, group);
        else hipLaunchKernelGGL((append_pages_kernel<128, FMT_F16>), grid, block, 0, st, p, group);
    } else {
        if (D == 64) hipLaunchKernelGGL((append_pages_kernel<64, FMT_BF16>), grid, block, 0, st, p, group);
        else hipLaunchKernelGGL((append_pages_kernel<128, FMT_BF16>), grid, block, 0, st, p, group);
    }
    IGGT_CHECK_LAUNCH();
    return 0;
}

}  // namespace

extern "C" {
int iggt_plan_pages(int* tables, long table_stride, int requests, int table_width, int* ring, int num_pages, const int* counters,
                    const int* lens, const int* new_lens, int page, int* starts, int* next_lens, int* next_counters, int* slots,
                    int num_slots, void* stream) {
    const int shift = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1;
    if (requests < 0 || requests > PLAN_MAX_REQUESTS || table_width < 0 || num_pages < 0 || num_slots < 0 || shift < 0) return -1;
    if (((long)table_width << shift) >= (1L << 31) - 1024 || ((long)num_pages << shift) >= (1L << 31)) return -1;
    // sums of pages over all requests and a thread's next slot (the grid has 2^17 threads at most) stay within 32 bits
    if ((long)requests * table_width >= (1L << 31) || num_slots >= 0x7fffffff - (1 << 20)) return -1;
    PlanParams p = {tables, table_stride, requests, table_width, ring, num_pages, counters, lens, new_lens, shift, starts,
                    next_lens, next_counters, slots, num_slots};
    // every workgroup repeats the prefix sums, and then a slot per thread is the shortest
    int blocks = (num_slots + PLAN_THREADS - 1) / PLAN_THREADS;
    blocks = blocks < 1 ? 1 : (blocks > 256 ? 256 : blocks);
    const size_t lds = (size_t)(requests > 0 ? requests : 1) * 4 * sizeof(int);
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)plan_pages_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 PLAN_MAX_REQUESTS * 4 * (int)sizeof(int));
        if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(plan_pages_kernel, dim3(blocks), dim3(PLAN_THREADS), lds, (hipStream_t)stream, p);
    IGGT_CHECK_LAUNCH();
    return 0;
}
int iggt_append_pages_bf16(const void* k, long k_rs, long k_hs, const void* v, long v_rs, long v_hs, const int* slots, int tokens,
                           void* k_codes, void* k_scale, void* v_codes, void* v_scale, int num_pages, int page, int Hkv, int D,
                           void* stream) {
    return append_h16(FMT_BF16, k, k_rs, k_hs, v, v_rs, v_hs, slots, tokens, k_codes, k_scale, v_codes, v_scale, num_pages, page, Hkv,
                      D, stream);
}
int iggt_append_pages_f16(const void* k, long k_rs, long k_hs, const void* v, long v_rs, long v_hs, const int* slots, int tokens,
                          void* k_codes, void* k_scale, void* v_codes, void* v_scale, int num_pages, int page, int Hkv, int D,
                          void* stream) {
    return append_h16(FMT_F16, k, k_rs, k_hs, v, v_rs, v_hs, slots, tokens, k_codes, k_scale, v_codes, v_scale, num_pages, page, Hkv, D,
                      stream);
}
}
