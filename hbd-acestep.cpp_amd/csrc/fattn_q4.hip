// fattn_q4.hip -- flash attention over Q4_0 K and V (mi_flash_attn_ext).
//
//   s_ij = scale q_i . k_j + mask_ij,  y_i = sum_j softmax(s_i)_j v_j
//
// with k, v = (level - 8) d per block of 32 elements. Unlike a Q8_0 cache's, the
// products take q as it is: a level has 4 bits, exact in fp16, so the matrix cores
// multiply levels by q in fp16 and the block's d is applied to the fp32 sum.
//  q      each row is scaled by a power of two so that its largest element lies in
//         [2^10, 2^11). BF16 y: held as one fp16 (BF16 q: exact but for elements under
//         2^-24 of the largest). F32 y: as a whole number and an fp16 remainder, 23 bits
//         of the row's largest; the matrix cores' sums of whole numbers are exact, where
//         sums of 24-bit terms are cut at each step (measured over the LM's decode size:
//         y off by 4.1e-6 with two fp16 of any size, 2-norm over 2-norm, torch's fp32 6e-7).
//         So elements far below their row's largest keep fewer bits than fp32: with one of the
//         row 10 / 100 / 1000 times the rest, on a channel that K hardly holds, y is off by
//         3.8e-7 / 1.9e-6 / 2.5e-5 (fp32 scores: 1.1e-7); a third part would be half as many
//         products again.
//  levels as fp16 numbers -8 .. 7, by one mask-and-or and one packed add each two (the
//         nibbles' bits as they are, subnormals n 2^-24, with the -8 in the accumulator's
//         start, took fewer instructions but 4 registers a block for that start).
//  P, V   F32 y: P and v = (level - 8) d as a high and a low fp16 each (v exact, P to
//         22 bits), three products; BF16 y: one fp16 each (2^-11 against y's 2^-8: the error
//         against 64 bits is 1 to 2 % above that of 32-bit operations rounded to BF16).
//         d above 8188 would leave fp16: tiles with one scale v by 2^-4, P by 2^4; there
//         a d below 2^-10 loses bits (held / 16 it leaves fp16's normal numbers: an absolute
//         2^-21 of d).
// Sums, maxima and the running output are fp32.
#include "launch.h"
#include "rules.h"

namespace mi {

typedef _Float16 fa4_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 fa4_h8 __attribute__((ext_vector_type(8)));
typedef float    fa4_f4 __attribute__((ext_vector_type(4)));
typedef int      fa4_v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) fa4_v2i fa4_lds_v2i;
typedef short fa4_v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) fa4_v4s fa4_lds_v4s;
typedef float    fa4_f4u __attribute__((ext_vector_type(4), aligned(4)));  // y at its element's alignment
typedef uint32_t fa4_u2u __attribute__((ext_vector_type(2), aligned(2)));

constexpr float FA4_LOG2E = 1.44269504088896340736f;
constexpr float FA4_OFF   = 8.0f;   // p = exp2(s - max + 8): fp16 parts of p keep absolute 2^-32 of the largest
constexpr float    FA4_BIG      = 8188.0f;  // past it a level times d leaves fp16
constexpr uint32_t FA4_BIG_BITS = 0x6fffu;  // as fp16
constexpr int      FA4_PRE_TILES = 4096;    // most tiles that a workgroup of the kernel for many rows walks

// the 18 bytes of a block (d, 16 bytes of levels) as loaded: 5 words from the 4-byte
// boundary at or before the block, 20 bytes that never leave the row
struct Fa4Raw {
    uint32_t w[5];
};

// The n keys of a tile from base on as a buffer: what lies past the last one (all of it for n <=
// 0) reads as zeros without a memory access, so that every load is unconditional and a lane's
// offset is the same in every tile (conditional loads had the compiler wait for each at once).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t fa4_rows(const char * base, int64_t stride, int n, int row_bytes) {
    const int bytes = n > 0 ? (n - 1) * (int) stride + row_bytes : 0;
    return __builtin_amdgcn_make_buffer_rsrc((void *) base, (short) 0, bytes, 0x00020000);
}

__device__ __forceinline__ Fa4Raw fa4_load(__amdgpu_buffer_rsrc_t rs, int off) {
    const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0);
    Fa4Raw      r;
    r.w[0] = x.x;
    r.w[1] = x.y;
    r.w[2] = x.z;
    r.w[3] = x.w;
    r.w[4] = __builtin_amdgcn_raw_buffer_load_b32(rs, off + 16, 0, 0);
    return r;
}

// odd blocks start 2 bytes after the boundary: (d, levels) sit at bytes 2 and 4, even ones at 0 and 2
__device__ __forceinline__ void fa4_block(const Fa4Raw & r, int blk, float & d, uint32_t * q) {
    const uint32_t sel = blk & 1 ? 0x07060504u : 0x05040302u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        q[i] = __builtin_amdgcn_perm(r.w[i + 1], r.w[i], sel);
    }
    d = f16_lo(blk & 1 ? r.w[0] >> 16 : r.w[0]);
}

// The scale of a block of K whose levels are summed before it is applied: an infinite one becomes NaN, as
// the block's zeros (level 8) times it are. A sum's sign would make the scores -inf, and leave the key out.
__device__ __forceinline__ float fa4_scale(float d) {
    return d + (d - d);
}

__device__ __forceinline__ uint32_t fa4_bits(fa4_h2 v) {
    return __builtin_bit_cast(uint32_t, v);
}

__device__ __forceinline__ fa4_h2 fa4_half2(uint32_t v) {
    return __builtin_bit_cast(fa4_h2, v);
}

// A lane's 8 elements of each block of a row of q: 4 from element at0 of the block on, 4 from
// at1 on. One branch on the type around all loads.
template <int NB, bool OS>
__device__ __forceinline__ void fa4_q(const char * p, int type, int at0, int at1, float (*f)[8]) {
    if (OS && type == MI_TYPE_F32) {
        fa4_f4u v[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            v[b][0] = *(const fa4_f4u *) (p + (b * 32 + at0) * 4);
            v[b][1] = *(const fa4_f4u *) (p + (b * 32 + at1) * 4);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[b][e] = v[b][e / 4][e % 4];
            }
        }
        return;
    }
    fa4_u2u v[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        v[b][0] = *(const fa4_u2u *) (p + (b * 32 + at0) * 2);
        v[b][1] = *(const fa4_u2u *) (p + (b * 32 + at1) * 2);
    }
    const bool bf = !OS || type == MI_TYPE_BF16;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const uint32_t w = e & 2 ? v[b][e / 4].y : v[b][e / 4].x;
            f[b][e]          = bf ? bf16_lo(w) : f16_lo(w);
            f[b][e + 1]      = bf ? bf16_hi(w) : f16_hi(w);
        }
    }
}

// Bytes 0 and 2 of a word as two fp16 numbers -8 .. 7: the low nibbles, or the high ones
// (bytes 1 and 3 of it: of w >> 8). 0x6400 | n is 1024 + n.
// One instruction takes both constants (the compiler, given literals, makes two).
__device__ __forceinline__ fa4_h2 fa4_magic(uint32_t w, uint32_t mask) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(0x64006400u));
    return fa4_half2(r);
}

__device__ __forceinline__ fa4_h2 fa4_low(uint32_t w) {
    const fa4_h2 c = { (_Float16) -1032.0f, (_Float16) -1032.0f };
    return fa4_magic(w, 0x000f000fu) + c;
}

__device__ __forceinline__ fa4_h2 fa4_high(uint32_t w) {
    const fa4_h2 m = { (_Float16) 0.0625f, (_Float16) 0.0625f }, c = { (_Float16) -72.0f, (_Float16) -72.0f };
    return __builtin_elementwise_fma(fa4_magic(w, 0x00f000f0u), m, c);
}

// 8 levels of a word of 4 bytes as an A operand: bytes 0 2 low, 0 2 high, 1 3 low, 1 3 high.
// Group g of the 4 lane groups takes bytes 4 g .. 4 g + 3 of a block's levels, so the slots
// are elements 4 g + { 0, 2, 16, 18, 1, 3, 17, 19 }.
__device__ __forceinline__ fa4_h8 fa4_levels(uint32_t w) {
    const uint32_t v = w >> 8;
    const u32x4    r = { fa4_bits(fa4_low(w)), fa4_bits(fa4_high(w)), fa4_bits(fa4_low(v)), fa4_bits(fa4_high(v)) };
    return __builtin_bit_cast(fa4_h8, r);
}

// slot e of them as an index into the 4 elements from 4 g on, then the 4 from 16 + 4 g on
__device__ __forceinline__ constexpr int fa4_slot(int e) {
    return (e & 2) * 2 + (e & 1) * 2 + (e >> 2);
}

__device__ __forceinline__ float fa4_max_groups(float v) {  // over the 4 lane groups of 16
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v            = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

typedef uint32_t fa4_u2h __attribute__((ext_vector_type(2), aligned(2)));  // 4 mask values

// Query rows (query position, head) of a KV head in tiles of 16, keys split over
// workgroups of W waves, a wave taking every (splits * W)-th tile of TK keys. With
// v_mfma_f32_16x16x32_f16 (lane l: A[l%16][8(l/16)+e], B[8(l/16)+e][l%16],
// C[4(l/16)+r][l%16]):
//   S^T = K Q^T   A = levels of 16 keys from LDS, B = the 16 rows; one product per block
//                 of 32 elements, each scaled by the keys' d. Lane l then holds the scores
//                 of row l%16 for keys 16 mt + 4 (l/16) + r.
//   O^T = V^T P^T B = those probabilities as they sit; A = the levels of V by transposed
//                 8-bit LDS reads (lane l: byte l%16 of 8 keys, low nibble dim j, high
//                 dim j + 16), times the keys' d.
// The raw blocks of the next tile are in flight under the current one's math. Tiles with
// no live key are not read where the 16 rows share a mask row (one query position), and
// a key that no row attends to counts as v = 0 whatever its bytes are.
// Bound by a tile's chain and its unpacking: a lone wave takes 1.5 us a tile (D = 128, BF16 y; F32 1.6),
// three on a SIMD 2.1 for a tile each. Three waves a SIMD (F32 y, a mask row each, left to itself takes 171
// registers and two waves: 5 positions on 20000 46.4 us instead of 39.0, 16 on 4016 66.4 instead of 55.9), two at
// D = 256 (one: 7 positions on 30177, BF16 y, 63 us instead of 52; 8 rows on 3001 23.3 instead of 24.0; F32 y then
// spills 3, 9 and 21 of 256 registers without a mask, with one mask row, with a row each). 2 rows
// of 60013 keys, 32 heads on 8, 128, BF16 y: 29 us, 3.7 TB/s; 8 of up to 6600, F32 y: 21 us, 1.8 TB/s.
// Tiles of 64 keys at D = 128 leave half as many waves a turn; 8 waves a workgroup: 257 positions on
// 387 keys 25.8 us instead of 19.0, 64 on 2064 29.6 instead of 22.8.
template <int D> struct Fa4 {
    static constexpr int NB   = D / 32;
    static constexpr int TK   = D == 64 ? 64 : 32;  // keys per tile
    static constexpr int IPL  = TK * NB / 64;        // blocks per lane and tile, of K and of V
    static constexpr int MT   = TK / 16;
    static constexpr int KROW = 16 * NB;             // bytes of levels per key
    static constexpr int RPP  = 16 / NB;             // keys per padding
    static constexpr int DS   = TK + 64 / NB;        // entries per block in the tables of d
    static constexpr int KB   = TK * KROW + TK / RPP * 4 * NB;
    static constexpr int VB   = TK * KROW + TK / RPP * 16;
    static constexpr int DKB  = NB * DS * 4;
    static constexpr int DVB  = NB * DS * 2;
    static constexpr int MB   = 8;                   // tiles whose mask is read at once
    static constexpr int WAVE = KB + VB + DKB + DVB; // LDS bytes per wave, without the mask
    static constexpr int DC   = 64;                  // columns merged at a time
    static __device__ __forceinline__ int koff(int key) { return key * KROW + key / RPP * 4 * NB; }
    static __device__ __forceinline__ int voff(int key) { return key * KROW + key / RPP * 16; }
};

// OS: F32 y (parts of q, P and V); MS: 0 no mask, 1 one mask row for all rows of the tile, 2 a mask row each
template <int D, bool OS, int MS, int W>
__global__ void __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(D == 256 ? 2 : D == 128 && OS && MS == 2 ? 3 : 1)))
k_fa4_dec(const FaArgs a) {
    using F           = Fa4<D>;
    constexpr int QP  = OS ? 2 : 1;
    constexpr int NB  = F::NB, TK = F::TK, IPL = F::IPL, MT = F::MT;
    constexpr int MSB = MS == 1 ? F::MB * TK * 4 : 0;
    constexpr int WB  = F::WAVE + MSB;
    static_assert(WB >= 16 * F::DC * 4, "the merge reuses the tiles' memory");
    __shared__ __align__(16) char lds[W * WB];
    __shared__ float              stat[W][16][2];

    const int      lane = threadIdx.x & 63;
    const int      wv   = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int      c16 = lane & 15, q4 = lane >> 4;
    const uint32_t item  = blockIdx.x / (uint32_t) a.splits;
    const uint32_t split = blockIdx.x - item * (uint32_t) a.splits;
    const uint32_t nbg   = (uint32_t) (a.nb * a.nkv);
    const int      rt    = (int) (item / nbg);  // the row tiles of a KV head nbg workgroups apart: one XCD's L2 where 8 divides it
    const uint32_t bg    = item - (uint32_t) rt * nbg;
    const uint32_t b     = bg / (uint32_t) a.nkv;
    const uint32_t g     = bg - b * (uint32_t) a.nkv;
    const int      row   = rt * 16 + c16 < a.rows ? rt * 16 + c16 : a.rows - 1;  // past the end: the last row again
    const int      iq    = row / a.rk;
    const int      h     = (int) g * a.rk + (row - iq * a.rk);
    const uint32_t kb    = b / (uint32_t) a.rk3;
    const char *   kg    = a.k + (int64_t) kb * a.k3 + (int64_t) g * a.k2;
    const char *   vg    = a.v + (int64_t) kb * a.v3 + (int64_t) g * a.v2;
    const char *   mrow  = nullptr;
    if constexpr (MS != 0) {
        mrow = a.mask + (int64_t) (b % (uint32_t) a.mne3) * a.m3 + (int64_t) (h % a.mne2) * a.m2 + (int64_t) iq * a.m1;
    }
    char *  kl  = lds + wv * WB;
    char *  vl  = kl + F::KB;
    float * dkl = (float *) (vl + F::VB);
    char *  dvl = (char *) dkl + F::DKB;
    float * ml  = (float *) (dvl + F::DVB);

    // q: this lane's 8 elements of each block, the row's largest magnitude over the 4 lane groups
    float qv[NB][8];
    {
        const char * qp = a.q + (int64_t) b * a.q3 + (int64_t) h * a.q2 + (int64_t) iq * a.q1;
        fa4_q<NB, OS>(qp, a.tq, 4 * q4, 16 + 4 * q4, qv);
    }
    float qmax = 0.0f;
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            qmax = fmaxf(qmax, fabsf(qv[blk][e]));
        }
    }
    qmax     = fa4_max_groups(qmax);
    int ex   = (int) (__float_as_uint(qmax) >> 23) - 127;  // 2^ex <= qmax < 2^(ex + 1)
    ex       = ex < -100 ? -100 : ex > 127 ? 10 : ex;      // a row that is not finite: as it is
    const float up = __uint_as_float((uint32_t) (127 + 10 - ex) << 23);
    const float qs = a.scale * FA4_LOG2E * __uint_as_float((uint32_t) (127 - 10 + ex) << 23);
    fa4_h8      qb[QP][NB];
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = qv[blk][fa4_slot(e)] * up, w = OS ? __builtin_rintf(v) : v;
            qb[0][blk][e] = (_Float16) w;
            if constexpr (OS) {
                qb[1][blk][e] = (_Float16) (v - w);
            }
        }
    }

    float  m = -INFINITY, l = 0.0f;
    fa4_f4 o[2 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
        o[i] = fa4_f4{ 0.0f, 0.0f, 0.0f, 0.0f };
    }

    const int ntile = (a.n_kv + TK - 1) / TK;
    const int step  = a.splits * W;
    Fa4Raw    kr[IPL], vr[IPL];
    fa4_u2h  mr[MS == 2 ? MT : 1];  // the lane's mask values, 4 keys each
    int       ko[IPL], vo[IPL];
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        const int idx = i * 64 + lane, blk = idx % NB, key = idx / NB;
        ko[i] = key * (int) a.k1 + ((18 * blk) & ~3);
        vo[i] = key * (int) a.v1 + ((18 * blk) & ~3);
    }
    // tile t; `on` false: no tile (zeros)
    auto load = [&](int t, bool on) {
        const int  t0 = t * TK, last = a.n_kv - 1 - t0;
        const int  n  = !on ? 0 : last + 1 < TK ? last + 1 : TK;
        const auto ks = fa4_rows(kg + (int64_t) t0 * a.k1, a.k1, n, 18 * NB);
        const auto vs = fa4_rows(vg + (int64_t) t0 * a.v1, a.v1, n, 18 * NB);
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            kr[i] = fa4_load(ks, ko[i]);
            vr[i] = fa4_load(vs, vo[i]);
        }
        if constexpr (MS == 2) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const int key = t0 + 16 * mt + 4 * q4;
                if (a.n_kv >= 4) {  // 4 keys in one load, the last ones from the row's end (shifted at their use)
                    const char * mp = mrow + (int64_t) (key < a.n_kv - 4 ? key : a.n_kv - 4) * 2;
                    mr[mt] = *(const fa4_u2h *) mp;
                } else {
                    for (int r = 0; r < 4; ++r) {
                        const int      at = key + r < a.n_kv ? key + r : a.n_kv - 1;
                        const uint32_t x  = *(const uint16_t *) (mrow + (int64_t) at * 2);
                        mr[mt][r / 2]     = r & 1 ? mr[mt][r / 2] | x << 16 : x;
                    }
                }
            }
        }
    };

    for (int base = (int) split * W + wv; base < ntile; base += F::MB * step) {
        uint32_t todo = 0;  // bit i: tile base + i * step is to be walked
        if constexpr (MS == 1) {
            uint16_t mv[F::MB];
#pragma unroll
            for (int i = 0; i < F::MB; ++i) {
                const int key = (base + i * step) * TK + (lane & (TK - 1));
                mv[i]         = *(const uint16_t *) (mrow + (int64_t) (key < a.n_kv ? key : a.n_kv - 1) * 2);
            }
#pragma unroll
            for (int i = 0; i < F::MB; ++i) {
                const int   key = (base + i * step) * TK + (lane & (TK - 1));
                const float x   = key < a.n_kv ? f16_lo(mv[i]) * FA4_LOG2E : -INFINITY;
                todo |= (uint32_t) (__builtin_amdgcn_ballot_w64(x != -INFINITY) != 0) << i;
                if (lane < TK) {
                    ml[i * TK + lane] = x;
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        } else {
            const int n = (ntile - base + step - 1) / step;
            todo        = n >= F::MB ? (1u << F::MB) - 1 : (1u << n) - 1;
        }
        if (todo) {
            load(base + (__builtin_ffs(todo) - 1) * step, true);
        }
        while (todo) {
            const int i = __builtin_ffs(todo) - 1;
            todo &= todo - 1;
            const int t0 = (base + i * step) * TK;
            // mask values of this lane's scores, and the keys that some row attends to
            float    ms[MT][4];
            uint64_t live = 0;
            if constexpr (MS == 1) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const fa4_f4 x = *(const fa4_f4 *) (ml + i * TK + 16 * mt + 4 * q4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        ms[mt][r] = x[r];
                    }
                }
                live = __builtin_amdgcn_ballot_w64(ml[i * TK + (lane & (TK - 1))] != -INFINITY);
            } else {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    uint64_t x = 0;
                    if constexpr (MS == 2) {
                        const int over = a.n_kv >= 4 ? t0 + 16 * mt + 4 * q4 + 4 - a.n_kv : 0;
                        x              = (uint64_t) mr[mt].y << 32 | mr[mt].x;
                        x              = over > 0 && over < 4 ? x >> (16 * over) : x;
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool in = t0 + 16 * mt + 4 * q4 + r < a.n_kv;
                        ms[mt][r]     = !in ? -INFINITY : MS == 2 ? f16_lo((uint32_t) (x >> (16 * r))) * FA4_LOG2E : 0.0f;
                        const uint64_t v = __builtin_amdgcn_ballot_w64(ms[mt][r] != -INFINITY);
#pragma unroll
                        for (int gr = 0; gr < 4; ++gr) {
                            live |= (uint64_t) ((v >> (16 * gr) & 0xffffu) != 0) << (16 * mt + 4 * gr + r);
                        }
                    }
                }
            }
            // raw blocks to LDS: K's levels as words [key][group][block], V's as rows, d by block and key
            bool big = false;
#pragma unroll
            for (int it = 0; it < IPL; ++it) {
                const int idx = it * 64 + lane, key = idx / NB, blk = idx % NB;
                float     d;
                uint32_t  q[4];
                fa4_block(kr[it], blk, d, q);
                char * kp = kl + F::koff(key) + blk * 4;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    *(uint32_t *) (kp + e * 4 * NB) = q[e];
                }
                dkl[blk * F::DS + key] = fa4_scale(d);
                fa4_block(vr[it], blk, d, q);
                *(uint4 *) (vl + F::voff(key) + blk * 16) = make_uint4(q[0], q[1], q[2], q[3]);
                d   = live >> key & 1 ? d : 0.0f;
                big = big || fabsf(d) > FA4_BIG;
                // in the order of the slots: keys 0, 2, 1, 3 of each four
                const int kp4 = (key & ~3) | (key & 1) << 1 | (key >> 1 & 1);
                *(_Float16 *) (dvl + (blk * F::DS + kp4) * 2) = (_Float16) d;
            }
            big = __builtin_amdgcn_ballot_w64(big) != 0;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            load(base + (todo ? __builtin_ffs(todo) - 1 : i) * step, todo != 0);

            // scores, in units of log2
            float s[MT][4], mx = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const uint32_t * kp = (const uint32_t *) (kl + F::koff(16 * mt + c16) + q4 * 4 * NB);
                uint32_t         kw[NB];
#pragma unroll
                for (int blk = 0; blk < NB; ++blk) {
                    kw[blk] = kp[blk];
                }
                fa4_f4 t = { 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
                for (int blk = 0; blk < NB; ++blk) {
                    const fa4_h8 x  = fa4_levels(kw[blk]);
                    const fa4_f4 dk = *(const fa4_f4 *) (dkl + blk * F::DS + 16 * mt + 4 * q4);
#pragma unroll
                    for (int p = QP - 1; p >= 0; --p) {
                        const fa4_f4 acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            x, qb[p][blk], fa4_f4{ 0.0f, 0.0f, 0.0f, 0.0f }, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            t[r] = __builtin_fmaf(acc[r], dk[r], t[r]);
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[mt][r] = ms[mt][r] == -INFINITY ? -INFINITY : __builtin_fmaf(t[r], qs, ms[mt][r]);
                    mx       = fmaxf(mx, s[mt][r]);
                }
            }
            // the maximum that p refers to moves only when a row's grows by more than 2^3: most tiles
            // need no reduction over lanes
            if (__builtin_amdgcn_ballot_w64(mx > m + 3.0f) != 0) {
                const float mnew = fmaxf(m, fa4_max_groups(mx));
                const float al   = m == mnew ? 1.0f : __builtin_amdgcn_exp2f(m - mnew);
                l *= al;
#pragma unroll
                for (int j = 0; j < 2 * NB; ++j) {
                    o[j] *= al;
                }
                m = mnew;
            }
            const float mu = (m == -INFINITY ? 0.0f : m) - FA4_OFF;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[mt][r] = __builtin_amdgcn_exp2f(s[mt][r] - mu);
                    l += s[mt][r];
                }
            }
            if (big) {  // d / 16 held in fp16, p * 16
#pragma unroll
                for (int it = 0; it < IPL; ++it) {
                    const int idx = it * 64 + lane, key = idx / NB, blk = idx % NB;
                    const int kp4 = (key & ~3) | (key & 1) << 1 | (key >> 1 & 1);
                    _Float16 * dp = (_Float16 *) (dvl + (blk * F::DS + kp4) * 2);
                    *dp           = *dp * (_Float16) 0.0625f;
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[mt][r] *= 16.0f;
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
#pragma unroll
            for (int kgp = 0; kgp < TK / 32; ++kgp) {
                fa4_h8 ph, pl;
#pragma unroll
                for (int e = 0; e < 8; ++e) {  // slots: keys 0, 2, 1, 3 of each four
                    const float p = s[2 * kgp + e / 4][(e & 1) * 2 + (e >> 1 & 1)];
                    ph[e]         = (_Float16) p;
                    if constexpr (OS) {
                        pl[e] = (_Float16) (p - (float) ph[e]);
                    }
                }
                // lane m of a group of 16 addresses key m / 2 of the group's 8, half m % 2 of a block's 16 bytes
                const int mk  = c16 >> 1;
                const int key = 32 * kgp + 4 * q4 + (mk & 3) + (mk & 4) * 4;
                char *    vp  = vl + F::voff(key) + 8 * (c16 & 1);
#pragma unroll
                for (int blk = 0; blk < NB; ++blk) {
                    const fa4_v2i  w  = __builtin_amdgcn_ds_read_tr8_b64_v2i32((fa4_lds_v2i *) (vp + blk * 16));
                    const uint32_t w0 = (uint32_t) w.x, w1 = (uint32_t) w.y;
                    const uint2    da = *(const uint2 *) (dvl + (blk * F::DS + 32 * kgp + 4 * q4) * 2);
                    const uint2    db = *(const uint2 *) (dvl + (blk * F::DS + 32 * kgp + 16 + 4 * q4) * 2);
                    const uint32_t dd[4] = { da.x, da.y, db.x, db.y };
                    const uint32_t ww[4] = { w0, w0 >> 8, w1, w1 >> 8 };
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        u32x4 vh, vlo;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const fa4_h2 x = half ? fa4_high(ww[e]) : fa4_low(ww[e]);
                            const fa4_h2 d = fa4_half2(dd[e]), v = x * d;
                            vh[e] = fa4_bits(v);
                            if constexpr (OS) {
                                vlo[e] = fa4_bits(__builtin_elementwise_fma(x, d, -v));
                            }
                        }
                        const fa4_h8 av = __builtin_bit_cast(fa4_h8, vh);
                        fa4_f4 &     oo = o[2 * blk + half];
                        oo              = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, ph, oo, 0, 0, 0);
                        if constexpr (OS) {
                            oo = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pl, oo, 0, 0, 0);
                            oo = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fa4_h8, vlo), ph, oo, 0, 0, 0);
                        }
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }

    // merge the waves: (m, l) of each row, then the outputs relative to the largest m
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (q4 == 0) {
        stat[wv][c16][0] = m;
        stat[wv][c16][1] = l;
    }
    __syncthreads();
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        mm = fmaxf(mm, stat[w][c16][0]);
    }
    const float wt = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mm);
    const int   nr = a.rows - rt * 16 < 16 ? a.rows - rt * 16 : 16;
    constexpr int DC = F::DC;
#pragma unroll
    for (int c = 0; c < D / DC; ++c) {
        if (c > 0) {
            __syncthreads();
        }
        float * om = (float *) (lds + wv * WB);
#pragma unroll
        for (int j = 0; j < DC / 16; ++j) {
            *(fa4_f4 *) (om + c16 * DC + j * 16 + 4 * q4) = o[c * (DC / 16) + j] * wt;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < nr * DC; i += 64 * W) {
            const int r = i / DC, d = i - r * DC;
            float     acc = 0.0f, mr2 = -INFINITY, ls = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                acc += ((const float *) (lds + w * WB))[i];
                mr2 = fmaxf(mr2, stat[w][r][0]);
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float mw = stat[w][r][0];  // -inf without a live score, or with NaN alone: l is 0 or NaN
                ls += stat[w][r][1] * (mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - mr2));
            }
            const int rr = rt * 16 + r;
            if (a.splits > 1) {
                float * p = a.ws + (((int64_t) bg * a.rows + rr) * a.splits + split) * (D + 4);
                if (c == 0 && d == 0) {
                    p[0] = mr2;
                    p[1] = ls;
                }
                p[4 + c * DC + d] = acc;
            } else {
                const int iq2 = rr / a.rk, h2 = (int) g * a.rk + (rr - iq2 * a.rk);
                char *    yp  = a.y + (int64_t) b * a.y3 + (int64_t) iq2 * a.y2 + (int64_t) h2 * a.y1;
                const float v = acc / ls;  // no live key: 0 / 0
                if (a.ty == MI_TYPE_F32) {
                    store_elem<MI_TYPE_F32>(yp + (size_t) (c * DC + d) * 4, v);
                } else {
                    store_elem<MI_TYPE_BF16>(yp + (size_t) (c * DC + d) * 2, v);
                }
            }
        }
    }
}

// The splits' partial results of a row: y = sum_i w_i o_i / sum_i w_i l_i with w_i =
// exp2(m_i - max m). A workgroup per row: D / 4 lanes take a float4 of the columns, the groups of
// them every SG-th split. The outputs of the first PRE splits of each group are loaded with the
// (m, l), before the weights are known: one round of memory latency for up to SG * PRE splits.
// A split without a live score has m = -inf and zeros; one whose live scores are all NaN has m = -inf
// too, and NaN: every split is added, with weight 0 as well, so that its NaN shows.
constexpr int FA4_MAX_SPLITS = 1024;

template <int D, int PRE>
__global__ void __launch_bounds__(256) k_fa4_combine(const FaArgs a) {
    constexpr int C4 = D / 4, SG = 256 / C4;
    __shared__ float                wsh[FA4_MAX_SPLITS];
    __shared__ float                red[8];
    __shared__ __align__(16) fa4_f4 part[SG][C4];
    const int      tid = threadIdx.x, c = tid % C4, sg = tid / C4;
    const uint32_t rec = blockIdx.x;
    const uint32_t bg  = rec / (uint32_t) a.rows;
    const int      row = (int) (rec - bg * (uint32_t) a.rows);
    const uint32_t b   = bg / (uint32_t) a.nkv;
    const uint32_t g   = bg - b * (uint32_t) a.nkv;
    const int      iq = row / a.rk, h = (int) g * a.rk + (row - iq * a.rk), last = a.splits - 1;
    const float *  p = a.ws + (int64_t) rec * a.splits * (D + 4);
    fa4_f4         pv[PRE];
#pragma unroll
    for (int j = 0; j < PRE; ++j) {  // past the last split: the last one again, never added
        const int s = sg + SG * j;
        pv[j]       = *(const fa4_f4 *) (p + (int64_t) (s < last ? s : last) * (D + 4) + 4 + 4 * c);
    }
    float ml[FA4_MAX_SPLITS / 256], ll[FA4_MAX_SPLITS / 256], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < FA4_MAX_SPLITS / 256; ++i) {
        const int    s = tid + 256 * i;
        const float2 x = *(const float2 *) (p + (int64_t) (s < last ? s : last) * (D + 4));
        ml[i]          = s <= last ? x.x : -INFINITY;
        ll[i]          = s <= last ? x.y : 0.0f;
        m              = fmaxf(m, ml[i]);
    }
    m = group_max<64>(m);
    if ((tid & 63) == 0) {
        red[tid >> 6] = m;
    }
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
#pragma unroll
    for (int i = 0; i < FA4_MAX_SPLITS / 256; ++i) {
        const int   s = tid + 256 * i;
        const float w = ml[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[i] - m);
        wsh[s]        = w;
        l             = __builtin_fmaf(w, ll[i], l);
    }
    l = group_sum<64>(l);
    if ((tid & 63) == 0) {
        red[4 + (tid >> 6)] = l;
    }
    __syncthreads();
    l          = (red[4] + red[5]) + (red[6] + red[7]);
    fa4_f4 acc = { 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
    for (int j = 0; j < PRE; ++j) {
        const int   s = sg + SG * j;
        const float w = wsh[s];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc[e] = s <= last ? __builtin_fmaf(w, pv[j][e], acc[e]) : acc[e];
        }
    }
    for (int s0 = SG * PRE + sg; s0 <= last; s0 += SG * PRE) {
#pragma unroll
        for (int j = 0; j < PRE; ++j) {
            const int s = s0 + SG * j;
            pv[j]       = *(const fa4_f4 *) (p + (int64_t) (s < last ? s : last) * (D + 4) + 4 + 4 * c);
        }
#pragma unroll
        for (int j = 0; j < PRE; ++j) {
            const int   s = s0 + SG * j;
            const float w = s <= last ? wsh[s] : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[e] = s <= last ? __builtin_fmaf(w, pv[j][e], acc[e]) : acc[e];
            }
        }
    }
    part[sg][c] = acc;
    __syncthreads();
    if (tid < C4) {
        fa4_f4 t = part[0][tid];
#pragma unroll
        for (int q = 1; q < SG; ++q) {
            t += part[q][tid];
        }
        t *= 1.0f / l;  // no live key: 0 * inf
        char * yp = a.y + (int64_t) b * a.y3 + (int64_t) iq * a.y2 + (int64_t) h * a.y1;
        if (a.ty == MI_TYPE_F32) {
            *(fa4_f4u *) (yp + 16 * tid) = t;
        } else {
            *(fa4_u2u *) (yp + 8 * tid) = fa4_u2u{ pack_bf16x2(t[0], t[1]), pack_bf16x2(t[2], t[3]) };
        }
    }
}

// The same for up to S splits: D / 4 lanes per row, a lane's columns of every split in registers,
// no exchange between lanes.
template <int D, int S>
__global__ void __launch_bounds__(256) k_fa4_combine_few(const FaArgs a) {
    constexpr int  C4   = D / 4, RW = 256 / C4;
    const int      c    = threadIdx.x % C4;
    const uint32_t nrec = (uint32_t) (a.nb * a.nkv) * (uint32_t) a.rows;
    const uint32_t rec  = blockIdx.x * RW + threadIdx.x / C4;
    if (rec >= nrec) {
        return;
    }
    const int     last = a.splits - 1;
    const float * p    = a.ws + (int64_t) rec * a.splits * (D + 4);
    fa4_f4        pv[S];
    float         m[S], l[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {  // past the last split: the last one again, never added
        const float * ps = p + (int64_t) (s < last ? s : last) * (D + 4);
        m[s]             = ps[0];
        l[s]             = ps[1];
        pv[s]            = *(const fa4_f4 *) (ps + 4 + 4 * c);
    }
    const uint32_t bg  = rec / (uint32_t) a.rows;
    const int      row = (int) (rec - bg * (uint32_t) a.rows);
    const uint32_t b   = bg / (uint32_t) a.nkv;
    const uint32_t g   = bg - b * (uint32_t) a.nkv;
    const int      iq = row / a.rk, h = (int) g * a.rk + (row - iq * a.rk);
    float          mm = m[0], lt = 0.0f;
#pragma unroll
    for (int s = 1; s < S; ++s) {
        mm = fmaxf(mm, m[s]);
    }
    fa4_f4 t = { 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const float w = s > last || m[s] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[s] - mm);
        lt            = s <= last ? __builtin_fmaf(w, l[s], lt) : lt;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            t[e] = s <= last ? __builtin_fmaf(w, pv[s][e], t[e]) : t[e];
        }
    }
    t *= 1.0f / lt;  // no live key: 0 * inf
    char * yp = a.y + (int64_t) b * a.y3 + (int64_t) iq * a.y2 + (int64_t) h * a.y1;
    if (a.ty == MI_TYPE_F32) {
        *(fa4_f4u *) (yp + 16 * c) = t;
    } else {
        *(fa4_u2u *) (yp + 8 * c) = fa4_u2u{ pack_bf16x2(t[0], t[1]), pack_bf16x2(t[2], t[3]) };
    }
}

// Many query rows: a workgroup of W waves owns W * 16 * RT rows (query position, head) of
// one KV head and walks the keys in tiles of T, K and V dequantized once per tile into LDS,
// double-buffered, the next tile's raw blocks in flight. A wave holds RT tiles of 16 rows;
// the products are those of k_fa4_dec (S^T = K Q^T, O^T = V^T P^T, 16x16x32), their A
// operands read from LDS once for all RT tiles.
//  K      BF16 y: (level - 8) d in fp16, one rounding (2^-11 of each term of q . k, where q
//         itself has 8 bits), so that the sum over blocks stays in the accumulator; F32 y: the
//         levels as whole numbers, the sums of each block scaled by d as in k_fa4_dec
//  V      (level - 8) d in fp16, F32 y: a high and a low part
//  order  a block's 32 elements lie in LDS as (half, group of 4, 0 2 1 3), the order in which
//         masks and shifts unpack the nibbles; q is read in the same order, and the output
//         lane's 4 values are one group of 4, put back when they are stored
// A tile in which some d would leave fp16 is held / 16, P or its scores taken * 16; in one with a
// block that is not finite the keys that no row of the workgroup attends to count as zeros. The
// waves tell each other at the barrier before they lay the tile out.
// The maximum that p refers to moves only when a row's grows by more than 2^3, so most tiles
// need no reduction over lanes; the row sums are products with ones. Masks are looked up per tile in
// k_fa_mask_summary's bytes.
// Bound by unpacking and exponentials beside the matrix cores (busy 33 % of the cycles, vector issue 58 %;
// two waves a SIMD is what the registers leave). 8 x 2048 positions, 32 heads on 8, 128: BF16 y without a mask
// 642 us, 856 TFLOP/s, causal 381 and 16 for the summary; F32 y 1292 and 752. 8 waves (256 rows) in BF16:
// 626 without a mask, but 2048 positions on 6144 keys 239 instead of 229.
template <int D, bool OS> struct Fa4P {
    static constexpr int NB = D / 32;
    static constexpr int T  = D == 256 ? 32 : 64;       // keys per tile
    static constexpr int RT = D == 256 ? 1 : 2;         // row tiles per wave
    static constexpr int W  = D == 256 || (OS && D == 128) ? 8 : 4;
    static constexpr int BQ = W * 16 * RT;
    static constexpr int KS = D * 2 + 16;               // K row stride: 16 keys on distinct banks
    static constexpr int VS = D * 2 + 32;               // V row stride: 8 keys on distinct banks, transposed reads
    static constexpr int VP = OS ? 2 : 1;
    static constexpr int DS = T + 16;                   // entries per block in the table of K's d (F32 y)
    static constexpr int KB = T * KS;
    static constexpr int VB = T * VS;
    static constexpr int DB = OS ? NB * DS * 4 : 0;
    static constexpr int BUF = KB + VP * VB + DB;
};

template <int D, bool OS, bool MSK>
__global__ void __launch_bounds__((64 * Fa4P<D, OS>::W)) __attribute__((amdgpu_waves_per_eu(2)))
k_fa4_pre(const FaArgs a) {
    using F          = Fa4P<D, OS>;
    constexpr int NB = F::NB, T = F::T, RT = F::RT, W = F::W, QP = OS ? 2 : 1;
    constexpr int NI = 2 * T * NB;                       // blocks per tile, K's then V's
    constexpr int IT = NI / (64 * W);                    // per thread
    static_assert(NI % (64 * W) == 0 && T * NB % 64 == 0, "a wave's blocks are K's or V's");
    __shared__ __align__(16) char lds[2 * F::BUF];
    __shared__ uint32_t           tflag[2][W];           // 1: V's d past fp16, 2: K's, 4: V not finite
    __shared__ uint64_t           lvw[W];
    __shared__ __align__(16) uint64_t wins[MSK ? FA4_PRE_TILES / 64 : 1][2];

    const int      tid = threadIdx.x, lane = tid & 63;
    const int      wv  = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int      c16 = lane & 15, q4 = lane >> 4;
    const uint32_t item  = blockIdx.x / (uint32_t) a.splits;
    const uint32_t split = blockIdx.x - item * (uint32_t) a.splits;
    const uint32_t nbg   = (uint32_t) (a.nb * a.nkv);
    const uint32_t bg    = item % nbg;
    const int      r0    = (a.rblocks - 1 - (int) (item / nbg)) * F::BQ;  // last rows first: the longest under a causal mask
    const uint32_t b     = bg / (uint32_t) a.nkv;
    const uint32_t g     = bg - b * (uint32_t) a.nkv;
    const uint32_t kb    = b / (uint32_t) a.rk3;
    const char *   kg    = a.k + (int64_t) kb * a.k3 + (int64_t) g * a.k2;
    const char *   vg    = a.v + (int64_t) kb * a.v3 + (int64_t) g * a.v2;

    // q: row tile rt, lane (row c16, group q4): positions 8 q4 .. 8 q4 + 7 of each block
    fa4_h8       qb[RT][QP][NB];
    float        qs[RT];
    const char * mrow[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r  = r0 + (wv * RT + rt) * 16 + c16;
        const int rc = r < a.rows ? r : a.rows - 1;
        const int iq = rc / a.rk, h = (int) g * a.rk + (rc - iq * a.rk);
        if constexpr (MSK) {
            mrow[rt] = a.mask + (int64_t) (b % (uint32_t) a.mne3) * a.m3 + (int64_t) (h % a.mne2) * a.m2 + (int64_t) iq * a.m1;
        }
        const char * qp = a.q + (int64_t) b * a.q3 + (int64_t) h * a.q2 + (int64_t) iq * a.q1;
        float        qv[NB][8], qmax = 0.0f;
        fa4_q<NB, OS>(qp, a.tq, 8 * q4, 8 * q4 + 4, qv);
#pragma unroll
        for (int blk = 0; blk < NB; ++blk) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                qmax = fmaxf(qmax, fabsf(qv[blk][e]));
            }
        }
        qmax           = fa4_max_groups(qmax);
        int ex         = (int) (__float_as_uint(qmax) >> 23) - 127;
        ex             = ex < -100 ? -100 : ex > 127 ? 10 : ex;
        const float up = __builtin_copysignf(__uint_as_float((uint32_t) (127 + 10 - ex) << 23), a.scale);
        qs[rt]         = fabsf(a.scale) * FA4_LOG2E * __uint_as_float((uint32_t) (127 - 10 + ex) << 23);
#pragma unroll
        for (int blk = 0; blk < NB; ++blk) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int   i = (e & 4) + ((e & 1) << 1 | (e >> 1 & 1));  // 0 2 1 3 of each four
                const float v = qv[blk][i] * up, w = OS ? __builtin_rintf(v) : v;
                qb[rt][0][blk][e] = (_Float16) w;
                if constexpr (OS) {
                    qb[rt][1][blk][e] = (_Float16) (v - w);
                }
            }
        }
    }

    float  m[RT];
    fa4_f4 o[RT][2 * NB], l[RT];  // l: the sum of p, in all 4 (A = ones)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = fa4_f4{ 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
            o[rt][i] = fa4_f4{ 0.0f, 0.0f, 0.0f, 0.0f };
        }
    }

    // thread: blocks i * 64 W + tid of the tile, of K (keys in order, a key's blocks together), then of V
    Fa4Raw raw[IT];
    int    off[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const bool isv = i * 64 * W + wv * 64 >= T * NB;  // uniform in the wave
        const int  j   = i * 64 * W + tid - (isv ? T * NB : 0);
        off[i]         = j / NB * (int) (isv ? a.v1 : a.k1) + ((18 * (j % NB)) & ~3);
    }
    auto load = [&](int i, int t, bool on) {  // block i of tile t; `on` false: no tile (zeros)
        const int     t0 = t * T, n = !on ? 0 : a.n_kv - t0 < T ? a.n_kv - t0 : T;
        const bool    isv = i * 64 * W + wv * 64 >= T * NB;
        const int64_t st  = isv ? a.v1 : a.k1;
        return fa4_load(fa4_rows((isv ? vg : kg) + (int64_t) t0 * st, st, n, 18 * NB), off[i]);
    };
    // flags of the blocks in raw: 1 a d of V past FA4_BIG, 2 of K, 4 one that is not finite
    auto flags = [&]() -> uint32_t {
        uint32_t fl = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const bool     isv = i * 64 * W + wv * 64 >= T * NB;
            const int      j   = i * 64 * W + tid - (isv ? T * NB : 0), blk = j % NB;
            const uint32_t mag = (blk & 1 ? raw[i].w[0] >> 16 : raw[i].w[0]) & 0x7fffu;
            if (__builtin_amdgcn_ballot_w64(mag > FA4_BIG_BITS) != 0) {
                fl |= (isv ? 1u : 2u) | (__builtin_amdgcn_ballot_w64(mag >= 0x7c00u) != 0 ? 4u : 0u);
            }
        }
        return fl;
    };
    // block i of a tile with the flags fl -> buffer bf: V's, K's d / 16 with flag 1, 2; zeros for keys
    // that are not in `live` with flag 4
    auto stage = [&](int i, const Fa4Raw & rw, int bf, uint32_t fl, uint64_t live) {
        char *     kl = lds + bf * F::BUF, *vl = kl + F::KB;
        float *    dl  = (float *) (vl + F::VP * F::VB);
        const bool isv = i * 64 * W + wv * 64 >= T * NB;
        const int  j   = i * 64 * W + tid - (isv ? T * NB : 0), blk = j % NB, key = j / NB;
        float      d;
        uint32_t   w[4];
        fa4_block(rw, blk, d, w);
        if (fl & 4) {
            d = live >> key & 1 ? d : 0.0f;
        }
        if (OS && !isv) {
            dl[blk * F::DS + key] = fa4_scale(d);  // fp32: nothing to scale
        }
        d *= fl & (isv ? 1u : 2u) ? 0.0625f : 1.0f;
        const _Float16 dh = (_Float16) d;
        const fa4_h2 dd = { dh, dh };
        uint32_t     q[16], ql[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // low (0 2), low (1 3), high (0 2), high (1 3)
                const uint32_t x  = k & 1 ? w[e] >> 8 : w[e];
                const fa4_h2   n  = k & 2 ? fa4_high(x) : fa4_low(x), v = n * dd;
                const int      at = (k & 2) * 4 + 2 * e + (k & 1);
                q[at] = OS && !isv ? fa4_bits(n) : fa4_bits(v);
                if constexpr (OS) {
                    ql[at] = fa4_bits(__builtin_elementwise_fma(n, dd, -v));
                }
            }
        }
        char * p = isv ? vl + key * F::VS + blk * 64 : kl + key * F::KS + blk * 64;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            *(uint4 *) (p + 16 * e) = make_uint4(q[4 * e], q[4 * e + 1], q[4 * e + 2], q[4 * e + 3]);
            if constexpr (OS) {
                if (isv) {
                    *(uint4 *) (p + F::VB + 16 * e) = make_uint4(ql[4 * e], ql[4 * e + 1], ql[4 * e + 2], ql[4 * e + 3]);
                }
            }
        }
    };

    const int ntile = (a.n_kv + T - 1) / T;
    const int tbeg  = (int) ((int64_t) ntile * split / a.splits), tend = (int) ((int64_t) ntile * (split + 1) / a.splits);
    const int iq0 = r0 / a.rk, iq1 = (r0 + F::BQ < a.rows ? r0 + F::BQ - 1 : a.rows - 1) / a.rk;
    // the tiles with a live key, and those with values that are not 0 (`dirty`), a bit per tile: a wave
    // reads the summary bytes of the workgroup's rows for 64 tiles at a time
    if constexpr (MSK) {
        const int nts = (a.n_kv + 63) / 64, nh = a.rk < a.mne2 ? a.rk : a.mne2;
        for (int w0 = tbeg + wv * 64; w0 < tend; w0 += 64 * W) {
            const int t = w0 + lane < tend ? w0 + lane : tend - 1;
            uint32_t  f = 0;
            for (int hh = 0; hh < nh; ++hh) {
                const int       mh = (int) (b % (uint32_t) a.mne3) * a.mne2 + ((int) g * a.rk + hh) % a.mne2;
                const uint8_t * mp = a.msum + ((int64_t) mh * a.ngq) * nts + t * T / 64;
#pragma unroll 4
                for (int gr = iq0 >> 4; gr <= iq1 >> 4; ++gr) {
                    f |= mp[(int64_t) gr * nts];
                }
            }
            const uint64_t x = __builtin_amdgcn_ballot_w64(w0 + lane < tend && (f & 1));
            const uint64_t y = __builtin_amdgcn_ballot_w64((f & 2) != 0);
            if (lane == 0) {
                wins[(w0 - tbeg) / 64][0] = x;
                wins[(w0 - tbeg) / 64][1] = y;
            }
        }
        __syncthreads();
    }
    int      wb = tbeg - 64;
    uint64_t lv = 0, nz = 0;
    auto     next = [&](bool & dirty) -> int {  // the next tile to walk, tend after the last
        if constexpr (MSK) {
            while (lv == 0) {
                wb += 64;
                if (wb >= tend) {
                    wb = tend;  // asked again: still none
                    return tend;
                }
                const uint4 x = *(const uint4 *) wins[(wb - tbeg) / 64];
                lv = (uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) x.y) << 32 |
                     (uint32_t) __builtin_amdgcn_readfirstlane((int) x.x);
                nz = (uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) x.w) << 32 |
                     (uint32_t) __builtin_amdgcn_readfirstlane((int) x.z);
            }
            const int i = (int) __builtin_ctzll(lv);
            lv &= lv - 1;
            dirty = nz >> i & 1;
            return wb + i;
        } else {
            dirty = false;
            wb    = wb < tbeg ? tbeg : wb + 1;
            return wb < tend ? wb : tend;
        }
    };
    // the flags that every wave found for a tile; the keys that some row of the workgroup attends to
    // where one is not finite
    auto agree = [&](int bf, int t, uint64_t & live) -> uint32_t {
        uint32_t fl = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            fl |= tflag[bf][w];
        }
        fl = __builtin_amdgcn_readfirstlane(fl);
        if (fl & 4) {
            live = 0;
#pragma unroll 1
            for (int k = 0; k < T; k += 4) {
                const int key = t * T + k + q4;
                bool      on  = false;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    bool x = key < a.n_kv;
                    if constexpr (MSK) {
                        x = x && *(const uint16_t *) (mrow[rt] + (int64_t) (x ? key : 0) * 2) != 0xFC00u;
                    }
                    on = on || x;
                }
                const uint64_t v = __builtin_amdgcn_ballot_w64(on);
#pragma unroll 1
                for (int gr = 0; gr < 4; ++gr) {
                    live |= (uint64_t) ((v >> (16 * gr) & 0xffffu) != 0) << (k + gr);
                }
            }
            if (lane == 0) {
                lvw[wv] = live;
            }
            __syncthreads();
            for (int w = 0; w < W; ++w) {
                live |= lvw[w];
            }
            __syncthreads();  // lvw may be written again
        }
        return fl;
    };
    bool dirty, dirty_n, dirty_2;
    int  t = next(dirty), bf = 0;
    if (t < tend) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            raw[i] = load(i, t, true);
        }
        tflag[0][wv] = flags();
        __syncthreads();
        uint64_t live = 0;
        uint32_t fl   = agree(0, t, live);
        int      tn   = next(dirty_n);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            stage(i, raw[i], 0, fl, live);
            raw[i] = load(i, tn, tn < tend);
        }
        tflag[1][wv] = flags();
        __syncthreads();
        while (true) {
            const int      t2 = next(dirty_2);
            const uint32_t fn = agree(bf ^ 1, tn, live);  // the next tile's
            const int    t0 = t * T;
            const char * kl = lds + bf * F::BUF;
            const char * vl = kl + F::KB;
            const float * dl = (const float *) (vl + F::VP * F::VB);
            const bool   clean = t0 + T <= a.n_kv && !dirty;
            const float  kf = !OS && (fl & 2) ? 16.0f : 1.0f;  // what the scores are to be multiplied by
            if constexpr (OS) {  // fewer registers are left for what the product's instructions could hide
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    stage(i, raw[i], bf ^ 1, fn, live);
                    raw[i] = load(i, t2, t2 < tend);
                }
            }
            const uint32_t one = fl & 1 ? 0x2c002c00u : 0x3c003c00u;  // 1/16 where V is held / 16 and P 16 times as large
            const fa4_h8   ones = __builtin_bit_cast(fa4_h8, make_uint4(one, one, one, one));
            const float poff = fl & 1 ? FA4_OFF + 4.0f : FA4_OFF;
            // 32 keys at a time: few enough scores and operands that the LDS reads of both products can be
            // in flight before the first is used
#pragma unroll
            for (int kk = 0; kk < T / 32; ++kk) {
                fa4_h8 kx[2][NB];
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                    for (int blk = 0; blk < NB; ++blk) {
                        kx[mt][blk] = *(const fa4_h8 *) (kl + (32 * kk + 16 * mt + c16) * F::KS + q4 * 16 + blk * 64);
                    }
                }
                // the mask of the lane's scores, 4 keys a load (rows lie at any 2 bytes)
                uint32_t mx[RT][2][2] = {};
                if (MSK && !clean) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const char * mp = mrow[rt] + (int64_t) (t0 + 32 * kk + 4 * q4) * 2;
                        if (t0 + T <= a.n_kv) {
                            const fa4_u2h y = *(const fa4_u2h *) mp, z = *(const fa4_u2h *) (mp + 32);
                            mx[rt][0][0] = y.x;
                            mx[rt][0][1] = y.y;
                            mx[rt][1][0] = z.x;
                            mx[rt][1][1] = z.y;
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const int      key = t0 + 32 * kk + 16 * (e / 4) + 4 * q4 + e % 4;
                                const int      at  = key < a.n_kv ? key : a.n_kv - 1;
                                const uint32_t y   = *(const uint16_t *) (mrow[rt] + (int64_t) at * 2);
                                mx[rt][e / 4][e % 4 / 2] |= y << (16 * (e % 2));
                            }
                        }
                    }
                }
                fa4_f4 s[RT][2];
                if constexpr (OS && D == 128) {  // the one workgroup's waves go in step: products before the others' exponentials
                    __builtin_amdgcn_s_setprio(1);  // (8 x 2048 positions, F32: 781 -> 752 us; BF16 and other D: slower)
                }
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        s[rt][mt] = fa4_f4{ 0.0f, 0.0f, 0.0f, 0.0f };
                    }
#pragma unroll
                    for (int blk = 0; blk < NB; ++blk) {
                        if constexpr (OS) {
                            const fa4_f4 dk = *(const fa4_f4 *) (dl + blk * F::DS + 32 * kk + 16 * mt + 4 * q4);
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                                for (int p = 1; p >= 0; --p) {
                                    const fa4_f4 acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                        kx[mt][blk], qb[rt][OS ? p : 0][blk], fa4_f4{ 0.0f, 0.0f, 0.0f, 0.0f }, 0, 0, 0);
#pragma unroll
                                    for (int r = 0; r < 4; ++r) {
                                        s[rt][mt][r] = __builtin_fmaf(acc[r], dk[r], s[rt][mt][r]);
                                    }
                                }
                            }
                        } else {
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
                                s[rt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kx[mt][blk], qb[rt][0][blk], s[rt][mt], 0, 0, 0);
                            }
                        }
                    }
                }
                if constexpr (OS && D == 128) {
                    __builtin_amdgcn_s_setprio(0);
                }
                // the next tile's blocks, while the product runs
                if (!OS && kk < IT) {
                    stage(kk, raw[kk], bf ^ 1, fn, live);  // past the last tile: zeros
                    raw[kk] = load(kk, t2, t2 < tend);
                }
                // scores in units of log2: s * fac
                float fac[RT], lm[RT];
                bool  grow = false;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    fac[rt] = qs[rt] * kf;
                }
                if (!clean) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const bool     in = t0 + 32 * kk + 16 * (e / 4) + 4 * q4 + e % 4 < a.n_kv;
                            const uint32_t w  = mx[rt][e / 4][e % 4 / 2];
                            const float    y  = in ? (e & 1 ? f16_hi(w) : f16_lo(w)) * FA4_LOG2E : -INFINITY;
                            s[rt][e / 4][e % 4] = __builtin_fmaf(s[rt][e / 4][e % 4], fac[rt], y);
                        }
                        fac[rt] = 1.0f;
                    }
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    float x = fmaxf(fmaxf(s[rt][0][0], s[rt][0][1]), s[rt][0][2]);
                    x       = fmaxf(fmaxf(x, s[rt][0][3]), s[rt][1][0]);
                    x       = fmaxf(fmaxf(x, s[rt][1][1]), s[rt][1][2]);
                    lm[rt]  = fmaxf(x, s[rt][1][3]) * fac[rt];
                    grow    = grow || lm[rt] > m[rt] + 3.0f;
                }
                if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const float mn = fmaxf(m[rt], fa4_max_groups(lm[rt]));
                        const float al = m[rt] == mn ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - mn);
                        m[rt]          = mn;
                        l[rt] *= al;
#pragma unroll
                        for (int i = 0; i < 2 * NB; ++i) {
                            o[rt][i] *= al;
                        }
                    }
                }
                fa4_h8 ph[RT], pl[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const float mu = poff - (m[rt] == -INFINITY ? 0.0f : m[rt]);
                    float       p[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][e / 4][e % 4], fac[rt], mu));
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        ph[rt][e] = (_Float16) p[e];
                        if constexpr (OS) {
                            pl[rt][e] = (_Float16) (p[e] - (float) ph[rt][e]);
                        }
                    }
                    l[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph[rt], l[rt], 0, 0, 0);
                    if constexpr (OS) {
                        l[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[rt], l[rt], 0, 0, 0);
                    }
                }
                // lane m of a group of 16 addresses key m / 4 of the group's 4, positions 4 (m % 4)
                const char * vp = vl + (32 * kk + 4 * q4 + (c16 >> 2)) * F::VS + (c16 & 3) * 8;
#pragma unroll
                for (int dt = 0; dt < 2 * NB; ++dt) {
                    fa4_h8 v[F::VP];
#pragma unroll
                    for (int p = 0; p < F::VP; ++p) {
                        const fa4_v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((fa4_lds_v4s *) (vp + p * F::VB + dt * 32));
                        const fa4_v4s z = __builtin_amdgcn_ds_read_tr16_b64_v4i16((fa4_lds_v4s *) (vp + p * F::VB + dt * 32 + 16 * F::VS));
                        v[p] = __builtin_bit_cast(fa4_h8, __builtin_shufflevector(x, z, 0, 1, 2, 3, 4, 5, 6, 7));
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        fa4_f4 & oo = o[rt][dt];
                        oo          = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[0], ph[rt], oo, 0, 0, 0);
                        if constexpr (OS) {
                            oo = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[0], pl[rt], oo, 0, 0, 0);
                            oo = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[F::VP - 1], ph[rt], oo, 0, 0, 0);
                        }
                    }
                }
            }
            if (tn >= tend) {
                break;
            }
            tflag[bf][wv] = flags();
            __syncthreads();
            fl      = fn;
            t       = tn;
            tn      = t2;
            dirty   = dirty_n;
            dirty_n = dirty_2;
            bf ^= 1;
        }
    }

#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float lr = l[rt][0];
        const int   r  = r0 + (wv * RT + rt) * 16 + c16;
        if (r >= a.rows) {
            continue;
        }
        const int iq = r / a.rk, h = (int) g * a.rk + (r - iq * a.rk);
        if (a.splits > 1) {
            float * p = a.ws + (((int64_t) bg * a.rows + r) * a.splits + split) * (D + 4);
            if (q4 == 0) {
                p[0] = m[rt];
                p[1] = lr;
            }
#pragma unroll
            for (int dt = 0; dt < 2 * NB; ++dt) {
                const fa4_f4 v = o[rt][dt];
                *(float4 *) (p + 4 + dt * 16 + 4 * q4) = make_float4(v[0], v[2], v[1], v[3]);
            }
        } else {
            char *      yp  = a.y + (int64_t) b * a.y3 + (int64_t) iq * a.y2 + (int64_t) h * a.y1;
            const float inv = 1.0f / lr;  // no live key: 0 * inf
#pragma unroll
            for (int dt = 0; dt < 2 * NB; ++dt) {
                const fa4_f4 v  = o[rt][dt] * inv;
                const int    at = dt * 16 + 4 * q4;
                if constexpr (OS) {
                    *(fa4_f4u *) (yp + (size_t) at * 4) = fa4_f4u{ v[0], v[2], v[1], v[3] };
                } else {
                    *(fa4_u2u *) (yp + (size_t) at * 2) = fa4_u2u{ pack_bf16x2(v[0], v[2]), pack_bf16x2(v[1], v[3]) };
                }
            }
        }
    }
}

constexpr int FA4_W        = 4;   // waves per workgroup of the kernel for few rows

// rows and threads of a workgroup of the kernel for many rows
struct Fa4Wg {
    int rows, threads;
};

template <int D> static Fa4Wg fa4_wg(bool f32) {
    return f32 ? Fa4Wg{ Fa4P<D, true>::BQ, 64 * Fa4P<D, true>::W } : Fa4Wg{ Fa4P<D, false>::BQ, 64 * Fa4P<D, false>::W };
}

static Fa4Wg fa4_wg(int D, bool f32) {
    switch (D) {
        case 64:
            return fa4_wg<64>(f32);
        case 128:
            return fa4_wg<128>(f32);
        default:
            return fa4_wg<256>(f32);
    }
}

// up to this many splits are merged by a lane for 4 columns of a row, more by a workgroup for a row
constexpr int FA4_FEW_SPLITS = 8;

// workgroups of 256 threads that the merge of `rows` rows takes
static int64_t fa4_merge_wgs(int64_t rows, int64_t splits, int D) {
    return splits <= FA4_FEW_SPLITS ? (rows + 1024 / D - 1) / (1024 / D) : rows;
}

void flash_attn_q4_plan(FaArgs & a, int D) {
    a.rows    = a.n_q * a.rk;
    a.rblocks = (a.rows + 15) / 16;
    a.splits  = 1;
    a.ngq     = (a.n_q + 15) / 16;
    if (a.nb == 0 || a.rows == 0 || a.n_kv == 0) {
        return;
    }
    if (a.n_kv > 1 << 27 || a.k1 >= 1 << 25 || a.v1 >= 1 << 25) {
        a.splits = 0;  // keys are counted in 32 bits, 8 tiles of every wave ahead; a tile's offsets too
        return;
    }
    const Fa4Plan p     = fa4_plan((int64_t) a.nb * a.nkv, a.rows, a.n_kv, D, a.ty == MI_TYPE_F32, a.n_q == 1, num_cus());
    a.mfma              = p.many && a.ngq <= 65535 && (int64_t) a.nb * a.nh <= 65535;
    const int64_t tiles = ((int64_t) a.n_kv + 63) / 64 * (D == 256 ? 2 : 1);
    const int64_t least = a.mfma ? (tiles + FA4_PRE_TILES - 1) / FA4_PRE_TILES : 1;
    const Fa4Wg wg = a.mfma ? fa4_wg(D, a.ty == MI_TYPE_F32) : Fa4Wg{ 16, 64 * FA4_W };
    a.rblocks      = (a.rows + wg.rows - 1) / wg.rows;
    const int64_t items = (int64_t) a.nb * a.nkv * a.rblocks, all = (int64_t) a.nb * a.nkv * a.rows;
    int64_t       want  = p.many == (a.mfma != 0) ? p.splits : 1;
    want                = want < FA4_MAX_SPLITS ? want : FA4_MAX_SPLITS;
    a.splits = (int) (want < least ? least : want);
    // more than the merge takes, or than a launch: its threads are counted in 32 bits
    const int64_t most = ((int64_t) 1 << 32) - 1;
    if (a.splits > FA4_MAX_SPLITS || items * a.splits > most / wg.threads || all >= ((int64_t) 1 << 31) ||
        (a.splits > 1 && fa4_merge_wgs(all, a.splits, D) > most / 256)) {
        a.splits = 0;
    }
}

// partial results of split keys, then the mask's summary bytes (for the largest mask a call may pass)
static size_t fa4_parts(const FaArgs & a, int D) {
    const size_t n = a.splits > 1 ? (size_t) a.splits * a.nb * a.nkv * a.rows * (D + 4) * sizeof(float) : 0;
    return (n + 255) / 256 * 256;
}

size_t flash_attn_q4_workspace(const FaArgs & a, int D) {
    size_t need = 0;
    for (const int ty : { MI_TYPE_F32, MI_TYPE_BF16 }) {  // whatever y is: a caller asks before there is one
        FaArgs t = a;
        t.ty     = ty;
        flash_attn_q4_plan(t, D);
        const size_t n = fa4_parts(t, D) + (t.mfma ? (size_t) t.nb * t.nh * t.ngq * ((t.n_kv + 63) / 64) : 0);
        need           = n > need ? n : need;
    }
    return need;
}

template <int D, bool OS>
static void launch_dec(const FaArgs & a, hipStream_t s) {
    const dim3 grid((uint32_t) ((int64_t) a.nb * a.nkv * a.rblocks * a.splits)), wg(64 * FA4_W);
    if (a.mfma) {
        const dim3 wp(64 * Fa4P<D, OS>::W);
        if (a.mask && a.n_kv > 0) {
            FaArgs m = a;
            m.msum   = (uint8_t *) a.ws + fa4_parts(a, D);
            launch_fa_mask_summary(m, s);
            MI_LAUNCH((k_fa4_pre<D, OS, true>), grid, wp, 0, s, m);
        } else {
            MI_LAUNCH((k_fa4_pre<D, OS, false>), grid, wp, 0, s, a);
        }
    } else if (a.mask == nullptr) {
        MI_LAUNCH((k_fa4_dec<D, OS, 0, FA4_W>), grid, wg, 0, s, a);
    } else if (a.n_q == 1 && a.mne2 == 1) {
        MI_LAUNCH((k_fa4_dec<D, OS, 1, FA4_W>), grid, wg, 0, s, a);
    } else {
        MI_LAUNCH((k_fa4_dec<D, OS, 2, FA4_W>), grid, wg, 0, s, a);
    }
    if (a.splits > 1) {
        const dim3 grid_m((uint32_t) fa4_merge_wgs((int64_t) a.nb * a.nkv * a.rows, a.splits, D));
        if (a.splits <= 2) {
            MI_LAUNCH((k_fa4_combine_few<D, 2>), grid_m, dim3(256), 0, s, a);
        } else if (a.splits <= 4) {
            MI_LAUNCH((k_fa4_combine_few<D, 4>), grid_m, dim3(256), 0, s, a);
        } else if (a.splits <= FA4_FEW_SPLITS) {
            MI_LAUNCH((k_fa4_combine_few<D, FA4_FEW_SPLITS>), grid_m, dim3(256), 0, s, a);
        } else if (a.splits <= 2 * 1024 / D) {
            MI_LAUNCH((k_fa4_combine<D, 2>), grid_m, dim3(256), 0, s, a);
        } else {
            MI_LAUNCH((k_fa4_combine<D, 8>), grid_m, dim3(256), 0, s, a);
        }
    }
}

template <int D>
static int launch_d(const FaArgs & a, hipStream_t s) {
    if (a.ty == MI_TYPE_BF16) {
        launch_dec<D, false>(a, s);
    } else {
        launch_dec<D, true>(a, s);
    }
    return MI_OK;
}

int launch_flash_attn_q4(const FaArgs & a, int D, hipStream_t s) {
    if (a.rows == 0 || a.nb == 0 || a.nkv == 0) {
        return MI_OK;
    }
    switch (D) {
        case 64:
            return launch_d<64>(a, s);
        case 128:
            return launch_d<128>(a, s);
        default:
            return launch_d<256>(a, s);
    }
}

}  // namespace mi
