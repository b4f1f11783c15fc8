// lora.hip -- low-rank adapters of many requests beside a shared projection (mi_lora_add):
//
//   y_t = y0_t + scale[id_t] B[id_t] (A[id_t] x_t),   id_t < 0: y_t = y0_t
//
// Two launches: h = A x (k_lora_down, keys split over waves and workgroups, partial sums to
// the workspace), then y = y0 + B (scale h) (k_lora_up). Both run on v_mfma_f32_16x16x32_bf16
// over tiles of 16 rows of x. A tile's rows may have 16 adapters: a wave walks the distinct
// ones, multiplies the whole tile by each and keeps the rows that have it (by selection, not
// by zeros: weights that are not finite stay with their own rows).
//
// x, h and y are fp32. Their factors of the products are held as three bf16 parts (24 bits),
// BF16 weights as they are, F16 weights as two exact bf16 parts: three or five products keep
// everything but 2^-24 of each term, at matrix-core rates that stay far above what the loads need.
// The parts of an infinity, and of an x that rounds past bf16's largest, multiply to NaN. So where a
// product's result is not finite the wave repeats it in fp32 (v_mfma_f32_16x16x4_f32) and takes those
// elements from there: they are what fp32 operations give, and every other element keeps its bits.
#include "launch.h"
#include "rules.h"

namespace mi {

typedef __bf16 lr_b8 __attribute__((ext_vector_type(8)));
typedef float  lr_f4 __attribute__((ext_vector_type(4)));
typedef float  lr_f4a __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t lr_u4a __attribute__((ext_vector_type(4), aligned(2)));

struct LrSplit {
    lr_b8 p[3];
};

__device__ __forceinline__ LrSplit lr_split(const float * x) {
    LrSplit s;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const __bf16 a = (__bf16) x[e];
        const float  r = x[e] - (float) a;
        const __bf16 b = (__bf16) r;
        s.p[0][e]      = a;
        s.p[1][e]      = b;
        s.p[2][e]      = (__bf16) (r - (float) b);
    }
    return s;
}

// whether some lane of the wave has a value that is not finite in c
template <typename V> __device__ __forceinline__ bool lr_bad(const V * c, int n) {
    constexpr int E = sizeof(V) / 4;
    float         t[4] = {};
#pragma unroll
    for (int i = 0; i < n; ++i) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            t[(i * E + e) % 4] = __builtin_fmaf(c[i][e], 0.0f, t[(i * E + e) % 4]);
        }
    }
    const float z = (t[0] + t[1]) + (t[2] + t[3]);  // 0 or NaN
    return __builtin_expect(__builtin_amdgcn_ballot_w64(z != z) != 0, false);
}

// v, for the compiler another value: what is derived from it is not kept from before
__device__ __forceinline__ int lr_again(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// the product of 8 elements of x a lane with 8 weights, in fp32
__device__ __forceinline__ lr_f4 lr_mul32(const float * x, const float * w, lr_f4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], w[e], c, 0, 0, 0);
    }
    return c;
}

// 8 weights as one or two bf16 parts
template <int WT> struct LrW;
template <> struct LrW<MI_TYPE_BF16> {
    uint4                           raw;
    lr_b8                           p;
    __device__ __forceinline__ void split() { p = __builtin_bit_cast(lr_b8, raw); }
    __device__ __forceinline__ lr_f4 mul(const LrSplit & x, lr_f4 c) const {
#pragma unroll
        for (int i = 2; i >= 0; --i) {
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.p[i], p, c, 0, 0, 0);
        }
        return c;
    }
};
template <> struct LrW<MI_TYPE_F16> {
    uint4                           raw;
    lr_b8                           hi, lo;
    __device__ __forceinline__ void split() {
        float f[8];
        unpack16<MI_TYPE_F16>(raw, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            hi[e] = (__bf16) f[e];
            lo[e] = (__bf16) (f[e] - (float) hi[e]);  // 11 significant bits less 8: exact
        }
    }
    __device__ __forceinline__ lr_f4 mul(const LrSplit & x, lr_f4 c) const {
#pragma unroll
        for (int i = 2; i >= 0; --i) {
            if (i < 2) {
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.p[i], lo, c, 0, 0, 0);
            }
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.p[i], hi, c, 0, 0, 0);
        }
        return c;
    }
};

// the adapter of row t of x: -1 for none (also for an id that names none)
__device__ __forceinline__ int32_t lr_id(const LoraArgs & a, uint32_t t) {
    if (t >= a.m) {
        return -1;
    }
    const int32_t id = *(const int32_t *) (a.ids + (int64_t) t * a.i0);
    return id < 0 || id >= a.n_ad ? -1 : id;
}

// h = A x. What bounds it: x once (4005 rows of 2560 at rank 32 16.2 us, 2.5 TB/s of x and the shares), or with few
// rows the chain of ids, weights, products and the sum in LDS (8 rows at rank 16 3.3 us, 48 rows of 24
// adapters at rank 64 from 4096 keys 7.4 us). A workgroup: 16 rows of x (blockIdx.x), one of a.ks shares of the keys (y), rank
// block of 16 NR and every a.slots-th distinct adapter of the tile (z). Its 4 waves take
// alternate steps of 32 keys and are summed in LDS. Five waves a SIMD for 4 rank blocks: left to itself the
// kernel takes registers for its fp32 repeat and runs four (4000 x 2560 at rank 64, 8 adapters in turn, both
// products 271 us instead of 236).
template <int WT, int NR>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NR == 4 ? 5 : 1))) k_lora_down(const LoraArgs a) {
    __shared__ lr_f4 part[3][NR][64];
    const int      lane = threadIdx.x & 63, c16 = lane & 15, q4 = lane >> 4;
    const int      wv   = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t t0   = blockIdx.x * 16;
    const uint32_t rb   = blockIdx.z / a.slots, slot = blockIdx.z - rb * a.slots;
    const int32_t  id   = lr_id(a, t0 + c16);  // of this lane's row of x
    if (blockIdx.y == 0 && blockIdx.z == 0 && wv == 0 && q4 == 0 && t0 + c16 < a.m && a.d_err &&
        *(const int32_t *) (a.ids + (int64_t) (t0 + c16) * a.i0) >= a.n_ad) {
        atomicAdd(a.d_err, 1);
    }
    const uint32_t tr  = t0 + c16 < a.m ? t0 + c16 : a.m - 1;
    const char *   xp  = a.x + (int64_t) tr * a.x1 + q4 * 32;
    const uint32_t s0  = blockIdx.y * a.kstep, s1 = s0 + a.kstep < a.k / 32 ? s0 + a.kstep : a.k / 32;
    uint64_t       todo = __builtin_amdgcn_ballot_w64(id >= 0) & 0xffffu;
    for (uint32_t j = 0; todo; ++j) {
        const int32_t  cur  = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        const uint64_t mine = __builtin_amdgcn_ballot_w64(id == cur) & 0xffffu;
        todo &= ~mine;
        if (j % a.slots != slot) {
            continue;
        }
        const char * wp[NR];
        lr_f4        c[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const uint32_t r = (rb * NR + i) * 16 + c16;  // past the rank: the last row again, never used
            wp[i] = a.a + (int64_t) cur * a.a2 + (int64_t) (r < a.r ? r : a.r - 1) * a.a1 + q4 * 16;
            c[i]  = lr_f4{ 0.0f, 0.0f, 0.0f, 0.0f };
        }
        for (uint32_t s = s0 + wv; s < s1; s += 4) {
            const lr_f4a x0 = *(const lr_f4a *) (xp + (int64_t) s * 128);
            const lr_f4a x1 = *(const lr_f4a *) (xp + (int64_t) s * 128 + 16);
            const float  xv[8] = { x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w };
            LrW<WT>      w[NR];
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const lr_u4a v = *(const lr_u4a *) (wp[i] + (int64_t) s * 64);
                w[i].raw = make_uint4(v.x, v.y, v.z, v.w);
            }
            const LrSplit xs = lr_split(xv);
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                w[i].split();
                c[i] = w[i].mul(xs, c[i]);
            }
        }
        if (lr_bad(c, NR)) {
            const int      l  = lr_again(lane);  // addresses made anew: no register holds them across the loop above
            const uint32_t tt = t0 + (l & 15) < a.m ? t0 + (l & 15) : a.m - 1;
            const char *   xb = a.x + (int64_t) tt * a.x1 + (l >> 4) * 32;
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const uint32_t r  = (rb * NR + i) * 16 + (l & 15);
                const char *   wb = a.a + (int64_t) cur * a.a2 + (int64_t) (r < a.r ? r : a.r - 1) * a.a1 + (l >> 4) * 16;
                lr_f4          f  = { 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll 1
                for (uint32_t s = s0 + wv; s < s1; s += 4) {
                    const lr_f4a x0 = *(const lr_f4a *) (xb + (int64_t) s * 128);
                    const lr_f4a x1 = *(const lr_f4a *) (xb + (int64_t) s * 128 + 16);
                    const float  xv[8] = { x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w };
                    const lr_u4a v = *(const lr_u4a *) (wb + (int64_t) s * 64);
                    float        wf[8];
                    unpack16<WT>(make_uint4(v.x, v.y, v.z, v.w), wf);
                    f = lr_mul32(xv, wf, f);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    c[i][e] = __builtin_isfinite(c[i][e]) ? c[i][e] : f[e];
                }
                __builtin_amdgcn_sched_barrier(0);  // one at a time: few registers
            }
        }
        __syncthreads();  // the previous adapter's sums are read
        if (wv > 0) {
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                part[wv - 1][i][lane] = c[i];
            }
        }
        __syncthreads();
        if (wv == 0) {
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                if ((rb * NR + i) * 16 >= a.rp) {
                    break;  // the last rank block's columns past the rank
                }
                const lr_f4 v = (c[i] + part[0][i][lane]) + (part[1][i][lane] + part[2][i][lane]);
                // lane: rank column c16, rows 4 q4 + e of the tile
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (mine >> (4 * q4 + e) & 1) {
                        a.h[((int64_t) blockIdx.y * a.m + t0 + 4 * q4 + e) * a.rp + (rb * NR + i) * 16 + c16] = v[e];
                    }
                }
            }
        }
    }
}

// y = y0 + B (scale h). A workgroup: 16 TT rows of x (blockIdx.x) and every gridDim.y-th block of
// 64 NT columns of y, a wave 16 NT of them. h is summed over the key shares, scaled and split
// once, into LDS; a block's y0 is loaded under the block before it. Many rows: memory bounds it
// (4005 x 19456 at rank 32 136 us, 4.6 TB/s of y0 and y). RS: steps of 32 ranks; U:
// adapters whose weights are loaded before the first is multiplied. With NT 1 (few rows) the distinct
// adapters of the tile are shared out over gridDim.z workgroups, each storing the rows of its own
// (and the first those without one): a row has one adapter, so there is nothing to sum.
// Column c of product i is column NT c + i of the wave's: a lane holds NT consecutive columns of
// 4 rows, and with NT 4 a load or store of y covers 256 consecutive bytes of a row (products of
// 16 consecutive columns each: 64, and 167 us instead of 138 for 4005 x 19456 at rank 32).
// The waves a SIMD are those that the registers of the product alone allow. The check for values that are
// not finite is one fma an element of y, once for all adapters of a tile (1 % at most; once for each: 6 % with 24).
template <int WT, int NT, int TT, int RS, int U>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NT == 4 ? 2 : RS == 1 ? 5 : RS == 4 ? 3 : 4))) k_lora_up(const LoraArgs a) {
    static_assert(NT == 1 || NT == 4, "a dword or a float4 of y per lane and row");
    constexpr int RQ = RS * 32 + 8;  // row of h in LDS: 16 rows on distinct banks
    constexpr int R  = 16 * TT;
    typedef float lr_y __attribute__((ext_vector_type(NT), aligned(4)));
    __shared__ __align__(16) __bf16 hs[3 * R * RQ];
    const int      lane = threadIdx.x & 63, c16 = lane & 15, q4 = lane >> 4;
    const int      wv   = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t t0   = blockIdx.x * R;
    const int32_t  idl  = lr_id(a, t0 + (lane < R ? lane : R));  // lanes 0 .. R - 1: the rows' adapters
    uint64_t       rows = __builtin_amdgcn_ballot_w64(idl >= 0 && lane < R), own = ~0ull;  // with an adapter; to be stored
    if constexpr (NT == 1) {
        own = blockIdx.z == 0 ? ~rows : 0;
        uint64_t left = rows;
        for (uint32_t j = 0; left; j = j + 1 < gridDim.z ? j + 1 : 0) {
            const uint64_t mine = __builtin_amdgcn_ballot_w64(idl == __builtin_amdgcn_readlane(idl, __builtin_ctzll(left)));
            left &= ~mine;
            own |= j == blockIdx.z ? mine : 0;
        }
        own &= t0 + R <= a.m ? (1ull << R) - 1 : (1ull << (a.m - t0)) - 1;
        rows &= own;
        if (own == 0) {
            return;  // the whole workgroup
        }
    }
    int32_t        id[TT][4];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            id[tt][e] = __shfl(idl, tt * 16 + 4 * q4 + e, 64);
        }
    }
    // element (row tt * 16 + 4 q4 + e, columns n ..); rows past the last: the last one again
    auto row = [&](int tt, int e) -> int64_t {
        const uint32_t t = t0 + tt * 16 + 4 * q4 + e;
        return t < a.m ? t : a.m - 1;
    };
    lr_y acc[TT][4], nxt[TT][4];
    auto load = [&](uint32_t n0) {  // columns past the last: the last ones again
        const uint32_t n = n0 + NT * c16;
        const int64_t  c = (int64_t) (n + NT <= a.n ? n : a.n - NT) * 4;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                nxt[tt][e] = *(const lr_y *) (a.y0 + row(tt, e) * a.y01 + c);
            }
        }
    };
    uint32_t n0 = (blockIdx.y * 4 + wv) * (16 * NT);
    load(n0);
    // G elements a thread and 16 key shares of each in flight
    constexpr int E = R * RS * 32 / 256, G = E < 4 ? E : 4;
    for (int i0 = threadIdx.x; i0 < R * RS * 32; i0 += 256 * G) {
        const float * hp[G];
        bool          on[G], any = false;
        float         sc[G], v[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int      i = i0 + 256 * g, t = i / (RS * 32), r = i - t * RS * 32;
            const int32_t  it = __shfl(idl, t, 64);
            const uint32_t tr = t0 + t < a.m ? t0 + t : a.m - 1;
            on[g] = it >= 0 && r < (int) a.r && (NT != 1 || own >> t & 1);
            any   = any || on[g];
            hp[g] = a.h + (int64_t) tr * a.rp + (r < (int) a.r ? r : 0);
            sc[g] = a.scales && on[g] ? *(const float *) (a.scales + (int64_t) it * a.s0) : 1.0f;
            v[g]  = 0.0f;
        }
        const int64_t st = (int64_t) a.m * a.rp;
        for (uint32_t s = 0; any && s < a.ks; s += 16) {
            float p[G][16];
#pragma unroll
            for (int g = 0; g < G; ++g) {
#pragma unroll
                for (int q = 0; q < 16; ++q) {  // past the last share: it again; rows without an adapter hold anything
                    p[g][q] = hp[g][(s + q < a.ks ? s + q : a.ks - 1) * st];
                }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    v[g] += s + q < a.ks ? p[g][q] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int    i = i0 + 256 * g, t = i / (RS * 32), r = i - t * RS * 32;
            const float  x = on[g] ? v[g] * sc[g] : 0.0f;
            // a finite x stays finite in its first part: no larger than bf16's largest
            const __bf16 x0 = (__bf16) (__builtin_isfinite(x) ? __builtin_amdgcn_fmed3f(x, -0x1.fep127f, 0x1.fep127f) : x);
            const float  r0 = x - (float) x0;
            const __bf16 x1 = (__bf16) r0;
            hs[t * RQ + r]           = x0;
            hs[(R + t) * RQ + r]     = x1;
            hs[(2 * R + t) * RQ + r] = (__bf16) (r0 - (float) x1);
        }
    }
    __syncthreads();
    const bool vec = a.r % 8 == 0;
    // 8 ranks from 32 s + 8 q4 on of a column of B; past the rank: zeros
    auto weights = [&](const char * p, int s) -> uint4 {
        const int r0 = s * 32 + 8 * q4;
        uint4     v  = make_uint4(0, 0, 0, 0);
        if (r0 + 8 <= (int) a.r) {
            const lr_u4a x = *(const lr_u4a *) (p + s * 64);
            v              = make_uint4(x.x, x.y, x.z, x.w);
        } else if (!vec && r0 < (int) a.r) {
            uint16_t x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = r0 + e < (int) a.r ? *(const uint16_t *) (p + s * 64 + e * 2) : 0;
            }
            v = make_uint4(x[0] | (uint32_t) x[1] << 16, x[2] | (uint32_t) x[3] << 16, x[4] | (uint32_t) x[5] << 16,
                           x[6] | (uint32_t) x[7] << 16);
        }
        return v;
    };
    // The elements of y named in `left` (bit (tt * 4 + e) NT + i), which hold y0: the product in fp32 is added.
    auto repeat = [&](uint32_t nb, uint32_t left) {
        uint64_t todo = rows;
        while (todo) {
            const int32_t cur = __builtin_amdgcn_readlane(idl, __builtin_ctzll(todo));
            todo &= ~__builtin_amdgcn_ballot_w64(idl == cur);
#pragma unroll 1
            for (int ti = 0; ti < TT * NT; ++ti) {
                const int      l = lr_again(lane), tt = ti / NT, i = ti - tt * NT;
                const uint32_t n = nb + NT * (l & 15) + i < a.n ? nb + NT * (l & 15) + i : a.n - 1;
                const char *   p = a.b + (int64_t) cur * a.b2 + (l >> 4) * 16 + (int64_t) n * a.b1;
                lr_f4          f = { 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll 1
                for (int s = 0; s < RS; ++s) {
                    const __bf16 * hp = hs + (tt * 16 + (l & 15)) * RQ + s * 32 + 8 * (l >> 4);
                    float          h[8], w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {  // an infinity's other parts are NaN
                        const float h0 = (float) hp[e], h1 = (float) hp[R * RQ + e] + (float) hp[2 * R * RQ + e];
                        h[e]           = __builtin_isinf(h0) ? h0 : h0 + h1;
                    }
                    unpack16<WT>(weights(p, s), w);
                    f = lr_mul32(h, w, f);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int     r  = tt * 16 + 4 * (l >> 4) + e;
                    const int32_t it = __shfl(idl, r, 64);
                    if (it == cur && left >> ((tt * 4 + e) * NT + i) & 1) {
                        float * yp = (float *) (a.y + (int64_t) (t0 + r) * a.y1 + (int64_t) n * 4);
                        *yp        = *yp + f[e];
                    }
                }
            }
        }
    };
    for (; n0 < a.n; n0 += gridDim.y * (64 * NT)) {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[tt][e] = nxt[tt][e];
            }
        }
        load(n0 + gridDim.y * (64 * NT));
        uint64_t todo = rows;
        while (todo) {
            int32_t cur[U];
            LrW<WT> w[U][RS][NT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                cur[u] = -2;  // no row's
                if (todo) {
                    cur[u] = __builtin_amdgcn_readlane(idl, __builtin_ctzll(todo));
                    todo &= ~__builtin_amdgcn_ballot_w64(idl == cur[u]);
                    const char * bp = a.b + (int64_t) cur[u] * a.b2 + q4 * 16;
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        const uint32_t n = n0 + NT * c16 + i;
                        const char *   p = bp + (int64_t) (n < a.n ? n : a.n - 1) * a.b1;
#pragma unroll
                        for (int s = 0; s < RS; ++s) {
                            w[u][s][i].raw = weights(p, s);
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (cur[u] == -2) {
                    break;
                }
                lr_f4 c[TT][NT] = {};
#pragma unroll
                for (int s = 0; s < RS; ++s) {
                    LrSplit h[TT];
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
                        for (int p = 0; p < 3; ++p) {
                            h[tt].p[p] = *(const lr_b8 *) (hs + (R * p + tt * 16 + c16) * RQ + s * 32 + 8 * q4);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        w[u][s][i].split();
#pragma unroll
                        for (int tt = 0; tt < TT; ++tt) {
                            c[tt][i] = w[u][s][i].mul(h[tt], c[tt][i]);
                        }
                    }
                }
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool mine = id[tt][e] == cur[u];
#pragma unroll
                        for (int i = 0; i < NT; ++i) {
                            acc[tt][e][i] = mine ? acc[tt][e][i] + c[tt][i][e] : acc[tt][e][i];
                        }
                    }
                }
            }
        }
        const uint32_t n = n0 + NT * c16;
        const bool     in  = n + NT <= a.n;
        const bool     bad = lr_bad(acc[0], TT * 4);
        uint32_t       left = 0;
        auto           mine = [&](int tt, int e) { return in && (NT == 1 ? own >> (4 * q4 + e) & 1 : t0 + tt * 16 + 4 * q4 + e < a.m); };
        if (bad) {
            const int      l = lr_again(lane);
            const uint32_t nn = n0 + NT * (l & 15);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t t  = t0 + tt * 16 + 4 * (l >> 4) + e;
                    const lr_y     y0 = *(const lr_y *) (a.y0 + (int64_t) (t < a.m ? t : a.m - 1) * a.y01 + (int64_t) (nn + NT <= a.n ? nn : a.n - NT) * 4);
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        if (!__builtin_isfinite(acc[tt][e][i])) {
                            left |= (mine(tt, e) ? 1u : 0u) << ((tt * 4 + e) * NT + i);
                            acc[tt][e][i] = y0[i];
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);  // few registers
                }
            }
        }
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (mine(tt, e)) {
                    *(lr_y *) (a.y + row(tt, e) * a.y1 + (int64_t) n * 4) = acc[tt][e];
                }
            }
        }
        if (bad) {
            repeat(n0, left);
        }
    }
}

// The columns past the last whole 4 (at most 3): a thread each, in fp32, the ranks in order.
__global__ void __launch_bounds__(256) k_lora_up_rest(const LoraArgs a, int f16) {
    const uint32_t left = a.n & 3u, i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.m * left) {
        return;
    }
    const uint32_t t = i / left, n = a.n - left + (i - t * left);
    const int32_t  id = lr_id(a, t);
    float          v  = *(const float *) (a.y0 + (int64_t) t * a.y01 + (int64_t) n * 4);
    if (id >= 0) {
        const char * bp = a.b + (int64_t) id * a.b2 + (int64_t) n * a.b1;
        float        c  = 0.0f;
        for (uint32_t r = 0; r < a.r; ++r) {
            float h = 0.0f;
            for (uint32_t s = 0; s < a.ks; ++s) {
                h += a.h[((int64_t) s * a.m + t) * a.rp + r];
            }
            c = __builtin_fmaf(h, f16 ? load_elem<MI_TYPE_F16>(bp + r * 2) : load_elem<MI_TYPE_BF16>(bp + r * 2), c);
        }
        v += c * (a.scales ? *(const float *) (a.scales + (int64_t) id * a.s0) : 1.0f);
    }
    *(float *) (a.y + (int64_t) t * a.y1 + (int64_t) n * 4) = v;
}

void lora_plan(LoraArgs & a) {
    a.rp                 = (a.r + 15) / 16 * 16;
    const uint32_t tiles = (a.m + 15) / 16, steps = a.k / 32;
    // key shares: workgroups for 4 per CU, a share of at least 8 steps (2 a wave)
    uint32_t ks = (uint32_t) (((uint64_t) num_cus() * 4 + tiles - 1) / (tiles ? tiles : 1));
    ks          = ks < 1 ? 1 : ks;
    a.kstep     = (steps + ks - 1) / ks;
    a.kstep     = a.kstep < 8 ? 8 : a.kstep;
    a.ks        = (steps + a.kstep - 1) / a.kstep;
    // rows of one tile can have 16 adapters: a workgroup each where few workgroups run
    a.slots = tiles * a.ks >= (uint32_t) num_cus() ? 1 : a.n_ad < 16 ? (uint32_t) (a.n_ad > 0 ? a.n_ad : 1) : 16;
    a.slots = a.slots > a.m && a.m > 0 ? a.m : a.slots;
}

size_t lora_workspace(const LoraArgs & a) {
    return (size_t) a.ks * a.m * a.rp * sizeof(float);
}

template <int WT, int NR> static void launch_down(const LoraArgs & a, hipStream_t s) {
    const uint32_t blocks = (a.rp + 16 * NR - 1) / (16 * NR);
    MI_LAUNCH((k_lora_down<WT, NR>), dim3((a.m + 15) / 16, a.ks, blocks * a.slots), dim3(256), 0, s, a);
}

template <int WT, int RS> static void launch_up(const LoraArgs & a, hipStream_t s) {
    if (lora_wide(a.m, a.n)) {
        // rows in tiles of 32 (16 at high ranks), column blocks of 256 over enough workgroups for 6 per CU: within 3 % of
        // the best at each size (both products, us, for 3 / 4 / 6 / 8 / 12: 4005 x 19456 155.4 / 158.2 / 153.0 / 154.9 / 156.6;
        // 793 x 19456 41.3 / 40.7 / 41.9 / 43.5 / 43.4; 1500 x 19456 65.2 / 62.2 / 63.0 / 63.1 / 65.4)
        constexpr int  TT    = RS < 8 ? 2 : 1;
        const uint32_t tiles = (a.m + 16 * TT - 1) / (16 * TT), blocks = (a.n + 255) / 256;
        const uint32_t want  = ((uint32_t) num_cus() * 6 + tiles - 1) / tiles;
        MI_LAUNCH((k_lora_up<WT, 4, TT, RS, 1>), dim3(tiles, want < blocks ? want : blocks), dim3(256), 0, s, a);
    } else {
        // the adapters of a tile over enough workgroups for 2 per CU (48 rows of 24 adapters, 2560
        // columns at rank 64, both launches: 1 workgroup 20.4 us, for 1 per CU 17.4, 2 16.9, 4 18.7, 8 19.7)
        const uint32_t wgs = (a.m + 15) / 16 * ((a.n + 63) / 64), most = a.n_ad < 16 ? (uint32_t) a.n_ad : 16;
        uint32_t       z   = ((uint32_t) num_cus() * 2 + wgs - 1) / wgs;
        z                  = z < most ? z : most;
        z                  = z < a.m ? z : a.m;
        MI_LAUNCH((k_lora_up<WT, 1, 1, RS, RS < 4 ? 4 : RS < 8 ? 2 : 1>), dim3((a.m + 15) / 16, (a.n + 63) / 64, z > 1 ? z : 1),
                  dim3(256), 0, s, a);
    }
}

template <int WT> static void launch_w(const LoraArgs & a, hipStream_t s) {
    if (a.rp <= 16) {
        launch_down<WT, 1>(a, s);
    } else if (a.rp <= 32) {
        launch_down<WT, 2>(a, s);
    } else {
        launch_down<WT, 4>(a, s);
    }
    if (!dry_run() && hipPeekAtLastError() != hipSuccess) {
        return;  // y, which may be y0, stays as it is: there is no A x to add
    }
    switch ((a.r + 31) / 32) {
        case 1: launch_up<WT, 1>(a, s); break;
        case 2: launch_up<WT, 2>(a, s); break;
        case 3:
        case 4: launch_up<WT, 4>(a, s); break;
        default: launch_up<WT, 8>(a, s); break;
    }
    if (lora_wide(a.m, a.n) && a.n % 4 != 0) {
        MI_LAUNCH(k_lora_up_rest, dim3((uint32_t) (((uint64_t) a.m * (a.n & 3u) + 255) / 256)), dim3(256), 0, s, a,
                  WT == MI_TYPE_F16 ? 1 : 0);
    }
}

int launch_lora(const LoraArgs & a, int type, hipStream_t s) {
    if (type == MI_TYPE_BF16) {
        launch_w<MI_TYPE_BF16>(a, s);
    } else {
        launch_w<MI_TYPE_F16>(a, s);
    }
    return MI_OK;
}

}  // namespace mi
