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
#include "launch.h"

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

// 8 weights as one or two bf16 parts
template <int WT> struct LrW;
template <> struct LrW<MI_TYPE_BF16> {
    lr_b8                           p;
    __device__ __forceinline__ void set(const uint4 & v) { p = __builtin_bit_cast(lr_b8, v); }
    __device__ __forceinline__ lr_f4 mul(const LrSplit & x, lr_f4 c, bool first) const {
        // weights as A, x as B, or the other way round
#pragma unroll
        for (int i = 2; i >= 0; --i) {
            c = first ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, x.p[i], c, 0, 0, 0)
                      : __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.p[i], p, c, 0, 0, 0);
        }
        return c;
    }
};
template <> struct LrW<MI_TYPE_F16> {
    lr_b8                           hi, lo;
    __device__ __forceinline__ void set(const uint4 & v) {
        float f[8];
        unpack16<MI_TYPE_F16>(v, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            hi[e] = (__bf16) f[e];
            lo[e] = (__bf16) (f[e] - (float) hi[e]);  // 11 significant bits less 8: exact
        }
    }
    __device__ __forceinline__ lr_f4 mul(const LrSplit & x, lr_f4 c, bool first) const {
#pragma unroll
        for (int i = 2; i >= 0; --i) {
            if (i < 2) {
                c = first ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, x.p[i], c, 0, 0, 0)
                          : __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.p[i], lo, c, 0, 0, 0);
            }
            c = first ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, x.p[i], c, 0, 0, 0)
                      : __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.p[i], hi, c, 0, 0, 0);
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

// h = A x. A workgroup: 16 rows of x (blockIdx.x), one of a.ks shares of the keys (y), rank
// block of 16 NR and every a.slots-th distinct adapter of the tile (z). Its 4 waves take
// alternate steps of 32 keys and are summed in LDS.
template <int WT, int NR>
__global__ void __launch_bounds__(256) k_lora_down(const LoraArgs a) {
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
                w[i].set(make_uint4(v.x, v.y, v.z, v.w));
            }
            const LrSplit xs = lr_split(xv);
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                c[i] = w[i].mul(xs, c[i], false);
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

// y = y0 + B (scale h). A workgroup: 16 rows of x (blockIdx.x) and 64 NT columns of y (y); a
// wave 16 NT of them. h is summed over the key shares, scaled and split once, into LDS.
template <int WT, int NT>
__global__ void __launch_bounds__(256) k_lora_up(const LoraArgs a) {
    extern __shared__ __align__(16) __bf16 hs[];  // [3][16][rq], rq = rank padded to 32, + 8
    const int      lane = threadIdx.x & 63, c16 = lane & 15, q4 = lane >> 4;
    const int      wv   = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t t0   = blockIdx.x * 16;
    const int      rk32 = (int) ((a.r + 31) / 32), rq = rk32 * 32 + 8;
    const int32_t  id   = lr_id(a, t0 + c16);
    for (int i = threadIdx.x; i < 16 * rk32 * 32; i += 256) {
        const int      t = i / (rk32 * 32), r = i - t * rk32 * 32;
        const int32_t  it = lr_id(a, t0 + t);
        float          v  = 0.0f;
        if (it >= 0 && r < (int) a.r) {
            for (uint32_t s = 0; s < a.ks; ++s) {
                v += a.h[((int64_t) s * a.m + t0 + t) * a.rp + r];
            }
            v *= a.scales ? *(const float *) (a.scales + (int64_t) it * a.s0) : 1.0f;
        }
        const __bf16 p0 = (__bf16) v;
        const float  r0 = v - (float) p0;
        const __bf16 p1 = (__bf16) r0;
        hs[t * rq + r]                = p0;
        hs[(16 + t) * rq + r]         = p1;
        hs[(32 + t) * rq + r]         = (__bf16) (r0 - (float) p1);
    }
    __syncthreads();
    const uint32_t n0 = (blockIdx.y * 4 + wv) * (16 * NT);
    if (n0 >= a.n) {
        return;
    }
    const uint32_t tr = t0 + c16 < a.m ? t0 + c16 : a.m - 1;
    const char *   y0 = a.y0 + (int64_t) tr * a.y01;
    lr_f4          acc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const uint32_t n = n0 + 16 * i + 4 * q4;
        if (n + 4 <= a.n) {
            acc[i] = *(const lr_f4a *) (y0 + (int64_t) n * 4);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[i][e] = n + e < a.n ? *(const float *) (y0 + (int64_t) (n + e) * 4) : 0.0f;
            }
        }
    }
    uint64_t todo = __builtin_amdgcn_ballot_w64(id >= 0) & 0xffffu;
    while (todo) {
        const int32_t  cur  = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        const uint64_t mine = __builtin_amdgcn_ballot_w64(id == cur) & 0xffffu;
        todo &= ~mine;
        const char * bp[NT];
        lr_f4        c[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint32_t n = n0 + 16 * i + c16;
            bp[i] = a.b + (int64_t) cur * a.b2 + (int64_t) (n < a.n ? n : a.n - 1) * a.b1;
            c[i]  = lr_f4{ 0.0f, 0.0f, 0.0f, 0.0f };
        }
        for (int s = 0; s < rk32; ++s) {
            LrSplit h;
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                h.p[p] = *(const lr_b8 *) (hs + (16 * p + c16) * rq + s * 32 + 8 * q4);
            }
            const int r0 = s * 32 + 8 * q4;
            LrW<WT>   w[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (r0 + 8 <= (int) a.r) {
                    const lr_u4a x = *(const lr_u4a *) (bp[i] + r0 * 2);
                    v              = make_uint4(x.x, x.y, x.z, x.w);
                } else if (r0 < (int) a.r) {
                    uint16_t x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[e] = r0 + e < (int) a.r ? *(const uint16_t *) (bp[i] + (r0 + e) * 2) : 0;
                    }
                    v = make_uint4(x[0] | (uint32_t) x[1] << 16, x[2] | (uint32_t) x[3] << 16,
                                   x[4] | (uint32_t) x[5] << 16, x[6] | (uint32_t) x[7] << 16);
                }
                w[i].set(v);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                c[i] = w[i].mul(h, c[i], true);
            }
        }
        if (id == cur) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                acc[i] += c[i];
            }
        }
    }
    if (t0 + c16 >= a.m) {
        return;
    }
    char * y = a.y + (int64_t) tr * a.y1;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const uint32_t n = n0 + 16 * i + 4 * q4;
        if (n + 4 <= a.n) {
            *(lr_f4a *) (y + (int64_t) n * 4) = acc[i];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (n + e < a.n) {
                    *(float *) (y + (int64_t) (n + e) * 4) = acc[i][e];
                }
            }
        }
    }
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

template <int WT> static void launch_w(const LoraArgs & a, hipStream_t s) {
    if (a.rp <= 16) {
        launch_down<WT, 1>(a, s);
    } else if (a.rp <= 32) {
        launch_down<WT, 2>(a, s);
    } else {
        launch_down<WT, 4>(a, s);
    }
    const size_t lb = (size_t) 48 * ((a.r + 31) / 32 * 32 + 8) * 2;
    MI_LAUNCH((k_lora_up<WT, 4>), dim3((a.m + 15) / 16, (a.n + 255) / 256), dim3(256), lb, s, a);
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
