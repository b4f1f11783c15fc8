// logits.hip -- what is done to a row of logits before a token is drawn (mi_logits_adjust):
// penalties for tokens of the row's history, a bias, a grammar's mask.
//
//   c  = times the token is in the history
//   l' = c == 0 ? l : (l > 0 ? l / rep : l * rep) - c freq - pres,  + bias,  -inf where not allowed
//
// A workgroup takes a tile of LG_TILE tokens of one row: its logits are loaded first, then the
// whole history is read and the tokens that fall into the tile are counted in LDS (integer
// atomics: their order does not show), then the tile is written. So one launch needs no
// memory but LDS; the history is read once a tile, from the cache.
#include "launch.h"

namespace mi {

constexpr int LG_TILE = 8192;  // tokens per workgroup

// rows of any vocabulary size: 16 bytes at the element's own alignment
typedef uint32_t lg_u4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t lg_u4a2 __attribute__((ext_vector_type(4), aligned(2)));

template <int T> __device__ __forceinline__ void lg_load(const char * p, float * f) {
    if constexpr (T == MI_TYPE_F32) {
        const lg_u4a4 v = __builtin_nontemporal_load((const lg_u4a4 *) p);
        unpack16<T>(make_uint4(v.x, v.y, v.z, v.w), f);
    } else {
        const lg_u4a2 v = __builtin_nontemporal_load((const lg_u4a2 *) p);
        unpack16<T>(make_uint4(v.x, v.y, v.z, v.w), f);
    }
}

template <int T> __device__ __forceinline__ void lg_store(char * p, const float * f) {
    const uint4 w = pack16<T>(f);
    if constexpr (T == MI_TYPE_F32) {
        const lg_u4a4 v = { w.x, w.y, w.z, w.w };
        __builtin_nontemporal_store(v, (lg_u4a4 *) p);
    } else {
        const lg_u4a2 v = { w.x, w.y, w.z, w.w };
        __builtin_nontemporal_store(v, (lg_u4a2 *) p);
    }
}

template <int T, bool HIST>
__global__ void __launch_bounds__(256) k_logits(const LogitsArgs a) {
    constexpr int VEC   = TT<T>::VEC;
    constexpr int ES    = TT<T>::ES;
    constexpr int STEPS = LG_TILE / (256 * VEC);
    __shared__ uint32_t count[HIST ? LG_TILE : 1];
    const int      tid = threadIdx.x;
    const uint32_t row = blockIdx.y;
    const int64_t  v0  = (int64_t) blockIdx.x * LG_TILE;
    const char *   xp  = a.x + (int64_t) row * a.x1;
    char *         yp  = a.y + (int64_t) row * a.y1;
    const int      nv  = a.n_vocab - v0 < LG_TILE ? (int) (a.n_vocab - v0) : LG_TILE;

    float f[STEPS][VEC];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int i = (s * 256 + tid) * VEC;
        if (i + VEC <= nv) {
            lg_load<T>(xp + (v0 + i) * ES, f[s]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                f[s][e] = i + e < nv ? load_elem<T>(xp + (v0 + i + e) * ES) : 0.0f;
            }
        }
    }
    int32_t state = -1;
    if (a.allowed) {
        state = a.state ? *(const int32_t *) (a.state + (int64_t) row * a.st0) : a.n_states == 1 ? 0 : (int32_t) row;
        if (state >= a.n_states) {
            if (blockIdx.x == 0 && tid == 0 && a.d_err) {
                atomicAdd(a.d_err, 1);
            }
            state = -1;
        }
    }
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if constexpr (HIST) {
#pragma unroll
        for (int i = 0; i < LG_TILE / 1024; ++i) {
            ((uint4 *) count)[i * 256 + tid] = make_uint4(0, 0, 0, 0);
        }
        const float * pp = (const float *) (a.pen + (int64_t) row * a.p1);
        rep              = pp[0];
        freq             = pp[1];
        pres             = pp[2];
        int32_t n        = a.len ? *(const int32_t *) (a.len + (int64_t) row * a.l0) : a.n_hist;
        n                = n < 0 ? 0 : n > a.n_hist ? a.n_hist : n;
        const int32_t * hp = (const int32_t *) (a.hist + (int64_t) row * a.h1);
        __syncthreads();
        for (int i = tid; i < n; i += 256) {
            const int32_t t = hp[i];
            if (t >= 0 && t < a.n_vocab) {
                const int64_t d = t - v0;
                if (d >= 0 && d < LG_TILE) {
                    atomicAdd(count + d, 1u);
                }
            } else if (blockIdx.x == 0 && a.d_err) {
                atomicAdd(a.d_err, 1);
            }
        }
        __syncthreads();
    }
    const float *    bp = a.bias ? (const float *) (a.bias + (int64_t) row * a.b1) : nullptr;
    const uint32_t * mp = state >= 0 ? (const uint32_t *) (a.allowed + (int64_t) state * a.m1) : nullptr;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int i = (s * 256 + tid) * VEC;
        if (i >= nv) {
            break;
        }
        const int64_t v = v0 + i;
        if constexpr (HIST) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const uint32_t c = count[i + e];
                if (c) {
                    const float l = f[s][e];
                    f[s][e]       = (l > 0.0f ? l / rep : l * rep) - (float) c * freq - pres;
                }
            }
        }
        if (bp) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                f[s][e] += bp[v + e < a.n_vocab ? v + e : a.n_vocab - 1];
            }
        }
        if (mp) {
            const uint32_t w = mp[v >> 5] >> (v & 31);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                f[s][e] = w >> e & 1u ? f[s][e] : -INFINITY;
            }
        }
        if (i + VEC <= nv) {
            lg_store<T>(yp + v * ES, f[s]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (i + e < nv) {
                    store_elem<T>(yp + (v + e) * ES, f[s][e]);
                }
            }
        }
    }
}

template <int T> static void launch_t(const LogitsArgs & a, hipStream_t s) {
    const dim3 grid((uint32_t) ((a.n_vocab + LG_TILE - 1) / LG_TILE), a.rows);
    if (a.hist) {
        MI_LAUNCH((k_logits<T, true>), grid, dim3(256), 0, s, a);
    } else {
        MI_LAUNCH((k_logits<T, false>), grid, dim3(256), 0, s, a);
    }
}

int launch_logits(const LogitsArgs & a, int type, hipStream_t s) {
    switch (type) {
        case MI_TYPE_F32:
            launch_t<MI_TYPE_F32>(a, s);
            return MI_OK;
        case MI_TYPE_BF16:
            launch_t<MI_TYPE_BF16>(a, s);
            return MI_OK;
        default:
            launch_t<MI_TYPE_F16>(a, s);
            return MI_OK;
    }
}

}  // namespace mi
