// logits.hip -- what is done to a row of logits before a token is drawn (mi_logits_adjust):
// penalties for tokens of the row's history, a bias, a grammar's mask.
//
//   c  = times the token is in the history
//   l' = c == 0 ? l : (l > 0 ? l / rep : l * rep) - c freq - pres,  + bias,  -inf where not allowed
//
// A workgroup takes a tile of 2048 or 4096 tokens of one row: its logits, bias and mask are loaded
// first, then the whole history is read and the tokens that fall into the tile are counted in LDS (integer
// atomics: their order does not show), then the tile is written. So one launch needs no
// memory but LDS; the history is read once a tile, from the cache.
#include "launch.h"
#include "rules.h"

namespace mi {

// rows of any vocabulary size: 16 bytes at the element's own alignment. Through the caches: a wave's
// access ends inside a line where rows do, and the next one reads or writes the rest (64 rows of
// 151669 F32 logits 18.5 us, 22.0 with streaming accesses).
typedef uint32_t lg_u4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t lg_u4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float    lg_f4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef int32_t  lg_i4a4 __attribute__((ext_vector_type(4), aligned(4)));

template <int T> __device__ __forceinline__ void lg_load(const char * p, float * f) {
    if constexpr (T == MI_TYPE_F32) {
        const lg_u4a4 v = *(const lg_u4a4 *) p;
        unpack16<T>(make_uint4(v.x, v.y, v.z, v.w), f);
    } else {
        const lg_u4a2 v = *(const lg_u4a2 *) p;
        unpack16<T>(make_uint4(v.x, v.y, v.z, v.w), f);
    }
}

template <int T> __device__ __forceinline__ void lg_store(char * p, const float * f) {
    const uint4 w = pack16<T>(f);
    if constexpr (T == MI_TYPE_F32) {
        const lg_u4a4 v = { w.x, w.y, w.z, w.w };
        *(lg_u4a4 *) p = v;
    } else {
        const lg_u4a2 v = { w.x, w.y, w.z, w.w };
        *(lg_u4a2 *) p = v;
    }
}

template <int T, int TILE, bool HIST>
__global__ void __launch_bounds__(256) k_logits(const LogitsArgs a) {
    constexpr int VEC   = TT<T>::VEC;
    constexpr int ES    = TT<T>::ES;
    constexpr int STEPS = TILE / (256 * VEC);
    __shared__ __align__(16) uint32_t count[HIST ? TILE : 4];
    const int      tid = threadIdx.x;
    const uint32_t row = blockIdx.y;
    const int64_t  v0  = (int64_t) blockIdx.x * TILE;
    const char *   xp  = a.x + (int64_t) row * a.x1;
    char *         yp  = a.y + (int64_t) row * a.y1;
    const int      nv  = a.n_vocab - v0 < TILE ? (int) (a.n_vocab - v0) : TILE;

    // everything the tile needs but the counts is asked for first
    int32_t state = -1, n = 0;
    if (a.allowed) {
        state = a.state ? *(const int32_t *) (a.state + (int64_t) row * a.st0) : a.n_states == 1 ? 0 : (int32_t) row;
    }
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if constexpr (HIST) {
        const float * pp = (const float *) (a.pen + (int64_t) row * a.p1);
        rep              = pp[0];
        freq             = pp[1];
        pres             = pp[2];
        n                = a.len ? *(const int32_t *) (a.len + (int64_t) row * a.l0) : a.n_hist;
        n                = n < 0 ? 0 : n > a.n_hist ? a.n_hist : n;
    }
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
    float bias[STEPS][VEC] = {};
    if (a.bias) {
        const float * bp = (const float *) (a.bias + (int64_t) row * a.b1) + v0;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int i = (s * 256 + tid) * VEC;
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                if (i + e + 4 <= nv) {
                    const lg_f4a4 b = *(const lg_f4a4 *) (bp + i + e);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        bias[s][e + k] = b[k];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        bias[s][e + k] = i + e + k < nv ? bp[i + e + k] : 0.0f;
                    }
                }
            }
        }
    }
    if (state >= a.n_states) {
        if (blockIdx.x == 0 && tid == 0 && a.d_err) {
            atomicAdd(a.d_err, 1);
        }
        state = -1;
    }
    uint32_t word[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        word[s] = ~0u;
    }
    if (state >= 0) {
        const uint32_t * mp = (const uint32_t *) (a.allowed + (int64_t) state * a.m1);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int i = (s * 256 + tid) * VEC;
            word[s]     = mp[(v0 + (i < nv ? i : 0)) >> 5];
        }
    }
    if constexpr (HIST) {
#pragma unroll
        for (int i = 0; i < TILE / 1024; ++i) {
            ((uint4 *) count)[i * 256 + tid] = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
        const int32_t * hp  = (const int32_t *) (a.hist + (int64_t) row * a.h1);
        uint32_t        bad = 0;
        auto            put = [&](int32_t t) {
            const uint32_t d = (uint32_t) t - (uint32_t) v0;  // a token before the tile, or negative, wraps past it
            if (d < (uint32_t) nv) {
                atomicAdd(count + d, 1u);
            }
            bad += (uint32_t) t >= (uint32_t) a.n_vocab;
        };
        int i = 0;
        for (; i + 4096 <= n; i += 4096) {  // 16 ids a thread in flight
            lg_i4a4 t[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                t[k] = *(const lg_i4a4 *) (hp + i + k * 1024 + tid * 4);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                put(t[k / 4][k % 4]);
            }
        }
        int32_t t[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int at = i + k * 256 + tid;
            t[k]         = at < n ? hp[at] : -1;
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (i + k * 256 + tid < n) {
                put(t[k]);
            }
        }
        if (bad && blockIdx.x == 0 && a.d_err) {
            atomicAdd(a.d_err, (int) bad);
        }
        __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int i = (s * 256 + tid) * VEC;
        if (i >= nv) {
            break;
        }
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
        if (a.bias) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                f[s][e] += bias[s][e];
            }
        }
        const uint32_t w = word[s] >> ((v0 + i) & 31);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            f[s][e] = w >> e & 1u ? f[s][e] : -INFINITY;
        }
        if (i + VEC <= nv) {
            lg_store<T>(yp + (v0 + i) * ES, f[s]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (i + e < nv) {
                    store_elem<T>(yp + (v0 + i + e) * ES, f[s][e]);
                }
            }
        }
    }
}

template <int T, int TILE> static void launch_tile(const LogitsArgs & a, hipStream_t s) {
    const dim3 grid((uint32_t) ((a.n_vocab + TILE - 1) / TILE), a.rows);
    if (a.hist) {
        MI_LAUNCH((k_logits<T, TILE, true>), grid, dim3(256), 0, s, a);
    } else {
        MI_LAUNCH((k_logits<T, TILE, false>), grid, dim3(256), 0, s, a);
    }
}

template <int T> static void launch_t(const LogitsArgs & a, hipStream_t s) {
    if (logits_small_tiles(a.rows, a.n_vocab, (uint32_t) num_cus())) {
        launch_tile<T, 2048>(a, s);
    } else {
        launch_tile<T, 4096>(a, s);
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
