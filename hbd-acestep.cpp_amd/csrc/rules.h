// rules.h -- dispatch rules as plain host functions of sizes, so that they can be
// checked without a GPU. Each says what was measured on both sides of its line.
#pragma once

#include <cstdint>

namespace mi {

// Q8_0 product of one row of x (nbk key blocks, ng groups of 64 weight rows): whether the
// prologue, the product and the key sum are one launch of a workgroup per row group. A
// wave takes an eighth of the keys (up to a block per split more), in sets of 4 blocks.
// us with the norm prologue, three launches / one, weights of 400 MB in turn:
//   1024 keys: 64 groups 8.0 / 5.6, 96 8.3 / 5.7, 256 7.4 / 6.5, 512 10.0 / 9.3, 2370 29.8 / 35.0
//   2048 keys: 96 groups 11.0 / 8.4, 192 13.4 / 9.5, 512 16.1 / 14.4; 6144 keys: 32 groups 12.0 / 14.2
// Past 256 row groups the product has no second sum to save, and a second round of
// workgroups stands against one: there it wins only with the sets near full (32 and 64
// blocks 0.93, 24 0.99, 48 0.99; 8 blocks 1.11, 16 1.03, 33 1.07, 40 1.07). Up to 128 row
// groups 33-80 blocks would win too (64 blocks 32 groups 7.8 / 7.2, 80 blocks 96 groups
// 11.5 / 9.2; 96 blocks 16 groups 8.9 / 9.3) but keep the three launches.
inline bool mmv_one_launch(uint32_t nbk, uint32_t ng) {
    if (ng > 512 || nbk > 64 || (nbk > 32 && ng < 128)) {
        return false;
    }
    const uint32_t share = (nbk + 7) / 8, sets = (share + 3) / 4;
    return ng <= 256 || share >= sets * 3;  // at most a quarter of the sets' slots empty
}

// Q8_0 product of more than 8 rows: whether the matrix kernel's 64 x 64 tiles (t64 of them,
// 512 threads each) take a product of nbk key blocks that 128 x 128 tiles would take with ks
// key splits; slots = resident workgroups. While they fit the slots they win everywhere
// measured (9 rows to 512 tiles; 592 weight rows x 498 blocks x 1625 rows 123 against 118 us
// is the one exception found). Past that, up to two and a half times over (us, 128 / 64):
//   64 key blocks: 1152 tiles 55 / 49, 1600 64 / 70; past 5 tiles per CU the times cross back
//     and forth (64-80 blocks: of the time, 1344-1536 tiles 0.88-0.97, 2016 0.91-0.94, 2432
//     1.08, 3344 0.93) and the 128 x 128 tiles stay
//   3 or 4 key splits stand against their second round: 640 tiles, 128 blocks 56 / 60
//   2 key splits: 0.85-0.95 of the time, at 800 tiles of 192 blocks or more 1.00-1.02 (304
//     blocks, 1217 rows 132 / 134; the 64 x 64 tiles all the same: they need no partials, and
//     the call without a workspace of its own takes sizes that partials would not leave room for)
//   short keys: the pipeline's start and the sum of the key groups weigh more the more tiles
//     a CU gets in turn: of the time, with 3 tiles per CU (768) 8 blocks 0.92, 6 1.0, 5 1.04,
//     1 1.11; with 4 (1024) 12 blocks 0.93, 10 1.0, 5 1.13; with 5 (1280) 16 blocks 0.97, 12 1.0,
//     5 1.22
inline bool mmq_small_tiles(uint64_t t64, uint64_t slots, uint64_t ks, uint32_t nbk) {
    if (t64 <= slots) {
        return true;
    }
    const uint64_t cu = (2 * t64 + slots - 1) / slots;  // tiles per CU
    return ks < 3 && cu <= 5 && nbk >= 4 * (cu - 1);
}

// APG: whether a workgroup takes a whole sample (its frames in rows of oc channels)
// instead of one or two channels of it (cg). The channel split fills the chip where
// there are few samples, but each of its workgroups takes a line request per frame for
// 16 bytes of it, so its time grows with n * oc; a workgroup per sample reads whole
// lines, and up to 256 samples take hardly longer than one. The line is where these
// two estimates cross (ns; 256 CUs, buffers of 500 MB in turn), us by sample / by channels:
//   64 channels:   1 x 6000 482 / 39, 8 x 750 59 / 11, 64 x 750 67 / 67, 128 x 750 77 / 131,
//                  256 x 1500 227 / 440, 16 x 100 8.2 / 8.1, 64 x 100 11.6 / 29.9, 1 x 12 3.3 / 4.2
//   1024 channels: 1 x 750 964 / 18, 16 x 750 1050 / 265, 8 x 12 12.8 / 50, 256 x 12 26 / 1553
inline bool apg_by_sample(uint32_t n, uint32_t t, uint32_t oc, uint32_t cg) {
    if (n > 65535) {
        return true;  // the channel split's grid has the samples in y
    }
    const uint32_t phases = 1024 / oc;  // frames that a sample's workgroup takes at a time
    const double   groups = (double) n * (oc / cg), rounds = (double) ((uint64_t) (groups + 255) / 256);
    const double   frames = (double) t / phases;  // of a thread
    const double   sample = 2000 + 30.0 * phases + (1100 + 6.0 * n) * frames;
    const double   over   = 0.03 * t * groups, chain = 4.5 * t;
    return sample < 1500 + 1400 * cg * rounds + (over > chain ? over : chain);
}

// Logits: whether a workgroup takes 2048 tokens of a row instead of 4096. Small tiles fill the
// chip where there are few rows; large ones read the history half as often (us, 151669 F32 logits:
// 8 rows, 1200 tokens of history 6.0 / 6.8; 64 rows, 8000 19.5 / 18.5).
inline bool logits_small_tiles(uint32_t rows, int64_t n_vocab, uint32_t cus) {
    return (int64_t) rows * ((n_vocab + 8191) / 8192) < 4 * (int64_t) cus;
}

// Adapters' second product, m rows of n columns: whether a lane takes 4 columns of each of its rows, in
// tiles of 32 rows (16 at high ranks) and 256 columns, not one column in tiles of 16 rows and 64
// columns whose adapters are shared out over workgroups. Wide tiles move y at the rate of memory, but
// multiply all their rows by each of their adapters; small ones give every adapter of few rows a
// workgroup. Which rows share an adapter is device memory, so the rule sees sizes only. us wide / narrow,
// both products: 64 x 6144, 8 adapters in turn 16.5 / 11.7; 200 x 6144 19.6 / 16.7; 500 x 6144 30.7 / 32.5; 64 x
// 19456, one 11.4 / 11.7; 100 x 19456 13.1 / 14.9; 200 x 2560, 24 of rank 64 62.4 / 36.5; 1000 x 1024 11.4 / 11.3;
// 600 x 2560 12.9 / 14.6; 2000 x 19456, 16 249 / 280; 4000 x 2560, 8 of rank 64 236 / 268; 1000 x 6144, 24 in runs of 40
// 24.3 / 27.8. What it loses: 24 adapters in turn at 300 to 1000 x 6144 and 100 to 200 x 19456, 9 to 16 % (1000 x
// 6144 82.1 / 70.6), 8 in turn right past the border, 11 % (250 x 6144 19.6 / 17.7).
inline bool lora_wide(int64_t m, int64_t n) {
    return n >= 4 && m * n >= 1500000;
}

// Attention over Q4_0 K and V: over how many of `items` workgroups each the keys are split, `slots`
// of them resident at once. A split saves tile_ns of every tile of a row's keys that is left to
// another workgroup, and costs a launch that joins the results (2300 ns) and the traffic of a partial
// result, row_ps picoseconds per row and split. us, 128 values, 16 heads on 8, unsplit / split in 2 /
// 3 / 4 / 6: one row per head of 256 keys 10.4 / 12.0, of 512 13.5 / - / 11.9; 64 positions on 2064
// keys 44.7 / 29.4 / 23.8 / 21.6 / 22.8; 512 on 512 23.5 / 34.4; many rows a workgroup: 1024 on 5120
// 418 / 224 / 162 / 139 / 174. Workgroups of a second round are waited for, so one round as full as it
// gets, or two where they are fuller: 64 sequences of up to 8000 keys, 32 heads on 8 (512 items, 768
// slots) unsplit 104, in 2 87, in 3 90; 3 of up to 60000 (24 items) in 32 31.6, in 42 35.1
inline int64_t fa4_splits(int64_t tiles, int64_t rows, int64_t items, int64_t slots, int64_t most, int64_t tile_ns, int64_t row_ps) {
    int64_t best = 1, least = tiles * tile_ns * ((items + slots - 1) / slots);
    for (int64_t rounds = 1; rounds <= 2; ++rounds) {
        const int64_t want = rounds * slots / items < most ? rounds * slots / items : most;
        int64_t       s    = 1;
        while (s < want && (s + 1) * (s + 1) * row_ps * rows <= tiles * tile_ns * 1000) {
            ++s;
        }
        const int64_t ns = tiles * tile_ns * ((items * s + slots - 1) / slots) / s + 2300 + row_ps * rows * s / 1000;
        if (s > 1 && ns < least) {
            best  = s;
            least = ns;
        }
    }
    return best;
}

struct Fa4Plan {
    bool    many;    // workgroups of many rows (k_fa4_pre), not of 16 (k_fa4_dec)
    int64_t splits;  // of a row's keys
};

// Which of the two kernels takes `rows` rows of each of `heads` KV heads (times sequences) on n_kv
// keys of d values, one: a single query position. The kernel for 16 rows per workgroup has the
// shorter way from the first key to the last (four waves share a tile's turn), the one for many
// rows unpacks a key once for 128 or 256 of them. Their times in ns as the sums of what was
// measured one by one; both sides, us, 16 rows / many, the kernel's best splits (F32 y, BF16 y):
//   16 heads on 8: 64 positions on 464 keys 13.3 / 22.8, 12.5 / 18.8; 257 on 387 18.9 / 35.8, 16.8 / 24.2;
//                  512 on 512 23.5 / 34.8, 20.9 / 26.3; 1024 on 1024 65 / 51, 52 / 37; 2048 on 2048 207 / 98, 146 / 58
//   32 on 8, 8 sequences: 16 on 4016 59 / 96, 48 / 40; 64 on 4064 194 / 108, 146 / 66; 128 on 128 45 / 28, 35 / 17
// What it loses where both were timed: 64 values, 32 on 8, 8 sequences, 16 on 4016 in F32 38.2 / 42.4 (many taken); 256
// values, 16 on 8, 512 on 512 39.5 / 41.2 (many taken); all others go to the quicker side or lie within 5 %.
inline Fa4Plan fa4_plan(int64_t heads, int64_t rows, int64_t n_kv, int d, bool f32, bool one, int64_t cus) {
    const int64_t all = heads * rows;
    // 16 rows a workgroup
    const int64_t tk = d == 64 ? 64 : 32, tiles = (n_kv + tk - 1) / tk, items = heads * ((rows + 15) / 16);
    const int64_t way = (one ? 1100 : 2200) / 4;  // a tile, one of four waves
    const int64_t most = (tiles + 7) / 8;         // two tiles a wave
    const int64_t room = (d == 256 ? 2 : 3) * cus;  // resident workgroups
    Fa4Plan       p{ false, fa4_splits(tiles, all, items, room, most, way, 800) };
    if (rows <= 32) {
        return p;
    }
    int64_t       work = (f32 ? 12 : 9) * items * p.splits + (f32 ? 142 : 108) * (d == 256 ? 7 : 4) * items * tiles / 400;
    const int64_t last = tiles * way / p.splits, wg = items * p.splits;
    work = wg <= room ? work : work / wg * ((wg + room - 1) / room * room);  // a last round that is not full
    const int64_t few  = 8500 + (work > last ? work : last) + (p.splits > 1 ? 2300 + all * p.splits * 8 / 10 : 0);
    // many
    const int64_t bq = f32 && d == 128 ? 256 : 128, tkm = d == 256 ? 32 : 64, tm = (n_kv + tkm - 1) / tkm;
    const int64_t wgs = heads * ((rows + bq - 1) / bq), slots = cus * (d == 256 || (f32 && d == 128) ? 1 : 2);
    const int64_t ns  = f32 ? (d == 64 ? 2600 : d == 128 ? 5100 : 3400) : (d == 64 ? 1000 : d == 128 ? 2000 : 1600);  // a tile
    const int64_t fit = (tm + 1) / 2;  // two tiles a workgroup
    const int64_t s    = fa4_splits(tm, all, wgs, slots, fit, ns, 250);
    const int64_t many = 14000 + tm * ns * ((wgs * s + slots - 1) / slots) / s + (s > 1 ? 2300 + all * s / 4 : 0);
    return many < few ? Fa4Plan{ true, s } : p;
}

}  // namespace mi
