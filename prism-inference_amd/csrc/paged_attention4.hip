// paged_attention4.hip -- grouped-query attention over the paged cache of 4 bits a value (gfx950), for
// single tokens, chunks and prompts of many requests in one call.
//
// Rows are (token, head of the group); a wavefront takes 16 * NT of them through blocks of 64 keys:
//   S^T = K Q^T     K as the A operand, 16 keys a matrix instruction
//   p = 2^(z - m), z = S * scale * log2 e, l = sum p
//   O^T += V^T P^T
// e2m1 codes times their group's power of two are exact in binary16, and one instruction makes two of them
// from a byte and the scale, so scales cost no arithmetic of their own and the products need no correction.
//
// Both operands come from rows of 4-bit codes without an exchange between lanes, since the sum over keys or dimensions
// may run in any order and rows and columns of a product may stand for any key or dimension:
//   K  lane (n, g) has the dimensions [g D/4, (g + 1) D/4) of four neighbouring keys, one for each of four tiles:
//      tile t's row 4 a + i is the block's key 16 a + 4 i + t.  Their scales of a group are one dword.
//   S  so lane (n, g) has the scores of row n for the 16 keys from 16 g on, in the order that makes them
//      the B operand of the second product as they stand.
//   V  lane (n, g) has the dimensions [n D/16, (n + 1) D/16) of the same 16 keys: its codes of two keys
//      are converted two dimensions at a time and their halves swapped (two byte permutations for four values).
#include <algorithm>
#include <type_traits>

#include "attend_common.hpp"

namespace prism {

namespace {

// The scale in byte i of a word; 0 stands for 2^-127, of which nothing is left in binary16.
template <int i>
__device__ __forceinline__ float scale_in(uint32_t w) {
    return __uint_as_float(i == 3 ? w >> 1 & 0x7f800000u : (w >> (8 * i) & 0xffu) << 23);
}
__device__ __forceinline__ float scale_in(uint32_t w, int i) {
    return i == 0 ? scale_in<0>(w) : i == 1 ? scale_in<1>(w) : i == 2 ? scale_in<2>(w) : scale_in<3>(w);
}
// Byte b of eight codes as two values.
__device__ __forceinline__ f16x2 pair_of(uint32_t w, float scale, int b) {
    return b == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)
           : b == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)
           : b == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)
                    : __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3);
}
union Halves {
    uint32_t u[4];
    f16x2 h[4];
    f16x8 v;
};
__device__ __forceinline__ f16x8 eight_of(uint32_t w, float scale) {
    Halves r;
#pragma unroll
    for (int b = 0; b < 4; ++b) r.h[b] = pair_of(w, scale, b);
    return r.v;
}
// The first halves of two pairs, and the second ones.
__device__ __forceinline__ uint32_t firsts(f16x2 a, f16x2 b) {
    return perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x05040100u);
}
__device__ __forceinline__ uint32_t seconds(f16x2 a, f16x2 b) {
    return perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}

// Scales of positions that no row sees, before a window, behind the keys or of a stand-in, may be no numbers, which zero
// probabilities do not silence: of 16 bytes those from `from` to `to` stay.
__device__ __forceinline__ void keep_scales(u32x4 &v, bool there, int32_t from, int32_t to) {
    keep_bytes(v, there ? to : 0);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int32_t gone = from - 4 * w;
        v[w] &= gone >= 4 ? 0u : gone <= 0 ? ~0u : ~0u << (8 * gone);
    }
}

// What both kernels below share: a wavefront's 16 * NT rows, their queries, statistics and sums.
// T: type of q and out; LIMBS: binary16 parts of q and of the probabilities (2 for binary32).
template <typename T, int D, int NT>
struct Rows4 {
    static constexpr int LIMBS = sizeof(T) == 4 ? 2 : 1;
    static constexpr int KS = D / 32, DT = D / 16;
    uint32_t token[NT], head[NT];  // of this lane's rows
    bool live[NT];
    int32_t lo[NT], hi[NT];        // the keys they see
    int32_t all_lo, all_hi;        // keys every row of the wavefront sees
    int32_t any_lo, any_hi;        // keys any row sees
    float kf[NT];                  // base-2 softmax scale of the row's scaled queries, not negative
    f16x8 qv[LIMBS][NT][KS];
    float m[NT], l[NT];
    f32x4 acc[NT][DT];             // tile d, row 4 g + i: dimension D/16 (4 g + i) + d

    __device__ __forceinline__ void load(const AttendArgs &p, const Request &q, uint32_t base_row, uint32_t last, uint32_t kvh) {
        const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane / 16;
        all_lo = 0, all_hi = 0x7fffffff, any_lo = 0x7fffffff, any_hi = 0;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t row = base_row + 16 * t + n;
            live[t] = row <= last;
            const uint32_t rr = live[t] ? row : last, i = rr / p.group;
            token[t] = q.first + i;
            head[t] = kvh * p.group + rr % p.group;
            visible(p, q, i, &lo[t], &hi[t]);
            all_lo = max(all_lo, lo[t]);
            all_hi = min(all_hi, hi[t]);
            any_lo = min(any_lo, lo[t]);
            any_hi = max(any_hi, hi[t]);
            // Lane group g has the dimensions [g D/4, (g + 1) D/4) of the row.
            const T *src = static_cast<const T *>(p.a.q) + token[t] * p.a.q_stride + static_cast<uint64_t>(head[t]) * D + g * (D / 4);
            f32x4 x[D / 16];
            float most = 0.0f;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                x[j] = load4(src + 4 * j);
#pragma unroll
                for (int k = 0; k < 4; ++k) most = fmaxf(most, fabsf(x[j][k]));
            }
            most = across_max(most);
            // A power of two, at most 2^113, takes the row's largest value to [2^13, 2^14); the sign of the scale goes along.
            int e = static_cast<int>(__float_as_uint(most) >> 23 & 255) - 127;
            e = !finite(most) ? 0 : max(e, -100);
            float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
            if (p.a.scale < 0.0f) up = -up;
            // Never 0: a masked score is -infinity, and 0 times it would be NaN.
            kf[t] = fmaxf(fabsf(p.a.scale) * kLog2e * __uint_as_float(static_cast<uint32_t>(127 - 13 + e) << 23), 0x1p-120f);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = x[2 * s + j / 4][j % 4] * up;
                    const _Float16 h = static_cast<_Float16>(v);
                    qv[0][t][s][j] = h;
                    if constexpr (LIMBS == 2) qv[LIMBS - 1][t][s][j] = static_cast<_Float16>(v - static_cast<float>(h));
                }
            m[t] = kNone;
            l[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int d = 1; d < 16; d *= 2) {
            all_lo = max(all_lo, __shfl_xor(all_lo, d));
            all_hi = min(all_hi, __shfl_xor(all_hi, d));
            any_lo = min(any_lo, __shfl_xor(any_lo, d));
            any_hi = max(any_hi, __shfl_xor(any_hi, d));
        }
        all_lo = uniform(all_lo), all_hi = uniform(all_hi), any_lo = uniform(any_lo), any_hi = uniform(any_hi);
    }

    // Scores s of the lane's 16 keys from `key` on (s[u][t][i]: key + 4 i + t) are masked where some row does not see some key
    // of the block (edge), and the statistics follow their maximum; p = 2^(s kf + off).
    __device__ __forceinline__ void scores(f32x4 (&s)[NT][4], bool there, bool edge, int32_t key, float (&off)[NT]) {
        float top[NT];
        bool grows = false;
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            if (edge)
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int32_t k = key + 4 * i + t;
                        s[u][t][i] = there && k >= lo[u] && k < hi[u] ? s[u][t][i] : kNone;
                    }
            float most = kNone;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) most = fmaxf(most, s[u][t][i]);
            top[u] = across_max(most * kf[u]);
            grows |= top[u] > m[u] + kSlack || m[u] == kNone;
        }
        if (__ballot(grows)) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                const float next = fmaxf(m[u], top[u]);
                const float alpha = __builtin_amdgcn_exp2f(next == kNone ? 0.0f : m[u] - next);
                m[u] = next;
                l[u] *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[u][d] *= alpha;
            }
        }
#pragma unroll
        for (int u = 0; u < NT; ++u) off[u] = kHeadroom - (m[u] == kNone ? 0.0f : m[u]);  // no key yet: scores of -inf
    }
    // Probabilities of half `c` of the keys: an operand of the second product.  Element j is the key 4 (j % 4) + 2 c + j / 4.
    template <int c>
    __device__ __forceinline__ void probabilities(const f32x4 (&s)[NT][4], f16x8 (&pv)[LIMBS][NT], const float (&off)[NT]) {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][2 * c + j / 4][j % 4], kf[u], off[u]));
                sum += e;
                const _Float16 h = static_cast<_Float16>(e);
                pv[0][u][j] = h;
                if constexpr (LIMBS == 2) pv[LIMBS - 1][u][j] = static_cast<_Float16>(e - static_cast<float>(h));
            }
            l[u] += sum;
        }
    }

    // l once the keys are done: the row's, of all four lanes, in the unit of the parts.
    __device__ __forceinline__ void total() {
#pragma unroll
        for (int u = 0; u < NT; ++u) l[u] = across_sum(l[u]) * kSumUnit;
    }

    // The rows, or with more than one part their unnormalised sums.
    __device__ __forceinline__ void write(const AttendArgs &p, uint32_t parts, uint32_t split, int *err) const {
        const uint32_t g = (threadIdx.x & 63) / 16;
        bool bad = false;
        const uint64_t all_rows = static_cast<uint64_t>(p.a.tokens) * p.a.heads;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (!live[t]) continue;
            const float inv = parts == 1 ? inverse(l[t]) : 1.0f;
            const uint64_t row = split * all_rows + static_cast<uint64_t>(token[t]) * p.a.heads + head[t];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d = 0; d < DT; d += 4) {
                    const f32x4 v = f32x4{acc[t][d][i], acc[t][d + 1][i], acc[t][d + 2][i], acc[t][d + 3][i]} * inv;
                    const uint32_t dim = DT * (4 * g + i) + d;
                    if (parts == 1) write_row<T>(p, token[t], head[t], dim, v, &bad);
                    else *reinterpret_cast<f32x4 *>(p.part + row * D + dim) = v;
                }
            if (parts > 1 && g == 0) {
                p.part_ml[2 * row] = m[t];
                p.part_ml[2 * row + 1] = l[t];
            }
        }
        if (bad) raise_error(err, kErrNonfinite);
    }
};

// The codes of a lane's dimensions of one key for the second product: D / 16 of them.
template <int D>
struct ValueCodes {
    uint32_t w[D == 256 ? 2 : 1];
    __device__ __forceinline__ void load(const uint8_t *p) {
        if constexpr (D == 64) {
            w[0] = *reinterpret_cast<const uint16_t *>(p);
        } else if constexpr (D == 128) {
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        } else {
            const u32x2 v = *reinterpret_cast<const u32x2 *>(p);
            w[0] = v[0], w[1] = v[1];
        }
    }
};

// Few rows (single tokens, drafts): the workgroup's four wavefronts share 16 * NT rows and split the
// keys.  Every code is used once, so they go from memory to registers, and memory is the bound: 64 requests of up to 16384 keys
// (8 heads of 128, 570 MB) 128 us, 4.5 TB/s, of one length 115 us, 5.0; 8 of up to 131072 (4 of 256) 156 us, 4.4, where
// conversions of 16 rows for the 6 of a group count too.  A single request's 1025 keys take 6.7 us and their join 3.7, a launch and
// four dependent loads each.  Keys through LDS, with half the accesses to L1, take as long; so do, but for heads
// of 256, the next block's codes loaded ahead, and a launch bound for four wavefronts a SIMD spills (130 against 116).
// WIDE: byte offsets into the keys or values pass 32 bits; else a lane's address is one register
// beside a scalar base.
template <typename T, int D, int NT, bool WIDE>
__global__ __launch_bounds__(256, D == 256 && sizeof(T) == 4 ? 1 : 2) void k_attend4_rows(AttendArgs p, int *err) {
    typedef Rows4<T, D, NT> R;
    constexpr int LIMBS = R::LIMBS, KS = R::KS, DT = R::DT, KG = D == 256 ? 2 : 1;
    __shared__ float join_ml[4][16 * NT][2];
    __shared__ f32x4 join_acc[3][NT * DT][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t n = lane & 15, g = lane / 16;
    Tile tile;
    if (!tile_of(p, 16 * NT, blockIdx.z, err, &tile)) return;
    const uint32_t kvh = tile.kvh;
    const uint32_t page_mask = p.c.page_size - 1;
    const int32_t *table = p.a.block_table + static_cast<uint64_t>(tile.r) * p.a.max_pages;
    const uint8_t *kc = static_cast<const uint8_t *>(p.c.k), *vc = static_cast<const uint8_t *>(p.c.v);
    const uint32_t kgroup = n / 4;  // 16-key group whose keys this lane loads for the first product
    int32_t id_k = 0, id_v = 0;
    uint32_t kraw[4][D / 32], ke[KG];
    ValueCodes<D> vraw[16];
    u32x4 ve;
    typedef std::conditional_t<WIDE, uint64_t, uint32_t> Offset;
    bool there_next = false, missing = false;
    auto look = [&](uint32_t b) {
        const int32_t base = static_cast<int32_t>(64 * b);
        id_k = entry_at(p, tile, table, base + 16 * static_cast<int32_t>(kgroup));
        id_v = entry_at(p, tile, table, base + 16 * static_cast<int32_t>(g));
    };
    auto fetch_k = [&](uint32_t b) {
        const int32_t key_k = static_cast<int32_t>(64 * b) + 16 * static_cast<int32_t>(kgroup);
        const Offset unit_k = static_cast<Offset>(is_page(p, tile, id_k, key_k) ? id_k : 0) * p.c.kv_heads + kvh;
        const uint32_t place_k = (static_cast<uint32_t>(key_k) & page_mask) + 4 * (n & 3);
#pragma unroll
        for (int j = 0; j < KG; ++j)
            ke[j] = *reinterpret_cast<const uint32_t *>(p.c.k_exponent + (((unit_k * (D / 32) + (D == 64 ? g / 2 : KG * g + j)) << p.page_log2) + place_k));
        const Offset k_at = ((unit_k << p.page_log2) + place_k) * (D / 2) + g * (D / 8);
#pragma unroll
        for (int t = 0; t < 4; ++t) __builtin_memcpy(kraw[t], __builtin_assume_aligned(kc + k_at + t * (D / 2), D == 64 ? 8 : 16), D / 8);
    };
    auto fetch_v = [&](uint32_t b) {
        const int32_t key_v = static_cast<int32_t>(64 * b) + 16 * static_cast<int32_t>(g);
        there_next = is_page(p, tile, id_v, key_v);
        missing |= !there_next && seen(tile, key_v);
        const Offset unit_v = static_cast<Offset>(there_next ? id_v : 0) * p.c.kv_heads + kvh;
        const uint32_t place_v = static_cast<uint32_t>(key_v) & page_mask;
        ve = *reinterpret_cast<const u32x4 *>(p.c.v_exponent + (((unit_v * (D / 32) + n / (512 / D)) << p.page_log2) + place_v));
        const Offset v_at = ((unit_v << p.page_log2) + place_v) * (D / 2) + n * (D / 32);
#pragma unroll
        for (int r = 0; r < 16; ++r) vraw[r].load(vc + v_at + r * (D / 2));
    };
    const uint32_t first = tile.b0 + wave;
    if (first < tile.b1) look(first);
    R rows;
    rows.load(p, tile.q, tile.row0, tile.last, kvh);
    // Heads of 256 leave two wavefronts a SIMD or one, so each product reloads the codes it used for its next block (8 requests of up
    // to 131072 keys 163 -> 153 us); others load both at the top of the block (64 of up to 16384, heads of 128, 128 us either way,
    // binary32 142 against 157, heads of 64 82 against 85).
    constexpr bool kAhead = D == 256;
    if (kAhead && first < tile.b1) {
        fetch_k(first);
        fetch_v(first);
        if (first + 4 < tile.b1) look(first + 4);
    }
    for (uint32_t b = first; b < tile.b1; b += 4) {
        if constexpr (!kAhead) {
            fetch_k(b);
            fetch_v(b);
            if (b + 4 < tile.b1) look(b + 4);
        }
        const int32_t base = static_cast<int32_t>(64 * b), key = base + 16 * static_cast<int32_t>(g);
        const bool there = there_next;
        const bool edge = base < rows.all_lo || base > rows.all_hi - 64 || __ballot(there) != ~0ull;
        f32x4 s[NT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int u = 0; u < NT; ++u) s[u][t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const f16x8 kv = eight_of(kraw[t][k], scale_in(ke[KG * k / KS], t));
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int i = 0; i < LIMBS; ++i) s[u][t] = mfma(kv, rows.qv[i][u][k], s[u][t]);
            }
        }
        if (kAhead && b + 4 < tile.b1) fetch_k(b + 4);
        f16x8 pv[2][LIMBS][NT];
        float off[NT];
        rows.scores(s, there, edge, key, off);
        rows.template probabilities<0>(s, pv[0], off);
        rows.template probabilities<1>(s, pv[1], off);
        if (edge) keep_scales(ve, there, tile.seen_lo - key, tile.seen_hi - key);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            // Element j of the operand is the key 4 (j % 4) + 2 c + j / 4.
            float vs[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) vs[j] = scale_in(ve[j % 4], 2 * c + j / 4);
#pragma unroll
            for (int b2 = 0; b2 < DT / 2; ++b2) {
                f16x2 x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = pair_of(vraw[4 * (j % 4) + 2 * c + j / 4].w[b2 / 4], vs[j], b2 % 4);
                Halves a, o;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    a.u[j] = firsts(x[2 * j], x[2 * j + 1]);
                    o.u[j] = seconds(x[2 * j], x[2 * j + 1]);
                }
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int i = 0; i < LIMBS; ++i) {
                        rows.acc[u][2 * b2] = mfma(a.v, pv[c][i][u], rows.acc[u][2 * b2]);
                        rows.acc[u][2 * b2 + 1] = mfma(o.v, pv[c][i][u], rows.acc[u][2 * b2 + 1]);
                    }
            }
        }
        if (kAhead && b + 4 < tile.b1) {
            fetch_v(b + 4);
            if (b + 8 < tile.b1) look(b + 8);
        }
    }
    if (missing) raise_error(err, kErrIndex);

    // The four wavefronts' rows join in the first.
    rows.total();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (g == 0) {
            join_ml[wave][16 * t + n][0] = rows.m[t];
            join_ml[wave][16 * t + n][1] = rows.l[t];
        }
        if (wave)
#pragma unroll
            for (int d = 0; d < DT; ++d) join_acc[wave - 1][t * DT + d][lane] = rows.acc[t][d];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float top = rows.m[t];
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, join_ml[w][16 * t + n][0]);
        const float ref = top == kNone ? 0.0f : top;
        const float mine = __builtin_amdgcn_exp2f(rows.m[t] - ref);
        rows.l[t] *= mine;
#pragma unroll
        for (int d = 0; d < DT; ++d) rows.acc[t][d] *= mine;
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            const float other = __builtin_amdgcn_exp2f(join_ml[w][16 * t + n][0] - ref);
            rows.l[t] = __builtin_fmaf(join_ml[w][16 * t + n][1], other, rows.l[t]);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const f32x4 v = join_acc[w - 1][t * DT + d][lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) rows.acc[t][d][i] = __builtin_fmaf(v[i], other, rows.acc[t][d][i]);
            }
        }
        rows.m[t] = top;
    }
    rows.write(p, tile.parts, blockIdx.z, err);
}

// Many rows (prompts, chunks): each of WAVES wavefronts has 16 * NT rows of its own and all keys.  A block's codes are
// converted to binary16 once by the workgroup, a quarter of the keys (or of eight wavefronts half the dimensions of one) by each
// wavefront, into LDS in the order of the operands; the next block's codes come from memory meanwhile and are converted after the products, so a
// block costs one barrier.  Bounds: conversions, exponentials and their like, at four cycles an instruction, fill 51 % of a SIMD's cycles and
// the matrix cores 39 %.  They add up: the conversions stand behind a block's last product (both ends of the branch below compile to one), where
// only the SIMD's other wavefront has products to issue beside them.  A prompt of 8192 tokens, 32 heads of 128, takes 580 to 705 us card by
// card, 780 to 950 TFLOP/s.
template <typename T, int D, int NT, int WAVES, bool WIDE>
__global__ __launch_bounds__(64 * WAVES, D == 256 && WAVES == 4 ? 1 : 2) void k_attend4_tile(AttendArgs p, int *err) {
    typedef Rows4<T, D, NT> R;
    typedef std::conditional_t<WIDE, uint64_t, uint32_t> Offset;
    constexpr int LIMBS = R::LIMBS, KS = R::KS, DT = R::DT;
    constexpr int H = WAVES / 4, HK = KS / H, HG = D == 256 ? 2 / H : 1, HB = DT / 2 / H;  // of one wavefront: its steps, scales and bytes
    static_assert(H == 1 || (H == 2 && D == 256));
    __shared__ f16x8 kf[2][4][KS][64];
    __shared__ f16x4 vf[2][DT][2][2][64];  // halves of an operand apart: writes of 8 bytes without bank conflicts
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t n = lane & 15, g = lane / 16;
    Tile tile;
    if (!tile_of(p, 16 * NT * WAVES, blockIdx.z, err, &tile)) return;
    const uint32_t kvh = tile.kvh, part = wave % 4, half = wave / 4;
    R rows;
    rows.load(p, tile.q, min(tile.row0 + wave * 16 * NT, tile.last), tile.last, kvh);
    const bool idle = tile.row0 + wave * 16 * NT > tile.last;  // converts only

    const uint32_t page_mask = p.c.page_size - 1, page_log2 = p.page_log2;
    const int32_t *table = p.a.block_table + static_cast<uint64_t>(tile.r) * p.a.max_pages;
    const uint8_t *kc = static_cast<const uint8_t *>(p.c.k), *vc = static_cast<const uint8_t *>(p.c.v);
    const uint32_t kgroup = n / 4;
    bool missing = false;

    // Codes of a block: this wavefront's key 4 i + part of each 16 (i: the lane's n & 3 for K, all four for V).
    uint32_t kraw[HK], ke[HG];
    ValueCodes<D / H> vraw[4];
    u32x4 ve;
    Offset k_at = 0, ke_at = 0, v_at = 0, ve_at = 0;
    bool there_found = false;
    int32_t id_k = 0, id_v = 0;
    // Three steps of a block, each in another's shadow: its table entries, the addresses that follow from them, its codes.
    auto look = [&](uint32_t b) {
        const int32_t base = static_cast<int32_t>(64 * b);
        id_k = entry_at(p, tile, table, base + 16 * static_cast<int32_t>(kgroup));
        id_v = entry_at(p, tile, table, base + 16 * static_cast<int32_t>(g));
    };
    auto find = [&](uint32_t b) {
        const int32_t base = static_cast<int32_t>(64 * b);
        const int32_t key_k = base + 16 * static_cast<int32_t>(kgroup), key_v = base + 16 * static_cast<int32_t>(g);
        there_found = is_page(p, tile, id_v, key_v);
        missing |= !there_found & seen(tile, key_v);
        const uint32_t page_k = is_page(p, tile, id_k, key_k) ? id_k : 0, page_v = there_found ? id_v : 0;
        // Below 2^32 bytes of codes there are fewer than 2^24 pages.
        Offset unit_k, unit_v;
        if constexpr (WIDE) {
            unit_k = static_cast<Offset>(page_k) * p.c.kv_heads + kvh, unit_v = static_cast<Offset>(page_v) * p.c.kv_heads + kvh;
        } else {
            unit_k = __umul24(page_k, p.c.kv_heads) + kvh, unit_v = __umul24(page_v, p.c.kv_heads) + kvh;
        }
        unit_k <<= page_log2, unit_v <<= page_log2;
        const uint32_t place_k = (static_cast<uint32_t>(key_k) & page_mask) + (4 * (n & 3) + part), place_v = static_cast<uint32_t>(key_v) & page_mask;
        ke_at = unit_k * (D / 32) + (place_k + (static_cast<uint32_t>(D == 64 ? g / 2 : D == 128 ? g : 2 * g + HG * half) << page_log2));
        ve_at = unit_v * (D / 32) + (place_v + (n / (512 / D) << page_log2));
        k_at = (unit_k + place_k) * (D / 2) + (g * (D / 8) + half * (4 * HK));
        v_at = (unit_v + place_v) * (D / 2) + (part * (D / 2) + n * (D / 32) + half * HB);
    };
    auto fetch = [&] {
#pragma unroll
        for (int j = 0; j < HG; ++j) ke[j] = p.c.k_exponent[ke_at + (static_cast<Offset>(j) << page_log2)];
        ve = *reinterpret_cast<const u32x4 *>(p.c.v_exponent + ve_at);
        __builtin_memcpy(kraw, __builtin_assume_aligned(kc + k_at, D == 64 ? 8 : 16), 4 * HK);
#pragma unroll
        for (int i = 0; i < 4; ++i) vraw[i].load(vc + v_at + 4 * i * (D / 2));
    };
    auto mend = [&](uint32_t b, bool there) {
        const int32_t key = static_cast<int32_t>(64 * b + 16 * g);
        if (__ballot(!there || key < tile.seen_lo || key > tile.seen_hi - 16)) keep_scales(ve, there, tile.seen_lo - key, tile.seen_hi - key);
    };
    const uint32_t pick = 0x000c0c0cu | part << 24;  // byte `part` of a word on top
    auto convert = [&](uint32_t at) {                // into buffer `at`
#pragma unroll
        for (int k = 0; k < HK; ++k) kf[at][part][HK * half + k][lane] = eight_of(kraw[k], scale_in<0>(ke[HG * k / HK]));
        float vs[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) vs[i] = __uint_as_float(perm(0u, ve[i], pick) >> 1);
#pragma unroll
        for (int b2 = 0; b2 < HB; ++b2) {
            const uint32_t d = 2 * (HB * half + b2);
            f16x2 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = pair_of(vraw[i].w[b2 / 4], vs[i], b2 % 4);
            vf[at][d][part / 2][part % 2][lane] = __builtin_bit_cast(f16x4, u32x2{firsts(x[0], x[1]), firsts(x[2], x[3])});
            vf[at][d + 1][part / 2][part % 2][lane] = __builtin_bit_cast(f16x4, u32x2{seconds(x[0], x[1]), seconds(x[2], x[3])});
        }
    };

    // At the top of block b its codes are in LDS, those of b + 1 on their way to registers, the addresses of b + 2
    // still to be found; past the last block the last one stands in.
    bool there_now = false, there_next = false;
    if (tile.b0 < tile.b1) {
        const uint32_t end = tile.b1 - 1;
        look(tile.b0);
        find(tile.b0);
        fetch();
        there_now = there_found;
        mend(tile.b0, there_now);
        convert(tile.b0 & 1);
        look(min(tile.b0 + 1, end));
        find(min(tile.b0 + 1, end));
        fetch();
        there_next = there_found;
        look(min(tile.b0 + 2, end));
    }
    for (uint32_t b = tile.b0; b < tile.b1; ++b) {
        const uint32_t end = tile.b1 - 1;
        __syncthreads();  // block b is in LDS, and every wavefront is done with block b - 1
        const int32_t base = static_cast<int32_t>(64 * b);
        const bool active = !idle && base < rows.any_hi && base > rows.any_lo - 64;  // base + 64 may be 2^31
        if (active) {
            const bool edge = base < rows.all_lo || base > rows.all_hi - 64 || __ballot(there_now) != ~0ull;
            // Products of one step of dimensions, four key tiles by NT row tiles, do not wait for each other.
            f32x4 s[NT][4];
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const f16x8 kv = kf[b & 1][t][k][lane];
#pragma unroll
                    for (int i = 0; i < LIMBS; ++i)
#pragma unroll
                        for (int u = 0; u < NT; ++u) s[u][t] = mfma(kv, rows.qv[i][u][k], k || i ? s[u][t] : f32x4{0, 0, 0, 0});
                }
            find(min(b + 2, end));
            float off[NT];
            rows.scores(s, there_now, edge, base + 16 * static_cast<int32_t>(g), off);
            mend(min(b + 1, end), there_next);
            f16x8 pv[2][LIMBS][NT];
            rows.template probabilities<0>(s, pv[0], off);
            rows.template probabilities<1>(s, pv[1], off);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const f16x8 vv = __builtin_shufflevector(vf[b & 1][d][c][0][lane], vf[b & 1][d][c][1][lane], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                    for (int i = 0; i < LIMBS; ++i)
#pragma unroll
                        for (int u = 0; u < NT; ++u) rows.acc[u][d] = mfma(vv, pv[c][i][u], rows.acc[u][d]);
                }
            }
            convert(~b & 1);
        } else {
            find(min(b + 2, end));
            mend(min(b + 1, end), there_next);
            convert(~b & 1);
        }
        fetch();
        look(min(b + 3, end));
        there_now = there_next;
        there_next = there_found;
    }
    if (missing) raise_error(err, kErrIndex);
    if (idle) return;
    rows.total();
    rows.write(p, tile.parts, blockIdx.z, err);
}

// How a call runs: rows a workgroup takes, whether its wavefronts share them, and the most splits.
struct Plan {
    uint32_t nt, M, slots, each, splits;
    bool shared;
};
Plan attend_plan(const prism_kv_cache &c, const prism_attention &a, uint32_t cus) {
    const uint32_t group = a.heads / c.kv_heads;
    const uint64_t typical = (static_cast<uint64_t>(a.tokens) * group + a.requests - 1) / a.requests;  // rows of a request
    Plan p;
    // Drafts of 17 to 32 rows a request are faster here than on tiles of 64 rows, most of which they leave empty (64 requests of up to 16384 keys,
    // 8 heads of 128, 24 / 32 rows each, bf16 168 / 254 us against 306 / 348, binary32 215 / 339 against 416 / 461; heads of 64 and 256 alike).
    p.shared = typical <= 32;
    auto slots_of = [&](uint32_t M) { return static_cast<uint32_t>(static_cast<uint64_t>(a.tokens) * group / M) + a.requests; };
    if (p.shared) {
        p.nt = c.head_dim == 256 || typical <= 16 ? 1 : 2;
    } else {
        // 128 rows a workgroup take fewer conversions and loads from LDS a row (a prompt of 8192 tokens, bf16, 620 us, with 64 rows
        // 860), 64 fill the chip from fewer rows and waste less of a short request's tile: taken for short keys on up to two tiles of 128
        // a CU (1000 tokens by themselves, bf16 49 -> 29 us, f32 62 -> 37), for requests of few rows (64 of one to 512 tokens, bf16, 166
        // -> 141), and in binary32, whose products outweigh the conversions, on up to four a CU.  Heads of 256, where 64 rows leave one
        // wavefront a SIMD, take them on up to one tile of 128 a CU (600 tokens by themselves, bf16, 35 -> 30; 1500 tokens 75 with 128
        // rows, 107 with 64).  Over 219 batches of 1 to 32 requests, heads of 64 and 128, the rule is 1 % behind the better of the two each
        // time, always 128 rows 15 %, always 64 4 %; over 156 with heads of 256 2 %, 9 % and 14 %.
        const uint64_t tiles = static_cast<uint64_t>(slots_of(128)) * c.kv_heads, keys = a.window ? std::min(a.window, a.max_length) : a.max_length;
        if (c.head_dim == 256) p.nt = tiles <= cus && keys < 1600 ? 1 : 2;
        else p.nt = typical <= 256 || (tiles <= 2ull * cus && keys < 1600) || (tiles <= 4ull * cus && a.dtype == PRISM_DTYPE_F32) ? 1 : 2;
    }
    p.M = p.shared ? 16 * p.nt : 64 * p.nt;
    p.slots = slots_of(p.M);
    uint64_t longest = a.max_length;
    if (a.window && longest > a.window + p.M / group) longest = a.window + p.M / group;  // what a tile sees of it
    const uint64_t tiles = static_cast<uint64_t>(p.slots) * c.kv_heads, blocks = longest / 64 + 1;
    uint64_t parts;
    if (p.shared) {
        // Four workgroups a CU were every request as long as max_length, so that long requests among short ones do not finish last,
        // where there are no more tiles than CUs, and for heads of 256, of which two fit a CU (with 8 and 4 workgroups, 8 heads of
        // 128: 4 requests of up to 16384 keys 22.7 -> 19.8 us, 8 31 -> 26.4, 16 of 4000 26 -> 23.4; 4 heads of 256: 3 requests of up to
        // 131072 110 -> 92, 64 of up to 2000 35 -> 31, but 8 of up to 131072 152 -> 156); else eight (64 requests of 8192 keys 125 ->
        // 115); four blocks a part at least, one for each wavefront.  Where the tiles alone fill the chip, up to twelve, as long as a
        // part has 48 blocks of 128 dimensions (64 requests of up to 16384 keys, heads of 128, with 8 / 12 / 16 workgroups a CU 138 /
        // 130 / 132 us, heads of 64 81 / 87 / 83).
        const uint64_t most = (tiles <= cus || c.head_dim == 256 ? 4ull : 8ull) * cus / tiles;
        parts = (blocks + 3) / 4;
        if (parts > most) parts = most;
        const uint64_t more = std::min<uint64_t>(12ull * cus / tiles, blocks * c.head_dim / 6144);
        if (tiles >= cus && parts < more) parts = more;
    } else {
        // A part writes and reads its rows' sums, as long as some five blocks take, so parts have 24 blocks or more until the
        // chip is full, and then up to eight workgroups a CU, eight blocks where the tiles leave CUs idle (33 blocks on 504
        // tiles: 141 us whole, 166 in two parts).
        parts = blocks / 24;
        if (parts > 8ull * cus / tiles) parts = 8ull * cus / tiles;
        uint64_t fill = 2ull * cus / tiles;
        if (fill > blocks / 8) fill = blocks / 8;
        if (parts < fill) parts = fill;
    }
    if (parts < 1) parts = 1;
    p.each = static_cast<uint32_t>((blocks + parts - 1) / parts);
    p.splits = static_cast<uint32_t>((blocks + p.each - 1) / p.each);
    return p;
}

template <typename T, int D>
int attend_launch(const AttendArgs &p, const Plan &plan, int *err, hipStream_t s) {
    const dim3 grid(p.slots * p.c.kv_heads, 1, p.splits);
    constexpr int most = D == 256 ? 1 : 2;  // row tiles of the kernel for few rows
    const bool wide = static_cast<uint64_t>(p.c.pages) * p.c.page_size * p.c.kv_heads * (D / 2) > 0xffffffffull;
    if (!plan.shared) {
        // 64 rows are four wavefronts' with 16 each; 128 are four with 32, or with heads of 256 eight with 16, whose registers
        // leave two on a SIMD (a prompt of 8192 tokens, 32 heads of 256, bf16, 2000 -> 1425 us, f32 2620 -> 1840).
        constexpr int nt = D == 256 ? 1 : 2, waves = D == 256 ? 8 : 4;
        if (plan.M == 64) {
            if (wide) k_attend4_tile<T, D, 1, 4, true><<<grid, 256, 0, s>>>(p, err);
            else k_attend4_tile<T, D, 1, 4, false><<<grid, 256, 0, s>>>(p, err);
        } else {
            if (wide) k_attend4_tile<T, D, nt, waves, true><<<grid, 64 * waves, 0, s>>>(p, err);
            else k_attend4_tile<T, D, nt, waves, false><<<grid, 64 * waves, 0, s>>>(p, err);
        }
    } else if (wide && plan.nt == 1) k_attend4_rows<T, D, 1, true><<<grid, 256, 0, s>>>(p, err);
    else if (wide) k_attend4_rows<T, D, most, true><<<grid, 256, 0, s>>>(p, err);
    else if (plan.nt == 1) k_attend4_rows<T, D, 1, false><<<grid, 256, 0, s>>>(p, err);
    else k_attend4_rows<T, D, most, false><<<grid, 256, 0, s>>>(p, err);
    int rc = launch_status();
    if (rc || p.splits == 1) return rc;
    const uint64_t rows = static_cast<uint64_t>(p.a.tokens) * p.a.heads;
    const uint32_t many = static_cast<uint32_t>(rows), quarter = static_cast<uint32_t>((rows + 3) / 4);
    if (p.splits > 8 && plan.shared) k_attend_join<T, D, 4, true><<<many, 256, 0, s>>>(p, plan.M, err);
    else if (p.splits > 8) k_attend_join<T, D, 4><<<many, 256, 0, s>>>(p, plan.M, err);
    else if (plan.shared) k_attend_join<T, D, 1, true><<<quarter, 256, 0, s>>>(p, plan.M, err);
    else k_attend_join<T, D, 1><<<quarter, 256, 0, s>>>(p, plan.M, err);
    return launch_status();
}
template <typename T>
int attend_headed(const AttendArgs &p, const Plan &plan, int *err, hipStream_t s) {
    switch (p.c.head_dim) {
    case 64: return attend_launch<T, 64>(p, plan, err, s);
    case 128: return attend_launch<T, 128>(p, plan, err, s);
    case 256: return attend_launch<T, 256>(p, plan, err, s);
    default: return kLaunchUnsupported;
    }
}

}  // namespace

size_t attention4_scratch_bytes(const prism_kv_cache &c, const prism_attention &a, uint32_t cus) {
    const Plan p = attend_plan(c, a, cus);
    return p.splits == 1 ? 0 : sizeof(float) * p.splits * (static_cast<size_t>(a.tokens) * a.heads) * (c.head_dim + 2);
}

int launch_attention4_paged(const prism_kv_cache &c, const prism_attention &a, void *scratch, uint32_t cus, int *err, hipStream_t s) {
    const Plan plan = attend_plan(c, a, cus);
    AttendArgs p{c, a, a.heads / c.kv_heads, 0, plan.slots, plan.each, plan.splits, static_cast<float *>(scratch), nullptr};
    p.page_log2 = static_cast<uint32_t>(__builtin_ctz(c.page_size));
    p.part_ml = p.part + static_cast<size_t>(plan.splits) * a.tokens * a.heads * c.head_dim;
    if (a.dtype == PRISM_DTYPE_F32) return attend_headed<float>(p, plan, err, s);
    if (a.dtype == PRISM_DTYPE_F16) return attend_headed<_Float16>(p, plan, err, s);
    return attend_headed<__bf16>(p, plan, err, s);
}

}  // namespace prism
