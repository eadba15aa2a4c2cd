// logprobs.hip -- log probabilities of given tokens, entropy and the most probable alternatives of rows of logits (gfx950).
//
// A part of a row is held as its largest logit m and, of all its others, s = sum exp(x - m) and t = sum exp(x - m) (x - m), so
// that log S = log1p(s) and the entropy log1p(s) - t / (1 + s) keep their digits where one word has nearly all the
// weight.  A wavefront keeps one m for all its lanes: a new largest is rare (the logarithm of the tiles), so the loop over the
// row has no exchange between lanes, only a look whether any lane has a logit above what is held.
// The alternatives ride along: a wavefront keeps the largest in a list, and that look is against the last of
// them.  One pass over the logits, whose bytes bound long rows.
#include "serve_common.hpp"

namespace prism {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kNone = -__builtin_inff();
constexpr uint32_t kEach = 16, kTile = 64 * kEach;  // logits a lane and a wavefront take at a time
constexpr uint32_t kRoom = 128;                     // of a wavefront's list, twice the most alternatives
constexpr uint32_t kMostParts = 64;

struct Softmax {
    float m, s, t;
};
__device__ __forceinline__ float exp_of(float y) { return __builtin_amdgcn_exp2f(y * kLog2e); }
__device__ __forceinline__ Softmax joined(Softmax a, Softmax b) {
    if (b.m > a.m) {
        const Softmax c = a;
        a = b;
        b = c;
    }
    // The second's largest counts as a word of weight exp(d) now.
    const float d = b.m - a.m, e = exp_of(d);
    const bool none = b.m == kNone;
    a.t += none ? b.t : e * (b.t + d * (b.s + 1.0f));
    a.s += none ? b.s : e * (b.s + 1.0f);  // a NaN of a part without a finite logit goes on
    return a;
}

// Larger logits have larger keys, and of equal ones the word of the lower id; 0 is none.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 as 0
    return x > kNone ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0;
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
    const uint32_t u = order_of(x);
    return u ? static_cast<uint64_t>(u) << 32 | (0xffffffffu - id) : 0;
}
__device__ __forceinline__ uint32_t id_of(uint64_t key) { return 0xffffffffu - static_cast<uint32_t>(key); }
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t u = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// What a wavefront's lanes wrote to LDS is there for the others.
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wavefront's largest keys: `count` of them in LDS, of which at most the k largest matter; keys up to `least` no longer do.
struct Largest {
    uint64_t *held;  // [kRoom]
    uint32_t k, count;
    uint64_t least;

    __device__ __forceinline__ void init(uint64_t *memory, uint32_t top) {
        held = memory;
        k = top;
        count = 0;
        least = 0;
    }
    // Down to the k largest, in order: a key's place is the number of larger ones.
    __device__ __forceinline__ void keep() {
        const uint32_t lane = threadIdx.x & 63;
        const uint64_t a = lane < count ? held[lane] : 0, b = 64 + lane < count ? held[64 + lane] : 0;
        settle();
        if (lane >= count) held[lane] = 0;
        if (64 + lane >= count) held[64 + lane] = 0;
        settle();
        uint32_t above_a = 0, above_b = 0;
        for (uint32_t i = 0; i < count; i += 4) {
            uint64_t other[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) other[j] = held[i + j];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                above_a += other[j] > a;
                above_b += other[j] > b;
            }
        }
        settle();
        if (a && above_a < k) held[above_a] = a;
        if (b && above_b < k) held[above_b] = b;
        settle();
        count = min(count, k);
        if (count == k) least = held[k - 1];
    }
    // With the largest order of each lane's keys: where k lanes or more have keys of account, none below the k-th
    // largest of those can be among the k largest of all.  Its bits from the top.
    __device__ __forceinline__ void raise(uint32_t order) {
        if (static_cast<uint32_t>(__builtin_popcountll(__ballot(order > static_cast<uint32_t>(least >> 32)))) < k) return;
        uint32_t at = 0;
#pragma unroll 1
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
            if (static_cast<uint32_t>(__builtin_popcountll(__ballot(order >= (at | bit)))) >= k) at |= bit;
        const uint64_t below = (static_cast<uint64_t>(at) << 32) - 1;
        if (at && below > least) least = below;
    }
    // The lanes whose key is above `least`, where there is room for them.
    __device__ __forceinline__ void put(uint64_t key) {
        const uint64_t on = __ballot(key > least);
        if (!on) return;
        if (key > least) held[count + __builtin_amdgcn_mbcnt_hi(on >> 32, __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(on), 0u))] = key;
        count += __builtin_popcountll(on);
        settle();
    }
    // All keys of a tile, key(i) for i < kEach, whose largest order in this lane is `order`.
    template <typename F>
    __device__ __forceinline__ void add(uint32_t order, F key) {
        raise(order);
        uint32_t some = 0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) some += __builtin_popcountll(__ballot(key(i) > least));
        if (count + some <= kRoom) {
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i) put(key(i));
            return;
        }
#pragma unroll 1
        for (uint32_t i = 0; i < kEach; ++i) {  // many of one size, or rows that rise: sorted as often as it takes
            uint64_t mine = key(0);
#pragma unroll
            for (uint32_t j = 1; j < kEach; ++j) mine = i == j ? key(j) : mine;
            if (count + __builtin_popcountll(__ballot(mine > least)) > kRoom) keep();
            put(mine);
        }
    }
};

// The lists of a workgroup's wavefronts, k ordered keys each, as one: into out[k].
template <int WAVES>
__device__ __forceinline__ void merge_lists(uint64_t (*held)[kRoom], uint64_t *out, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    if (threadIdx.x < k) out[threadIdx.x] = 0;
    __syncthreads();
    const uint64_t key = lane < k ? held[wave][lane] : 0;
    uint32_t above = lane;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
        const uint64_t *other = held[(wave + w) % WAVES];
        for (uint32_t i = 0; i < k; i += 4)
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) above += i + j < k && other[i + j] > key;
    }
    if (key && above < k) out[above] = key;
    __syncthreads();
}

struct LogprobsArgs {
    prism_logprobs a;
    uint32_t parts, each;  // parts of a row, their logits
    uint64_t *keys;        // [tokens][parts][top]
    Softmax *sums;         // [tokens][parts]
};

// A row's results from its sums and ordered alternatives; one wavefront.
template <typename T>
__device__ __forceinline__ void write_row(const prism_logprobs &a, uint64_t row, Softmax w, const uint64_t *keys, int *err) {
    const uint32_t lane = threadIdx.x & 63;
    const float nan = __builtin_nanf(""), log_s = log1pf(w.s);
    const bool wrong = !(w.m < __builtin_inff()) || !(w.s >= 0.0f);
    if (lane == 0) {
        if (wrong) raise_error(err, kErrNonfinite);
        if (a.logprobs) {
            const int32_t id = a.targets[row];
            float lp = 0.0f;
            if (id < -1 || id >= static_cast<int64_t>(a.vocab)) {
                raise_error(err, kErrIndex);
                lp = nan;
            } else if (id >= 0) {
                const float v = static_cast<float>(static_cast<const T *>(a.logits)[row * a.stride + id]);
                lp = v == kNone ? kNone : (v - w.m) - log_s;
            }
            a.logprobs[row] = wrong ? nan : lp;
        }
        if (a.entropy) a.entropy[row] = wrong ? nan : w.m == kNone ? 0.0f : log_s - w.t / (1.0f + w.s);
    }
    if (lane < a.top) {
        const uint64_t key = keys[lane];
        a.top_ids[row * a.top + lane] = wrong || !key ? -1 : static_cast<int32_t>(id_of(key));
        a.top_logprobs[row * a.top + lane] = wrong ? nan : !key ? kNone : (logit_of(key) - w.m) - log_s;
    }
}

// One lane's logits of a tile.
template <typename T>
struct Logits {
    static constexpr uint32_t kRun = 16 / sizeof(T);  // neighbours, in one load
    float v[kEach];
    static __device__ __forceinline__ uint32_t id(uint32_t base, uint32_t i) {
        return base + i / kRun * (64 * kRun) + (threadIdx.x & 63) * kRun + i % kRun;
    }
    __device__ __forceinline__ void load(const T *x, uint32_t base, uint32_t end) {
        if (base + kTile <= end) {
            typedef T Run __attribute__((ext_vector_type(kRun)));
            Run r[kEach / kRun];
#pragma unroll
            for (uint32_t j = 0; j < kEach / kRun; ++j) r[j] = load_any<Run>(x + id(base, kRun * j));
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i) v[i] = static_cast<float>(r[i / kRun][i % kRun]);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i) v[i] = id(base, i) < end ? static_cast<float>(x[id(base, i)]) : kNone;
        }
    }
};

// A workgroup takes a part of a row, its wavefronts every WAVES-th tile of it.
template <typename T, int WAVES, bool TOP>
__global__ __launch_bounds__(64 * WAVES) void k_logprobs(LogprobsArgs p, int *err) {
    __shared__ uint64_t held[TOP ? WAVES : 1][kRoom], merged[64];
    __shared__ float part[WAVES][3];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint64_t row = blockIdx.x / p.parts;
    const uint32_t which = blockIdx.x % p.parts;
    const uint32_t begin = which * p.each, end = min(p.a.vocab, begin + p.each);
    const T *x = static_cast<const T *>(p.a.logits) + row * p.a.stride;
    Softmax w{kNone, 0.0f, 0.0f};  // s and t of this lane
    Largest top;
    top.init(held[TOP ? wave : 0], p.a.top);
    Logits<T> next;
    uint32_t base = begin + wave * kTile;
    if (base < end) next.load(x, base, end);
    for (; base < end; base += WAVES * kTile) {
        Logits<T> now = next;
        if (base + WAVES * kTile < end) next.load(x, base + WAVES * kTile, end);
        float most = now.v[0];
#pragma unroll
        for (uint32_t i = 1; i < kEach; ++i) most = fmaxf(most, now.v[i]);
        // A later word of the size of the last alternative has a higher id.
        if (__ballot(TOP ? order_of(most) > static_cast<uint32_t>(top.least >> 32) : most > w.m)) {
            if constexpr (TOP) top.add(order_of(most), [&](uint32_t i) { return key_of(now.v[i], Logits<T>::id(base, i)); });
            if (__ballot(most > w.m)) {
                float m = most;
#pragma unroll
                for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
                if (w.m != kNone) {  // the former largest counts as another word, of lane 0
                    const float d = w.m - m, e = exp_of(d);
                    w.t = e * (w.t + d * w.s);
                    w.s *= e;
                    if (lane == 0) {
                        w.s += e;
                        w.t += e * d;
                    }
                }
                w.m = m;
                uint64_t owner = 0;  // one logit of this size stands for m and is left out
#pragma unroll
                for (uint32_t i = 0; i < kEach; ++i) {
                    const uint64_t on = owner ? 0 : __ballot(now.v[i] == m);
                    if (on) {
                        owner = on;
                        if (lane == static_cast<uint32_t>(__builtin_ctzll(on))) now.v[i] = kNone;
                    }
                }
            }
        }
        const float ref = w.m == kNone ? 0.0f : w.m;
        float s[4] = {}, t[4] = {};
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const float y = now.v[i] - ref, e = exp_of(y);
            s[i % 4] += e;
            t[i % 4] = __builtin_fmaf(e, fmaxf(y, -200.0f), t[i % 4]);  // e is 0 there; a masked word's y is -infinity
        }
        w.s += (s[0] + s[1]) + (s[2] + s[3]);
        w.t += (t[0] + t[1]) + (t[2] + t[3]);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        w.s += __shfl_xor(w.s, d);
        w.t += __shfl_xor(w.t, d);
    }
    if constexpr (TOP) {
        top.keep();
        if (top.count < p.a.top && lane >= top.count) held[wave][lane] = 0;
    }
    const uint64_t *keys = held[0];
    if constexpr (WAVES > 1) {
        if (lane == 0) {
            part[wave][0] = w.m;
            part[wave][1] = w.s;
            part[wave][2] = w.t;
        }
        if constexpr (TOP) {
            __syncthreads();
            merge_lists<WAVES>(held, merged, p.a.top);
            keys = merged;
        } else {
            __syncthreads();
        }
        if (wave) return;
        w = Softmax{part[0][0], part[0][1], part[0][2]};
#pragma unroll
        for (int i = 1; i < WAVES; ++i) w = joined(w, Softmax{part[i][0], part[i][1], part[i][2]});
    } else {
        settle();
    }
    if (p.parts == 1) {
        write_row<T>(p.a, row, w, keys, err);
        return;
    }
    if (lane == 0) p.sums[blockIdx.x] = w;
    if (TOP && lane < p.a.top) p.keys[static_cast<uint64_t>(blockIdx.x) * p.a.top + lane] = keys[lane];
}

// A workgroup joins the parts of a row, each wavefront a quarter of their lists first.
template <typename T, bool TOP>
__global__ __launch_bounds__(256) void k_logprobs_join(LogprobsArgs p, int *err) {
    __shared__ uint64_t held[4][kRoom], merged[64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint64_t row = blockIdx.x;
    if constexpr (TOP) {
        const uint32_t some = (p.parts + 3) / 4, from = min(p.parts, wave * some), n = (min(p.parts, from + some) - from) * p.a.top;
        const uint64_t *keys = p.keys + (row * p.parts + from) * p.a.top;
        uint64_t key[kEach];
        uint32_t most = 0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            key[i] = 64 * i + lane < n ? keys[64 * i + lane] : 0;
            most = max(most, static_cast<uint32_t>(key[i] >> 32));
        }
        Largest top;
        top.init(held[wave], p.a.top);
        top.add(most, [&](uint32_t i) { return key[i]; });
        top.keep();
        if (lane >= top.count) held[wave][lane] = 0;
        __syncthreads();
        merge_lists<4>(held, merged, p.a.top);
    }
    if (wave) return;
    Softmax w{kNone, 0.0f, 0.0f};
    if (lane < p.parts) w = p.sums[row * p.parts + lane];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) w = joined(w, Softmax{__shfl_xor(w.m, d), __shfl_xor(w.s, d), __shfl_xor(w.t, d)});
    write_row<T>(p.a, row, w, merged, err);
}

struct Parts {
    uint32_t parts, each;
};
// Rows are split until some 1024 workgroups share the logits, a tile for each wavefront at least.
Parts parts_of(const prism_logprobs &a) {
    const uint32_t tiles = (a.vocab + 4 * kTile - 1) / (4 * kTile);
    uint32_t parts = (1024 + a.tokens - 1) / a.tokens;
    if (parts > tiles) parts = tiles;
    if (parts > kMostParts) parts = kMostParts;
    const uint32_t some = (tiles + parts - 1) / parts;
    return Parts{(tiles + some - 1) / some, some * 4 * kTile};
}

template <typename T, bool TOP>
int logprobs_launch(const LogprobsArgs &p, int *err, hipStream_t s) {
    const uint32_t grid = p.a.tokens * p.parts;
    if (p.a.vocab <= 2 * kTile) k_logprobs<T, 1, TOP><<<grid, 64, 0, s>>>(p, err);
    else k_logprobs<T, 4, TOP><<<grid, 256, 0, s>>>(p, err);
    const int rc = launch_status();
    if (rc || p.parts == 1) return rc;
    k_logprobs_join<T, TOP><<<p.a.tokens, 256, 0, s>>>(p, err);
    return launch_status();
}
template <typename T>
int logprobs_typed(const LogprobsArgs &p, int *err, hipStream_t s) {
    return p.a.top ? logprobs_launch<T, true>(p, err, s) : logprobs_launch<T, false>(p, err, s);
}

}  // namespace

size_t logprobs_scratch_bytes(const prism_logprobs &a, uint32_t) {
    const Parts q = parts_of(a);
    return q.parts == 1 ? 0 : static_cast<size_t>(a.tokens) * q.parts * (sizeof(uint64_t) * a.top + sizeof(Softmax));
}

int launch_logprobs(const prism_logprobs &a, void *scratch, uint32_t, int *err, hipStream_t s) {
    const Parts q = parts_of(a);
    LogprobsArgs p{a, q.parts, q.each, static_cast<uint64_t *>(scratch), nullptr};
    p.sums = reinterpret_cast<Softmax *>(p.keys + static_cast<size_t>(a.tokens) * q.parts * a.top);
    if (a.dtype == PRISM_DTYPE_F32) return logprobs_typed<float>(p, err, s);
    if (a.dtype == PRISM_DTYPE_F16) return logprobs_typed<_Float16>(p, err, s);
    return logprobs_typed<__bf16>(p, err, s);
}

}  // namespace prism
