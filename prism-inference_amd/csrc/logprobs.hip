// logprobs.hip -- log probabilities of given tokens, entropy and the most probable alternatives of rows of logits (gfx950).
//
// A part of a row is held as its largest logit m and, of all its others, s = sum exp(x - m) and t = sum exp(x - m) (x - m), so
// that log S = log1p(s) and the entropy log1p(s) - t / (1 + s) keep their digits where one word has nearly all the
// weight.  A wavefront keeps one m for all its lanes: a new largest is rare (the logarithm of the tiles), so the loop over the
// row has no exchange between lanes, only a look whether any lane has a logit above m.
//
// The alternatives cost that loop one number for each 16 to 256 logits: the largest of a lane's group of them.  The k largest logits
// are among the groups whose largest is no smaller than the k-th largest of the lanes' largest, a few more than k groups unless
// many logits are equal, and only these are read again.
#include "serve_common.hpp"

namespace prism {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kNone = -__builtin_inff();
constexpr uint32_t kEach = 16, kTile = 64 * kEach;  // logits a lane and a wavefront take at a time
constexpr uint32_t kRoom = 128;                     // of a wavefront's list, twice the most alternatives
constexpr uint32_t kMostParts = 64;
constexpr uint32_t kGroups = 16;       // of a lane in a part
constexpr uint32_t kCandidates = 512;  // groups to read again that a workgroup notes down

struct Softmax {
    float m, s, t;
};
__device__ __forceinline__ float exp_of(float y) { return __builtin_amdgcn_exp2f(y * kLog2e); }
// a - b for a smaller a, no lower than where its exponential is 0 long since: the other factor of a 0 stays finite.
__device__ __forceinline__ float difference(float a, float b) { return fmaxf(a - b, -200.0f); }
__device__ __forceinline__ Softmax joined(Softmax a, Softmax b) {
    if (b.m > a.m) {
        const Softmax c = a;
        a = b;
        b = c;
    }
    // The second's largest counts as a word of weight exp(d) now.
    const float d = difference(b.m, a.m), e = exp_of(d);
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
    // The lanes whose key is above `least`.
    __device__ __forceinline__ void add(uint64_t key) {
        uint64_t on = __ballot(key > least);
        if (!on) return;
        if (count + __builtin_popcountll(on) > kRoom) {
            keep();
            on = __ballot(key > least);
        }
        if (key > least) held[count + __builtin_amdgcn_mbcnt_hi(on >> 32, __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(on), 0u))] = key;
        count += __builtin_popcountll(on);
        settle();
    }
};

// The keys that a workgroup's wavefronts hold, at most 64 each, as one ordered list of the k largest: a key's place is the
// number of larger ones.  counts[w] of held[w]; all[] has room for them and for seven zeros.
template <int WAVES>
__device__ __forceinline__ void merge_lists(const uint64_t (*held)[kRoom], const uint32_t *counts, uint64_t *all, uint64_t *out, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    uint32_t before = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) {
        before += w < wave ? counts[w] : 0;
        total += counts[w];
    }
    const uint64_t key = lane < counts[wave] ? held[wave][lane] : 0;
    if (key) all[before + lane] = key;
    if (threadIdx.x < 7) all[total + threadIdx.x] = 0;
    if (threadIdx.x < k) out[threadIdx.x] = 0;
    __syncthreads();
    uint32_t above = 0;
    if (__ballot(key != 0))
        for (uint32_t i = 0; i < total; i += 8) {
            uint64_t other[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) other[j] = all[i + j];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) above += other[j] > key;
        }
    if (key && above < k) out[above] = key;
    __syncthreads();
}

struct LogprobsArgs {
    prism_logprobs a;
    uint32_t parts, each;    // parts of a row, their logits
    uint32_t tiles, groups;  // tiles of a lane's group, groups of a lane in a part
    float *largest;          // [tokens][parts][groups][threads], of rows in parts
    Softmax *sums;           // [tokens][parts]
};

// The token that a row's log probability is asked of, and its logit; loaded before there is anything to wait for.
struct Given {
    int32_t id;
    float logit;
};
template <typename T>
__device__ __forceinline__ Given given_of(const prism_logprobs &a, uint64_t row) {
    Given g{-1, 0.0f};
    if (a.targets) g.id = a.targets[row];
    if (g.id >= 0 && g.id < static_cast<int64_t>(a.vocab)) g.logit = static_cast<float>(static_cast<const T *>(a.logits)[row * a.stride + g.id]);
    return g;
}

// What a row's log probabilities are taken from.
struct Scale {
    float m, log_s;
    bool wrong;
};
// A row's log probability and entropy from its sums, by one wavefront.
__device__ __forceinline__ Scale write_sums(const prism_logprobs &a, uint64_t row, Softmax w, Given g, int *err) {
    const float nan = __builtin_nanf("");
    const Scale r{w.m, log1pf(w.s), !(w.m < __builtin_inff()) || !(w.s >= 0.0f)};
    if ((threadIdx.x & 63) == 0) {
        if (r.wrong) raise_error(err, kErrNonfinite);
        if (a.logprobs) {
            const bool outside = g.id < -1 || g.id >= static_cast<int64_t>(a.vocab);
            if (outside) raise_error(err, kErrIndex);
            const float lp = g.logit == kNone ? kNone : (g.logit - r.m) - r.log_s;
            a.logprobs[row] = r.wrong || outside ? nan : g.id < 0 ? 0.0f : lp;
        }
        if (a.entropy) a.entropy[row] = r.wrong ? nan : r.m == kNone ? 0.0f : r.log_s - w.t / (1.0f + w.s);
    }
    return r;
}
// Its alternatives in order; threads 0 to top - 1.
__device__ __forceinline__ void write_top(const prism_logprobs &a, uint64_t row, const Scale &r, const uint64_t *keys) {
    if (threadIdx.x >= a.top) return;
    const uint64_t key = keys[threadIdx.x], at = row * a.top + threadIdx.x;
    a.top_ids[at] = r.wrong || !key ? -1 : static_cast<int32_t>(id_of(key));
    a.top_logprobs[at] = r.wrong ? __builtin_nanf("") : !key ? kNone : (logit_of(key) - r.m) - r.log_s;
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

constexpr uint32_t kBuckets = 256;  // of lanes, whose largest bound the k-th largest of all

// What finding the alternatives takes of LDS, for WAVES wavefronts.
template <int WAVES>
struct Shared {
    uint64_t held[WAVES][kRoom], all[64 * WAVES + 7], merged[64];
    uint32_t order[64 * WAVES < kBuckets ? 64 * WAVES : kBuckets], found[kCandidates], counts[WAVES], count, least;
    Scale scale;
};

// The row's alternatives, from the largest of its groups: largest[group][thread], `n` groups of the lanes of FROM
// wavefronts.  Meanwhile the second wavefront (or the only one) makes sh.scale by `sums`.
template <typename T, int WAVES, int FROM, typename F>
__device__ __forceinline__ void alternatives(const LogprobsArgs &p, uint64_t row, const float *largest, uint32_t n, Shared<WAVES> &sh, F sums) {
    constexpr uint32_t kThreads = 64 * WAVES, kSide = 64 * FROM, kFlight = 16;  // loads in flight
    constexpr uint32_t kShare = kThreads / kBuckets > 1 ? kThreads / kBuckets : 1, kOrders = kThreads / kShare / 64;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid / 64), k = p.a.top, all = n * kSide;
    const T *x = static_cast<const T *>(p.a.logits) + row * p.a.stride;
    uint32_t most = 0, here[kFlight];  // of the first groups, which are all of most rows
    auto look = [&](uint32_t i, uint32_t(&o)[kFlight]) {
        float v[kFlight];
#pragma unroll
        for (uint32_t j = 0; j < kFlight; ++j) v[j] = largest[min(i + j * kThreads + tid, all - 1)];
#pragma unroll
        for (uint32_t j = 0; j < kFlight; ++j) o[j] = i + j * kThreads + tid < all ? order_of(v[j]) : 0;
    };
    auto most_of = [&](const uint32_t(&o)[kFlight]) {
#pragma unroll
        for (uint32_t j = 0; j < kFlight; ++j) most = max(most, o[j]);
    };
    look(0, here);
    most_of(here);
    for (uint32_t i = kFlight * kThreads; i < all; i += kFlight * kThreads) {
        uint32_t more[kFlight];
        look(i, more);
        most_of(more);
    }
    uint32_t bucket = most;
#pragma unroll
    for (uint32_t d = 1; d < kShare; d *= 2) bucket = max(bucket, static_cast<uint32_t>(__shfl_xor(static_cast<int>(bucket), d)));
    if (tid % kShare == 0) sh.order[tid / kShare] = bucket;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    // The k-th largest of the buckets' largest, its bits from the top, two at a time (18 of them: sign, exponent and nine more;
    // what is left out only lets some more groups in).
    if (wave == 0) {
        uint32_t order[kOrders], bound = 0;
#pragma unroll
        for (uint32_t w = 0; w < kOrders; ++w) order[w] = sh.order[64 * w + lane];
#pragma unroll 1
        for (uint32_t bit = 1u << 30; bit >= 1u << 14; bit >>= 2) {
            uint32_t some[3] = {};
#pragma unroll
            for (uint32_t i = 0; i < 3; ++i)
#pragma unroll
                for (uint32_t w = 0; w < kOrders; ++w) some[i] += __builtin_popcountll(__ballot(order[w] >= (bound | (i + 1) * bit)));
            bound |= some[2] >= k ? 3 * bit : some[1] >= k ? 2 * bit : some[0] >= k ? bit : 0;
        }
        if (lane == 0) sh.least = max(bound, 1u);
    }
    if (wave == (WAVES > 1 ? 1 : 0)) {
        const Scale r = sums();
        if (lane == 0) sh.scale = r;
    }
    __syncthreads();
    const uint32_t least = sh.least;
    auto note = [&](uint32_t i, const uint32_t(&o)[kFlight]) {
#pragma unroll
        for (uint32_t j = 0; j < kFlight; ++j)
            if (o[j] >= least) {
                const uint32_t at = atomicAdd(&sh.count, 1u);
                if (at < kCandidates) sh.found[at] = i + j * kThreads + tid;
            }
    };
    if (__ballot(most >= least)) {
        note(0, here);
        for (uint32_t i = kFlight * kThreads; i < all; i += kFlight * kThreads) {
            uint32_t more[kFlight];
            look(i, more);
            note(i, more);
        }
    }
    __syncthreads();
    const uint32_t found = sh.count;
    Largest top;
    top.init(sh.held[wave], k);
    top.least = (static_cast<uint64_t>(least) << 32) - 1;
    const uint32_t log2_tiles = p.tiles <= 1 ? 0 : 32 - __builtin_clz(p.tiles - 1), log2_each = 4 + log2_tiles;
    // Logit e of a group: its id, and its key.
    auto id_at = [&](uint32_t code, uint32_t e) -> uint32_t {
        const uint32_t i = code / kSide, t = code % kSide, run = 16 / sizeof(T), j = e % kEach;
        const uint32_t tile = i % p.groups * p.tiles + e / kEach;
        return i / p.groups * p.each + (tile * FROM + t / 64) * kTile + j / run * (64 * run) + t % 64 * run + j % run;
    };
    auto key_at = [&](uint32_t code, uint32_t e) -> uint64_t {
        const uint32_t id = id_at(code, e), end = min(p.a.vocab, (code / kSide / p.groups + 1) * p.each);
        return e / kEach < p.tiles && id < end ? key_of(static_cast<float>(x[id]), id) : 0;
    };
    if (found <= kCandidates) {
        const uint32_t units = found << log2_each;
        for (uint32_t u = tid; u < (units + kThreads - 1) / kThreads * kThreads; u += 4 * kThreads) {
            uint64_t key[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t v = u + j * kThreads;
                key[j] = v < units ? key_at(sh.found[v >> log2_each], v & ((1u << log2_each) - 1)) : 0;
            }
#pragma unroll 1
            for (uint32_t j = 0; j < 4; ++j) top.add(j == 0 ? key[0] : j == 1 ? key[1] : j == 2 ? key[2] : key[3]);
        }
    } else {
        // Many of one size (words left out by a large negative logit, where fewer than k others are): each wavefront goes
        // through every WAVES-th run of groups by ascending id and passes those whose best could not be among the k largest.
        for (uint32_t i = 0; i < all; i += kThreads) {
            const uint32_t mine = i + tid, order_i = mine < all ? order_of(largest[mine]) : 0;
            const uint64_t best = order_i ? static_cast<uint64_t>(order_i) << 32 | (0xffffffffu - id_at(mine, 0)) : 0;
            uint64_t todo = ~0ull;
            for (;;) {
                const uint64_t on = __ballot(best > top.least) & todo;
                if (!on) break;
                const uint32_t l = static_cast<uint32_t>(__builtin_ctzll(on));
                todo &= ~(1ull << l);
                for (uint32_t e = lane; e - lane < 1u << log2_each; e += 64) top.add(e >> log2_each == 0 ? key_at(i + 64 * wave + l, e) : 0);
            }
        }
    }
    if (top.count > 64) top.keep();
    if (lane == 0) sh.counts[wave] = top.count;
    __syncthreads();
    merge_lists<WAVES>(sh.held, sh.counts, sh.all, sh.merged, k);
    write_top(p.a, row, sh.scale, sh.merged);
}

// A workgroup takes a part of a row, its wavefronts every WAVES-th tile of it, the next tile's loads in flight.  Memory bounds it:
// 1024 rows of 151936 binary32 logits, 20 alternatives, take 116 us, 5.4 TB/s (none 107, 64 of them 128; bf16 72), 4096 of 32000
// 100.  One row of 151936 takes 4.5 us in 38 parts, and its join 6.4.
template <typename T, int WAVES, bool TOP>
__global__ __launch_bounds__(64 * WAVES) void k_logprobs(LogprobsArgs p, int *err) {
    __shared__ float group_largest[TOP ? kGroups : 1][64 * WAVES], part[WAVES][3];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const uint64_t row = blockIdx.x / p.parts;
    const uint32_t which = blockIdx.x % p.parts;
    const uint32_t begin = which * p.each, end = min(p.a.vocab, begin + p.each);
    const T *x = static_cast<const T *>(p.a.logits) + row * p.a.stride;
    Softmax w{kNone, 0.0f, 0.0f};  // s and t of this lane
    Logits<T> next;
    uint32_t base = begin + wave * kTile, left = p.tiles, group = 0;
    float largest = kNone;
    auto note = [&] {  // the largest of a group
        if (p.parts == 1) group_largest[group][tid] = largest;
        else p.largest[(static_cast<uint64_t>(blockIdx.x) * p.groups + group) * (64 * WAVES) + tid] = largest;
        ++group;
        left = p.tiles;
        largest = kNone;
    };
    if (base < end) next.load(x, base, end);
    for (; base < end; base += WAVES * kTile) {
        Logits<T> now = next;
        if (base + WAVES * kTile < end) next.load(x, base + WAVES * kTile, end);
        float most = now.v[0];
#pragma unroll
        for (uint32_t i = 1; i < kEach; ++i) most = fmaxf(most, now.v[i]);
        if constexpr (TOP) {
            largest = fmaxf(largest, most);
            if (--left == 0) note();
        }
        if (__ballot(most > w.m)) {
            float m = most;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
            if (w.m != kNone) {  // the former largest counts as another word, of lane 0
                const float d = difference(w.m, m), e = exp_of(d);
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
    if constexpr (TOP)
        while (group < p.groups) note();
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        w.s += __shfl_xor(w.s, d);
        w.t += __shfl_xor(w.t, d);
    }
    if constexpr (WAVES > 1) {
        if (lane == 0) {
            part[wave][0] = w.m;
            part[wave][1] = w.s;
            part[wave][2] = w.t;
        }
    }
    __syncthreads();
    auto joined_parts = [&] {
        if constexpr (WAVES > 1) {
            w = Softmax{part[0][0], part[0][1], part[0][2]};
#pragma unroll
            for (int i = 1; i < WAVES; ++i) w = joined(w, Softmax{part[i][0], part[i][1], part[i][2]});
        }
        return w;
    };
    if (p.parts > 1) {
        if (tid == 0) p.sums[blockIdx.x] = joined_parts();
        return;
    }
    const Given given = given_of<T>(p.a, row);
    auto sums = [&] { return write_sums(p.a, row, joined_parts(), given, err); };
    if constexpr (TOP) {
        __shared__ Shared<WAVES> sh;
        alternatives<T, WAVES, WAVES>(p, row, &group_largest[0][0], p.groups, sh, sums);
    } else {
        if (wave == 0) sums();
    }
}

// A workgroup finishes a row that was in parts, with sixteen wavefronts, since what it waits for is the chain from the groups'
// largest to the logits read again: 6.4 us for one row.
constexpr int kJoinWaves = 16;
template <typename T, bool TOP>
__global__ __launch_bounds__(TOP ? 64 * kJoinWaves : 64) void k_logprobs_join(LogprobsArgs p, int *err) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t row = blockIdx.x;
    const Given given = given_of<T>(p.a, row);
    Softmax w{kNone, 0.0f, 0.0f};
    if (lane < p.parts) w = p.sums[row * p.parts + lane];
    auto sums = [&] {
#pragma unroll
        for (int d = 1; d < 64; d *= 2) w = joined(w, Softmax{__shfl_xor(w.m, d), __shfl_xor(w.s, d), __shfl_xor(w.t, d)});
        return write_sums(p.a, row, w, given, err);
    };
    if constexpr (TOP) {
        __shared__ Shared<kJoinWaves> sh;
        alternatives<T, kJoinWaves, 4>(p, row, p.largest + row * p.parts * p.groups * 256, p.parts * p.groups, sh, sums);
    } else {
        sums();
    }
}

// How a call runs: wavefronts of a workgroup, parts of a row, and groups.
struct Plan {
    uint32_t waves, parts, each, tiles, groups;
};
Plan plan_of(const prism_logprobs &a, uint32_t cus) {
    Plan p;
    p.waves = a.vocab <= 4 * kTile ? 1 : 4;
    const uint32_t tiles = (a.vocab + p.waves * kTile - 1) / (p.waves * kTile);
    // Up to a row a CU are split until some four workgroups a CU share the logits, a tile for each wavefront at least; more keep the
    // memory busy whole (rows of 151936 binary32 logits, 20 alternatives, 256 CUs, whole / split: 200 rows 36 / 32 us, 256 42 / 38,
    // 400 52 / 70, 900 106 / 145).
    uint32_t parts = p.waves == 1 || a.tokens > cus ? 1 : (4 * cus + a.tokens - 1) / a.tokens;
    if (parts > tiles) parts = tiles;
    if (parts > kMostParts) parts = kMostParts;
    uint32_t some = (tiles + parts - 1) / parts;
    if (some > kGroups * 16) some = kGroups * 16;  // groups of 256 logits at most
    p.parts = (tiles + some - 1) / some;
    p.each = some * p.waves * kTile;
    p.tiles = (some + kGroups - 1) / kGroups;
    p.groups = (some + p.tiles - 1) / p.tiles;
    return p;
}

template <typename T, bool TOP>
int logprobs_launch(const LogprobsArgs &p, uint32_t waves, int *err, hipStream_t s) {
    const uint32_t grid = p.a.tokens * p.parts;
    if (waves == 1) k_logprobs<T, 1, TOP><<<grid, 64, 0, s>>>(p, err);
    else k_logprobs<T, 4, TOP><<<grid, 256, 0, s>>>(p, err);
    const int rc = launch_status();
    if (rc || p.parts == 1) return rc;
    k_logprobs_join<T, TOP><<<p.a.tokens, TOP ? 64 * kJoinWaves : 64, 0, s>>>(p, err);
    return launch_status();
}
template <typename T>
int logprobs_typed(const LogprobsArgs &p, uint32_t waves, int *err, hipStream_t s) {
    return p.a.top ? logprobs_launch<T, true>(p, waves, err, s) : logprobs_launch<T, false>(p, waves, err, s);
}

}  // namespace

size_t logprobs_scratch_bytes(const prism_logprobs &a, uint32_t cus) {
    const Plan q = plan_of(a, cus);
    return q.parts == 1 ? 0 : static_cast<size_t>(a.tokens) * q.parts * (sizeof(Softmax) + (a.top ? 4ull * q.groups * 256 : 0));
}

int launch_logprobs(const prism_logprobs &a, void *scratch, uint32_t cus, int *err, hipStream_t s) {
    const Plan q = plan_of(a, cus);
    LogprobsArgs p{a, q.parts, q.each, q.tiles, q.groups, static_cast<float *>(scratch), nullptr};
    p.sums = reinterpret_cast<Softmax *>(p.largest + (a.top ? static_cast<size_t>(a.tokens) * q.parts * q.groups * 256 : 0));
    if (a.dtype == PRISM_DTYPE_F32) return logprobs_typed<float>(p, q.waves, err, s);
    if (a.dtype == PRISM_DTYPE_F16) return logprobs_typed<_Float16>(p, q.waves, err, s);
    return logprobs_typed<__bf16>(p, q.waves, err, s);
}

}  // namespace prism
