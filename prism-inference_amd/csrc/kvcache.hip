// kvcache.hip -- what keeps the paged 8-bit cache of many requests (gfx950): pages and slots
// of a step's new tokens, rotary positions, and the append that quantizes keys and values.
#include "serve_common.hpp"

namespace prism {

namespace {

// ---- plan -------------------------------------------------------------------------------
// Exclusive sums over the requests of their new tokens, of the pages they need and of those
// they give back; everything else follows from these per token.  One workgroup makes the
// sums (a few thousand requests are a few loads a thread); the tokens are filled by the same
// workgroup, or by a grid where they are many.

constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kPlanOwnFill = 4096;  // tokens the summing workgroup fills by itself

struct PlanScratch {
    int32_t *need_base, *back_base;  // [requests + 1]
    int32_t *head;                   // {tokens, stack height before pages are taken, refused}
};
PlanScratch plan_scratch(void *p, uint32_t requests) {
    int32_t *i = static_cast<int32_t *>(p);
    return PlanScratch{i, i + requests + 1, i + 2 * (requests + 1)};
}

__device__ __forceinline__ int64_t pages_of(int64_t tokens, uint32_t page) { return (tokens + page - 1) / page; }

// The last r in [0, n) with base[r] <= x, for base ascending with base[0] <= x.
__device__ __forceinline__ uint32_t last_at_most(const int32_t *base, uint32_t n, int32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (base[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void plan_fill(const prism_kv_plan &p, const PlanScratch &sc, uint32_t t, int32_t tokens,
                                          int32_t height) {
    int32_t position = 0, slot = -1, owner = -1;
    if (static_cast<int32_t>(t) < tokens) {
        // Requests without new tokens share their offset with the next: the last of equals has it.
        const uint32_t r = last_at_most(p.offsets, p.requests, static_cast<int32_t>(t));
        const int32_t old = p.new_lengths[r] - p.added[r];
        const int32_t page = static_cast<int32_t>(p.page_size);
        position = old + static_cast<int32_t>(t) - p.offsets[r];
        owner = static_cast<int32_t>(r);
        const int32_t held = static_cast<int32_t>(pages_of(old, p.page_size)), j = position / page, place = position % page;
        int32_t *entry = p.block_table + static_cast<uint64_t>(r) * p.max_pages + j;
        int32_t id;
        if (j < held) {
            id = *entry;
        } else {
            id = p.free_pages[height - 1 - (sc.need_base[r] + j - held)];
            if (place == 0) *entry = id;  // a new page begins with a new token
        }
        const int64_t s = static_cast<int64_t>(id) * page + place;
        slot = id >= 0 && s <= 0x7fffffff ? static_cast<int32_t>(s) : -1;
    }
    p.positions[t] = position;
    p.slots[t] = slot;
    p.owners[t] = owner;
}

__device__ __forceinline__ int64_t wave_inclusive(int64_t v) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int64_t o = __shfl_up(v, d);
        if (lane >= static_cast<uint32_t>(d)) v += o;
    }
    return v;
}

__global__ __launch_bounds__(kPlanThreads) void k_plan(prism_kv_plan p, PlanScratch sc, int fill, int *err) {
    __shared__ int64_t part[3][kPlanThreads / 64];
    __shared__ int bad_any;
    const uint32_t tid = threadIdx.x, wave = tid / 64, waves = blockDim.x / 64;
    if (tid == 0) bad_any = 0;
    __syncthreads();
    const uint32_t each = (p.requests + blockDim.x - 1) / blockDim.x;
    const uint32_t r0 = min(p.requests, tid * each), r1 = min(p.requests, r0 + each);
    int64_t sum[3] = {0, 0, 0};  // tokens, pages needed, pages given back
    bool bad = false;
    for (uint32_t r = r0; r < r1; ++r) {
        const int64_t n = p.lengths[r], a = p.added[r];
        const bool ended = a == -1;
        bad |= n < 0 || a < -1 || pages_of(n + (ended ? 0 : a), p.page_size) > p.max_pages;
        const int64_t held = pages_of(n, p.page_size);
        sum[0] += ended ? 0 : a;
        sum[1] += ended ? 0 : pages_of(n + a, p.page_size) - held;
        sum[2] += ended ? held : 0;
    }
    if (bad) bad_any = 1;
    const int32_t count = *p.free_count;
    int64_t before[3], total[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int64_t inc = wave_inclusive(sum[i]);
        before[i] = inc - sum[i];
        if ((tid & 63) == 63) part[i][wave] = inc;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        total[i] = 0;
        for (uint32_t w = 0; w < waves; ++w) {
            if (w < wave) before[i] += part[i][w];
            total[i] += part[i][w];
        }
    }
    const bool wrong = bad_any || count < 0 || static_cast<uint32_t>(count) > p.free_capacity ||
                       total[2] > static_cast<int64_t>(p.free_capacity) - count || total[0] > p.max_tokens;
    const int64_t height = count + total[2];
    const int64_t missing = wrong || total[1] <= height ? 0 : total[1] - height;
    const bool refused = wrong || missing > 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const int32_t n = p.lengths[r], a = p.added[r];
        p.offsets[r] = refused ? 0 : static_cast<int32_t>(before[0]);
        if (refused) {
            p.new_lengths[r] = n;
            continue;
        }
        sc.need_base[r] = static_cast<int32_t>(before[1]);
        sc.back_base[r] = static_cast<int32_t>(before[2]);
        p.new_lengths[r] = a == -1 ? 0 : n + a;
        const int64_t held = pages_of(n, p.page_size);
        before[0] += a == -1 ? 0 : a;
        before[1] += a == -1 ? 0 : pages_of(static_cast<int64_t>(n) + a, p.page_size) - held;
        before[2] += a == -1 ? held : 0;
    }
    const int32_t tokens = refused ? 0 : static_cast<int32_t>(total[0]);
    if (tid == 0) {
        p.offsets[p.requests] = tokens;
        p.counts[0] = static_cast<int32_t>(refused ? count : height - total[1]);
        p.counts[1] = tokens;
        p.counts[2] = static_cast<int32_t>(refused ? 0 : total[1]);
        p.counts[3] = static_cast<int32_t>(missing < 0x7fffffff ? missing : 0x7fffffff);
        sc.head[0] = tokens;
        sc.head[1] = static_cast<int32_t>(refused ? 0 : height);
        if (wrong) raise_error(err, kErrIndex);
        if (missing) raise_error(err, kErrPages);
    }
    __syncthreads();
    if (!refused)
        for (int32_t b = static_cast<int32_t>(tid); b < total[2]; b += static_cast<int32_t>(blockDim.x)) {
            const uint32_t r = last_at_most(sc.back_base, p.requests, b);
            p.free_pages[count + b] = p.block_table[static_cast<uint64_t>(r) * p.max_pages + (b - sc.back_base[r])];
        }
    if (!fill) return;
    __syncthreads();
    for (uint32_t t = tid; t < p.max_tokens; t += blockDim.x) plan_fill(p, sc, t, tokens, static_cast<int32_t>(height));
}

__global__ __launch_bounds__(256) void k_plan_fill(prism_kv_plan p, PlanScratch sc) {
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    if (t < p.max_tokens) plan_fill(p, sc, t, sc.head[0], sc.head[1]);
}

// ---- rotary positions -------------------------------------------------------------------
// One workgroup rotates kRopeTokens tokens of some heads: it first makes their cosines and
// sines in binary64 (one pair of them serves every head), then a lane takes four consecutive
// elements of a row and their partners.  binary64 FMAs run at the binary32 rate here, so
// the exact rotation costs no more than a rounded one; memory bounds it.

constexpr uint32_t kRopeTokens = 4;

template <typename T, int D>
__global__ __launch_bounds__(256) void k_rope(RopeRows a, RopeRows b, Rotation rot, const int32_t *positions, uint32_t tokens,
                                              uint32_t heads_each, double eps, int *err) {
    constexpr uint32_t kLanes = D / 4, kRows = 64 / kLanes;  // lanes of a row, rows of a wavefront
    __shared__ double cs[kRopeTokens][D / 2], sn[kRopeTokens][D / 2];
    const uint32_t tid = threadIdx.x, lane = tid & 63, half = rot.dims / 2;
    const uint32_t t0 = blockIdx.x * kRopeTokens, nt = min(kRopeTokens, tokens - t0);
    for (uint32_t i = tid; i < nt * half; i += 256) {
        const uint32_t t = i / half, k = i % half;
        double s, c;
        sincos(static_cast<double>(positions[t0 + t]) * rot.freq[k], &s, &c);
        cs[t][k] = c * rot.magnitude;
        sn[t][k] = s * rot.magnitude;
    }
    __syncthreads();
    const uint32_t all = a.heads + b.heads, h0 = blockIdx.y * heads_each, h1 = min(all, h0 + heads_each);
    const uint32_t groups = (h1 - h0 + kRows - 1) / kRows;
    const uint32_t e0 = 4 * (lane % kLanes);
    bool bad = false;
    for (uint32_t it = tid / 64; it < nt * groups; it += 4) {
        const uint32_t t = it / groups, h = h0 + it % groups * kRows + lane / kLanes;
        const bool live = h < h1;
        const RopeRows &m = h < a.heads ? a : b;
        const uint32_t hh = min(h, h1 - 1) - (h < a.heads ? 0 : a.heads);
        const T *x = static_cast<const T *>(m.x) + (t0 + t) * m.x_stride + static_cast<uint64_t>(hh) * D;
        f32x4 v{0, 0, 0, 0};
        if (live) v = load4(x + e0);
        double scale = 1.0;
        if (m.norm) {
            double q = 0.0;
#pragma unroll
            for (int j = 0; j < 4; ++j) q = __builtin_fma(static_cast<double>(v[j]), static_cast<double>(v[j]), q);
#pragma unroll
            for (uint32_t d = 1; d < kLanes; d *= 2) q += __shfl_xor(q, d);
            scale = 1.0 / sqrt(q / D + eps);
        }
        if (!live) continue;
        f32x4 out;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t e = e0 + j;
            bad |= !finite(v[j]);
            double y = v[j];
            if (m.norm) y = y * scale * m.norm[e];
            if (e < rot.dims) {
                const bool first = rot.interleaved ? !(e & 1) : e < half;
                const uint32_t o = rot.interleaved ? e ^ 1 : first ? e + half : e - half;
                const uint32_t k = rot.interleaved ? e / 2 : first ? e : o;
                double z = rot.interleaved ? v[j ^ 1] : static_cast<float>(x[o]);
                if (m.norm) z = z * scale * m.norm[o];
                y = y * cs[t][k] + (first ? -z : z) * sn[t][k];
            }
            out[j] = static_cast<float>(y);
        }
        store4(static_cast<T *>(m.out) + (t0 + t) * m.out_stride + static_cast<uint64_t>(hh) * D + e0, out);
    }
    if (bad) raise_error(err, kErrInput);
}

// ---- append -----------------------------------------------------------------------------
// A run is the new tokens of one page: consecutive tokens on consecutive slots.  One
// wavefront takes one run's keys or values of one head, so a page's scale and codes have
// one writer and no result depends on timing.  It reads the run twice (the magnitudes, then
// the codes; the second time from cache), and rewrites the page's earlier codes where the
// scale grew.

template <int FMT>
__device__ __forceinline__ float least_scale(float most) {  // 2^e, most <= qmax 2^e
    const uint32_t u = __float_as_uint(most);
    // qmax is 0.9921875 * 2^7, or 0.875 * 2^9: compare the significand with its.
    constexpr uint32_t significand = FMT == kInt8 ? 0x7e0000u : 0x600000u;
    int e = static_cast<int>(u >> 23) - 126 - (FMT == kInt8 ? 7 : 9) + ((u & 0x7fffffu) > significand ? 1 : 0);
    if (e < -100) e = -100;
    return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

template <int FMT>
__device__ __forceinline__ uint32_t rescale4(uint32_t c, float by) {
    return code4<FMT>(value4<FMT>(c) * by);
}

struct AppendArgs {
    prism_kv_cache c;
    const void *k, *v;
    uint64_t k_stride, v_stride;
    const int32_t *slots;
    uint32_t tokens;
};

template <typename T, int FMT, int D>
__device__ void append_run(const prism_kv_cache &c, const T *x, uint64_t stride, bool is_v, uint32_t head, uint32_t page,
                           uint32_t first, uint32_t n, int *err) {
    constexpr uint32_t kLanes = D / 4, kRows = 64 / kLanes;
    const uint32_t lane = threadIdx.x & 63, e0 = 4 * (lane % kLanes), ps = c.page_size;
    float most = 0.0f;
    bool bad = false;
    for (uint32_t i = lane / kLanes; i < n; i += kRows) {
        const f32x4 v = load4(x + i * stride + e0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bad |= !finite(v[j]);
            most = fmaxf(most, finite(v[j]) ? fabsf(v[j]) : 0.0f);
        }
    }
#pragma unroll
    for (uint32_t d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
    if (bad) raise_error(err, kErrInput);
    const uint64_t unit = static_cast<uint64_t>(page) * c.kv_heads + head;
    float *scale = (is_v ? c.v_scale : c.k_scale) + unit;
    const float old = first ? *scale : 0.0f, s = fmaxf(old, least_scale<FMT>(most));
    const float inv = 1.0f / s, by = old * inv;
    const bool grew = first && s != old;
    uint8_t *codes = static_cast<uint8_t *>(is_v ? c.v : c.k) + unit * ps * D;
    if (!is_v) {
        if (grew)
            for (uint32_t i = 4 * lane; i < first * D; i += 256) {
                uint32_t *w = reinterpret_cast<uint32_t *>(codes + i);
                *w = rescale4<FMT>(*w, by);
            }
        for (uint32_t i = lane / kLanes; i < n; i += kRows)
            *reinterpret_cast<uint32_t *>(codes + (first + i) * D + e0) = code4<FMT>(load4(x + i * stride + e0) * inv);
    } else {
        // Four places of a dimension at a time.
        const uint32_t end = first + n;
        for (uint32_t g = grew ? 0 : first & ~3u; g < end; g += 4)
            for (uint32_t d = lane; d < D; d += 64) {
                f32x4 v{0, 0, 0, 0};
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    if (g + j >= first && g + j < end) v[j] = static_cast<float>(x[(g + j - first) * stride + d]);
                uint32_t *w = reinterpret_cast<uint32_t *>(codes + d * ps + g);
                uint32_t r = code4<FMT>(v * inv);
                if (g < first || g + 4 > end) {  // keep, or rescale, what the page held beside the run
                    const uint32_t had = *w, again = grew ? rescale4<FMT>(had, by) : had;
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t mask = 255u << (8 * j);
                        if (g + j < first) r = (r & ~mask) | (again & mask);
                        else if (g + j >= end) r = (r & ~mask) | (had & mask);
                    }
                }
                *w = r;
            }
    }
    if (lane == 0) *scale = s;
}

// A wavefront looks for the runs that begin among `each` (at most 32) tokens.
template <typename T, int FMT, int D>
__global__ __launch_bounds__(256) void k_append(AppendArgs a, uint32_t each, int *err) {
    const uint32_t lane = threadIdx.x & 63, task = blockIdx.y * 4 + threadIdx.x / 64;
    if (task >= 2 * a.c.kv_heads) return;
    const uint32_t t0 = blockIdx.x * each, ps = a.c.page_size;
    const int32_t slots = static_cast<int32_t>(a.c.pages * ps);
    // Lane l holds the slot of token t0 - 1 + l.
    const int64_t mine = static_cast<int64_t>(t0) + lane - 1;
    int32_t s = -1;
    if (lane <= each && mine >= 0 && mine < a.tokens) s = a.slots[mine];
    const bool here = lane >= 1 && lane <= each;
    bool bad = here && (s < -1 || s >= slots);
    if (s < 0 || s >= slots) s = -1;
    const int32_t prev = __shfl_up(s, 1);
    const bool follows = prev >= 0 && s == prev + 1 && s % static_cast<int32_t>(ps) != 0;
    bool leads = here && s >= 0 && !follows;
    if (leads && prev >= 0 && prev / static_cast<int32_t>(ps) == s / static_cast<int32_t>(ps)) {
        bad = true;  // a second run in the page
        leads = false;
    }
    if (bad && task == 0) raise_error(err, kErrIndex);
    const bool is_v = task >= a.c.kv_heads;
    const uint32_t head = is_v ? task - a.c.kv_heads : task;
    const uint64_t stride = is_v ? a.v_stride : a.k_stride;
    uint64_t left = __ballot(leads);
    while (left) {
        const int l = __builtin_ctzll(left);
        left &= left - 1;
        const uint32_t t = t0 + l - 1, slot = static_cast<uint32_t>(__shfl(s, l));
        const uint32_t page = slot / ps, first = slot % ps, most = min(ps - first, a.tokens - t);
        uint32_t n = 0;
        for (uint32_t base = 0; base < most; base += 64) {  // how many tokens follow
            const uint32_t i = base + lane;
            const uint64_t on = __ballot(i < most && static_cast<uint32_t>(a.slots[t + i]) == slot + i);
            const uint32_t run = ~on ? __builtin_ctzll(~on) : 64;
            n += run;
            if (run < 64) break;
        }
        const T *x = static_cast<const T *>(is_v ? a.v : a.k) + t * stride + static_cast<uint64_t>(head) * D;
        append_run<T, FMT, D>(a.c, x, stride, is_v, head, page, first, n, err);
    }
}

template <typename T, int D>
int rope_typed(const Rotation &rot, const RopeRows &a, const RopeRows &b, const int32_t *positions, uint32_t tokens, float eps,
               int *err, hipStream_t s) {
    const uint32_t tiles = (tokens + kRopeTokens - 1) / kRopeTokens, heads = a.heads + b.heads;
    // Heads are split over workgroups until some 1024 of them share the rows.
    uint32_t parts = (1024 + tiles - 1) / tiles;
    constexpr uint32_t least = 4 * 64 / (D / 4);  // rows of a workgroup's four wavefronts
    if (parts > (heads + least - 1) / least) parts = (heads + least - 1) / least;
    const uint32_t each = (heads + parts - 1) / parts;
    k_rope<T, D><<<dim3(tiles, (heads + each - 1) / each), 256, 0, s>>>(a, b, rot, positions, tokens, each, eps, err);
    return launch_status();
}
template <typename T>
int rope_headed(const Rotation &rot, const RopeRows &a, const RopeRows &b, const int32_t *positions, uint32_t tokens,
                uint32_t head_dim, float eps, int *err, hipStream_t s) {
    switch (head_dim) {
    case 64: return rope_typed<T, 64>(rot, a, b, positions, tokens, eps, err, s);
    case 128: return rope_typed<T, 128>(rot, a, b, positions, tokens, eps, err, s);
    case 256: return rope_typed<T, 256>(rot, a, b, positions, tokens, eps, err, s);
    default: return kLaunchUnsupported;
    }
}

template <typename T, int FMT>
int append_headed(const AppendArgs &a, uint32_t each, dim3 grid, int *err, hipStream_t s) {
    switch (a.c.head_dim) {
    case 64: k_append<T, FMT, 64><<<grid, 256, 0, s>>>(a, each, err); break;
    case 128: k_append<T, FMT, 128><<<grid, 256, 0, s>>>(a, each, err); break;
    case 256: k_append<T, FMT, 256><<<grid, 256, 0, s>>>(a, each, err); break;
    default: return kLaunchUnsupported;
    }
    return launch_status();
}
template <typename T>
int append_typed(const AppendArgs &a, uint32_t each, dim3 grid, int *err, hipStream_t s) {
    return a.c.format == PRISM_CACHE_INT8 ? append_headed<T, kInt8>(a, each, grid, err, s)
                                          : append_headed<T, kE4m3>(a, each, grid, err, s);
}

}  // namespace

size_t plan_scratch_bytes(uint32_t requests) { return sizeof(int32_t) * (2 * (static_cast<size_t>(requests) + 1) + 4); }

int launch_kv_plan(const prism_kv_plan &p, void *scratch, int *err, hipStream_t s) {
    const PlanScratch sc = plan_scratch(scratch, p.requests);
    const bool own = p.max_tokens <= kPlanOwnFill;
    k_plan<<<1, kPlanThreads, 0, s>>>(p, sc, own, err);
    const int rc = launch_status();
    if (rc || own) return rc;
    k_plan_fill<<<(p.max_tokens + 255) / 256, 256, 0, s>>>(p, sc);
    return launch_status();
}

int launch_rope(int dtype, const Rotation &rot, const RopeRows &a, const RopeRows &b, const int32_t *positions,
                uint32_t tokens, uint32_t head_dim, float eps, int *err, hipStream_t s) {
    if (dtype == PRISM_DTYPE_F32) return rope_headed<float>(rot, a, b, positions, tokens, head_dim, eps, err, s);
    if (dtype == PRISM_DTYPE_F16) return rope_headed<_Float16>(rot, a, b, positions, tokens, head_dim, eps, err, s);
    return rope_headed<__bf16>(rot, a, b, positions, tokens, head_dim, eps, err, s);
}

int launch_kv_append(const prism_kv_cache &cache, int dtype, const void *k, uint64_t k_stride, const void *v,
                     uint64_t v_stride, const int32_t *slots, uint32_t tokens, int *err, hipStream_t s) {
    const AppendArgs a{cache, k, v, k_stride, v_stride, slots, tokens};
    const uint32_t each = tokens <= 512 ? 1 : tokens <= 4096 ? 4 : 16;
    const dim3 grid((tokens + each - 1) / each, (2 * cache.kv_heads + 3) / 4);
    if (dtype == PRISM_DTYPE_F32) return append_typed<float>(a, each, grid, err, s);
    if (dtype == PRISM_DTYPE_F16) return append_typed<_Float16>(a, each, grid, err, s);
    return append_typed<__bf16>(a, each, grid, err, s);
}

}  // namespace prism
