// logprobs.hip -- log probabilities of given tokens, entropy and the most probable alternatives of rows of logits (gfx950).
//
// A row's softmax is held as its largest logit m and, of all others, s = sum exp(x - m) and t = sum exp(x - m) (x - m), so that
//   log S = log1p(s), entropy = log1p(s) - t / (1 + s)
// keep their digits where one word has nearly all the weight.
#include "serve_common.hpp"

namespace prism {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kNone = -__builtin_inff();

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
    if (b.m == kNone) return a;
    // The second's largest counts as a word of weight exp(d) now.
    const float d = b.m - a.m, e = exp_of(d);
    a.t += e * (b.t + d * (b.s + 1.0f));
    a.s += e * (b.s + 1.0f);
    return a;
}

// Larger logits have larger keys, and of equal ones the word of the lower id; 0 is none.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
    if (!(x > kNone)) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 as 0
    return static_cast<uint64_t>(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - id);
}
__device__ __forceinline__ uint32_t id_of(uint64_t key) { return 0xffffffffu - static_cast<uint32_t>(key); }
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t u = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// A workgroup has a row; each alternative is another look at it.
template <typename T>
__global__ __launch_bounds__(256) void k_logprobs(prism_logprobs a, int *err) {
    __shared__ Softmax part[4];
    __shared__ uint64_t best[4];
    __shared__ int bad_any;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const uint64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    if (threadIdx.x == 0) bad_any = 0;
    __syncthreads();
    Softmax w{kNone, 0.0f, 0.0f};
    bool bad = false;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += 256) {
        const float v = static_cast<float>(x[i]);
        bad |= !(v < __builtin_inff());
        w = joined(w, Softmax{v, 0.0f, 0.0f});
    }
    if (bad) bad_any = 1;
    for (int d = 1; d < 64; d *= 2) w = joined(w, Softmax{__shfl_xor(w.m, d), __shfl_xor(w.s, d), __shfl_xor(w.t, d)});
    if (lane == 0) part[wave] = w;
    __syncthreads();
    w = joined(joined(part[0], part[1]), joined(part[2], part[3]));
    const float nan = __builtin_nanf(""), log_s = log1pf(w.s);
    const bool wrong = bad_any != 0;
    if (threadIdx.x == 0) {
        if (wrong) raise_error(err, kErrNonfinite);
        if (a.logprobs) {
            const int32_t id = a.targets[row];
            float lp = 0.0f;
            if (id < -1 || id >= static_cast<int64_t>(a.vocab)) {
                raise_error(err, kErrIndex);
                lp = nan;
            } else if (id >= 0) {
                const float v = static_cast<float>(x[id]);
                lp = v == kNone ? kNone : (v - w.m) - log_s;
            }
            a.logprobs[row] = wrong ? nan : lp;
        }
        if (a.entropy) a.entropy[row] = wrong ? nan : w.m == kNone ? 0.0f : log_s - w.t / (1.0f + w.s);
    }
    uint64_t below = ~0ull;
    for (uint32_t i = 0; i < a.top; ++i) {
        uint64_t most = 0;
        for (uint32_t j = threadIdx.x; j < a.vocab; j += 256) {
            const uint64_t k = key_of(static_cast<float>(x[j]), j);
            if (k < below && k > most) most = k;
        }
        for (int d = 1; d < 64; d *= 2) {
            const uint64_t o = __shfl_xor(static_cast<unsigned long long>(most), d);
            most = o > most ? o : most;
        }
        if (lane == 0) best[wave] = most;
        __syncthreads();
        for (int k = 0; k < 4; ++k) most = best[k] > most ? best[k] : most;
        __syncthreads();
        below = most ? most : 1;
        if (threadIdx.x == 0) {
            a.top_ids[row * a.top + i] = wrong || !most ? -1 : static_cast<int32_t>(id_of(most));
            a.top_logprobs[row * a.top + i] = wrong ? nan : !most ? kNone : (logit_of(most) - w.m) - log_s;
        }
    }
}

}  // namespace

size_t logprobs_scratch_bytes(const prism_logprobs &, uint32_t) { return 0; }

int launch_logprobs(const prism_logprobs &a, void *, uint32_t, int *err, hipStream_t s) {
    if (a.dtype == PRISM_DTYPE_F32) k_logprobs<float><<<a.tokens, 256, 0, s>>>(a, err);
    else if (a.dtype == PRISM_DTYPE_F16) k_logprobs<_Float16><<<a.tokens, 256, 0, s>>>(a, err);
    else k_logprobs<__bf16><<<a.tokens, 256, 0, s>>>(a, err);
    return launch_status();
}

}  // namespace prism
