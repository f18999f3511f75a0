// Routes by scores with a balance bias and expert groups: router_topk with scoring, bias, groups, top_groups, group_best, renormalize and scale.
//
//   s_e = 1 / (1 + exp(-l_e)) or softmax(l)_e;  c_e = s_e + b_e;  the score of a group of E / groups neighbours is the sum of its group_best largest c;
//   the top_groups best groups stay, the top_k largest c of their experts are the routes, the lower id first on ties;
//   p = s / (sum of the routes' s) * scale, without renormalize p = s * scale.
// The choice is the one of 64-bit arithmetic: scores of 32 bits tell apart what is closer than their rounding at random.
// An expert whose c is NaN or -infinity (a bias can close experts so) comes behind all others of the groups that stay, counts nothing in its group's score and has
// weight 0; a logit of NaN does the same to its expert, infinite ones count as the largest finite ones.  Where the routes' scores are all 0, so are their weights.
#include <cfloat>

#include "moe_device.h"
#include "orx_internal.h"

namespace orx {
namespace {

struct ScoreParams {
    const float *logits, *bias;
    int* ids;
    float* prob;
    int m, e, top_k, groups, top_groups, group_best, sigmoid, renormalize;
    int lanes;         // to a group, a power of two
    uint32_t inverse;  // ceil(2^21 / experts of a group): ids below 1024 divided by it
    float scale;
};

// Larger key, larger value, in two words; 0 is left for what is never chosen, 1 for what is chosen last.
struct Key {
    uint32_t high, low;
};
__device__ __forceinline__ Key key_of(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v), key = bits >> 63 ? ~bits : bits | 0x8000000000000000ull;
    return {(uint32_t)(key >> 32), (uint32_t)key};
}

// Moves of 64-bit values between lanes, as wave_sum makes them of 32-bit ones.
__device__ __forceinline__ double join(uint32_t low, uint32_t high) { return __builtin_bit_cast(double, ((uint64_t)high << 32) | low); }
template <int CONTROL>
__device__ __forceinline__ double moved(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    return join(__builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, CONTROL, 0xF, 0xF, true), __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(bits >> 32), CONTROL, 0xF, 0xF, true));
}
// a lane's value and its partner's, 16 or 32 lanes away, in the same order for both
template <int LANES>
__device__ __forceinline__ void both(double v, double& one, double& other) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    if constexpr (LANES == 16) {
        auto low = __builtin_amdgcn_permlane16_swap((uint32_t)bits, (uint32_t)bits, false, false), high = __builtin_amdgcn_permlane16_swap((uint32_t)(bits >> 32), (uint32_t)(bits >> 32), false, false);
        one = join(low[0], high[0]), other = join(low[1], high[1]);
    } else {
        auto low = __builtin_amdgcn_permlane32_swap((uint32_t)bits, (uint32_t)bits, false, false), high = __builtin_amdgcn_permlane32_swap((uint32_t)(bits >> 32), (uint32_t)(bits >> 32), false, false);
        one = join(low[0], high[0]), other = join(low[1], high[1]);
    }
}
__device__ __forceinline__ double wave_sum_double(double v) {
    double one, other;
    both<32>(v, one, other), v = one + other;
    both<16>(v, one, other), v = one + other;
    v += moved<0x128>(v);  // row_ror:8
    v += moved<0x124>(v);  // row_ror:4
    v += moved<0x4E>(v);   // quad_perm [2,3,0,1]
    v += moved<0xB1>(v);   // quad_perm [1,0,3,2]
    return v;
}
// the two largest of two pairs
__device__ __forceinline__ void two_of(double& first, double& second, double a, double b) {
    second = fmax(fmin(first, a), fmax(second, b));
    first = fmax(first, a);
}
// The two largest of LANES neighbouring lanes, known to all of them (mirrors: lane i's partner is 7 - i, 15 - i of its group).
__device__ __forceinline__ void two_of_lanes(double& first, double& second, int lanes) {
    if (lanes > 1) two_of(first, second, moved<0xB1>(first), moved<0xB1>(second));
    if (lanes > 2) two_of(first, second, moved<0x4E>(first), moved<0x4E>(second));
    if (lanes > 4) two_of(first, second, moved<0x141>(first), moved<0x141>(second));
    if (lanes > 8) two_of(first, second, moved<0x140>(first), moved<0x140>(second));
    double a, b, c, d;
    if (lanes > 16) {
        both<16>(first, a, b), both<16>(second, c, d);
        first = a, second = c, two_of(first, second, b, d);
    }
    if (lanes > 32) {
        both<32>(first, a, b), both<32>(second, c, d);
        first = a, second = c, two_of(first, second, b, d);
    }
}
// A wave's LDS accesses run in their order; this keeps the compiler to it where lanes read what others wrote.
__device__ __forceinline__ void lane_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// A wave to a token, LOCAL scores to a lane (expert j * 64 + lane).
// With many tokens bound by instructions, with few by one chain: 64-bit exponentials, then ranks.  A rank is one maximum of the keys' high words and one ballot for every held key; only
// where several lanes have it do the low words decide.  8192 tokens of 256 experts, 8 groups, top 8: 32.6 us with 64-bit shuffles, 16.2 now; 5 tokens of 128: 7.0, 3.6 now.
template <int LOCAL>
__global__ __launch_bounds__(256) void router_scores_kernel(ScoreParams p) {
    __shared__ double held[4][LOCAL * 64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= p.m) return;
    double* const mine = held[wave];
    double score[LOCAL];
    float bias[LOCAL];
    bool known[LOCAL];  // the expert is there and its logit is a number
    float largest = -FLT_MAX;
#pragma unroll
    for (int j = 0; j < LOCAL; ++j) {
        const int id = j * 64 + lane;
        const float l = p.logits[row * p.e + min(id, p.e - 1)];
        bias[j] = p.bias != nullptr ? p.bias[min(id, p.e - 1)] : 0.f;
        known[j] = id < p.e && l == l;
        const float finite = fminf(fmaxf(l, -FLT_MAX), FLT_MAX);
        score[j] = finite;
        largest = known[j] ? fmaxf(largest, finite) : largest;
    }
    if (p.sigmoid) {
#pragma unroll
        for (int j = 0; j < LOCAL; ++j) score[j] = 1.0 / (1.0 + exp(-score[j]));
    } else {
        const double top = key_value(wave_max_u32(ordered_key(largest)));
        double sum = 0;
#pragma unroll
        for (int j = 0; j < LOCAL; ++j) {
            score[j] = exp(score[j] - top);
            sum += known[j] ? score[j] : 0.0;
        }
        const double inverse = 1.0 / wave_sum_double(sum);
#pragma unroll
        for (int j = 0; j < LOCAL; ++j) score[j] *= inverse;
    }
    Key key[LOCAL];
#pragma unroll
    for (int j = 0; j < LOCAL; ++j) {
        const int id = j * 64 + lane;
        const double choice = score[j] + (double)bias[j];
        const bool open = known[j] && choice > -__builtin_inf();  // (false for NaN too)
        key[j] = key_of(choice);
        if (!open) key[j] = Key{0, id < p.e ? 1u : 0u};
        mine[id] = open ? choice : -__builtin_inf();
    }
    lane_order();
    if (p.top_groups < p.groups) {
        // LANES lanes to a group; then a group stays if fewer than top_groups are in front of it
        const int size = p.e / p.groups, lanes = p.lanes, group = lane / lanes;
        double first = -__builtin_inf(), second = -__builtin_inf();
        if (group < p.groups)
            for (int i = lane & (lanes - 1); i < size; i += lanes) two_of(first, second, mine[group * size + i], -__builtin_inf());
        two_of_lanes(first, second, lanes);
        const Key own = key_of(p.group_best > 1 && second > -__builtin_inf() ? first + second : first);
        const uint64_t own_key = (uint64_t)own.high << 32 | own.low;
        int in_front = 0;
        for (int g = 0; g < p.groups; ++g) {
            const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)own.high, g * lanes) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)own.low, g * lanes);
            in_front += other > own_key || (other == own_key && g < group) ? 1 : 0;
        }
        const uint64_t kept = __ballot(group < p.groups && in_front < p.top_groups);
#pragma unroll
        for (int j = 0; j < LOCAL; ++j) {
            const int of = (int)((uint32_t)(j * 64 + lane) * p.inverse >> 21);  // id / size
            if (!(kept >> (min(of, p.groups - 1) * lanes) & 1)) key[j] = Key{0, 0};
        }
        lane_order();
    }
#pragma unroll
    for (int j = 0; j < LOCAL; ++j) mine[j * 64 + lane] = score[j];
    lane_order();
    int my_id = 0;
    bool my_last = false;  // chosen for want of another
    for (int rank = 0; rank < p.top_k; ++rank) {
        uint32_t best = key[0].high;
#pragma unroll
        for (int j = 1; j < LOCAL; ++j) best = max(best, key[j].high);
        best = wave_max_u32(best);
        uint64_t having[LOCAL];
        int count = 0;
#pragma unroll
        for (int j = 0; j < LOCAL; ++j) having[j] = __ballot(key[j].high == best), count += __popcll(having[j]);
        uint32_t low = 2;
        if (count > 1) {
            low = 0;
#pragma unroll
            for (int j = 0; j < LOCAL; ++j) low = max(low, key[j].high == best ? key[j].low : 0u);
            low = wave_max_u32(low);
#pragma unroll
            for (int j = 0; j < LOCAL; ++j) having[j] &= __ballot(key[j].low == low);
        }
        int chosen = 0;
        uint64_t lowest = 0;
#pragma unroll
        for (int j = LOCAL - 1; j >= 0; --j)
            if (having[j] != 0) chosen = j, lowest = having[j];
        lowest &= 0 - lowest;
        const int id = chosen * 64 + __builtin_ctzll(lowest);
        const bool last = best == 0 && low == 1;
#pragma unroll
        for (int j = 0; j < LOCAL; ++j)
            if (j == chosen && (lowest >> lane & 1)) key[j] = Key{0, 0};
        if (lane == rank) my_id = id, my_last = last;
    }
    const bool route = lane < p.top_k;
    const double s = route && !my_last ? mine[my_id] : 0.0;
    const double sum = p.renormalize ? wave_sum_double(s) : 1.0;
    if (route) {
        p.ids[row * p.top_k + lane] = my_id;
        p.prob[row * p.top_k + lane] = (float)(sum > 0 ? s / sum * (double)p.scale : 0.0);
    }
}

int geometry(const orx_function&, int rows, Geometry* g) {
    g->grid[0] = ceil_div((uint32_t)rows, 4u);
    g->block[0] = 256;
    return ORX_OK;
}
// [Bias,] IDs, Logits, Prob[, m].  slots used: M, E, top_k, group (groups), slots (top_groups), tiles (group_best), flags, weight_scale
enum { kBias = 1, kSigmoid = 2, kRenormalize = 4 };
int launch(const orx_function& f, int rows, const Geometry& g, hipStream_t s, void** args) {
    const int bias = f.flags & kBias ? 1 : 0;
    ScoreParams p;
    p.bias = bias ? pointer_arg<const float>(args, 0) : nullptr;
    p.ids = pointer_arg<int>(args, bias), p.logits = pointer_arg<const float>(args, bias + 1), p.prob = pointer_arg<float>(args, bias + 2);
    p.m = rows, p.e = f.E, p.top_k = f.top_k, p.groups = f.group, p.top_groups = f.slots, p.group_best = f.tiles;
    p.lanes = 1;
    while (2 * p.lanes * f.group <= 64) p.lanes *= 2;
    p.inverse = ceil_div(1u << 21, (uint32_t)(f.E / f.group));
    p.sigmoid = f.flags & kSigmoid, p.renormalize = f.flags & kRenormalize, p.scale = f.weight_scale;
    const dim3 grid(g.grid[0]), block(256);
    if (f.E <= 64) ORX_LAUNCH(router_scores_kernel<1>, grid, block, 0, s, p);
    else if (f.E <= 128) ORX_LAUNCH(router_scores_kernel<2>, grid, block, 0, s, p);
    else if (f.E <= 256) ORX_LAUNCH(router_scores_kernel<4>, grid, block, 0, s, p);
    else if (f.E <= 512) ORX_LAUNCH(router_scores_kernel<8>, grid, block, 0, s, p);
    else ORX_LAUNCH(router_scores_kernel<16>, grid, block, 0, s, p);
    return hip_check(hipGetLastError(), "launch router_topk by scores");
}

}  // namespace

// The keys that ask for scores, a bias, groups or a factor; M, E, top_k, dynamic_rows and renormalize are read by the caller (`f` holds their values).
int make_router_scores(const Variant& v, bool renormalize, orx_function* f) {
    bool bad = false;
    const std::string scoring = v.string("scoring", "softmax", &bad);
    const bool bias = v.boolean("bias", false, &bad);
    f->group = (int)v.integer("groups", 1, &bad);
    f->slots = (int)v.integer("top_groups", f->group, &bad);
    f->tiles = (int)v.integer("group_best", 2, &bad);
    const double scale = v.real("scale", 1.0, &bad);
    if (bad) return ORX_ERR_BAD_VARIANT;
    if (scoring != "softmax" && scoring != "sigmoid") {
        set_error("router_topk: scoring must be softmax or sigmoid");
        return ORX_ERR_BAD_VARIANT;
    }
    if (f->group < 1 || f->group > 64 || f->E % f->group || f->slots < 1 || f->slots > f->group || (int64_t)f->E / f->group * f->slots < f->top_k ||
        (f->tiles != 1 && f->tiles != 2)) {
        set_error("router_topk: need groups of up to 64 that divide E, 1 <= top_groups <= groups, top_k experts among them and group_best 1 or 2");
        return ORX_ERR_BAD_VARIANT;
    }
    if (!(scale > 0 && scale <= FLT_MAX)) {
        set_error("router_topk: scale must be a positive number");
        return ORX_ERR_BAD_VARIANT;
    }
    f->weight_scale = (float)scale;
    f->flags = (bias ? kBias : 0) | (scoring == "sigmoid" ? kSigmoid : 0) | (renormalize ? kRenormalize : 0);
    f->args.clear();
    if (bias) f->args.push_back({"Bias", ArgPointer, 4});
    for (const ArgSpec& a : std::initializer_list<ArgSpec>{{"IDs", ArgPointer, 4}, {"Logits", ArgPointer, 4}, {"Prob", ArgPointer, 4}}) f->args.push_back(a);
    if (f->dynamic_rows) f->args.push_back({"m", ArgI32, 4});
    f->geometry = geometry;
    f->launch = launch;
    f->device_function = f->E <= 64    ? reinterpret_cast<const void*>(&router_scores_kernel<1>)
                         : f->E <= 128 ? reinterpret_cast<const void*>(&router_scores_kernel<2>)
                         : f->E <= 256 ? reinterpret_cast<const void*>(&router_scores_kernel<4>)
                         : f->E <= 512 ? reinterpret_cast<const void*>(&router_scores_kernel<8>)
                                       : reinterpret_cast<const void*>(&router_scores_kernel<16>);
    return ORX_OK;
}

}  // namespace orx
