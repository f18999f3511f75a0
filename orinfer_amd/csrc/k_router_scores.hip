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
    float scale;
};

// Larger key, larger value; 0 is left for what is never chosen, 1 for what is chosen last.
__device__ __forceinline__ uint64_t key_of(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    return bits >> 63 ? ~bits : bits | 0x8000000000000000ull;
}
constexpr uint64_t kLast = 1;

__device__ __forceinline__ double wave_sum_double(double v) {
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
// The largest key of the wave and the lowest id that has it.
__device__ __forceinline__ void wave_best(uint64_t& key, int& id) {
    for (int d = 32; d > 0; d >>= 1) {
        const uint64_t other = __shfl_xor(key, d);
        const int other_id = __shfl_xor(id, d);
        if (other > key || (other == key && other_id < id)) key = other, id = other_id;
    }
}

// A wave's LDS accesses run in their order; this keeps the compiler to it where lanes read what others wrote.
__device__ __forceinline__ void lane_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// A wave to a token, LOCAL scores to a lane (expert j * 64 + lane).
template <int LOCAL>
__global__ __launch_bounds__(256) void router_scores_kernel(ScoreParams p) {
    __shared__ double held[4][LOCAL * 64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= p.m) return;
    double* const mine = held[wave];
    double score[LOCAL];
    bool known[LOCAL];  // the expert is there and its logit is a number
    float largest = -FLT_MAX;
#pragma unroll
    for (int j = 0; j < LOCAL; ++j) {
        const int id = j * 64 + lane;
        const float l = id < p.e ? p.logits[row * p.e + id] : 0.f;
        known[j] = id < p.e && l == l;
        score[j] = fminf(fmaxf(l, -FLT_MAX), FLT_MAX);
        if (known[j]) largest = fmaxf(largest, (float)score[j]);
    }
    if (p.sigmoid) {
#pragma unroll
        for (int j = 0; j < LOCAL; ++j) score[j] = 1.0 / (1.0 + exp(-score[j]));
    } else {
        for (int d = 32; d > 0; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
        double sum = 0;
#pragma unroll
        for (int j = 0; j < LOCAL; ++j) {
            score[j] = exp(score[j] - (double)largest);
            sum += known[j] ? score[j] : 0.0;
        }
        sum = wave_sum_double(sum);
#pragma unroll
        for (int j = 0; j < LOCAL; ++j) score[j] /= sum;
    }
    uint64_t key[LOCAL];
#pragma unroll
    for (int j = 0; j < LOCAL; ++j) {
        const int id = j * 64 + lane;
        const double choice = score[j] + (p.bias != nullptr && id < p.e ? (double)p.bias[id] : 0.0);
        const bool open = known[j] && choice > -__builtin_inf();  // (false for NaN too)
        key[j] = id >= p.e ? 0 : open ? key_of(choice) : kLast;
        mine[id] = open ? choice : -__builtin_inf();
    }
    lane_order();
    if (p.top_groups < p.groups) {
        // a lane to a group: its two largest
        const int size = p.e / p.groups;
        double first = -__builtin_inf(), second = -__builtin_inf();
        if (lane < p.groups)
            for (int i = 0; i < size; ++i) {
                const double c = mine[lane * size + i];
                second = fmax(second, fmin(first, c)), first = fmax(first, c);
            }
        const double total = p.group_best > 1 && second > -__builtin_inf() ? first + second : first;
        uint64_t group_key = lane < p.groups ? key_of(total) : 0;
        uint64_t kept = 0;
        for (int i = 0; i < p.top_groups; ++i) {
            uint64_t best = group_key;
            int at = lane;
            wave_best(best, at);
            kept |= 1ull << at;
            if (lane == at) group_key = 0;
        }
#pragma unroll
        for (int j = 0; j < LOCAL; ++j)
            if (j * 64 + lane < p.e && !(kept >> ((j * 64 + lane) / size) & 1)) key[j] = 0;
    }
    lane_order();
#pragma unroll
    for (int j = 0; j < LOCAL; ++j) mine[j * 64 + lane] = score[j];
    lane_order();
    int my_id = 0;
    uint64_t my_key = 0;
    for (int rank = 0; rank < p.top_k; ++rank) {
        uint64_t best = 0;
        int at = 0x7FFFFFFF;
#pragma unroll
        for (int j = 0; j < LOCAL; ++j)
            if (key[j] > best) best = key[j], at = j * 64 + lane;
        wave_best(best, at);
#pragma unroll
        for (int j = 0; j < LOCAL; ++j)
            if (j * 64 + lane == at) key[j] = 0;
        if (lane == rank) my_id = at, my_key = best;
    }
    const bool route = lane < p.top_k;
    const double s = route && my_key != kLast ? mine[my_id] : 0.0;
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
