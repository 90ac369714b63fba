// sample.hip — a token for each row of logits: temperature, top-k, top-p, min-p
// and inverse sampling by a given random number (gfx950).
//
//   w_i = exp((x_i - max) / T)
//   the k largest (of equal ones those of the lowest index);
//   of these, from the largest on, those with less than p sum(w) before them;
//   of these the w_i >= min_p;  the token: the first, in the tokens' order, with
//   sum_{j <= i} w_j > u sum(w)
//
// Weights are whole numbers, round(2^s w'), s up to 50 and s + log2(n) at most 62,
// so that every sum is exact and the same in any order: sums meet in atomics
// without the token depending on timing.  (w' is w times a factor for all of a row
// that puts the largest between 1/2 and 1; at 152064 tokens a step is 2^-44, and
// what is below half of it is none.)  A row is cut into chunks over workgroups, by
// n and the number of rows.  Top-p's bound alone knows how: a chunk's bins are
// whole numbers of its own largest weight, so that their sums are off the row's by
// up to a step a logit.
//
// The row is never sorted.  Four launches: each chunk's maximum and its
// histogram over the logarithm of w, ten bins a factor of two, from one reading
// into registers; the bins summed for the row, which gives those that are kept
// whole and those (one, mostly) where a cut falls; each chunk's sum of what is
// kept whole, and the elements of the bins between as a list; the cuts in the
// list (through finer bins where it is long), the chunk of the token, and the
// token.  A list that is too long (many equal logits) is cut by radix selection
// over the row instead.  Short rows take one launch (sample_one_kernel).
//
// Few rows are bound by the launches' latency (one row of 152064 logits 23 us, 9
// of 50257 25 us), many by the two readings of the logits: 64 rows of 152064 (39
// MB) 53 us, of which the histograms 15 and the second reading 15.
#include "frq_internal.h"

namespace frq {
namespace smp {
namespace {

constexpr int NT = 512;            // threads
constexpr int NB = 512, PER = 10;  // bins, bins a factor of two: 51 of them
constexpr int MAX_S = 50;          // E - v <= s + 1 where a weight is not zero
constexpr int CAP = 16384;         // elements of a row's list
constexpr int FT = 512;            // threads of a row's last launch
constexpr int FEW = FT;            // elements that are put in order
constexpr int LISTED = 2048;        // top-k up to this: the list holds all of them
constexpr int MAX_N = 1 << 24;
constexpr int MAX_V = 8;           // quads a thread at most
constexpr int MAX_CHUNKS = MAX_N / (4 * NT * MAX_V);
static_assert(NB == NT && NB == FT && MAX_CHUNKS <= 2 * FT, "");
constexpr int ERR_NAN_BIT = 1, ERR_ARG_BIT = 2;

struct __attribute__((packed, aligned(4))) F4 {
    float v[4];
};

struct Chunk {    // a chunk's maximum
    double e;     // the whole number above the logarithm of its largest weight
    float most;
    int at;       // its first index; -1: the chunk holds a NaN
};
struct Row {
    double c;           // log2(e) / T
    double e;           // the largest of the chunks'
    double least;       // v = x c of min_p
    uint64_t below;     // weight of the bins before lo
    uint64_t all;       // of all bins
    int done;           // the token is written
    int lo, hi;         // bins < lo are kept whole, bins lo .. hi are the list
    int count_below;
    int k;              // 0: no bound
    float p;            // 1: no bound
    int listed;         // the list's length (may pass CAP)
};

struct Args {
    const float* x;
    int64_t pitch;
    int n, s;          // logits a row; log2 of the scale
    int chunks, len;   // chunks a row, logits a chunk (a multiple of 4)
    const float *temp, *topp, *minp, *u;
    const int32_t* topk;
    int64_t* token;
    float* prob;
    Row* row;
    Chunk* chunk;      // [m][chunks]
    uint64_t* weight;  // [m][chunks][NB]
    uint32_t* count;
    uint64_t* kept;    // [m][chunks] of the bins kept whole
    uint64_t* list;    // [m][CAP]
    int* err;
};

struct Ask {  // a row's parameters
    double c;
    float p, minp;
    int k;
    bool greedy, bad;
    // which histograms the row needs: up to LISTED of the largest are all listed,
    // and their weights are taken from the list
    __device__ __forceinline__ bool counts() const { return k > 0; }
    __device__ __forceinline__ bool weights() const { return p < 1.0f && (k == 0 || k > LISTED); }
};
__device__ __forceinline__ Ask ask_of(const Args& a, int r) {
    Ask q;
    const float t = a.temp ? a.temp[r] : 1.0f;
    const int k = a.topk ? a.topk[r] : 0;
    const float p = a.topp ? a.topp[r] : 1.0f, mp = a.minp ? a.minp[r] : 0.0f, u = a.u[r];
    q.greedy = t == 0.0f;
    q.bad = !(t >= 0.0f && t < __builtin_inff()) || (!q.greedy && (p != p || mp != mp || u != u));
    q.c = 1.4426950408889634074 / (double)t;
    q.k = k > 0 && k < a.n ? k : 0;
    q.p = p < 1.0f ? fmaxf(p, 0.0f) : 1.0f;
    q.minp = fminf(fmaxf(mp, 0.0f), 1.0f);
    return q;
}

// round(2^y) for y up to 50: 2^f by its Taylor series, |f| <= 1/2, whose next
// term is below 2^-52; the sum with 2^52 rounds.
__device__ __forceinline__ uint64_t weight_of(double y) {
    if (!(y > -1.0)) return 0;
    const double i = __builtin_rint(y), f = (y - i) * 0.69314718055994530942;
    double p = 1.0 / 479001600.0;
    p = __builtin_fma(p, f, 1.0 / 39916800.0);
    p = __builtin_fma(p, f, 1.0 / 3628800.0);
    p = __builtin_fma(p, f, 1.0 / 362880.0);
    p = __builtin_fma(p, f, 1.0 / 40320.0);
    p = __builtin_fma(p, f, 1.0 / 5040.0);
    p = __builtin_fma(p, f, 1.0 / 720.0);
    p = __builtin_fma(p, f, 1.0 / 120.0);
    p = __builtin_fma(p, f, 1.0 / 24.0);
    p = __builtin_fma(p, f, 1.0 / 6.0);
    p = __builtin_fma(p, f, 0.5);
    p = __builtin_fma(p, f, 1.0);
    p = __builtin_fma(p, f, 1.0);
    const double r = __builtin_ldexp(p, (int)i) + 4503599627370496.0;
    return __builtin_bit_cast(uint64_t, r) & 0xFFFFFFFFFFFFFull;
}
// The bin of v against e >= v; NB and more: no weight.
__device__ __forceinline__ int bin_of(double e, double v) {
    const double d = (e - v) * (double)PER;
    return d < (double)NB ? (int)d : NB;
}
// A number that every x with x c above v (in log2, give or take the roundings of
// numbers as large as e) is not below.
__device__ __forceinline__ float floor_of(double v, double e, double c) {
    const float f = (float)((v - 0.01 - __builtin_fabs(e) * 0x1p-48) / c);
    return f - __builtin_fabsf(f) * 0x1p-22f - 1e-37f;
}
// The order of finite floats as whole numbers (both zeros alike).
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
// (order, index) as one key: larger is taken earlier.
__device__ __forceinline__ uint64_t key_of(float x, int i) { return (uint64_t)order_of(x) << 32 | (uint32_t)~i; }

__device__ __forceinline__ F4 load4(const float* x, int i, int end) {
    if (i + 3 < end) return *reinterpret_cast<const F4*>(x + i);
    F4 f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.v[j] = i + j < end ? x[i + j] : -__builtin_inff();
    return f;
}

// Sums over the lanes up to and with each (DPP: within rows of 16, then the
// rows' ends), and over the workgroup.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_add(uint64_t x) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, false);
    return x + ((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ uint64_t lane_sums(uint64_t x) {
    x = dpp_add<0x111, 0xF>(x);
    x = dpp_add<0x112, 0xF>(x);
    x = dpp_add<0x114, 0xF>(x);
    x = dpp_add<0x118, 0xF>(x);
    x = dpp_add<0x142, 0xA>(x);
    return dpp_add<0x143, 0xC>(x);
}
__device__ __forceinline__ uint64_t last_lane(uint64_t x) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, 63);
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), 63) << 32 | lo;
}
template <int T>
__device__ __forceinline__ uint64_t group_sum(uint64_t v, uint64_t* tmp) {  // tmp: [T / 64]
    v = lane_sums(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v += tmp[i];
    return v;
}
// The sum of the threads before, and of all.
template <int T>
__device__ __forceinline__ uint64_t group_before(uint64_t v, uint64_t* tmp, uint64_t* all = nullptr) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t x = lane_sums(v);
    __syncthreads();
    if (lane == 63) tmp[w] = x;
    __syncthreads();
    uint64_t before = x - v, total = 0;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) {
        const uint64_t t = tmp[i];
        total += t;
        if (i < w) before += t;
    }
    if (all) *all = total;
    return before;
}

// A thread's quads of a chunk: quad i of thread t lies at beg + 4 (i NT + t).  Held
// in registers, or (one launch for all: its code is run once, and loops are shorter)
// in LDS.
template <int NV>
struct Held {
    F4 f[NV];
    template <typename F>
    __device__ __forceinline__ void each(F&& use) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) use(i, f[i]);
    }
};
struct Staged {
    const F4* x;
    int quads;
    template <typename F>
    __device__ __forceinline__ void each(F&& use) const {
#pragma unroll 1
        for (int i = 0; i < quads; ++i) use(i, x[i * NT + threadIdx.x]);
    }
};
__device__ __forceinline__ float top_of(const F4& f) { return fmaxf(fmaxf(f.v[0], f.v[1]), fmaxf(f.v[2], f.v[3])); }

// The largest of a chunk's numbers and its first index; whether one is a NaN.
struct Most {
    float wave[NT / 64];
    int at[NT / 64];
};
template <typename H>
__device__ __forceinline__ bool most_of(const H& held, int beg, Most& L, float& most, int& at) {
    const int tid = threadIdx.x;
    float top = -__builtin_inff();
    int where = beg;
    bool nan = false;
    held.each([&](int i, const F4& f) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            nan |= f.v[j] != f.v[j];
            if (f.v[j] > top) {
                top = f.v[j];
                where = beg + 4 * (i * NT + tid) + j;
            }
        }
    });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float o = __shfl_xor(top, d, 64);
        const int oa = __shfl_xor(where, d, 64);
        if (o > top || (o == top && oa < where)) {
            top = o;
            where = oa;
        }
    }
    if ((tid & 63) == 0) {
        L.wave[tid >> 6] = top;
        L.at[tid >> 6] = where;
    }
    nan = __syncthreads_or(nan);
#pragma unroll
    for (int i = 0; i < NT / 64; ++i)
        if (L.wave[i] > top || (L.wave[i] == top && L.at[i] < where)) {
            top = L.wave[i];
            where = L.at[i];
        }
    most = top;
    at = where;
    return nan;
}
// The chunk's histograms, added to weight and count (as the row needs them).
template <typename H>
__device__ __forceinline__ void add_bins(const H& held, const Ask& q, double e, int s, unsigned long long* weight,
                                         uint32_t* count) {
    const float least = floor_of(e - (double)(s + 1), e, q.c);  // below: no weight
    const bool counts = q.counts();
    if (q.weights()) {
        held.each([&](int, const F4& f) {
            if (!__builtin_amdgcn_ballot_w64(top_of(f) >= least)) return;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double v = (double)f.v[j] * q.c;
                const uint64_t w = weight_of(v - e + (double)s);
                if (w) {
                    const int b = min(bin_of(e, v), NB - 1);
                    atomicAdd(&weight[b], (unsigned long long)w);
                    if (counts) atomicAdd(&count[b], 1u);
                }
            }
        });
    } else {
        held.each([&](int, const F4& f) {
            if (!__builtin_amdgcn_ballot_w64(top_of(f) >= least)) return;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = bin_of(e, (double)f.v[j] * q.c);
                if (b < NB) atomicAdd(&count[b], 1u);
            }
        });
    }
}

// A workgroup a chunk, its logits in registers between the maximum and the bins.  64
// rows of 152064 (39 MB) in 15 us: the weights, some 35 operations of 64 bits a
// logit, take as long as the reading beside them.  Two or four copies of the
// histograms against colliding atomics: the same; half the chunks, twice as long: 56
// us the call against 49.
template <int NV>
__global__ __launch_bounds__(NT) void sample_bins_kernel(const Args a) {
    __shared__ unsigned long long weight[NB];
    __shared__ uint32_t count[NB];
    __shared__ Most tops;
    const int r = blockIdx.x / a.chunks, ch = blockIdx.x % a.chunks, tid = threadIdx.x;
    const float* x = a.x + (int64_t)r * a.pitch;
    const int beg = ch * a.len, end = min(beg + a.len, a.n);
    Held<NV> held;
#pragma unroll
    for (int i = 0; i < NV; ++i) held.f[i] = load4(x, beg + 4 * (i * NT + tid), end);
    const Ask q = ask_of(a, r);
    weight[tid] = 0;
    count[tid] = 0;
    float most;
    int at;
    const bool nan = most_of(held, beg, tops, most, at);
    const double e = __builtin_ceil((double)most * q.c);
    if (tid == 0) a.chunk[(int64_t)r * a.chunks + ch] = Chunk{e, most, nan ? -1 : at};
    if ((!q.counts() && !q.weights()) || q.greedy || q.bad) return;
    if (!nan && most > -__builtin_inff() && most < __builtin_inff()) add_bins(held, q, e, a.s, weight, count);
    __syncthreads();
    const int64_t to = ((int64_t)r * a.chunks + ch) * NB;
    if (q.weights()) a.weight[to + tid] = weight[tid];
    if (q.counts()) a.count[to + tid] = count[tid];
}

// f total for f of [0, 1), down to a whole number and whether it is more; exact
// (a sum of many equal weights has more bits than a double).
__device__ __forceinline__ uint64_t part_of(float f, uint64_t total, bool* more) {
    const uint32_t u = __float_as_uint(f), e = u >> 23, m = e ? (u & 0x7FFFFFu) | 0x800000u : u & 0x7FFFFFu;
    const int sh = 150 - (int)(e ? e : 1);  // f = m 2^-sh, sh of 24 and more
    // m total = hi 2^32 + lo, hi below 2^54
    const uint64_t a = (uint64_t)(uint32_t)total * m, hi = (total >> 32) * m + (a >> 32);
    const uint32_t lo = (uint32_t)a;
    if (sh >= 96) {
        *more = hi || lo;
        return 0;
    }
    if (sh >= 32) {
        *more = lo || (hi & (((uint64_t)1 << (sh - 32)) - 1));
        return hi >> (sh - 32);
    }
    *more = lo & ((1u << sh) - 1);
    return hi << (32 - sh) | lo >> sh;
}
// ceil(p total), at least one: what lies before an element is less than that
// where the element is kept.
__device__ __forceinline__ uint64_t share_of(float p, uint64_t total) {
    bool more;
    const uint64_t t = part_of(p, total, &more) + more;
    return t > 0 ? t : 1;
}

// Where the cuts fall: weight w and number n of this thread's bin (the first NB
// threads have one each; the others keep to the barriers).
struct Cuts {
    uint64_t tmp[NB / 64], klo, below;
    uint32_t tmp_n[NB / 64];
    int kbin, lo, hi, count_below;
};
struct Cut {
    uint64_t below, all;
    int lo, hi, count_below, k;
};
__device__ __forceinline__ void cut_start(Cuts& L) {  // by one thread, a barrier before cut_bins
    L.kbin = NB;
    L.lo = NB;
    L.hi = -1;
    L.klo = 0;
    L.below = 0;
    L.count_below = 0;
}
__device__ __forceinline__ Cut cut_bins(const Ask& q, Cuts& L, uint64_t w, uint32_t n) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bin = tid % NB;
    const bool on = tid < NB, ws = q.weights(), ns = q.counts();
    const uint64_t x = lane_sums(w);
    const uint32_t c = (uint32_t)lane_sums(n);
    if (on && lane == 63) {
        L.tmp[wave] = x;
        L.tmp_n[wave] = c;
    }
    __syncthreads();
    uint64_t before = x - w, all = 0;
    uint32_t cbefore = c - n;
#pragma unroll
    for (int i = 0; i < NB / 64; ++i) {
        all += L.tmp[i];
        if (i < wave) {
            before += L.tmp[i];
            cbefore += L.tmp_n[i];
        }
    }
    // the bin where the k largest end
    if (on && ns && cbefore < (uint32_t)q.k && cbefore + n >= (uint32_t)q.k) {
        L.kbin = bin;
        L.klo = before;
    }
    __syncthreads();
    int k = L.kbin < NB ? q.k : 0;
    if (on && ws && w) {
        const uint64_t t = share_of(q.p, k ? L.klo : all);
        if (before <= t && before + w > t) atomicMin(&L.lo, bin);
        if (before < t) atomicMax(&L.hi, bin);
    }
    __syncthreads();
    int lo = L.lo, hi = L.hi;
    if (k) {
        lo = ws ? min(lo, L.kbin) : q.p < 1.0f ? 0 : L.kbin;
        hi = L.kbin;
    } else if (ws && lo > hi) {
        lo = hi + 1;  // the cut falls between two bins
    } else if (q.p < 1.0f && !ws) {
        lo = 0;  // fewer than k are in the bins: all of them are listed
        hi = NB - 1;
        k = q.k;
    }
    if (on && bin == lo) {  // what lies before the list
        L.below = before;
        L.count_below = (int)cbefore;
    }
    __syncthreads();
    return Cut{L.below, ws ? all : 0, lo, hi, L.count_below, k};
}
// v = x c of min_p.
__device__ __forceinline__ double least_of(const Ask& q, float most) {
    return q.minp > 0.0f ? (double)most * q.c + log2((double)q.minp) : -__builtin_inf();
}
// A row that needs no weights, or has none: its token, by one thread.
__device__ __forceinline__ void told(const Args& a, int r, const Ask& q, bool ok, int at) {
    a.token[r] = ok ? at : -1;
    if (a.prob) a.prob[r] = ok ? 1.0f : 0.0f;
    if (!ok) atomicOr(a.err, q.bad ? ERR_ARG_BIT : ERR_NAN_BIT);
}

__device__ __forceinline__ Row row_of(const Ask& q, double e, double least, const Cut& c) {
    return Row{q.c, e, least, c.below, c.all, 0, c.lo, c.hi, c.count_below, c.k, q.p, 0};
}

// A workgroup a row.  Bound by latency, the loads of the chunks' histograms and
// the fetching of its own code, which is run once: one row of 38 chunks 7 us; 10 and
// 20 loads a thread in flight instead of 4 and 8, 2 KB of code more, 4 us longer.
constexpr int RT = 1024;  // threads: two a bin
__global__ __launch_bounds__(RT) void sample_row_kernel(const Args a) {
    __shared__ uint64_t half_w[NB];
    __shared__ uint32_t half_n[NB];
    __shared__ Cuts cuts;
    __shared__ float wmost[RT / 64];
    __shared__ int wat[RT / 64];
    __shared__ int shift[MAX_CHUNKS];  // whole factors of two between a chunk's scale and the row's; -1: too many
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Ask q = ask_of(a, r);
    Row* row = a.row + r;
    static_assert(MAX_CHUNKS <= RT && MAX_CHUNKS <= 64 * (RT / 64), "");
    float most = -__builtin_inff();
    int at = 0;
    double mine = 0.0;
    if (tid < a.chunks) {
        const Chunk c = a.chunk[(int64_t)r * a.chunks + tid];
        most = c.most;
        at = c.at;
        mine = c.e;
    }
    // the first chunk with the largest number holds its first index
    float top = most;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    const int who = __builtin_ctzll(__builtin_amdgcn_ballot_w64(most == top) | (1ull << 63));
    if (lane == who) {
        wmost[wave] = top;
        wat[wave] = at;
    }
    if (tid == 0) cut_start(cuts);
    const bool nan = __syncthreads_or(at < 0);
    most = wmost[0];
    at = wat[0];
    for (int i = 1; i < (a.chunks + 63) / 64; ++i)
        if (wmost[i] > most) {
            most = wmost[i];
            at = wat[i];
        }
    const bool finite = most > -__builtin_inff() && most < __builtin_inff();
    if (q.bad || nan || !finite || q.greedy) {
        if (tid == 0) {
            told(a, r, q, !q.bad && !nan && finite, at);
            row->done = 1;
        }
        return;
    }
    const double e = __builtin_ceil((double)most * q.c);
    const bool ws = q.weights(), ns = q.counts();
    Cut cut{0, 0, NB, -1, 0, 0};
    if (ws || ns) {
        if (tid < a.chunks) {
            const double de = e - mine;  // whole, or infinite
            shift[tid] = de <= 51.0 ? (int)de : -1;
        }
        __syncthreads();
        uint64_t w = 0;
        uint32_t n = 0;
        const int bin = tid % NB;
        const int64_t base = (int64_t)r * a.chunks * NB;
        // (loads without a branch: all in flight)
        if (ws) {
#pragma unroll 4
            for (int i = tid / NB; i < a.chunks; i += RT / NB) {
                const int sh = shift[i], b = bin - PER * sh;
                const bool in = sh >= 0 && b >= 0;
                const uint64_t wb = a.weight[base + i * NB + (in ? b : 0)];
                w += in ? wb >> sh : 0;
            }
        }
        if (ns) {
#pragma unroll 8
            for (int i = tid / NB; i < a.chunks; i += RT / NB) {
                const int sh = shift[i], b = bin - PER * sh;
                const bool in = sh >= 0 && b >= 0;
                const uint32_t nb = a.count[base + i * NB + (in ? b : 0)];
                n += in ? nb : 0;
            }
        }
        if (tid >= NB) {
            half_w[bin] = w;
            half_n[bin] = n;
        }
        __syncthreads();
        if (tid < NB) {
            w += half_w[bin];
            n += half_n[bin];
        }
        cut = cut_bins(q, cuts, w, n);
    }
    if (tid == 0) *row = row_of(q, e, least_of(q, most), cut);
}

// Adds up what of a chunk is kept whole; returns which of the thread's elements go
// to the list (bit 4 i + j: element j of quad i).
template <typename H>
__device__ __forceinline__ uint32_t split_chunk(const H& held, int beg, int end, double c, double e, double ce,
                                                double least, int lo, int hi, int s, uint64_t& sum) {
    const int sh = PER * (int)(e - ce);
    // what lies past the bins, or has no weight, or (without a list) is below
    // min_p, by whole waves
    double past = fmax(e - (double)(hi >= lo ? hi + 1 : lo) / (double)PER, e - (double)(s + 1));
    if (hi < lo) past = fmax(past, least);
    const float skip = floor_of(past, e, c);
    uint32_t in = 0;
    held.each([&](int i, const F4& f) {
        if (!__builtin_amdgcn_ballot_w64(top_of(f) >= skip)) return;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double v = (double)f.v[j] * c;  // (past the end: -inf)
            const int b = bin_of(ce, v) + sh;
            if (b < lo && v >= least) sum += weight_of(v - e + (double)s);
            in |= b >= lo && b <= hi && beg + 4 * (i * NT + (int)threadIdx.x) + j < end ? 1u << (4 * i + j) : 0u;
        }
    });
    return in;
}
// The thread's elements of the list, from place `to` on, up to CAP.
template <typename H>
__device__ __forceinline__ void put_list(const H& held, int beg, uint32_t in, int to, uint64_t* list) {
    held.each([&](int i, const F4& f) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (in >> (4 * i + j) & 1) {
                if (to < CAP) list[to] = key_of(f.v[j], beg + 4 * (i * NT + (int)threadIdx.x) + j);
                ++to;
            }
    });
}

// A workgroup a chunk again (15 us there): the weights of what is kept whole, by the
// row's scale, and the list's elements, one atomic a workgroup.
template <int NV>
__global__ __launch_bounds__(NT) void sample_take_kernel(const Args a) {
    __shared__ uint64_t tmp[NT / 64];
    __shared__ int place;
    const int r = blockIdx.x / a.chunks, ch = blockIdx.x % a.chunks, tid = threadIdx.x;
    Row* rp = a.row + r;
    const float* x = a.x + (int64_t)r * a.pitch;
    const int beg = ch * a.len, end = min(beg + a.len, a.n);
    Held<NV> held;
#pragma unroll
    for (int i = 0; i < NV; ++i) held.f[i] = load4(x, beg + 4 * (i * NT + tid), end);
    if (rp->done) return;
    const double c = rp->c, e = rp->e, least = rp->least;
    const int lo = rp->lo, hi = rp->hi;
    const double ce = a.chunk[(int64_t)r * a.chunks + ch].e, de = e - ce;
    uint64_t sum = 0;
    uint32_t in = 0;
    if (de <= 51.0) in = split_chunk(held, beg, end, c, e, ce, least, lo, hi, a.s, sum);
    sum = group_sum<NT>(sum, tmp);
    if (tid == 0) a.kept[(int64_t)r * a.chunks + ch] = sum;
    if (hi < lo) return;
    uint64_t mine;  // one atomic a workgroup
    int to = (int)group_before<NT>((uint64_t)__builtin_popcount(in), tmp, &mine);
    if (tid == 0 && mine) place = atomicAdd(&rp->listed, (int)mine);
    __syncthreads();
    if (!in) return;
    put_list(held, beg, in, to + place, a.list + (int64_t)r * CAP);
}

struct Last {  // the row's last launch
    uint64_t kept[MAX_CHUNKS];
    double e[MAX_CHUNKS];
    uint64_t few[FEW], order[FEW];
    uint64_t tmp[FT / 64];
    unsigned long long weight[NB];
    uint32_t count[NB];
    uint64_t rest, before;
    int at, chunk, bin, n;
    uint64_t list[1];  // CAP, where it is needed
};

// few[0 .. n - 1], n up to FEW different keys, in descending order.
__device__ __forceinline__ void put_in_order(Last& L, int n) {
    __syncthreads();
    const int tid = threadIdx.x;
    if (tid < (n + 63) / 64 * 64) {  // whole waves
        const uint64_t mine = tid < n ? L.few[tid] : 0;
        int place = 0;
#pragma unroll 4
        for (int i = 0; i < n; ++i) place += L.few[i] > mine;
        if (tid < n) L.order[place] = mine;
    }
    __syncthreads();
}

// Runs f(key, v, chunk) over the row's elements of the list's bins.
template <typename F>
__device__ __forceinline__ void over_row(const Args& a, const Row& row, const Last& L, const float* x, F&& f) {
#pragma unroll 1
    for (int ch = 0; ch < a.chunks; ++ch) {
        const int end = min((ch + 1) * a.len, a.n);
        const double ce = L.e[ch], de = row.e - ce;
        if (!(de <= 51.0)) continue;
        const int sh = PER * (int)de;
#pragma unroll 1
        for (int i = ch * a.len + 4 * (int)threadIdx.x; i < end; i += 4 * FT) {
            const F4 v4 = load4(x, i, end);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double v = (double)v4.v[j] * row.c;
                const int b = bin_of(ce, v) + sh;
                if (i + j < end && b >= row.lo && b <= row.hi) f(key_of(v4.v[j], i + j), v, ch);
            }
        }
    }
}
__device__ __forceinline__ double v_of(const Row& row, uint64_t key) {
    return (double)value_of((uint32_t)(key >> 32)) * row.c;
}

// The last key that is kept of the elements of the list's bins with keys of
// `limit` and more: of the first `want`, or (by_weight) of those with less than
// `want` before them, `before` with the bins before.  *sum: the weight kept, with
// `before`.  Over the row: eight bits of the order at a time, then the index among
// equal ones.
__device__ __forceinline__ uint64_t cut_row(const Args& a, const Row& row, const float* x, Last& L, bool by_weight,
                                            uint64_t before, uint64_t want, uint64_t limit, uint64_t* sum) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    uint64_t total = before, n = 0;  // of larger keys
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        L.count[tid] = 0;
        L.weight[tid] = 0;
        __syncthreads();
        over_row(a, row, L, x, [&](uint64_t key, double v, int) {
            const uint32_t o = (uint32_t)(key >> 32);
            if (key < limit || (shift < 24 && o >> (shift + 8) != prefix)) return;
            atomicAdd(&L.weight[o >> shift & 255], (unsigned long long)weight_of(v - row.e + (double)a.s));
            atomicAdd(&L.count[o >> shift & 255], 1u);
        });
        __syncthreads();
        int d = 255;
        for (; d > 0; --d) {
            if (by_weight ? total + L.weight[d] >= want : n + L.count[d] >= want) break;
            total += L.weight[d];
            n += L.count[d];
        }
        prefix = prefix << 8 | (uint32_t)d;
    }
    // equal ones: how many of them, then the index of the last
    const uint64_t w = weight_of((double)value_of(prefix) * row.c - row.e + (double)a.s), ties = L.count[prefix & 255];
    uint64_t take = by_weight ? (total >= want ? 0 : w ? (want - total + w - 1) / w : ties) : want - n;
    if (take > ties) take = ties;
    *sum = total + take * w;
    if (!take) return prefix == 0xFFFFFFFFu ? ~0ull : (uint64_t)(prefix + 1) << 32;  // none of them
    uint64_t seen = 0;
    __syncthreads();
    if (tid == 0) L.at = -1;
    for (int base = 0; base < a.n && seen < take; base += FT) {
        const int i = base + tid;
        const uint64_t mine = i < a.n && order_of(x[i]) == prefix && key_of(x[i], i) >= limit;
        uint64_t all;
        const uint64_t prior = seen + group_before<FT>(mine, L.tmp, &all);
        if (mine && prior + 1 == take) L.at = i;
        seen += all;
    }
    __syncthreads();
    return (uint64_t)prefix << 32 | (uint32_t)~L.at;
}

// The same over the list (FEW < n <= CAP, in LDS): bins of equal width over the
// list's, then the elements of one in order.  False where that one has too many.
__device__ __forceinline__ bool cut_list(const Args& a, const Row& row, int n, Last& L, bool by_weight, uint64_t before,
                                         uint64_t want, uint64_t limit, uint64_t* sum, uint64_t* cut) {
    const int tid = threadIdx.x;
    if (by_weight && before >= want) {  // none
        *sum = before;
        *cut = ~0ull;
        return true;
    }
    const double scale = (double)NB / (double)(row.hi - row.lo + 1);
    auto bin = [&](uint64_t key) {  // (falls with the key)
        const double d = ((row.e - v_of(row, key)) * (double)PER - (double)row.lo) * scale;
        return d < (double)(NB - 1) ? d > 0.0 ? (int)d : 0 : NB - 1;
    };
    auto weight = [&](uint64_t key) { return weight_of(v_of(row, key) - row.e + (double)a.s); };
    __syncthreads();
    L.count[tid] = 0;
    L.weight[tid] = 0;
    if (tid == 0) {
        L.bin = -1;
        L.n = 0;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < n; i += FT) {
        const uint64_t key = L.list[i];
        if (key < limit) continue;
        const int b = bin(key);
        atomicAdd(&L.weight[b], (unsigned long long)weight(key));
        atomicAdd(&L.count[b], 1u);
    }
    __syncthreads();
    const uint64_t w = L.weight[tid], c = L.count[tid];
    uint64_t all;
    const uint64_t wb = before + group_before<FT>(w, L.tmp, &all), cb = group_before<FT>(c, L.tmp);
    if (c && (by_weight ? wb < want && wb + w >= want : cb < want && cb + c >= want)) {
        L.bin = tid;
        L.before = wb;
        L.chunk = (int)cb;
    }
    __syncthreads();
    const int at = L.bin;
    if (at < 0) {  // all of them
        *sum = before + all;
        *cut = limit;
        return true;
    }
    if (L.count[at] > FEW) return false;
    const uint64_t start = L.before, first = (uint64_t)L.chunk;
#pragma unroll 1
    for (int i = tid; i < n; i += FT) {
        const uint64_t key = L.list[i];
        if (key >= limit && bin(key) == at) L.few[atomicAdd(&L.n, 1)] = key;
    }
    __syncthreads();
    const int m = L.n;
    put_in_order(L, m);
    const uint64_t mine = tid < m ? weight(L.order[tid]) : 0;
    const uint64_t prior = start + group_before<FT>(mine, L.tmp);
    const bool in = tid < m && (by_weight ? prior < want : first + (uint64_t)tid < want);
    const int taken = __syncthreads_count(in);
    *sum = start + group_sum<FT>(in ? mine : 0, L.tmp);
    *cut = L.order[taken - 1];  // (the bin holds the last one)
    __syncthreads();
    return true;
}

// The cuts in the row's list of n (in few where it is short, else in list where
// that holds it), its token and share; kept, e: of the chunks, what of them is kept
// whole and their scales.  Bound by latency: one chain of a dozen barriers, whose
// code is run once, and so is kept short.
__device__ __forceinline__ void finish_row(const Args& a, const float* x, const Row& row, int r, int n, Last& L) {
    const int tid = threadIdx.x;
    const double s = (double)a.s;
    uint64_t two[2];
    uint64_t cut = 0;  // the last key of the list that is kept
    auto weight = [&](uint64_t key) { return weight_of(v_of(row, key) - row.e + s); };
    auto keep = [&](uint64_t key) {
        if (v_of(row, key) >= row.least)
            atomicAdd((unsigned long long*)&L.kept[(int)~(uint32_t)key / a.len], (unsigned long long)weight(key));
    };
    if (n > 0 && n <= FEW) {
        put_in_order(L, n);
        const uint64_t key = L.order[tid < n ? tid : 0], w = tid < n ? weight(key) : 0;
        const bool first = tid < (row.k ? min(n, row.k - row.count_below) : n);
        uint64_t total = row.all;
        const uint64_t before = row.below + group_before<FT>(w, L.tmp);
        if (row.k) total = row.below + group_sum<FT>(first ? w : 0, L.tmp);
        const bool in = first && (row.p == 1.0f || before < share_of(row.p, total));
        const int taken = __syncthreads_count(in);
        cut = taken ? L.order[taken - 1] : ~0ull;
        if (in) keep(key);
    } else if (n > FEW) {
        const bool here = n <= CAP;
        __syncthreads();
        // by the number, then by the share
        uint64_t total = row.all;
#pragma unroll 1
        for (int by = row.k ? 0 : 1; by < (row.p < 1.0f ? 2 : 1); ++by) {
            const uint64_t want = by ? share_of(row.p, total) : (uint64_t)(row.k - row.count_below), limit = cut;
            uint64_t sum;
            if (!here || !cut_list(a, row, n, L, by, row.below, want, limit, &sum, &cut))
                cut = cut_row(a, row, x, L, by, row.below, want, limit, &sum);
            cut = cut > limit ? cut : limit;
            total = sum;
        }
        __syncthreads();
        if (here) {
#pragma unroll 1
            for (int i = tid; i < n; i += FT)
                if (L.list[i] >= cut) keep(L.list[i]);
        } else {
            over_row(a, row, L, x, [&](uint64_t key, double, int) {
                if (key >= cut) keep(key);
            });
        }
    }
    if (tid == 0) {
        L.chunk = 0;
        L.rest = ~0ull;
    }
    __syncthreads();
    // the chunk of the token (two a thread)
#pragma unroll
    for (int j = 0; j < 2; ++j) two[j] = 2 * tid + j < a.chunks ? L.kept[2 * tid + j] : 0;
    uint64_t total;
    uint64_t before = group_before<FT>(two[0] + two[1], L.tmp, &total);
    const float u = fminf(fmaxf(a.u[r], 0.0f), 0.999999940395355225f);  // below 1: 1 - 2^-24
    bool more;
    const uint64_t target = part_of(u, total, &more);  // below total, which holds the largest weight
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if (target >= before && target - before < two[j]) {
            L.chunk = 2 * tid + j;
            L.rest = target - before;
        }
        before += two[j];
    }
    __syncthreads();
    // the token: the chunk in runs of four a thread
    const int ch = L.chunk, end = min((ch + 1) * a.len, a.n);
    const double ce = L.e[ch];
    const int sh = PER * (int)(row.e - ce);
    uint64_t rest = L.rest;
    int i = ch * a.len + 4 * tid;
    F4 f = load4(x, i, end);
#pragma unroll 1
    for (;;) {
        const F4 next = load4(x, i + 4 * FT, end);
        uint64_t w[4], mine = 0, sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double v = (double)f.v[j] * row.c;
            const int b = bin_of(ce, v) + sh;
            const bool in = i + j < end && v >= row.least && (b < row.lo || (b <= row.hi && key_of(f.v[j], i + j) >= cut));
            w[j] = in ? weight_of(v - row.e + s) : 0;
            mine += w[j];
        }
        before = group_before<FT>(mine, L.tmp, &sum);
        if (rest < sum || i - 4 * tid + 4 * FT >= end) {
            if (rest >= before && rest - before < mine) {
                rest -= before;
                int j = 0;
                uint64_t wj = w[0];
#pragma unroll
                for (int k = 1; k < 4; ++k)
                    if (j == k - 1 && rest >= wj) {
                        rest -= wj;
                        wj = w[k];
                        j = k;
                    }
                a.token[r] = i + j;
                if (a.prob) a.prob[r] = (float)((double)wj / (double)total);
            }
            return;
        }
        rest -= sum;
        i += 4 * FT;
        f = next;
    }
}

// A workgroup a row (finish_row): one row 7 us, 64 rows 11, those with the longest lists.
__global__ __launch_bounds__(FT) void sample_token_kernel(const Args a) {
    extern __shared__ __align__(16) char lds[];
    Last& L = *reinterpret_cast<Last*>(lds);
    const int r = blockIdx.x, tid = threadIdx.x;
    const Row row = a.row[r];
    const uint64_t* list = a.list + (int64_t)r * CAP;
    const uint64_t ahead = list[tid];  // (memory of the list, whatever its length)
    uint64_t two[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) two[j] = tid + j * FT < a.chunks ? a.kept[(int64_t)r * a.chunks + tid + j * FT] : 0;
    if (row.done) return;
    const int n = row.listed;
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (tid + j * FT < a.chunks) {
            L.kept[tid + j * FT] = two[j];
            L.e[tid + j * FT] = a.chunk[(int64_t)r * a.chunks + tid + j * FT].e;
        }
    if (n <= FEW) {
        L.few[tid] = ahead;
    } else if (n <= CAP) {
        L.list[tid] = ahead;
#pragma unroll 4
        for (int i = tid + FT; i < n; i += FT) L.list[i] = list[i];
    }
    finish_row(a, a.x + (int64_t)r * a.pitch, row, r, n, L);
}

// Rows of up to ONE logits: all of it in one launch, a workgroup a row, the logits
// in LDS and nothing else read.  Latency bounds it.  Against the four launches, in us:
// a row of 1000 14 -> 6, 7 rows of 5000 22 -> 19, 256 rows of 2000 24 -> 15; 64 rows
// of 16384 in one chunk 26 -> 29, so ONE lies below that.
constexpr int ONE = 8192;
__global__ __launch_bounds__(NT) void sample_one_kernel(const Args a) {
    extern __shared__ __align__(16) char lds[];
    __shared__ Most tops;
    __shared__ Cuts cuts;
    Last& L = *reinterpret_cast<Last*>(lds);
    static_assert(NT == FT && ONE / (4 * NT) * 4 <= 32 && offsetof(Last, list) % 16 == 0, "");
    const int r = blockIdx.x, tid = threadIdx.x;
    const float* x = a.x + (int64_t)r * a.pitch;
    F4* quad = reinterpret_cast<F4*>(L.list + (a.n > FEW ? (a.n + 1) / 2 * 2 : 0));
    const Staged held{quad, a.len / (4 * NT)};
#pragma unroll 4
    for (int i = 0; i < held.quads; ++i) quad[i * NT + tid] = load4(x, 4 * (i * NT + tid), a.n);  // (each thread its own)
    const Ask q = ask_of(a, r);
    L.weight[tid] = 0;
    L.count[tid] = 0;
    if (tid == 0) cut_start(cuts);
    float most;
    int at;
    const bool nan = most_of(held, 0, tops, most, at), finite = most > -__builtin_inff() && most < __builtin_inff();
    if (q.bad || nan || !finite || q.greedy) {
        if (tid == 0) told(a, r, q, !q.bad && !nan && finite, at);
        return;
    }
    const double e = __builtin_ceil((double)most * q.c), least = least_of(q, most);
    Cut cut{0, 0, NB, -1, 0, 0};
    if (q.weights() || q.counts()) {
        add_bins(held, q, e, a.s, L.weight, L.count);
        __syncthreads();
        cut = cut_bins(q, cuts, L.weight[tid], L.count[tid]);
    }
    uint64_t sum = 0, n = 0;
    const uint32_t in = split_chunk(held, 0, a.n, q.c, e, e, least, cut.lo, cut.hi, a.s, sum);
    sum = group_sum<NT>(sum, L.tmp);
    if (cut.hi >= cut.lo) {
        const int to = (int)group_before<NT>((uint64_t)__builtin_popcount(in), L.tmp, &n);
        if (in) put_list(held, 0, in, to, n <= FEW ? L.few : L.list);
    }
    if (tid == 0) {
        L.kept[0] = sum;
        L.e[0] = e;
    }
    finish_row(a, reinterpret_cast<const float*>(quad), row_of(q, e, least, cut), r, (int)n, L);
}

// How a call's rows are cut, and its workspace.
struct Plan {
    int quads, chunks, len, s;  // quads a thread; logits a chunk
    size_t row, chunk, weight, count, kept, list, bytes;
};
int s_of(size_t n) {
    int bits = 0;
    while (((size_t)1 << bits) < n) ++bits;
    return std::min(MAX_S, 62 - bits);
}
Plan plan_of(size_t m, size_t n) {
    Plan p{};
    p.quads = MAX_V;
    auto cut = [&]() {
        p.len = 4 * NT * p.quads;
        p.chunks = (int)((n + p.len - 1) / p.len);
    };
    cut();
    p.s = s_of(n);
    if (n <= (size_t)ONE) {
        p.quads = (int)((n + 4 * NT - 1) / (4 * NT));
        cut();
        p.bytes = 256;  // nothing is kept between launches
        return p;
    }
    while (p.quads > 1 && m * p.chunks < 1024 && p.chunks < 20) {
        p.quads /= 2;
        cut();
    }
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t q = at;
        at += round_up(bytes, 256);
        return q;
    };
    const size_t all = m * (size_t)p.chunks;
    p.row = take(m * sizeof(Row));
    p.chunk = take(all * sizeof(Chunk));
    p.weight = take(all * NB * 8);
    p.count = take(all * NB * 4);
    p.kept = take(all * 8);
    p.list = take(m * CAP * 8);
    p.bytes = at;
    return p;
}

int bad(const char* msg) { return set_error(FRQ_ERR_ARG, msg); }

struct Guard {
    int prev = -1;
    explicit Guard(int d) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev != d) (void)hipSetDevice(d);
    }
    ~Guard() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

constexpr size_t MAX_M = 1 << 20;

template <typename K>
hipError_t with_lds(K kernel, int lds) {
    if (lds <= 48 * 1024) return hipSuccess;
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
}
hipError_t launch_one(const Args& a, size_t m, hipStream_t s) {
    static_assert(sizeof(Last) + ONE * 8 + ONE * 4 + 1024 <= 160 * 1024, "LDS of a CU");
    const int lds = (int)sizeof(Last) + (a.n > FEW ? (a.n + 1) / 2 * 16 : 0) + a.len * 4;
    if (const hipError_t e = with_lds(sample_one_kernel, lds); e != hipSuccess) return e;
    sample_one_kernel<<<dim3((unsigned)m), dim3(NT), lds, s>>>(a);
    return hipGetLastError();
}
template <int NV>
hipError_t launch(const Args& a, size_t m, hipStream_t s) {
    static_assert(sizeof(Last) + CAP * 8 + 1024 <= 160 * 1024, "LDS of a CU");
    const dim3 rows((unsigned)m), all((unsigned)(m * a.chunks));
    const int lds = (int)sizeof(Last) + CAP * 8;
    if (const hipError_t e = with_lds(sample_token_kernel, lds); e != hipSuccess) return e;
    sample_bins_kernel<NV><<<all, dim3(NT), 0, s>>>(a);
    sample_row_kernel<<<rows, dim3(RT), 0, s>>>(a);
    sample_take_kernel<NV><<<all, dim3(NT), 0, s>>>(a);
    sample_token_kernel<<<rows, dim3(FT), lds, s>>>(a);
    return hipGetLastError();
}

}  // namespace
}  // namespace smp
}  // namespace frq

using namespace frq;
using namespace frq::smp;

extern "C" {

size_t frq_sample_ws(size_t m, size_t n) {
    if (!m || !n || n > (size_t)MAX_N || m > MAX_M) return 0;
    return plan_of(m, n).bytes;
}

int frq_sample_dev(frq_ctx* ctx, const float* d_logits, size_t pitch, size_t m, size_t n, const float* d_temp,
                   const int32_t* d_topk, const float* d_topp, const float* d_minp, const float* d_u, int64_t* d_token,
                   float* d_prob, void* d_ws, size_t ws_bytes) {
    if (!n || n > (size_t)MAX_N) return bad("frq_sample_dev: n must be in [1, 2^24]");
    if (m > MAX_M) return bad("too many rows");
    if (pitch < n || pitch > ((size_t)1 << 40)) return bad("pitch is below the row's width");
    if (m && (!d_logits || !d_u || !d_token)) return bad("null pointer");
    if (d_ws && ((uintptr_t)d_ws & 15)) return bad("the workspace must be 16-byte aligned");
    if (!ctx) return bad("null context");
    if (!m) return FRQ_OK;
    const Plan p = plan_of(m, n);
    if (d_ws && ws_bytes < p.bytes) return bad("the workspace is below frq_sample_ws");
    Guard g(ctx_device(ctx));
    hipStream_t s = (hipStream_t)frq_get_stream(ctx);
    if (!d_ws) {
        // the context's workspace may move with a later call: a graph would
        // keep its old address
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        const hipError_t e = hipStreamIsCapturing(s, &st);
        if (e != hipSuccess) return set_error(FRQ_ERR_HIP, std::string("hipStreamIsCapturing: ") + hipGetErrorString(e));
        if (st != hipStreamCaptureStatusNone) return bad("under graph capture the caller gives the workspace");
        if (int rc = ctx_ws(ctx, p.bytes, &d_ws)) return rc;
    }
    char* ws = (char*)d_ws;
    const Args a{d_logits, (int64_t)pitch, (int)n, p.s, p.chunks, p.len, d_temp, d_topp, d_minp, d_u, d_topk, d_token, d_prob,
                 (Row*)(ws + p.row), (Chunk*)(ws + p.chunk), (uint64_t*)(ws + p.weight), (uint32_t*)(ws + p.count),
                 (uint64_t*)(ws + p.kept), (uint64_t*)(ws + p.list), ctx_err(ctx)};
    hipError_t e = hipSuccess;
    if (n <= (size_t)ONE) e = launch_one(a, m, s);
    else if (p.quads == 1) e = launch<1>(a, m, s);
    else if (p.quads == 2) e = launch<2>(a, m, s);
    else if (p.quads == 4) e = launch<4>(a, m, s);
    else e = launch<8>(a, m, s);
    return e == hipSuccess ? FRQ_OK : set_error(FRQ_ERR_HIP, std::string("launch sample: ") + hipGetErrorString(e));
}

}  // extern "C"
