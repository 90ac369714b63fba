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
// so that every sum is exact and the same in any order: a row is cut over
// workgroups, and their sums meet in atomics, without the token depending on it.
// (w' is w times a factor for all of a row that puts the largest between 1/2 and
// 1; at 152064 tokens a step is 2^-44, and what is below half of it is none.)
//
// Nothing is sorted but a few candidates.  Three launches: each chunk's maximum
// and its histogram over the logarithm of w, ten bins a factor of two; the bins
// summed for the row, which gives those that are kept whole and those (one, mostly)
// where a cut falls; then each chunk's sum of what is kept whole, and the elements
// of the bins between as a list, which the row's last workgroup sorts, cuts, and
// walks to the token.  A list that is too long (many equal logits) is cut by
// radix selection over the row instead.
#include "frq_internal.h"

namespace frq {
namespace smp {
namespace {

constexpr int NT = 256;           // threads
constexpr int NB = 512, PER = 10; // bins, bins a factor of two: 51 of them
constexpr int MAX_S = 50;         // E - v <= s + 1 where a weight is not zero
constexpr int CAP = 2048;         // candidates of a row's list
constexpr int MAX_N = 1 << 24;
constexpr int MAX_CHUNKS = 64;
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
    int listed, ticket; // the list's length (may pass CAP), workgroups done
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

// Over the workgroup.
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor((unsigned long long)v, d, 64);
    return v;
}
__device__ uint64_t group_sum(uint64_t v, uint64_t* tmp) {  // tmp: [NT / 64]
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) v += tmp[i];
    return v;
}
// The sum of the threads before.
__device__ uint64_t group_before(uint64_t v, uint64_t* tmp) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint64_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up((unsigned long long)x, d, 64);
        if (lane >= d) x += o;
    }
    __syncthreads();
    if (lane == 63) tmp[w] = x;
    __syncthreads();
    uint64_t before = x - v;
    for (int i = 0; i < w; ++i) before += tmp[i];
    return before;
}

__global__ __launch_bounds__(NT) void sample_bins_kernel(const Args a) {
    __shared__ unsigned long long weight[NB];
    __shared__ uint32_t count[NB];
    __shared__ float wmost[NT / 64];
    __shared__ int wat[NT / 64];
    const int r = blockIdx.x / a.chunks, ch = blockIdx.x % a.chunks, tid = threadIdx.x;
    const float* x = a.x + (int64_t)r * a.pitch;
    const int beg = ch * a.len, end = min(beg + a.len, a.n);
    const Ask q = ask_of(a, r);
    float most = -__builtin_inff();
    int at = beg < end ? beg : 0;
    bool nan = false;
    for (int i = beg + 4 * tid; i < end; i += 4 * NT) {
        const F4 f = load4(x, i, end);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            nan |= f.v[j] != f.v[j];
            if (f.v[j] > most) {
                most = f.v[j];
                at = i + j;
            }
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float o = __shfl_xor(most, d, 64);
        const int oa = __shfl_xor(at, d, 64);
        if (o > most || (o == most && oa < at)) {
            most = o;
            at = oa;
        }
    }
    if ((tid & 63) == 0) {
        wmost[tid >> 6] = most;
        wat[tid >> 6] = at;
    }
    nan = __syncthreads_or(nan);
#pragma unroll
    for (int i = 0; i < NT / 64; ++i)
        if (wmost[i] > most || (wmost[i] == most && wat[i] < at)) {
            most = wmost[i];
            at = wat[i];
        }
    const double e = __builtin_ceil((double)most * q.c);
    if (tid == 0) a.chunk[(int64_t)r * a.chunks + ch] = Chunk{e, most, nan ? -1 : at};
    if ((!q.k && q.p == 1.0f) || q.greedy || q.bad) return;
    for (int i = tid; i < NB; i += NT) {
        weight[i] = 0;
        count[i] = 0;
    }
    __syncthreads();
    if (!nan && most > -__builtin_inff() && most < __builtin_inff()) {
        for (int i = beg + 4 * tid; i < end; i += 4 * NT) {
            const F4 f = load4(x, i, end);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double v = (double)f.v[j] * q.c;
                const uint64_t w = weight_of(v - e + (double)a.s);
                if (w) {
                    const int b = min(bin_of(e, v), NB - 1);
                    atomicAdd(&weight[b], (unsigned long long)w);
                    atomicAdd(&count[b], 1u);
                }
            }
        }
    }
    __syncthreads();
    const int64_t to = ((int64_t)r * a.chunks + ch) * NB;
    for (int i = tid; i < NB; i += NT) {
        a.weight[to + i] = weight[i];
        a.count[to + i] = count[i];
    }
}

// f total for f of [0, 1), down to a whole number and whether it is more; exact
// (a sum of many equal weights has more bits than a double).
__device__ __forceinline__ uint64_t part_of(float f, uint64_t total, bool* more) {
    const uint32_t u = __float_as_uint(f), e = u >> 23, m = e ? (u & 0x7FFFFFu) | 0x800000u : u & 0x7FFFFFu;
    const int sh = 150 - (int)(e ? e : 1);  // f = m 2^-sh, sh of 24 and more
    const unsigned __int128 x = (unsigned __int128)total * m;
    if (sh >= 128) {
        *more = x != 0;
        return 0;
    }
    *more = (x & (((unsigned __int128)1 << sh) - 1)) != 0;
    return (uint64_t)(x >> sh);
}
// ceil(p total), at least one: what lies before an element is less than that
// where the element is kept.
__device__ __forceinline__ uint64_t share_of(float p, uint64_t total) {
    bool more;
    const uint64_t t = part_of(p, total, &more) + more;
    return t > 0 ? t : 1;
}

__global__ __launch_bounds__(NT) void sample_row_kernel(const Args a) {
    __shared__ uint64_t tmp[NT / 64];
    __shared__ int kbin, lo, hi;
    __shared__ uint64_t klo;
    __shared__ int shift[MAX_CHUNKS];  // whole factors of two between a chunk's scale and the row's; -1: too many
    const int r = blockIdx.x, tid = threadIdx.x;
    const Ask q = ask_of(a, r);
    const Chunk* chunk = a.chunk + (int64_t)r * a.chunks;
    Row* row = a.row + r;
    float most = -__builtin_inff();
    int at = 0;
    bool nan = false;
    double e = -__builtin_inf();
    for (int i = 0; i < a.chunks; ++i) {
        const Chunk c = chunk[i];
        nan |= c.at < 0;
        if (c.most > most) {
            most = c.most;
            at = c.at;
        }
        e = fmax(e, c.e);
    }
    const bool finite = most > -__builtin_inff() && most < __builtin_inff();
    if (q.bad || nan || !finite || q.greedy) {
        if (tid == 0) {
            const bool ok = !q.bad && !nan && finite;
            a.token[r] = ok ? at : -1;
            if (a.prob) a.prob[r] = ok ? 1.0f : 0.0f;
            if (!ok) atomicOr(a.err, q.bad ? ERR_ARG_BIT : ERR_NAN_BIT);
            row->done = 1;
        }
        return;
    }
    uint64_t before[2] = {0, 0}, w[2] = {0, 0}, all = 0, below = 0;
    uint32_t cbefore[2] = {0, 0}, n[2] = {0, 0};
    int count_below = 0, k = 0;
    if (tid == 0) {
        kbin = NB;
        lo = NB;
        hi = -1;
        klo = 0;
    }
    __syncthreads();
    if (q.k || q.p < 1.0f) {
        if (tid < a.chunks) {
            const double de = e - chunk[tid].e;  // whole, or infinite
            shift[tid] = de <= 51.0 ? (int)de : -1;
        }
        __syncthreads();
#pragma unroll 8
        for (int i = 0; i < a.chunks; ++i) {
            const int sh = shift[i];
            const int64_t from = ((int64_t)r * a.chunks + i) * NB;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int b = 2 * tid + j - PER * sh;
                const bool in = sh >= 0 && b >= 0;
                const int64_t at = from + (in ? b : 0);  // (loads without a branch, to be in flight together)
                const uint64_t wb = a.weight[at];
                const uint32_t nb = a.count[at];
                w[j] += in ? wb >> sh : 0;
                n[j] += in ? nb : 0;
            }
        }
        before[0] = group_before(w[0] + w[1], tmp);
        cbefore[0] = (uint32_t)group_before(n[0] + n[1], tmp);
        before[1] = before[0] + w[0];
        cbefore[1] = cbefore[0] + n[0];
        all = group_sum(w[0] + w[1], tmp);
        // the bin where the k largest end
        if (q.k) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (cbefore[j] < (uint32_t)q.k && cbefore[j] + n[j] >= (uint32_t)q.k) {
                    kbin = 2 * tid + j;
                    klo = before[j];
                }
        }
        __syncthreads();
        k = kbin < NB ? q.k : 0;
        const int kb = kbin;
        const uint64_t sure = k ? klo : all;
        if (q.p < 1.0f) {
            const uint64_t t = share_of(q.p, sure);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (w[j] && before[j] <= t) {
                    if (before[j] + w[j] > t) atomicMin(&lo, 2 * tid + j);
                    if (before[j] < t) atomicMax(&hi, 2 * tid + j);
                }
        }
        __syncthreads();
        if (tid == 0) {
            if (k) {
                lo = min(lo, kb);
                hi = kb;
            } else if (q.p < 1.0f && lo > hi) {
                lo = hi + 1;  // the cut falls between two bins
            }
        }
        __syncthreads();
        // what lies before the list
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (2 * tid + j < lo) {
                below += w[j];
                count_below += (int)n[j];
            }
        }
        below = group_sum(below, tmp);
        count_below = (int)group_sum((uint64_t)count_below, tmp);
    }
    if (tid == 0) {
        *row = Row{q.c, e, q.minp > 0.0f ? (double)most * q.c + log2((double)q.minp) : -__builtin_inf(),
                   below, all, 0, lo, hi, count_below, k, q.p, 0, 0};
    }
}

struct Last {  // the row's last workgroup
    unsigned long long list[CAP];
    uint64_t kept[MAX_CHUNKS];
    uint64_t tmp[NT / 64];
    uint32_t count[256];
    unsigned long long weight[256];
    uint64_t cut, target;
    int at, last;
};

// Descending, `size` (a power of two) keys.
__device__ void sort_list(unsigned long long* v, int size) {
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += NT) {
                const int lo = 2 * j * (i / j) + i % j, hi = lo + j;
                const unsigned long long x = v[lo], y = v[hi];
                if ((x < y) == !(lo & k)) {
                    v[lo] = y;
                    v[hi] = x;
                }
            }
        }
    __syncthreads();
}

// Runs f(key, weight) over the row's elements of the list's bins.
template <typename F>
__device__ __forceinline__ void over_list(const Args& a, const Row& row, const Chunk* chunk, const float* x, F&& f) {
    for (int ch = 0; ch < a.chunks; ++ch) {
        const int end = min((ch + 1) * a.len, a.n);
        const double ce = chunk[ch].e, de = row.e - ce;
        if (!(de <= 51.0)) continue;
        const int sh = PER * (int)de;
        for (int i = ch * a.len + 4 * (int)threadIdx.x; i < end; i += 4 * NT) {
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

// The last key of the list's elements that is kept, where they do not fit: of
// the first `want` (weight 0), or of those with less than `want` before them,
// `before` with the bins before.  Eight bits of the order at a time, then the
// index among equal ones.  Adds up what is kept into *sum.
__device__ uint64_t select_cut(const Args& a, const Row& row, const Chunk* chunk, const float* x, Last& L, bool by_weight,
                               uint64_t before, uint64_t want, uint64_t limit, uint64_t* sum) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    uint64_t total = before, n = 0;  // of larger keys
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        L.count[tid] = 0;
        L.weight[tid] = 0;
        __syncthreads();
        over_list(a, row, chunk, x, [&](uint64_t key, double v, int) {
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
    *sum = total + take * w - before;
    if (!take) return prefix == 0xFFFFFFFFu ? ~0ull : (uint64_t)(prefix + 1) << 32;  // none of them
    uint64_t seen = 0;
    __syncthreads();
    if (tid == 0) L.at = -1;
    for (int base = 0; base < a.n && seen < take; base += NT) {
        const int i = base + tid;
        const uint64_t mine = i < a.n && order_of(x[i]) == prefix && key_of(x[i], i) >= limit;
        const uint64_t prior = seen + group_before(mine, L.tmp);
        if (mine && prior + 1 == take) L.at = i;
        seen += group_sum(mine, L.tmp);
    }
    __syncthreads();
    return (uint64_t)prefix << 32 | (uint32_t)~L.at;
}

__device__ void finish_row(const Args& a, int r, Last& L) {
    const int tid = threadIdx.x;
    const Row row = a.row[r];
    const float* x = a.x + (int64_t)r * a.pitch;
    const Chunk* chunk = a.chunk + (int64_t)r * a.chunks;
    const int n = row.listed;
    const double s = (double)a.s;
    for (int i = tid; i < a.chunks; i += NT) L.kept[i] = a.kept[(int64_t)r * a.chunks + i];
    uint64_t cut = 0;  // the last key of the list that is kept
    if (n > 0 && n <= CAP) {
        int size = 2;
        while (size < n) size <<= 1;
        for (int i = tid; i < size; i += NT) L.list[i] = i < n ? a.list[(int64_t)r * CAP + i] : 0;
        sort_list(L.list, size);
        const int per = (size + NT - 1) / NT;  // a run of the order a thread
        const int beg = tid * per, end = min(beg + per, n), held = row.k ? row.k - row.count_below : n;
        auto weight = [&](int i) { return weight_of((double)value_of((uint32_t)(L.list[i] >> 32)) * row.c - row.e + s); };
        uint64_t mine = 0, got = 0;
        for (int i = beg; i < end; ++i) {
            const uint64_t w = weight(i);
            mine += w;
            if (i < held) got += w;
        }
        uint64_t before = row.below + group_before(mine, L.tmp);
        const uint64_t total = row.k ? row.below + group_sum(got, L.tmp) : row.all;
        const uint64_t want = row.p < 1.0f ? share_of(row.p, total) : ~0ull;
        uint64_t taken = 0;
        for (int i = beg; i < end; ++i) {
            taken += i < held && before < want;
            before += weight(i);
        }
        taken = group_sum(taken, L.tmp);
        cut = taken ? L.list[taken - 1] : ~0ull;
        __syncthreads();
        for (int i = tid; i < (int)taken; i += NT) {
            const float v = value_of((uint32_t)(L.list[i] >> 32));
            const int at = (int)~(uint32_t)L.list[i];
            if ((double)v * row.c >= row.least)
                atomicAdd((unsigned long long*)&L.kept[at / a.len], (unsigned long long)weight(i));
        }
    } else if (n > CAP) {
        uint64_t total = row.all, sum = 0;
        if (row.k) {
            cut = select_cut(a, row, chunk, x, L, false, row.below, (uint64_t)(row.k - row.count_below), 0, &sum);
            total = row.below + sum;
        }
        if (row.p < 1.0f) {
            const uint64_t pcut = select_cut(a, row, chunk, x, L, true, row.below, share_of(row.p, total), cut, &sum);
            cut = cut > pcut ? cut : pcut;
        }
        __syncthreads();
        over_list(a, row, chunk, x, [&](uint64_t key, double v, int ch) {
            if (key >= cut && v >= row.least)
                atomicAdd((unsigned long long*)&L.kept[ch], (unsigned long long)weight_of(v - row.e + s));
        });
    }
    __syncthreads();
    // the chunk, then the token
    uint64_t total = 0;
    for (int i = 0; i < a.chunks; ++i) total += L.kept[i];
    const float u = fminf(fmaxf(a.u[r], 0.0f), 0.999999940395355225f);  // below 1: 1 - 2^-24
    bool more;
    uint64_t target = part_of(u, total, &more);  // below total, which holds the largest weight
    int ch = 0;
    while (ch + 1 < a.chunks && target >= L.kept[ch]) target -= L.kept[ch++];
    const int first = ch * a.len, end = min(first + a.len, a.n);
    const double ce = chunk[ch].e;
    const int sh = PER * (int)(row.e - ce);
    if (tid == 0) L.at = -1;
    __syncthreads();
    for (int base = first; base < end; base += 4 * NT) {
        const int i = base + 4 * tid;
        uint64_t w[4] = {0, 0, 0, 0}, mine = 0;
        if (i < end) {
            const F4 f = load4(x, i, end);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double v = (double)f.v[j] * row.c;
                const int b = bin_of(ce, v) + sh;
                const bool in = i + j < end && v >= row.least &&
                                (b < row.lo || (b <= row.hi && key_of(f.v[j], i + j) >= cut));
                w[j] = in ? weight_of(v - row.e + s) : 0;
                mine += w[j];
            }
        }
        uint64_t before = group_before(mine, L.tmp);
        const uint64_t sum = group_sum(mine, L.tmp);
        if (target < sum) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (w[j] && target >= before && target < before + w[j]) {
                    a.token[r] = i + j;
                    if (a.prob) a.prob[r] = (float)((double)w[j] / (double)total);
                }
                before += w[j];
            }
            break;
        }
        target -= sum;
    }
}

__global__ __launch_bounds__(NT) void sample_take_kernel(const Args a) {
    __shared__ Last L;
    const int r = blockIdx.x / a.chunks, ch = blockIdx.x % a.chunks, tid = threadIdx.x, lane = tid & 63;
    Row* rp = a.row + r;
    if (rp->done) return;
    const double c = rp->c, e = rp->e, least = rp->least;
    const int lo = rp->lo, hi = rp->hi;
    const float* x = a.x + (int64_t)r * a.pitch;
    const int beg = ch * a.len, end = min(beg + a.len, a.n);
    const double ce = a.chunk[(int64_t)r * a.chunks + ch].e, de = e - ce;
    uint64_t sum = 0;
    if (de <= 51.0) {
        const int sh = PER * (int)de;
        for (int i = beg + 4 * tid; i - 4 * lane < end; i += 4 * NT) {  // whole waves
            F4 f;
            if (i < end) f = load4(x, i, end);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double v = i + j < end ? (double)f.v[j] * c : -__builtin_inf();
                const int b = bin_of(ce, v) + sh;
                if (b < lo && v >= least) sum += weight_of(v - e + (double)a.s);
                const bool in = b >= lo && b <= hi;
                const uint64_t who = __builtin_amdgcn_ballot_w64(in);
                if (who) {  // one place a wave
                    int at = 0;
                    if (lane == __builtin_ctzll(who)) at = atomicAdd(&rp->listed, __builtin_popcountll(who));
                    at = __builtin_amdgcn_readlane(at, __builtin_ctzll(who)) +
                         __builtin_popcountll(who & (((uint64_t)1 << lane) - 1));
                    if (in && at < CAP) a.list[(int64_t)r * CAP + at] = key_of(f.v[j], i + j);
                }
            }
        }
    }
    sum = group_sum(sum, L.tmp);
    if (tid == 0) a.kept[(int64_t)r * a.chunks + ch] = sum;
    // the row's last workgroup goes on
    __threadfence();
    __syncthreads();
    if (tid == 0) L.last = __hip_atomic_fetch_add(&rp->ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == a.chunks - 1;
    __syncthreads();
    if (!L.last) return;
    __threadfence();
    finish_row(a, r, L);
}

// How a call's rows are cut, and its workspace.
struct Plan {
    int chunks, len, s;
    size_t row, chunk, weight, count, kept, list, bytes;
};
Plan plan_of(size_t m, size_t n) {
    Plan p{};
    size_t want = (768 + m - 1) / m;
    want = std::min(want, (n + 2047) / 2048);
    want = std::max<size_t>(1, std::min<size_t>(want, 40));
    p.len = (int)round_up((n + want - 1) / want, 4);
    p.chunks = (int)((n + p.len - 1) / p.len);
    int bits = 0;
    while (((size_t)1 << bits) < n) ++bits;
    p.s = std::min(MAX_S, 62 - bits);
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
    const dim3 all((unsigned)(m * p.chunks)), rows((unsigned)m), b(NT);
    sample_bins_kernel<<<all, b, 0, s>>>(a);
    sample_row_kernel<<<rows, b, 0, s>>>(a);
    sample_take_kernel<<<all, b, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FRQ_OK : set_error(FRQ_ERR_HIP, std::string("launch sample: ") + hipGetErrorString(e));
}

}  // extern "C"
