// A paged cache of keys and values, and what is done with it: writing new tokens, attention of one new token per sequence, choosing
// the tokens that stay when it has to shrink, and moving them to the front.
//
// Layout: k, v [pages_total][kv_heads][page][hd]; table [batch][pages] names the pages of a sequence in order; token t of sequence b
// and head h lives at row t % page of (table[b][t / page], h).  Page ids outside the pool are never dereferenced: their tokens count as
// masked, writes to them are dropped.  Lengths are clamped to 0 .. pages * page.  All row offsets are 64-bit.
#include "seq16.h"

#include "interactron_hip.h"

namespace {

constexpr int kBlock = 256;
constexpr int64_t kMostGroups = 1 << 24;   // workgroups along x: a launch counts its threads in 32 bits

struct Cache {   // (the launch argument form of ix_paged_cache)
    unsigned char *k, *v;
    const int* table;
    int* lens;
    float* weight;
    int64_t pages_total;
    int kv, shift, hd, batch, pages;
    __device__ __forceinline__ int cap() const { return pages << shift; }
    __device__ __forceinline__ int len(int b) const { return min(max(lens[b], 0), cap()); }
    // first row of the page that holds token t (its row in the page is t & (page - 1)), or -1
    __device__ __forceinline__ int64_t page_row(int b, int h, int t) const {
        const int id = table[(int64_t)b * pages + (t >> shift)];
        return (unsigned)id < (uint64_t)pages_total ? (((int64_t)id * kv + h) << shift) : -1;
    }
};

// ====================================================================================================================================
// append: a copy, 16 bytes per thread and step.  4 x 2 060 tokens of 8 heads of 64 in bf16 (25 MB): 8.5 us, 3.0 TB/s with its launch; 32 x 1
// token: 3.1 us, a launch
// ====================================================================================================================================
struct AppendArgs {
    Cache c;
    const unsigned char *nk, *nv;     // new rows, [batch][T][kv][hd] by byte strides
    int64_t sb_k, st_k, sh_k, sb_v, st_v, sh_v;
    const int *counts, *at;           // null: T, the cache's lengths
    int T, chunks, per_block;         // 16-byte chunks of a row; items (token, head, chunk) of one workgroup
    int set_lens;                     // this launch also writes the lengths (only where no other workgroup can still read the old ones)
};

__global__ __launch_bounds__(kBlock) void append_kernel(AppendArgs p) {
    const int b = blockIdx.y, cap = p.c.cap();
    const int start = min(max((p.at ? p.at : p.c.lens)[b], 0), cap), count = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
    const int64_t items = (int64_t)count * p.c.kv * p.chunks, i1 = min(items, (int64_t)(blockIdx.x + 1) * p.per_block);
    for (int64_t i = (int64_t)blockIdx.x * p.per_block + threadIdx.x; i < i1; i += kBlock) {
        const int c = (int)(i % p.chunks), h = (int)((i / p.chunks) % p.c.kv), t = (int)(i / ((int64_t)p.chunks * p.c.kv));
        if (start + t >= cap) continue;
        const int slot = start + t;
        if (p.c.weight && c == 0) p.c.weight[((int64_t)b * p.c.kv + h) * cap + slot] = 0.f;
        const int64_t row = p.c.page_row(b, h, slot);
        if (row < 0) continue;
        const int64_t to = ((row + (slot & ((1 << p.c.shift) - 1))) * p.chunks + c) * 16;
        *reinterpret_cast<u32x4*>(p.c.k + to) = *reinterpret_cast<const u32x4*>(p.nk + b * p.sb_k + t * p.st_k + h * p.sh_k + c * 16);
        *reinterpret_cast<u32x4*>(p.c.v + to) = *reinterpret_cast<const u32x4*>(p.nv + b * p.sb_v + t * p.st_v + h * p.sh_v + c * 16);
    }
    if (p.set_lens && blockIdx.x == 0) {
        __syncthreads();   // (every thread of the only workgroup that reads this length has read it)
        if (threadIdx.x == 0) p.c.lens[b] = min(start + count, cap);
    }
}

__global__ __launch_bounds__(kBlock) void append_lens_kernel(Cache c, const int* counts, const int* at, int T) {
    const int b = blockIdx.x * kBlock + threadIdx.x;
    if (b >= c.batch) return;
    const int start = min(max((at ? at : c.lens)[b], 0), c.cap()), count = counts ? min(max(counts[b], 0), T) : T;
    c.lens[b] = min(start + count, c.cap());
}

// ====================================================================================================================================
// attention of one new token
// ====================================================================================================================================
// The keys that a query at the last of n tokens sees, as tiles of KT keys that start at multiples of KT: the tiles of the first
// `sinks` tokens, then those from the first token of the window on.  (KT <= page size, so a tile's keys lie in few pages.)
struct Tiles {
    int n, lo, first, head, t_lo, count, per;   // per: tiles of one split
    __device__ __forceinline__ Tiles(int n_, int window, int sinks, int KT, int splits, int least) {
        n = n_;
        lo = window > 0 ? max(0, n - window) : 0;
        first = min(sinks, lo);
        t_lo = lo / KT;
        head = min((first + KT - 1) / KT, t_lo);
        count = n > 0 ? head + (n + KT - 1) / KT - t_lo : 0;
        per = max(least, (count + splits - 1) / splits);
    }
    __device__ __forceinline__ int base(int t, int KT) const { return (t < head ? t : t - head + t_lo) * KT; }
    __device__ __forceinline__ bool sees(int j) const { return (j < n) & ((j >= lo) | (j < first)); }
    __device__ __forceinline__ bool whole(int j0, int KT) const { return j0 + KT <= n && (j0 >= lo || j0 + KT <= first); }
    __device__ __forceinline__ int used() const { return (count + per - 1) / per; }   // splits that have tiles
};

struct AttnArgs {
    Cache c;
    const unsigned char* q;   // [batch][heads][hd] by byte strides
    int64_t sq_b, sq_h;
    unsigned char* out;       // [batch][heads][hd], dense
    float *part_o, *part_ml, *logits;
    int heads, group, qtiles, window, sinks, splits, least, max_tiles;
    float c2;                 // scale log2(e)
    int accumulate;
};

template <int DT> constexpr int tile_keys() { return DT == 0 ? 16 : 32; }
template <int DT> constexpr float up_exponent() { return DT == 2 ? 15.f : 0.f; }

template <int N> __device__ __forceinline__ void load_words(unsigned* w, const unsigned char* p) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(p + 4 * i);
            w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
        }
    } else if constexpr (N == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        w[0] = x.x; w[1] = x.y;
    } else {
        w[0] = *reinterpret_cast<const unsigned*>(p);
    }
}

// One workgroup: the keys of one split for up to 16 query heads that share a key head.  Everything goes from HBM to registers in the
// layout in which the matrix instructions take it; only the join of the four waves passes through LDS.
//   scores  S^T[key][q] = K Q^T: lane (n, g) reads 8 elements of key n per step, 64 bytes of a key row per instruction and four lanes;
//   outputs O^T[d][q] = V^T P^T: rows of V^T may stand in any order, so lane (m, g) takes the D / 16 neighbouring d = m D / 16 + db of
//   the keys 4 g + r (and 16 + 4 g + r): a wave reads whole rows, and with 16-bit values one v_perm_b32 per register turns two rows
//   into the pairs of keys that the matrix instruction wants.  P comes out of the scores' accumulator in exactly that key order.
// P is carried as two 16-bit terms (hi + the rest), so that the sum keeps the precision of the f32 weights: the launch is bound by the
// bytes of K and V, the second matrix instruction is free.  fp16: carried 2^15 times as large, so that the type's smallest step, 2^-24, is 2^-39
// of the largest weight and not a share of what a row has besides one dominant key.
// bf16, 32 heads over 8 of 128: one sequence of 131 071 tokens (537 MB) 94 us = 5.7 TB/s, 32 of 700 to 8 192 (583 MB) 111 us = 5.3 TB/s, where
// a kernel that only reads reaches 6.2; 411 tokens of 8 heads in f32: 8.8 us, the chain length -> page -> rows -> join in a launch.
template <int DT, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void cache_attn_kernel(AttnArgs p) {
    constexpr int KT = tile_keys<DT>(), NS = KT / 16, EB = SeqT<DT>::bytes, KSTEPS = D / 32, DB = D / 16;
    constexpr int VK = KT / 4, VW = DB * EB / 4;   // keys of V per lane, registers of one of them
    __shared__ float lds_o[WAVES][16][D + 4];
    __shared__ float lds_m[WAVES][16], lds_l[WAVES][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
    const int split = blockIdx.x, b = blockIdx.z, h = blockIdx.y % p.c.kv, qt = blockIdx.y / p.c.kv;
    const int rows = min(16, p.group - 16 * qt), head0 = h * p.group + 16 * qt;   // this workgroup's query heads
    const Tiles tl(p.c.len(b), p.window, p.sinks, KT, p.splits, p.least);
    const int t0 = split * tl.per, t1 = min(tl.count, t0 + tl.per);
    if (t0 >= t1 && p.splits > 1) return;   // (the join counts the splits that have tiles)

    Frag<DT> qf[KSTEPS];
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
#pragma unroll
        for (int w = 0; w < SeqT<DT>::words; ++w) qf[ks].w[w] = 0;
        if (n < rows) load_words<SeqT<DT>::words>(qf[ks].w, p.q + b * p.sq_b + (head0 + n) * p.sq_h + (ks * 32 + g * 8) * EB);
    }
    f32x4 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    const int page_mask = (1 << p.c.shift) - 1;
    Frag<DT> kf[NS][KSTEPS];
    unsigned vf[VK][VW];
    // a tile's page rows are looked up while the tile in front of it is requested, its keys and values while that one is worked on
    int64_t row[NS];
    unsigned bad = 0, bad_now = 0;   // bit s: sub-tile s lies in no page of the pool
    auto find = [&](int t) {
        const int j0 = tl.base(t, KT);
        bad = 0;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int j = j0 + 16 * s;
            const int64_t r = j < p.c.cap() ? p.c.page_row(b, h, j) : -1;
            if (r < 0) bad |= 1u << s;
            row[s] = r < 0 ? 0 : r + (j & page_mask);   // (row 0 is in the pool: its values are masked)
        }
    };
    auto load = [&](int t) {
        int64_t at[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) at[s] = row[s];
        bad_now = bad;
        if (t + WAVES < t1) find(t + WAVES);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const unsigned char* kr = p.c.k + (at[s] + n) * (D * EB) + g * (8 * EB);
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) load_words<SeqT<DT>::words>(kf[s][ks].w, kr + ks * (32 * EB));
        }
#pragma unroll
        for (int i = 0; i < VK; ++i) load_words<VW>(vf[i], p.c.v + (at[i / 4] + 4 * g + i % 4) * (D * EB) + n * (DB * EB));
    };
    int t = t0 + wave;
    if (t < t1) {
        find(t);
        load(t);
    }
    for (; t < t1; t += WAVES) {
        const int j0 = tl.base(t, KT);
        f32x4 x[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            x[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) x[s] = seq_mma<DT>(kf[s][ks], qf[ks], x[s]);
            x[s] *= p.c2;
        }
        unsigned vc[VK][VW];
#pragma unroll
        for (int i = 0; i < VK; ++i)
#pragma unroll
            for (int w = 0; w < VW; ++w) vc[i][w] = vf[i][w];
        if (bad_now || !tl.whole(j0, KT)) {   // masked keys: no score, and zeros for values (what lies there may be anything)
#pragma unroll
            for (int i = 0; i < VK; ++i) {
                const int s = i / 4, j = j0 + 16 * s + 4 * g + i % 4;
                // (selects, no branch: ROCm 7.2's compiler lost the first element's store of a short-circuit form of this)
                const bool see = tl.sees(j) & !(bad_now >> s & 1);
                x[s][i % 4] = see ? x[s][i % 4] : -INFINITY;
#pragma unroll
                for (int w = 0; w < VW; ++w) vc[i][w] = see ? vc[i][w] : 0;
            }
        }
        if (t + WAVES < t1) load(t + WAVES);
        if (p.accumulate && n < rows) {
            float* dst = p.logits + (((int64_t)b * p.heads + head0 + n) * p.max_tiles + t) * KT + 4 * g;
#pragma unroll
            for (int s = 0; s < NS; ++s) *reinterpret_cast<f32x4*>(dst + 16 * s) = x[s];
        }
        float top = -INFINITY;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, x[s][r]);
        const float mn = fmaxf(m, seq_max_g(top)), ref = mn == -INFINITY ? 0.f : mn, alpha = seq_exp2(m - ref);
        float sum = 0.f;
        float pr[VK];
        const float low = ref - up_exponent<DT>();
#pragma unroll
        for (int i = 0; i < VK; ++i) {
            pr[i] = seq_exp2(x[i / 4][i % 4] - low);
            sum += pr[i];
        }
        m = mn;
        l = l * alpha + sum;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= alpha;
        if constexpr (DT == 0) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[db] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vc[r][db]), pr[r], o[db], 0, 0, 0);
        } else {
            Frag<DT> hi, lo;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                hi.w[w] = seq_pack<DT>(pr[2 * w], pr[2 * w + 1]);
                lo.w[w] = seq_pack<DT>(pr[2 * w] - seq_lo<DT>(hi.w[w]), pr[2 * w + 1] - seq_hi<DT>(hi.w[w]));
            }
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                Frag<DT> a;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    a.w[w] = __builtin_amdgcn_perm(vc[2 * w + 1][db / 2], vc[2 * w][db / 2], db & 1 ? 0x07060302u : 0x05040100u);
                o[db] = seq_mma<DT>(a, lo, o[db]);
                o[db] = seq_mma<DT>(a, hi, o[db]);
            }
        }
    }
    l = seq_sum_g(l);
    if (g == 0) { lds_m[wave][n] = m; lds_l[wave][n] = l; }
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) lds_o[wave][n][(4 * g + r) * DB + db] = o[db][r];
    __syncthreads();
    for (int i = tid; i < rows * D; i += 64 * WAVES) {
        const int q = i / D, d = i % D;
        float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, lds_m[w][q]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = seq_exp2(lds_m[w][q] - ref);
            sum += f * lds_l[w][q];
            acc += f * lds_o[w][q][d];
        }
        const int64_t at = (int64_t)b * p.heads + head0 + q;
        if (DT == 2) {
            acc *= 1.f / 32768.f;
            sum *= 1.f / 32768.f;
        }
        if (p.part_ml) {
            p.part_o[(at * p.splits + split) * D + d] = acc;
            if (d == 0) { p.part_ml[(at * p.splits + split) * 2] = top; p.part_ml[(at * p.splits + split) * 2 + 1] = sum; }
        } else {
            seq_store1<DT>(p.out, at * D + d, sum == 0.f ? 0.f : acc / sum);
        }
    }
}

// Joins the splits of one query head; with `accumulate` further workgroups add the weights P_j of 1024 tile slots each, summed over the
// query heads of the key head in their order, to the cache's accumulated weights.  Bound by a launch and the chain maxima -> factors -> rows:
// 5 us for 256 heads in 17 splits or 32 heads in 64, 6 us for 1 024 heads in 8.
constexpr int kJoinSplits = 1024;   // split factors that are in LDS at a time

template <int DT>
__global__ __launch_bounds__(kBlock) void cache_join_kernel(AttnArgs p, int D, int out_blocks, int weight_blocks) {
    constexpr int KT = tile_keys<DT>(), WAVES = kBlock / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ float red[kBlock], stat[2 * 64], factor[kJoinSplits];
    // (maximum, 1 / sum) of query head `at` over its splits, by one wave
    auto stats = [&](int64_t at, int used) {
        const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + at * p.splits;
        float top = -INFINITY, sum = 0.f;
        for (int s = lane; s < used; s += 64) {   // (rescaled as it goes: one pass)
            const float2 x = ml[s];
            const float up = fmaxf(top, x.x), ref = up == -INFINITY ? 0.f : up;
            sum = sum * seq_exp2(top - ref) + x.y * seq_exp2(x.x - ref);
            top = up;
        }
        const float all = ix_wave_max(top), ref = all == -INFINITY ? 0.f : all;
        sum = ix_wave_sum(sum * seq_exp2(top - ref));
        return float2{ref, sum == 0.f ? 0.f : 1.f / sum};
    };
    if ((int)blockIdx.x < out_blocks) {
        const int64_t at = blockIdx.x;
        const int b = (int)(at / p.heads);
        const Tiles tl(p.c.len(b), p.window, p.sinks, KT, p.splits, p.least);
        const int used = tl.used();
        const float2 st = stats(at, used);   // (every wave for itself)
        const int d = tid % D, part = tid / D, parts = kBlock / D;
        float acc = 0.f;
        for (int s0 = 0; s0 < used; s0 += kJoinSplits) {
            const int here = min(kJoinSplits, used - s0);
            __syncthreads();
            for (int s = tid; s < here; s += kBlock) factor[s] = seq_exp2(p.part_ml[(at * p.splits + s0 + s) * 2] - st.x) * st.y;
            __syncthreads();
            const float* src = p.part_o + (at * p.splits + s0) * D + d;
            int s = part;
            for (; s + 7 * parts < here; s += 8 * parts) {   // eight loads in flight
                float x[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) x[u] = src[(int64_t)(s + u * parts) * D];
#pragma unroll
                for (int u = 0; u < 8; ++u) acc += x[u] * factor[s + u * parts];
            }
            for (; s < here; s += parts) acc += src[(int64_t)s * D] * factor[s];
        }
        red[tid] = acc;
        __syncthreads();
        if (part == 0) {
            for (int k = 1; k < parts; ++k) acc += red[k * D + d];
            seq_store1<DT>(p.out, at * D + d, acc);
        }
        return;
    }
    const int item = blockIdx.x - out_blocks, chunk = item % weight_blocks, h = (item / weight_blocks) % p.c.kv, b = item / weight_blocks / p.c.kv;
    const Tiles tl(p.c.len(b), p.window, p.sinks, KT, p.splits, p.least);
    if (chunk * 1024 >= tl.count * KT) return;
    const int used = tl.used(), i0 = chunk * 1024 + 4 * tid;   // four neighbouring slots (of one tile)
    const bool live = i0 < tl.count * KT;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int q0 = 0; q0 < p.group; q0 += 64) {
        const int qn = min(64, p.group - q0);
        __syncthreads();
        for (int q = wave; q < qn; q += WAVES) {
            const float2 st = stats((int64_t)b * p.heads + h * p.group + q0 + q, used);
            if (lane == 0) { stat[2 * q] = st.x; stat[2 * q + 1] = st.y; }
        }
        __syncthreads();
        if (live) {
            const float* src = p.logits + ((int64_t)b * p.heads + h * p.group + q0) * p.max_tiles * KT + i0;
            for (int q = 0; q < qn; ++q) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(src + (int64_t)q * p.max_tiles * KT);
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[u] += seq_exp2(x[u] - stat[2 * q]) * stat[2 * q + 1];
            }
        }
    }
    if (!live) return;
    const int j = tl.base(i0 / KT, KT) + i0 % KT;
    float* dst = p.c.weight + ((int64_t)b * p.c.kv + h) * p.c.cap() + j;
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (tl.sees(j + u)) dst[u] += acc[u];
}

// ====================================================================================================================================
// select: the tokens that stay
// ====================================================================================================================================
// One workgroup of 16 waves per (sequence, key head).  The r-th largest weight of the middle is found digit by digit (up to four passes of
// eight bits over keys whose unsigned order is the weights' order; three are enough where the weights differ in 24 bits).  Every wave has a
// stretch of tokens of its own, up to 2048 of them in registers for all passes (longer stretches are read again); at the end it counts what
// stays of it, the counts are summed in wave order, and it writes its kept indexes with ballots: ascending, and of equal weights the lowest
// indexes.
// Bound by the chain of its steps: 12 us for 4 352 weights of 128 rows (2.2 MB, 0.5 us at the rate of a copy), of which the launch and the
// first loads take 6, a pass 1, counting and writing 1 each; 17 us for 12 755 of 16 rows.
constexpr int kSelBlock = 1024, kSelWaves = 16, kSelHeld = 32, kSelCopies = 2;

__device__ __forceinline__ unsigned weight_key(float w) {
    if (w != w) return 0u;   // a NaN counts less than every number
    const unsigned u = __float_as_uint(w + 0.f);   // (-0 and 0 are equal)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// the sum over this lane and those below it: within rows of 16 lanes, then the rows' last sums into the rows above
__device__ __forceinline__ unsigned upto_lane(unsigned x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15 into rows 1 and 3, row_bcast 31 into 2 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}

__global__ __launch_bounds__(kSelBlock) void select_kernel(const float* weight, const int* lens, int* kept, int* left, int kv, int cap, int budget,
                                                           int sinks, int recent) {
    // counts by pass, in two copies of every other lane (on different banks): weights share few values of the first digit (two / four / eight
    // copies 11.9 / 12.2 / 12.8 us with 4 352 tokens of 128 rows, 16.9 / 17.0 / 17.2 us with 12 755 of 16)
    __shared__ __attribute__((aligned(16))) unsigned hist[4][kSelCopies][256 + 16];
    __shared__ int more[kSelWaves], same[kSelWaves];
    const int b = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = min(max(lens[b], 0), cap);
    const float* w = weight + ((int64_t)b * kv + h) * cap;
    int* out = kept + ((int64_t)b * kv + h) * budget;
    if (h == 0 && tid == 0) left[b] = min(n, budget);
    if (n <= budget) {
        for (int i = tid; i < budget; i += kSelBlock) out[i] = i < n ? i : -1;
        return;
    }
    const int m0 = sinks, m1 = n - recent;   // (sinks + recent <= budget < n)
    unsigned need = budget - sinks - recent;
    const int span = m1 - m0, each = ((span + kSelWaves - 1) / kSelWaves + 63) / 64 * 64, w0 = m0 + wave * each, w1 = min(m1, w0 + each);
    unsigned held[kSelHeld];
    // the keys of this wave's tokens from `from` on, 64 a register; places behind its stretch hold no token
    auto fetch = [&](int from) {
#pragma unroll
        for (int u = 0; u < kSelHeld; ++u) {
            const int i = from + 64 * u + lane;
            held[u] = i < w1 ? __float_as_uint(w[i]) : 0u;
        }
#pragma unroll
        for (int u = 0; u < kSelHeld; ++u) held[u] = weight_key(__uint_as_float(held[u]));
    };
    constexpr int kPart = 64 * kSelHeld;
    const bool once = each <= kPart;
    if (need && once) fetch(w0);
    for (int i = tid; i < sinks; i += kSelBlock) out[i] = i;
    for (int i = tid; i < recent; i += kSelBlock) out[budget - recent + i] = m1 + i;
    if (need == 0) return;
    for (int i = tid; i < 4 * kSelCopies * 272; i += kSelBlock) (&hist[0][0][0])[i] = 0;
    __syncthreads();
    unsigned prefix = 0, mask = 0;
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
        unsigned* mine = hist[pass][lane & (kSelCopies - 1)];
        for (int from = w0; from < w1; from += kPart) {
            if (!once) fetch(from);
#pragma unroll
            for (int u = 0; u < kSelHeld; ++u) {
                if (from + 64 * u >= w1) break;   // (uniform)
                if (from + 64 * u + lane < w1 && (held[u] & mask) == prefix) atomicAdd(&mine[(held[u] >> shift) & 255], 1u);
            }
        }
        __syncthreads();   // (the only one of a pass: every wave finds the digit by itself)
        // the digit at which the count from above reaches `need`: lane l holds digits 255 - 4 l down to 252 - 4 l
        unsigned c[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < kSelCopies; ++k) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(&hist[pass][k][252 - 4 * lane]);
            c[0] += x.w; c[1] += x.z; c[2] += x.y; c[3] += x.x;
        }
        const unsigned own = c[0] + c[1] + c[2] + c[3];
        const unsigned upto = upto_lane(own);
        unsigned before = upto - own, digit = 0, rest = 0, held_by = 0;
        const unsigned long long hit = __ballot(before < need && need <= upto);   // (one lane: at least `need` keys carry the prefix)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (before < need && need <= before + c[k]) { digit = 255 - 4 * lane - k; rest = need - before; held_by = c[k]; }
            before += c[k];
        }
        const int from = __ffsll((long long)hit) - 1;
        prefix |= __builtin_amdgcn_readlane(digit, from) << shift;
        need = __builtin_amdgcn_readlane(rest, from);
        mask |= 255u << shift;
        if (need == __builtin_amdgcn_readlane(held_by, from)) break;   // (all that carry the prefix stay: most often one, after three digits)
    }
    // nothing below `prefix` stays; of the weights that equal it the first `need`
    int a = 0, e = 0;
    for (int from = w0; from < w1; from += kPart) {
        if (!once) fetch(from);
#pragma unroll
        for (int u = 0; u < kSelHeld; ++u) {
            if (from + 64 * u >= w1) break;
            const bool in = from + 64 * u + lane < w1;
            a += __popcll(__ballot(in && held[u] > prefix));
            e += __popcll(__ballot(in && held[u] == prefix));
        }
    }
    if (lane == 0) { more[wave] = a; same[wave] = e; }
    __syncthreads();
    int at = sinks, eq = 0;
    for (int k = 0; k < wave; ++k) { at += more[k] + min(same[k], max(0, (int)need - eq)); eq += same[k]; }
    const unsigned long long below = (1ull << lane) - 1;
    for (int from = w0; from < w1; from += kPart) {
        if (!once) fetch(from);
#pragma unroll
        for (int u = 0; u < kSelHeld; ++u) {
            if (from + 64 * u >= w1) break;
            const int i = from + 64 * u + lane;
            const unsigned long long equal = __ballot(i < w1 && held[u] == prefix);
            const bool stay = i < w1 && (held[u] > prefix || (held[u] == prefix && eq + __popcll(equal & below) < (int)need));
            const unsigned long long all = __ballot(stay);
            if (stay) out[at + __popcll(all & below)] = i;
            at += __popcll(all);
            eq += __popcll(equal);
        }
    }
}

// ====================================================================================================================================
// compact: kept rows to the front, in place
// ====================================================================================================================================
// Row i takes what row kept[i] >= i held.  A workgroup walks one column slice of K or V (or the weights) of one (sequence, head) in
// ascending chunks of a row a thread: all rows of a chunk are in registers before the first of them is written, and no later chunk reads a row
// that an earlier one has written, because kept[] ascends and is nowhere below its own place.  So the move needs no second copy of the
// cache, and the next chunk's rows are on their way while this one is stored, its places (kept index, two page look-ups) a chunk before
// that, the kept indexes themselves another one.  HBM-bound: 16 sequences of 8 heads of 128, 4 096 of 4 200 to 4 352 tokens kept, bf16: 103-118
// us = 4.6-5.2 TB/s (a copy: 4.7); 2 060 of 12 755 of two sequences of 8 heads of 64 in f32 (34 MB): 11.5 us = 2.9 TB/s, a chain of steps.
struct CompactArgs {
    Cache c;
    const int *kept, *left;
    int budget, row_bytes, slices;   // slices of 16 LANES bytes in a row
};

__device__ __forceinline__ int64_t row_at(const Cache& c, int b, int h, int t) {
    const int64_t r = c.page_row(b, h, t);
    return r < 0 ? -1 : r + (t & ((1 << c.shift) - 1));
}

template <int LANES, int THREADS>   // threads of a row's slice, of the workgroup
__global__ __launch_bounds__(THREADS) void compact_kernel(CompactArgs p) {
    constexpr int PER = THREADS / LANES, kChunk = THREADS;   // rows of one pass; LANES passes a chunk
    __shared__ int64_t place[4][kChunk][2];
    const int b = blockIdx.z, h = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, cap = p.c.cap();
    const int n = min(max(p.left[b], 0), min(p.budget, cap));
    const int* kept = p.kept + ((int64_t)b * p.c.kv + h) * p.budget;
    auto kept_at = [&](int i) { return i < n ? kept[i] : -1; };
    if (part == 2 * p.slices) {   // the weights, and the length
        if (h == 0 && tid == 0) p.c.lens[b] = n;
        if (!p.c.weight) return;
        float* w = p.c.weight + ((int64_t)b * p.c.kv + h) * cap;
        for (int i0 = 0; i0 < n; i0 += THREADS * 8) {
            float x[8];
            bool move[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = i0 + u * THREADS + tid, from = kept_at(i);
                move[u] = from > i && from < cap;
                x[u] = move[u] ? w[from] : 0.f;
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (move[u]) w[i0 + u * THREADS + tid] = x[u];
        }
        return;
    }
    unsigned char* pool = (part < p.slices ? p.c.k : p.c.v) + (int64_t)(part % p.slices) * (16 * LANES) + (tid % LANES) * 16;
    const int chunks = (n + kChunk - 1) / kChunk, r0 = tid / LANES;
    auto find = [&](int c, int from, int64_t& src, int64_t& dst) {   // where row c kChunk + tid comes from and goes to
        const int i = c * kChunk + tid;
        src = dst = -1;
        if (from > i && from < cap) {
            src = row_at(p.c, b, h, from);
            dst = row_at(p.c, b, h, i);
            if (src < 0 || dst < 0) src = dst = -1;
        }
    };
    u32x4 x[LANES], y[LANES];
    auto load = [&](int c, u32x4 (&r)[LANES]) {
#pragma unroll
        for (int u = 0; u < LANES; ++u) {
            const int64_t src = place[c & 3][u * PER + r0][0];
            r[u] = src >= 0 ? *reinterpret_cast<const u32x4*>(pool + src * p.row_bytes) : u32x4{0, 0, 0, 0};
        }
    };
    int64_t src, dst;
    int next = kept_at(2 * kChunk + tid);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        find(c, kept_at(c * kChunk + tid), src, dst);
        place[c][tid][0] = src;
        place[c][tid][1] = dst;
    }
    __syncthreads();
    load(0, x);
    for (int c = 0; c < chunks; ++c) {
        find(c + 2, next, src, dst);
        next = kept_at((c + 3) * kChunk + tid);
        if (c + 1 < chunks) load(c + 1, y);
#pragma unroll
        for (int u = 0; u < LANES; ++u) asm volatile("" : "+v"(x[u]));   // this thread's rows of the chunk are in registers ...
        place[(c + 2) & 3][tid][0] = src;
        place[(c + 2) & 3][tid][1] = dst;
        __syncthreads();                                                  // ... and so are everybody's
#pragma unroll
        for (int u = 0; u < LANES; ++u) {
            const int64_t to = place[c & 3][u * PER + r0][1];
            if (to >= 0) *reinterpret_cast<u32x4*>(pool + to * p.row_bytes) = x[u];
        }
#pragma unroll
        for (int u = 0; u < LANES; ++u) x[u] = y[u];
    }
}

// ====================================================================================================================================
// host side
// ====================================================================================================================================
int cache_of(Cache& c, const ix_paged_cache* s, const char* who) {
    IX_CHECK_ARG(s && s->k && s->v && s->table && s->lens, "%s: null cache", who);
    IX_CHECK_ARG(s->dtype >= 0 && s->dtype <= 2, "%s: dtype %d is none of 0 (f32), 1 (bf16), 2 (fp16)", who, s->dtype);
    IX_CHECK_ARG(s->hd == 32 || s->hd == 64 || s->hd == 128, "%s: head dim %d is none of 32, 64, 128", who, s->hd);
    IX_CHECK_ARG(s->page >= 16 && s->page <= 1024 && (s->page & (s->page - 1)) == 0, "%s: page size %d is no power of two from 16 to 1024", who, s->page);
    IX_CHECK_ARG(s->batch > 0 && s->batch <= 65535 && s->kv_heads > 0 && s->kv_heads <= 1024 && s->pages > 0 && s->pages_total > 0,
                 "%s: bad sizes (batch %d, key heads %d, pages %d of %lld)", who, s->batch, s->kv_heads, s->pages, (long long)s->pages_total);
    IX_CHECK_ARG((int64_t)s->pages * s->page < (1ll << 30) && s->pages_total < (1ll << 31), "%s: a cache row or pool of 2^30 tokens or more", who);
    IX_CHECK_ARG(ix_al16(s->k) && ix_al16(s->v), "%s: unaligned pool", who);
    int shift = 0;
    while ((1 << shift) < s->page) ++shift;
    c = Cache{static_cast<unsigned char*>(s->k), static_cast<unsigned char*>(s->v), s->table, s->lens, s->weight, s->pages_total, s->kv_heads, shift,
              s->hd, s->batch, s->pages};
    return IX_OK;
}

// Memory of the pools, and of rows [batch][T][kv][row] by byte strides: whether they share any.
struct Span { const unsigned char *from, *to; };
Span pool_span(const ix_paged_cache* s, const void* pool) {
    const unsigned char* p = static_cast<const unsigned char*>(pool);
    return Span{p, p + s->pages_total * s->kv_heads * s->page * s->hd * (s->dtype == 0 ? 4 : 2)};
}
Span row_span(const ix_paged_cache* s, const void* rows, int64_t T, int64_t sb, int64_t st, int64_t sh) {
    Span r{static_cast<const unsigned char*>(rows), static_cast<const unsigned char*>(rows) + s->hd * (s->dtype == 0 ? 4 : 2)};
    for (int64_t far : {(s->batch - 1) * sb, (T - 1) * st, (s->kv_heads - 1) * sh}) (far < 0 ? r.from : r.to) += far;
    return r;
}
bool meet(const Span& a, const Span& b) { return a.from < b.to && b.from < a.to; }

struct Plan {   // of one attention launch
    int max_tiles, splits, least, qtiles, kt, waves;
    bool join;
    size_t o, ml, logits;   // floats
};

// Splits.  A cache of up to 32 tiles is one piece for eight waves: no join, one launch.  Longer ones are cut into about 512 workgroups of
// four waves (two are resident on a compute unit at head dim 128), or 1 024 where several sequences may differ in length; in pieces of at
// least one tile a wave and at most 2 048 (1 024) keys.  A workgroup costs some microseconds before and after its keys, a rest of the
// last round as much as a piece: 32 sequences of up to 8 192 tokens in pieces of 256 / 512 / 1 024 keys 125 / 111 / 111 us (join 8 / 7 / 6);
// one of 131 071 tokens in 512 / 1 024 / 2 048 workgroups 94 / 96 / 99 us (join 5 / 7 / 14).
Plan plan_of(const ix_paged_cache* s, int heads, int window, int sinks, int accumulate) {
    Plan r;
    r.kt = s->dtype == 0 ? 16 : 32;
    const int64_t cap = (int64_t)s->pages * s->page;
    const int64_t all = (cap + r.kt - 1) / r.kt;
    int64_t seen = all;
    if (window > 0) {
        const int64_t some = ((int64_t)sinks + r.kt - 1) / r.kt + ((int64_t)window + r.kt - 1) / r.kt + 1;
        seen = some < all ? some : all;
    }
    r.max_tiles = (int)seen;
    const int group = heads / s->kv_heads;
    r.qtiles = (group + 15) / 16;
    const int64_t rows = (int64_t)s->batch * s->kv_heads * r.qtiles;
    r.waves = seen <= 32 ? 8 : 4;
    r.least = r.waves;
    if (seen <= 32) {
        r.splits = 1;
    } else {
        const int64_t most = (s->batch > 1 ? 1024 : 2048) / r.kt;
        int64_t per = rows * seen / (s->batch > 1 ? 1024 : 512);
        if (per < r.least) per = r.least;
        if (per > most) per = rows * seen / most <= 65536 ? most : rows * seen / 65536;
        r.splits = (int)((seen + per - 1) / per);
    }
    r.join = r.splits > 1 || accumulate;
    const int64_t parts = (int64_t)s->batch * heads * r.splits;
    r.o = r.join ? (size_t)parts * s->hd : 0;
    r.ml = r.join ? ((size_t)parts * 2 + 3) / 4 * 4 : 0;
    r.logits = accumulate ? (size_t)s->batch * heads * r.max_tiles * r.kt : 0;
    return r;
}

int attn_check(const ix_paged_cache* s, int heads, int window, int sinks, const char* who) {
    IX_CHECK_ARG(heads > 0 && heads % s->kv_heads == 0 && heads <= 4096, "%s: %d query heads over %d key heads", who, heads, s->kv_heads);
    IX_CHECK_ARG(window >= 0 && sinks >= 0, "%s: negative window or sinks", who);
    return IX_OK;
}

}  // namespace

extern "C" int ix_cache_append(const struct ix_paged_cache* cache, const void* k, const void* v, int T, int64_t sb_k, int64_t st_k, int64_t sh_k,
                               int64_t sb_v, int64_t st_v, int64_t sh_v, const int* counts, const int* at, hipStream_t stream) {
    Cache c;
    if (int rc = cache_of(c, cache, "ix_cache_append")) return rc;
    const int eb = cache->dtype == 0 ? 4 : 2;
    IX_CHECK_ARG(T >= 0 && T < (1 << 30), "ix_cache_append: T=%d", T);
    IX_CHECK_ARG(T == 0 || (k && v && ix_al16(k) && ix_al16(v)), "ix_cache_append: null or unaligned rows");
    for (int64_t s : {sb_k, st_k, sh_k, sb_v, st_v, sh_v}) IX_CHECK_ARG(s * eb % 16 == 0, "ix_cache_append: rows that do not start on 16 bytes");
    for (const int* x : {counts, at})   // (the lengths themselves may be named; another part of their memory would change under the call)
        IX_CHECK_ARG(!x || x == c.lens || x + c.batch <= c.lens || c.lens + c.batch <= x, "ix_cache_append: counts or at overlap the lengths");
    const Span pool_k = pool_span(cache, cache->k), pool_v = pool_span(cache, cache->v);
    IX_CHECK_ARG(!meet(pool_k, pool_v), "ix_cache_append: keys and values share memory");
    for (const Span& x : {row_span(cache, k, T, sb_k * eb, st_k * eb, sh_k * eb), row_span(cache, v, T, sb_v * eb, st_v * eb, sh_v * eb)})
        IX_CHECK_ARG(T == 0 || !(meet(x, pool_k) || meet(x, pool_v)), "ix_cache_append: the new rows are parts of the cache's own pools");
    AppendArgs p{c, static_cast<const unsigned char*>(k), static_cast<const unsigned char*>(v), sb_k * eb, st_k * eb, sh_k * eb, sb_v * eb, st_v * eb,
                 sh_v * eb, counts, at, T, cache->hd * eb / 16, 0, 0};
    // a workgroup moves up to 1 024 16-byte chunks of K and as many of V: four of each per thread
    const int64_t items = (int64_t)T * c.kv * p.chunks;
    p.per_block = 1024;
    const bool one = items <= p.per_block;
    int64_t blocks = (items + p.per_block - 1) / p.per_block;
    if (blocks < 1) blocks = 1;
    IX_CHECK_ARG(blocks < kMostGroups, "ix_cache_append: too many rows");
    // (lengths that are read as starts must not change under the other workgroups of the sequence)
    p.set_lens = one || (at && at != c.lens && counts != c.lens);
    append_kernel<<<dim3((unsigned)blocks, c.batch), kBlock, 0, stream>>>(p);
    IX_CHECK_LAUNCH("ix_cache_append");
    if (!p.set_lens) {
        append_lens_kernel<<<ix_div_up(c.batch, kBlock), kBlock, 0, stream>>>(c, counts, at, T);
        IX_CHECK_LAUNCH("ix_cache_append (lengths)");
    }
    return IX_OK;
}

extern "C" int ix_workspace_bytes_cache_attn(const struct ix_paged_cache* cache, int heads, int window, int sinks, int accumulate, size_t* out_host) {
    Cache c;
    if (int rc = cache_of(c, cache, "ix_workspace_bytes_cache_attn")) return rc;
    if (int rc = attn_check(cache, heads, window, sinks, "ix_workspace_bytes_cache_attn")) return rc;
    IX_CHECK_ARG(out_host, "ix_workspace_bytes_cache_attn: null output");
    const Plan r = plan_of(cache, heads, window, sinks, accumulate);
    *out_host = 4 * (r.o + r.ml + r.logits);
    return IX_OK;
}

extern "C" int ix_cache_attn(const struct ix_paged_cache* cache, const void* q, int64_t sq_b, int64_t sq_h, void* out, int heads, float scale, int window,
                             int sinks, int accumulate, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    AttnArgs p;
    if (int rc = cache_of(p.c, cache, "ix_cache_attn")) return rc;
    if (int rc = attn_check(cache, heads, window, sinks, "ix_cache_attn")) return rc;
    const int eb = cache->dtype == 0 ? 4 : 2, hd = cache->hd;
    IX_CHECK_ARG(q && out && ix_al16(q) && ix_al16(out) && sq_b * eb % 16 == 0 && sq_h * eb % 16 == 0, "ix_cache_attn: null or unaligned query or output");
    IX_CHECK_ARG(!accumulate || cache->weight, "ix_cache_attn: accumulate without weights in the cache");
    IX_CHECK_ARG(seq_scale_ok(scale), "ix_cache_attn: the scale is no number, or too large");
    const Plan r = plan_of(cache, heads, window, sinks, accumulate);
    const size_t need = 4 * (r.o + r.ml + r.logits);
    if (need && (!workspace || workspace_bytes < need)) {
        ix_set_error("ix_cache_attn: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
        return IX_ERR_WORKSPACE;
    }
    IX_CHECK_ARG(ix_al16(workspace), "ix_cache_attn: unaligned workspace");
    p.q = static_cast<const unsigned char*>(q);
    p.sq_b = sq_b * eb;
    p.sq_h = sq_h * eb;
    p.out = static_cast<unsigned char*>(out);
    float* ws = static_cast<float*>(workspace);
    p.part_o = r.join ? ws : nullptr;
    p.part_ml = r.join ? ws + r.o : nullptr;
    p.logits = accumulate ? ws + r.o + r.ml : nullptr;
    p.heads = heads;
    p.group = heads / cache->kv_heads;
    p.qtiles = r.qtiles;
    p.window = window;
    p.sinks = sinks;
    p.splits = r.splits;
    p.least = r.least;
    p.max_tiles = r.max_tiles;
    p.c2 = scale * SEQ_LOG2E;
    p.accumulate = accumulate != 0;
    const int64_t wblocks = accumulate ? ((int64_t)r.max_tiles * r.kt + 1023) / 1024 : 0, oblocks = (int64_t)cache->batch * heads;
    const int64_t jblocks = oblocks + wblocks * cache->batch * cache->kv_heads;
    IX_CHECK_ARG((int64_t)cache->kv_heads * r.qtiles <= 65535 && jblocks < kMostGroups, "ix_cache_attn: too many heads or tokens for one launch");
    const dim3 grid(r.splits, cache->kv_heads * r.qtiles, cache->batch);
#define CACHE_GO(DT, D)                                                                       \
    { if (r.waves == 8) cache_attn_kernel<DT, D, 8><<<grid, 512, 0, stream>>>(p);             \
      else cache_attn_kernel<DT, D, 4><<<grid, 256, 0, stream>>>(p); }
#define CACHE_HD(DT) { if (hd == 32) CACHE_GO(DT, 32) else if (hd == 64) CACHE_GO(DT, 64) else CACHE_GO(DT, 128) }
    if (cache->dtype == 0) CACHE_HD(0) else if (cache->dtype == 1) CACHE_HD(1) else CACHE_HD(2)
    IX_CHECK_LAUNCH("ix_cache_attn");
    if (r.join) {
        if (cache->dtype == 0) cache_join_kernel<0><<<(unsigned)jblocks, kBlock, 0, stream>>>(p, hd, (int)oblocks, (int)wblocks);
        else if (cache->dtype == 1) cache_join_kernel<1><<<(unsigned)jblocks, kBlock, 0, stream>>>(p, hd, (int)oblocks, (int)wblocks);
        else cache_join_kernel<2><<<(unsigned)jblocks, kBlock, 0, stream>>>(p, hd, (int)oblocks, (int)wblocks);
        IX_CHECK_LAUNCH("ix_cache_attn (join)");
    }
    return IX_OK;
}

extern "C" int ix_cache_select(const float* weight, const int* lens, int* kept, int* left, int batch, int kv_heads, int capacity, int budget, int sinks,
                               int recent, hipStream_t stream) {
    IX_CHECK_ARG(weight && lens && kept && left, "ix_cache_select: null pointer");
    IX_CHECK_ARG(batch > 0 && batch <= 65535 && kv_heads > 0 && kv_heads < (1 << 20) && capacity > 0 && capacity < (1 << 30), "ix_cache_select: bad sizes");
    IX_CHECK_ARG(budget > 0 && sinks >= 0 && recent >= 0 && (int64_t)sinks + recent <= budget, "ix_cache_select: %d first and %d last tokens do not fit into %d",
                 sinks, recent, budget);
    IX_CHECK_ARG(budget <= capacity, "ix_cache_select: a budget of %d for a capacity of %d", budget, capacity);
    IX_CHECK_ARG(left + batch <= lens || lens + batch <= left, "ix_cache_select: the lengths are still read while the new ones are written");
    select_kernel<<<dim3(kv_heads, batch), kSelBlock, 0, stream>>>(weight, lens, kept, left, kv_heads, capacity, budget, sinks, recent);
    IX_CHECK_LAUNCH("ix_cache_select");
    return IX_OK;
}

extern "C" int ix_cache_compact(const struct ix_paged_cache* cache, const int* kept, const int* left, int budget, hipStream_t stream) {
    CompactArgs p;
    if (int rc = cache_of(p.c, cache, "ix_cache_compact")) return rc;
    IX_CHECK_ARG(kept && left && budget > 0, "ix_cache_compact: null pointer or empty budget");
    IX_CHECK_ARG(left + cache->batch <= cache->lens || cache->lens + cache->batch <= left, "ix_cache_compact: the new lengths overlap the cache's own");
    IX_CHECK_ARG(!meet(pool_span(cache, cache->k), pool_span(cache, cache->v)), "ix_cache_compact: keys and values share memory: rows would move twice");
    p.kept = kept;
    p.left = left;
    p.budget = budget;
    p.row_bytes = cache->hd * (cache->dtype == 0 ? 4 : 2);
    // slices of 128 bytes (a cache line); of 64 where a row has no more, or where that leaves compute units without a workgroup (then with
    // four times the rows a step: what is left is a chain of steps)
    const bool narrow = p.row_bytes < 128 || (int64_t)cache->batch * cache->kv_heads * 2 * (p.row_bytes / 128) < 256;
    p.slices = p.row_bytes / (narrow ? 64 : 128);
    const dim3 grid(2 * p.slices + 1, cache->kv_heads, cache->batch);
    if (narrow) compact_kernel<4, 1024><<<grid, 1024, 0, stream>>>(p);
    else compact_kernel<8, 256><<<grid, 256, 0, stream>>>(p);
    IX_CHECK_LAUNCH("ix_cache_compact");
    return IX_OK;
}
