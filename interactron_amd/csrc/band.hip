// Band attention: query i of a sequence of m queries and n keys stands at p = i + n - m and sees the keys j < n of its band
// p - left <= j <= p + right and the first `sinks` ones (with `causal` only up to p):
//     z_ij = scale q_i k_j     P = softmax over the visible j     o_i = sum_j P_ij v_j
//     dv_j = sum_i P_ij do_i   delta_i = do_i o_i   dz_ij = P_ij (do_i v_j - delta_i)   dq_i = scale sum_j dz_ij k_j   dk_j = scale sum_i dz_ij q_i
// q, do, out, dq [B][Lq][H][D], k, v, dk, dv [B][Lk][kv][D]; query head h reads key head h / (H / kv), so dk, dv sum over the group.
// Rows behind a sequence's lengths are not read (they may hold anything) and come back as zeros; a query that sees nothing gives zeros.
//
// Three products' loops, all of one shape: a workgroup of four waves OWNS rows (queries: forward and dq; keys: dk / dv) that live in registers as
// the matrix instructions' B operands, and STREAMS tiles of the other side through LDS.  A tile of products comes out of the matrix
// instructions with owner rows in the lanes' columns and streamed rows in the registers: softmax statistics and the row constants of the
// gradients are per lane, and the accumulator of one product is, rounded, the B operand of the next (contracting over streamed rows) --
// no [L, S] value passes through LDS.  The streamed operand is staged once, as rows: products over the head dim read 16 bytes of a row,
// products over rows read the same image transposed (ds_read_b64_tr_b16; with f32 one value a lane).
#include "seq16.h"

#include "interactron_hip.h"

namespace {

constexpr int kBlock = 256, kWaves = 4;
constexpr int kFar = 1 << 30;   // an unlimited band (lengths stay below 2^28)

// owner rows of a wave: two blocks of 16 with 16-bit operands, one with f32 (twice the registers an element)
constexpr int owner_blocks(int dt) { return dt == 0 ? 1 : 2; }
constexpr int owner_rows(int dt) { return 16 * owner_blocks(dt) * kWaves; }
constexpr int key_tile(int dt) { return dt == 0 ? 32 : 64; }
constexpr int query_tile(int dt, int hd) { return dt == 0 || hd == 128 ? 32 : 64; }

// ---- the LDS image of a tile of rows ------------------------------------------------------------------------------------------------
// 32-byte pairs of a row change places by the row's number, so that eight neighbouring rows' pieces lie in different banks for both ways
// of reading.  f32: also the four rows 4 apart that a transposed read takes at once.
template <int DT, int D> struct Img {
    static constexpr int EB = SeqT<DT>::bytes, ROW = D * EB, PAIRS = ROW / 32, SWEEP = ROW >= 256 ? 1 : 256 / ROW, KS = D / 32, DB = D / 16;
    __device__ static __forceinline__ int turn(int row) {
        if constexpr (DT == 0) return (((row >> 2) & 3) << 1 | (row & 1)) & (PAIRS - 1);
        else return (row / SWEEP) & (PAIRS - 1);
    }
    __device__ static __forceinline__ int chunk(int row, int c) { return row * ROW + (((c >> 1) ^ turn(row)) << 5) + ((c & 1) << 4); }
    // eight elements d = 32 ks + 8 g .. of `row` (row = a multiple of 16, plus n)
    __device__ static __forceinline__ Frag<DT> row_frag(const unsigned char* img, int row, int ks, int g) {
        Frag<DT> f;
        if constexpr (DT == 0) {
            const unsigned char* p = img + row * ROW + (((4 * ks + g) ^ turn(row)) << 5);
            const u32x4 a = *reinterpret_cast<const u32x4*>(p), b = *reinterpret_cast<const u32x4*>(p + 16);
            f.w[0] = a.x; f.w[1] = a.y; f.w[2] = a.z; f.w[3] = a.w;
            f.w[4] = b.x; f.w[5] = b.y; f.w[6] = b.z; f.w[7] = b.w;
        } else {
            const u32x4 a = *reinterpret_cast<const u32x4*>(img + chunk(row, 4 * ks + g));
            f.w[0] = a.x; f.w[1] = a.y; f.w[2] = a.z; f.w[3] = a.w;
        }
        return f;
    }
    // column d = 16 db + n of rows row0 + 4 g + i and row0 + 16 + 4 g + i (row0 a multiple of 32)
    __device__ static __forceinline__ Frag<DT> col_frag(const unsigned char* img, int row0, int db, int n, int g) {
        Frag<DT> f;
        if constexpr (DT == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = row0 + 16 * (i / 4) + 4 * g + i % 4;
                f.w[i] = *reinterpret_cast<const unsigned*>(img + row * ROW + (((2 * db + (n >> 3)) ^ turn(row)) << 5) + ((n & 7) << 2));
            }
        } else {
            const int row = row0 + 4 * g + (n >> 2);
            const unsigned char* p = img + row * ROW + ((db ^ turn(row)) << 5) + ((n & 3) << 3);
            typedef s16x4 __attribute__((address_space(3))) lds4;
            const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p)));
            const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 16 * ROW)));
            f.w[0] = a.x; f.w[1] = a.y; f.w[2] = b.x; f.w[3] = b.y;
        }
        return f;
    }
};
static_assert(Img<1, 128>::PAIRS == 8 && Img<1, 32>::SWEEP == 4, "image geometry");

// a tile of ROWS rows on its way from memory to LDS: requested before the arithmetic of the tile in front of it, stored after it
template <int DT, int D, int ROWS> struct Stage {
    static constexpr int CH = Img<DT, D>::ROW / 16, N = ROWS * CH / kBlock;
    static_assert(ROWS * CH % kBlock == 0, "a tile is whole passes of the workgroup");
    u32x4 r[N];
    __device__ __forceinline__ void load(const unsigned char* base, int64_t stride, int row0, int rows) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int c = threadIdx.x + u * kBlock, row = row0 + c / CH;
            r[u] = row < rows ? *reinterpret_cast<const u32x4*>(base + row * stride + (c % CH) * 16) : u32x4{0, 0, 0, 0};
        }
    }
    __device__ __forceinline__ void store(unsigned char* img) const {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int c = threadIdx.x + u * kBlock;
            *reinterpret_cast<u32x4*>(img + Img<DT, D>::chunk(c / CH, c % CH)) = r[u];
        }
    }
};

struct BandArgs {
    const unsigned char *q, *k, *v, *go, *o, *o_rest;
    int64_t qb, ql, qh, kb, kl, kh, vb, vl, vh, gb, gl, gh;   // bytes
    unsigned char *out, *rest, *dq, *dk, *dv;                 // dense; rest: what rounding the output to 16 bits took away, in 16 bits
    float *lse, *delta, *part;                                // [B][H][Lp] base-2 normalisers (+inf: nothing visible) and delta; partial sums
    const int *q_lens, *kv_lens;
    int B, Lq, Lk, Lp, H, kv, left, right, sinks, causal;
    int wide_blocks, wide_splits, splits, key_groups;         // dk / dv: see the host side; workgroups of theirs
    float c2, scale;                                          // |scale| log2(e), scale
    unsigned flip;                                            // sign bits of a fragment's register where scale < 0
    __device__ __forceinline__ int m(int b) const { return q_lens ? min(max(q_lens[b], 0), Lq) : Lq; }
    __device__ __forceinline__ int n(int b) const { return kv_lens ? min(max(kv_lens[b], 0), Lk) : Lk; }
    __device__ __forceinline__ bool sees(int p_, int j, int n_) const {
        return (j < n_) & (((j >= p_ - left) & (j <= p_ + right)) | ((j < sinks) & (!causal | (j <= p_))));
    }
    // every pair of p0 .. p1 and j0 .. j1 sees each other (apart from j < n)
    __device__ __forceinline__ bool all_see(int p0, int p1, int j0, int j1) const {
        return (j0 >= p1 - left && j1 <= p0 + right) || (j1 < sinks && (!causal || j1 <= p0));
    }
    __device__ __forceinline__ bool none_sees(int p0, int p1, int j0, int j1) const {
        return (j1 < p0 - left || j0 > p1 + right) && (j0 >= sinks || (causal && j0 > p1));
    }
};

// (batch, head) of workgroup x of `total`: neighbouring heads -- which share keys -- on one XCD (workgroups go round the eight of them)
__device__ __forceinline__ int spread_heads(int x, int total) { return total % 8 == 0 ? (x % 8) * (total / 8) + x / 8 : x; }

// the key tiles that queries at p0 .. p1 see: the first keys' tiles, then the band's
struct KeyTiles {
    int head, first, count;
    __device__ __forceinline__ KeyTiles(const BandArgs& a, int p0, int p1, int n, int TB) {
        const int lo = max(0, p0 - a.left), hi = min(n - 1, p1 + a.right);
        const int sk = max(0, a.causal ? min(min(a.sinks, n), p1 + 1) : min(a.sinks, n));
        const bool band = lo <= hi;
        first = band ? lo / TB : 0;
        head = (sk + TB - 1) / TB;
        const int last = band ? hi / TB + 1 : 0;
        if (first <= head) count = head = max(head, last);   // one run of tiles
        else count = head + last - first;
    }
    __device__ __forceinline__ int tile(int t) const { return t < head ? t : t - head + first; }
};

template <int DT, int D, int NB>
__device__ __forceinline__ void owner_frags(Frag<DT> (&f)[NB][D / 32], const unsigned char* base, int64_t stride, int row0, int rows, int n, int g, unsigned flip) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int row = row0 + 16 * nb + n;
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
            const unsigned char* p = base + row * stride + (32 * ks + 8 * g) * SeqT<DT>::bytes;
#pragma unroll
            for (int w = 0; w < SeqT<DT>::words; w += 4) {
                const u32x4 x = row < rows ? *reinterpret_cast<const u32x4*>(p + 4 * w) : u32x4{0, 0, 0, 0};
                f[nb][ks].w[w] = x.x ^ flip; f[nb][ks].w[w + 1] = x.y ^ flip; f[nb][ks].w[w + 2] = x.z ^ flip; f[nb][ks].w[w + 3] = x.w ^ flip;
            }
        }
    }
}

// accumulators of two neighbouring 16-row blocks (this lane: rows 4 g + r of each) -> B operand over those 32 rows
template <int DT> __device__ __forceinline__ Frag<DT> as_frag(const f32x4& a, const f32x4& b) {
    Frag<DT> f;
    if constexpr (DT == 0) {
#pragma unroll
        for (int r = 0; r < 4; ++r) { f.w[r] = __float_as_uint(a[r]); f.w[4 + r] = __float_as_uint(b[r]); }
    } else {
        f.w[0] = seq_pack<DT>(a[0], a[1]); f.w[1] = seq_pack<DT>(a[2], a[3]);
        f.w[2] = seq_pack<DT>(b[0], b[1]); f.w[3] = seq_pack<DT>(b[2], b[3]);
    }
    return f;
}

// four neighbouring values of a row
template <int DT> __device__ __forceinline__ void store4(unsigned char* p, const f32x4& x) {
    if constexpr (DT == 0) *reinterpret_cast<f32x4*>(p) = x;
    else *reinterpret_cast<u32x2*>(p) = u32x2{seq_pack<DT>(x[0], x[1]), seq_pack<DT>(x[2], x[3])};
}

// fp16: gradients of scores may lie anywhere in the f32 range.  They are rounded as dz F, F a power of two of the accumulator's column
// that only falls: where a value would reach 2^15 it is lowered until the value lies in [2^14, 2^15) and the sum so far is rescaled.
template <int DB> __device__ __forceinline__ void fit16(float top, float& F, f32x4 (&acc)[DB]) {
    if (__builtin_amdgcn_ballot_w64(top * F >= 32768.f)) {
        top = seq_max_g(top);   // (the four lanes of a column agree)
        if (top * F >= 32768.f && top < INFINITY) {
            const unsigned e = __float_as_uint(top) >> 23;
            const float f = __uint_as_float((268u - e) << 23);   // top 2^(141 - e) lies in [2^14, 2^15)
            const float down = f / F;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] *= down;
            F = f;
        }
    }
}
constexpr float kFirstF = 1099511627776.f;   // 2^40

// ====================================================================================================================================
// forward
// ====================================================================================================================================
// The running maximum is raised only where a tile exceeds it by more than 2^8 (a weight may then reach 256, exact in all types' ranges):
// most tiles leave the accumulators alone.  16-bit types: a weight is rounded once to the type for the second product (half a step, like
// the result itself: against 64 bits the two add up to sqrt(2) times the result's own rounding); the sum takes the unrounded weights.
constexpr float kSlack = 8.f;

template <int DT, int D, int NB, int TB>
__global__ __launch_bounds__(kBlock, 2) void band_fwd_kernel(BandArgs a) {
    typedef Img<DT, D> I;
    constexpr int ROWS = 16 * NB * kWaves, SB = TB / 16, BYTES = TB * I::ROW;
    __shared__ __attribute__((aligned(256))) unsigned char lds[2][2][BYTES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g = lane >> 4;
    const int bh = spread_heads(blockIdx.x, a.B * a.H), b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.kv);
    const int blk = a.causal ? gridDim.y - 1 - blockIdx.y : blockIdx.y, i0 = blk * ROWS;   // (causal: the longest rows first)
    const int m = a.m(b), n = a.n(b), shift = n - m;
    const int iw = i0 + wave * 16 * NB;   // this wave's queries
    f32x4 o[NB][I::DB];
    float top[NB], sum[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        top[nb] = -INFINITY;
        sum[nb] = 0.f;
#pragma unroll
        for (int db = 0; db < I::DB; ++db) o[nb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (i0 < m) {
        const KeyTiles kt(a, i0 + shift, min(i0 + ROWS, m) - 1 + shift, n, TB);
        Frag<DT> qf[NB][I::KS];
        owner_frags<DT, D, NB>(qf, a.q + b * a.qb + h * a.qh, a.ql, iw, m, n16, g, a.flip);
        const unsigned char *kp = a.k + b * a.kb + hk * a.kh, *vp = a.v + b * a.vb + hk * a.vh;
        const int pw0 = iw + shift, pw1 = min(iw + 16 * NB, m) - 1 + shift;
        Stage<DT, D, TB> sk, sv;
        if (kt.count) {
            sk.load(kp, a.kl, kt.tile(0) * TB, n);
            sv.load(vp, a.vl, kt.tile(0) * TB, n);
            sk.store(lds[0][0]);
            sv.store(lds[0][1]);
        }
        __syncthreads();
        for (int t = 0; t < kt.count; ++t) {
            const unsigned char *ki = lds[t & 1][0], *vi = lds[t & 1][1];
            const int j0 = kt.tile(t) * TB;
            const bool more = t + 1 < kt.count;
            if (more) {
                sk.load(kp, a.kl, kt.tile(t + 1) * TB, n);
                sv.load(vp, a.vl, kt.tile(t + 1) * TB, n);
            }
            if (iw < m && !a.none_sees(pw0, pw1, j0, j0 + TB - 1)) {
                f32x4 s[NB][SB];
#pragma unroll
                for (int sb = 0; sb < SB; ++sb) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) s[nb][sb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < I::KS; ++ks) {
                        const Frag<DT> kf = I::row_frag(ki, 16 * sb + n16, ks, g);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) s[nb][sb] = seq_mma<DT>(kf, qf[nb][ks], s[nb][sb]);
                    }
                }
                if (j0 + TB > n || !a.all_see(pw0, pw1, j0, j0 + TB - 1)) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int sb = 0; sb < SB; ++sb)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const bool see = a.sees(iw + 16 * nb + n16 + shift, j0 + 16 * sb + 4 * g + r, n);
                                s[nb][sb][r] = see ? s[nb][sb][r] : -INFINITY;
                            }
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int sb = 0; sb < SB; ++sb)
#pragma unroll
                        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[nb][sb][r]);
                    mx = seq_max_g(mx) * a.c2;
                    if (__builtin_amdgcn_ballot_w64(mx > top[nb] + kSlack)) {
                        const float up = fmaxf(top[nb], mx), down = up == -INFINITY ? 1.f : seq_exp2(top[nb] - up);
                        top[nb] = up;
                        sum[nb] *= down;
#pragma unroll
                        for (int db = 0; db < I::DB; ++db) o[nb][db] *= down;
                    }
                    const float ref = top[nb] == -INFINITY ? 0.f : top[nb];
#pragma unroll
                    for (int sb = 0; sb < SB; ++sb)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            s[nb][sb][r] = seq_exp2(fmaf(s[nb][sb][r], a.c2, -ref));
                            sum[nb] += s[nb][sb][r];
                        }
                }
#pragma unroll
                for (int kk = 0; kk < SB / 2; ++kk) {
                    Frag<DT> pf[NB];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) pf[nb] = as_frag<DT>(s[nb][2 * kk], s[nb][2 * kk + 1]);
#pragma unroll
                    for (int db = 0; db < I::DB; ++db) {
                        const Frag<DT> vf = I::col_frag(vi, 32 * kk, db, n16, g);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) o[nb][db] = seq_mma<DT>(vf, pf[nb], o[nb][db]);
                    }
                }
            }
            if (more) {
                sk.store(lds[(t + 1) & 1][0]);
                sv.store(lds[(t + 1) & 1][1]);
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int i = iw + 16 * nb + n16;
        const float total = seq_sum_g(sum[nb]);
        const bool none = i >= m || total == 0.f;
        const float inv = 1.f / total;
        if (a.lse && g == 0 && i < a.Lp) a.lse[(int64_t)bh * a.Lp + i] = none ? INFINITY : top[nb] + __log2f(total);
        if (i >= a.Lq) continue;
        const int64_t at = (((int64_t)b * a.Lq + i) * a.H + h) * I::ROW;
#pragma unroll
        for (int db = 0; db < I::DB; ++db) {
            const f32x4 x = none ? f32x4{0.f, 0.f, 0.f, 0.f} : o[nb][db] * inv;
            store4<DT>(a.out + at + (16 * db + 4 * g) * I::EB, x);
            if constexpr (DT != 0) {
                if (a.rest) {
                    f32x4 y;
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const unsigned w = seq_pack<DT>(x[r], x[r + 1]);
                        y[r] = x[r] - seq_lo<DT>(w);
                        y[r + 1] = x[r + 1] - seq_hi<DT>(w);
                    }
                    store4<DT>(a.rest + at + (16 * db + 4 * g) * I::EB, y);
                }
            }
        }
    }
}

// ====================================================================================================================================
// gradients
// ====================================================================================================================================
// delta_i = do_i o_i, a row by the lanes that hold 16 bytes of it each.  16-bit: o is the stored output and the rest its rounding took, so
// that delta -- which is subtracted from every do_i v_j of the row -- is as good as from the 32-bit output.
template <int DT, int D>
__global__ __launch_bounds__(kBlock) void band_delta_kernel(BandArgs a) {
    constexpr int EB = SeqT<DT>::bytes, LANES = D * EB / 16;
    const int64_t row = ((int64_t)blockIdx.x * kBlock + threadIdx.x) / LANES;   // (batch, query, head)
    const int c = threadIdx.x % LANES, h = (int)(row % a.H);
    const int64_t bi = row / a.H;
    const int i = (int)(bi % a.Lp), b = (int)(bi / a.Lp);
    if (b >= a.B) return;   // (whole rows: the lanes of a row leave together)
    float d = 0.f;
    if (i < a.m(b)) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(a.go + b * a.gb + i * a.gl + h * a.gh + 16 * c);
        const int64_t at = (((int64_t)b * a.Lq + i) * a.H + h) * (D * EB) + 16 * c;
        const u32x4 y = *reinterpret_cast<const u32x4*>(a.o + at);
        if constexpr (DT == 0) {
#pragma unroll
            for (int w = 0; w < 4; ++w) d += __uint_as_float(x[w]) * __uint_as_float(y[w]);
        } else {
            const u32x4 z = *reinterpret_cast<const u32x4*>(a.o_rest + at);
#pragma unroll
            for (int w = 0; w < 4; ++w)
                d += seq_lo<DT>(x[w]) * (seq_lo<DT>(y[w]) + seq_lo<DT>(z[w])) + seq_hi<DT>(x[w]) * (seq_hi<DT>(y[w]) + seq_hi<DT>(z[w]));
        }
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) d += __shfl_xor(d, o, 64);
    if (c == 0) a.delta[((int64_t)b * a.H + h) * a.Lp + i] = d;
}

// dq: query-owning, streams k (both ways) and v (rows).  Tiles are taken 32 keys at a time.
template <int DT, int D, int NB, int TB>
__device__ __forceinline__ void band_dq(const BandArgs& a, unsigned char* mem, int group) {
    typedef Img<DT, D> I;
    constexpr int ROWS = 16 * NB * kWaves, BYTES = TB * I::ROW;
    auto lds = reinterpret_cast<unsigned char (*)[2][BYTES]>(mem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g = lane >> 4;
    const int bh = spread_heads(group % (a.B * a.H), a.B * a.H), b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.kv);
    const int blocks = (a.Lq + ROWS - 1) / ROWS, y = group / (a.B * a.H), i0 = (a.causal ? blocks - 1 - y : y) * ROWS;
    const int m = a.m(b), n = a.n(b), shift = n - m, iw = i0 + wave * 16 * NB;
    f32x4 acc[NB][I::DB];
    float lse[NB], delta[NB], F[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        lse[nb] = INFINITY;
        delta[nb] = 0.f;
        F[nb] = kFirstF;
#pragma unroll
        for (int db = 0; db < I::DB; ++db) acc[nb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (i0 < m) {
        const KeyTiles kt(a, i0 + shift, min(i0 + ROWS, m) - 1 + shift, n, TB);
        Frag<DT> qf[NB][I::KS], gf[NB][I::KS];
        owner_frags<DT, D, NB>(qf, a.q + b * a.qb + h * a.qh, a.ql, iw, m, n16, g, a.flip);
        owner_frags<DT, D, NB>(gf, a.go + b * a.gb + h * a.gh, a.gl, iw, m, n16, g, 0u);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int i = iw + 16 * nb + n16;
            if (i < m) {
                lse[nb] = a.lse[(int64_t)bh * a.Lp + i];
                delta[nb] = a.delta[(int64_t)bh * a.Lp + i];
            }
        }
        const unsigned char *kp = a.k + b * a.kb + hk * a.kh, *vp = a.v + b * a.vb + hk * a.vh;
        const int pw0 = iw + shift, pw1 = min(iw + 16 * NB, m) - 1 + shift;
        Stage<DT, D, TB> sk, sv;
        if (kt.count) {
            sk.load(kp, a.kl, kt.tile(0) * TB, n);
            sv.load(vp, a.vl, kt.tile(0) * TB, n);
            sk.store(lds[0][0]);
            sv.store(lds[0][1]);
        }
        __syncthreads();
        for (int t = 0; t < kt.count; ++t) {
            const unsigned char *ki = lds[t & 1][0], *vi = lds[t & 1][1];
            const int j0 = kt.tile(t) * TB;
            const bool more = t + 1 < kt.count;
            if (more) {
                sk.load(kp, a.kl, kt.tile(t + 1) * TB, n);
                sv.load(vp, a.vl, kt.tile(t + 1) * TB, n);
            }
            if (iw < m && !a.none_sees(pw0, pw1, j0, j0 + TB - 1)) {
                const bool part = j0 + TB > n || !a.all_see(pw0, pw1, j0, j0 + TB - 1);
#pragma unroll
                for (int kk = 0; kk < TB / 32; ++kk) {
                    f32x4 s[NB][2], z[NB][2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) s[nb][u] = z[nb][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int ks = 0; ks < I::KS; ++ks) {
                            const Frag<DT> kf = I::row_frag(ki, 32 * kk + 16 * u + n16, ks, g), vf = I::row_frag(vi, 32 * kk + 16 * u + n16, ks, g);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                s[nb][u] = seq_mma<DT>(kf, qf[nb][ks], s[nb][u]);
                                z[nb][u] = seq_mma<DT>(vf, gf[nb][ks], z[nb][u]);
                            }
                        }
                    }
                    Frag<DT> zf[NB];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                float p = seq_exp2(fmaf(s[nb][u][r], a.c2, -lse[nb]));
                                if (part) p = a.sees(iw + 16 * nb + n16 + shift, j0 + 32 * kk + 16 * u + 4 * g + r, n) ? p : 0.f;
                                z[nb][u][r] = p * (z[nb][u][r] - delta[nb]);
                            }
                        if constexpr (DT == 2) {
                            float mx = 0.f;
#pragma unroll
                            for (int u = 0; u < 2; ++u)
#pragma unroll
                                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, fabsf(z[nb][u][r]));
                            fit16<I::DB>(mx, F[nb], acc[nb]);
                            z[nb][0] *= F[nb];
                            z[nb][1] *= F[nb];
                        }
                        zf[nb] = as_frag<DT>(z[nb][0], z[nb][1]);
                    }
#pragma unroll
                    for (int db = 0; db < I::DB; ++db) {
                        const Frag<DT> kf = I::col_frag(ki, 32 * kk, db, n16, g);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) acc[nb][db] = seq_mma<DT>(kf, zf[nb], acc[nb][db]);
                    }
                }
            }
            if (more) {
                sk.store(lds[(t + 1) & 1][0]);
                sv.store(lds[(t + 1) & 1][1]);
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int i = iw + 16 * nb + n16;
        if (i >= a.Lq) continue;
        const float f = DT == 2 ? a.scale / F[nb] : a.scale;
        unsigned char* dst = a.dq + (((int64_t)b * a.Lq + i) * a.H + h) * I::ROW;
#pragma unroll
        for (int db = 0; db < I::DB; ++db) store4<DT>(dst + (16 * db + 4 * g) * I::EB, acc[nb][db] * f);
    }
}

// dk and dv: key-owning, streams q and do of every query head of the group (both ways, 32 queries at a time) with their lse and delta.
// A block of keys that is cut into splits leaves f32 partial sums [2][ROWS][D]; band_sum_kernel adds them in order.
struct KeyItem {
    int block, split, splits;
    __device__ __forceinline__ KeyItem(const BandArgs& a, int item) {
        const int wide = a.wide_blocks * a.wide_splits;
        if (item < wide) {
            block = item / a.wide_splits; split = item % a.wide_splits; splits = a.wide_splits;
        } else {
            block = a.wide_blocks + (item - wide) / a.splits; split = (item - wide) % a.splits; splits = a.splits;
        }
    }
};

template <int DT, int D, int NB, int TB>
__device__ __forceinline__ void band_dkv(const BandArgs& a, unsigned char* mem, int group) {
    typedef Img<DT, D> I;
    constexpr int ROWS = 16 * NB * kWaves, BYTES = TB * I::ROW;
    auto lds = reinterpret_cast<unsigned char (*)[2][BYTES]>(mem);
    auto row_c = reinterpret_cast<float (*)[2][TB]>(mem + 4 * BYTES);   // lse, delta of the tile's queries
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g = lane >> 4;
    const int bk = spread_heads(group % (a.B * a.kv), a.B * a.kv), b = bk / a.kv, hk = bk % a.kv, G = a.H / a.kv, item = group / (a.B * a.kv);
    const KeyItem it(a, item);
    const int m = a.m(b), n = a.n(b), shift = n - m, j0 = it.block * ROWS, jw = j0 + wave * 16 * NB;
    f32x4 ak[NB][I::DB], av[NB][I::DB];
    float F[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        F[nb] = kFirstF;
#pragma unroll
        for (int db = 0; db < I::DB; ++db) ak[nb][db] = av[nb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int tiles = 0, first = 0;   // query tiles of one head
    if (j0 < n && m > 0) {
        const int j1 = min(j0 + ROWS, n) - 1;
        const bool to_all = j0 < a.sinks;
        const int p0 = to_all ? (a.causal ? j0 : -kFar) : j0 - a.right, p1 = to_all ? kFar : j1 + a.left;
        const int lo = max(0, p0 - shift), hi = min(m - 1, p1 - shift);
        first = lo / TB;
        tiles = lo <= hi ? hi / TB - first + 1 : 0;
    }
    const int64_t all = (int64_t)tiles * G;
    const int u0 = (int)(all * it.split / it.splits), u1 = (int)(all * (it.split + 1) / it.splits);
    if (u0 < u1) {
        Frag<DT> kf[NB][I::KS], vf[NB][I::KS];
        owner_frags<DT, D, NB>(kf, a.k + b * a.kb + hk * a.kh, a.kl, jw, n, n16, g, a.flip);
        owner_frags<DT, D, NB>(vf, a.v + b * a.vb + hk * a.vh, a.vl, jw, n, n16, g, 0u);
        const int jw1 = min(jw + 16 * NB, n) - 1;
        Stage<DT, D, TB> sq, sg;
        float rc = 0.f;
        auto load = [&](int u) {
            const int h = hk * G + u / tiles, i0 = (first + u % tiles) * TB;
            sq.load(a.q + b * a.qb + h * a.qh, a.ql, i0, m);
            sg.load(a.go + b * a.gb + h * a.gh, a.gl, i0, m);
            if (tid < 2 * TB) rc = (tid < TB ? a.lse : a.delta)[((int64_t)b * a.H + h) * a.Lp + i0 + tid % TB];
        };
        auto store = [&](int buf) {
            sq.store(lds[buf][0]);
            sg.store(lds[buf][1]);
            if (tid < 2 * TB) row_c[buf][tid / TB][tid % TB] = rc;
        };
        load(u0);
        store(0);
        __syncthreads();
        for (int u = u0; u < u1; ++u) {
            const int buf = (u - u0) & 1;
            const unsigned char *qi = lds[buf][0], *gi = lds[buf][1];
            const int p0 = (first + u % tiles) * TB + shift, p1 = p0 + TB - 1;   // (queries behind m: do = 0 and P = 0)
            const bool more = u + 1 < u1;
            if (more) load(u + 1);
            if (jw < n && !a.none_sees(p0, p1, jw, jw1)) {
                const bool part = !a.all_see(p0, p1, jw, jw1);
#pragma unroll
                for (int kk = 0; kk < TB / 32; ++kk) {
                    f32x4 s[NB][2], z[NB][2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) s[nb][x] = z[nb][x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int ks = 0; ks < I::KS; ++ks) {
                            const Frag<DT> qf = I::row_frag(qi, 32 * kk + 16 * x + n16, ks, g), gf = I::row_frag(gi, 32 * kk + 16 * x + n16, ks, g);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                s[nb][x] = seq_mma<DT>(qf, kf[nb][ks], s[nb][x]);
                                z[nb][x] = seq_mma<DT>(gf, vf[nb][ks], z[nb][x]);
                            }
                        }
                    }
                    Frag<DT> pf[NB], zf[NB];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const f32x4 lse = *reinterpret_cast<const f32x4*>(&row_c[buf][0][32 * kk + 16 * x + 4 * g]);
                        const f32x4 del = *reinterpret_cast<const f32x4*>(&row_c[buf][1][32 * kk + 16 * x + 4 * g]);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                float p = seq_exp2(fmaf(s[nb][x][r], a.c2, -lse[r]));
                                if (part) p = a.sees(p0 + 32 * kk + 16 * x + 4 * g + r, jw + 16 * nb + n16, n) ? p : 0.f;
                                s[nb][x][r] = p;
                                z[nb][x][r] = p * (z[nb][x][r] - del[r]);
                            }
                    }
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        if constexpr (DT == 2) {
                            float mx = 0.f;
#pragma unroll
                            for (int x = 0; x < 2; ++x)
#pragma unroll
                                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, fabsf(z[nb][x][r]));
                            fit16<I::DB>(mx, F[nb], ak[nb]);
                            z[nb][0] *= F[nb];
                            z[nb][1] *= F[nb];
                            s[nb][0] *= 1024.f;   // (weights of long rows stay clear of the type's smallest steps)
                            s[nb][1] *= 1024.f;
                        }
                        pf[nb] = as_frag<DT>(s[nb][0], s[nb][1]);
                        zf[nb] = as_frag<DT>(z[nb][0], z[nb][1]);
                    }
#pragma unroll
                    for (int db = 0; db < I::DB; ++db) {
                        const Frag<DT> gf = I::col_frag(gi, 32 * kk, db, n16, g), qf = I::col_frag(qi, 32 * kk, db, n16, g);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            av[nb][db] = seq_mma<DT>(gf, pf[nb], av[nb][db]);
                            ak[nb][db] = seq_mma<DT>(qf, zf[nb], ak[nb][db]);
                        }
                    }
                }
            }
            if (more) store(buf ^ 1);
            __syncthreads();
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int row = wave * 16 * NB + 16 * nb + n16, j = j0 + row;
        const float fk = DT == 2 ? a.scale / F[nb] : a.scale, fv = DT == 2 ? 1.f / 1024.f : 1.f;
        if (j >= n) {   // (padding: columns beside the valid ones of this block)
#pragma unroll
            for (int db = 0; db < I::DB; ++db) ak[nb][db] = av[nb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (it.splits > 1) {
            float* dst = a.part + (((int64_t)bk * (a.key_groups / (a.B * a.kv)) + item) * 2 * ROWS + row) * D;
#pragma unroll
            for (int db = 0; db < I::DB; ++db) {
                *reinterpret_cast<f32x4*>(dst + 16 * db + 4 * g) = ak[nb][db] * fk;
                *reinterpret_cast<f32x4*>(dst + (int64_t)ROWS * D + 16 * db + 4 * g) = av[nb][db] * fv;
            }
        } else if (j < a.Lk) {
            const int64_t at = (((int64_t)b * a.Lk + j) * a.kv + hk) * I::ROW;
#pragma unroll
            for (int db = 0; db < I::DB; ++db) {
                store4<DT>(a.dk + at + (16 * db + 4 * g) * I::EB, ak[nb][db] * fk);
                store4<DT>(a.dv + at + (16 * db + 4 * g) * I::EB, av[nb][db] * fv);
            }
        }
    }
}

// Both in one launch, the key blocks first: either alone would leave compute units empty at the sizes where time counts, and at its end.
template <int DT, int D> constexpr int bwd_bytes() {
    constexpr int q = 4 * key_tile(DT) * Img<DT, D>::ROW, k = 4 * query_tile(DT, D) * Img<DT, D>::ROW + 16 * query_tile(DT, D);
    return q > k ? q : k;
}
template <int DT, int D, int NB>
__global__ __launch_bounds__(kBlock, D == 128 && DT != 0 ? 1 : 2) void band_bwd_kernel(BandArgs a) {
    __shared__ __attribute__((aligned(256))) unsigned char mem[bwd_bytes<DT, D>()];
    if ((int)blockIdx.x < a.key_groups) band_dkv<DT, D, NB, query_tile(DT, D)>(a, mem, blockIdx.x);
    else band_dq<DT, D, NB, key_tile(DT)>(a, mem, blockIdx.x - a.key_groups);
}

// dk, dv of the blocks that were cut into splits: the partial sums in split order, four values a thread
template <int DT, int D>
__global__ __launch_bounds__(kBlock) void band_sum_kernel(BandArgs a, int items, int rows) {
    typedef Img<DT, D> I;
    const int bk = blockIdx.x, b = bk / a.kv, hk = bk % a.kv;
    const bool wide = (int)blockIdx.y < a.wide_blocks;
    const int splits = wide ? a.wide_splits : a.splits;
    if (splits == 1) return;
    const int block = blockIdx.y, item = wide ? block * splits : a.wide_blocks * a.wide_splits + (block - a.wide_blocks) * splits;
    for (int e = (blockIdx.z * kBlock + threadIdx.x) * 4; e < 2 * rows * D; e += gridDim.z * kBlock * 4) {
        const int which = e / (rows * D), row = e / D % rows, d = e % D, j = block * rows + row;
        if (j >= a.Lk) continue;
        const float* src = a.part + ((int64_t)bk * items + item) * 2 * rows * D + e;
        f32x4 x = *reinterpret_cast<const f32x4*>(src);
        for (int s = 1; s < splits; ++s) x += *reinterpret_cast<const f32x4*>(src + (int64_t)s * 2 * rows * D);
        store4<DT>((which ? a.dv : a.dk) + (((int64_t)b * a.Lk + j) * a.kv + hk) * I::ROW + d * I::EB, x);
    }
}

// ====================================================================================================================================
// host side
// ====================================================================================================================================
struct KeyPlan { int blocks, wide, wide_splits, splits, items; };

// Splits of dk / dv.  A block of keys streams the queries of its band; a block with some of the first `sinks` keys streams all of them, and
// would run long after the others: it is cut into pieces of about the others' length.  Where all blocks together are fewer than the
// compute units (few key heads, many query heads), every block is cut until they are not.
KeyPlan key_plan(const ix_band* s) {
    KeyPlan r;
    const int rows = owner_rows(s->dtype), group = s->heads / s->kv_heads;
    r.blocks = (s->Lk + rows - 1) / rows;
    r.wide = s->sinks > 0 ? (s->sinks < s->Lk ? (s->sinks + rows - 1) / rows : r.blocks) : 0;
    const int64_t far = s->window > 0 ? s->window : (int64_t)s->Lq + s->Lk;
    const int tb = query_tile(s->dtype, s->hd);
    const int64_t all = (s->Lq + tb - 1) / tb, band = ((s->causal ? far : 2 * far) + rows + tb - 1) / tb + 1, each = (band < all ? band : all) * group;
    const int64_t wgs = (int64_t)s->batch * s->kv_heads * r.blocks;
    int64_t sp = wgs < 256 ? (256 + wgs - 1) / wgs : 1;
    if (sp > (each + 3) / 4) sp = (each + 3) / 4;   // (no piece under four tiles)
    r.splits = (int)(sp < 1 ? 1 : sp);
    const int64_t piece = (each + r.splits - 1) / r.splits;
    int64_t ws = (all * group + piece - 1) / piece;
    if (ws > 64) ws = 64;
    r.wide_splits = (int)(ws < 1 ? 1 : ws);
    r.items = r.wide * r.wide_splits + (r.blocks - r.wide) * r.splits;
    return r;
}

size_t part_bytes(const ix_band* s, const KeyPlan& r) {
    if (r.splits == 1 && (r.wide_splits == 1 || r.wide == 0)) return 0;
    return (size_t)s->batch * s->kv_heads * r.items * 2 * owner_rows(s->dtype) * s->hd * 4;
}

int64_t lse_pitch(const ix_band* s) { return ((int64_t)s->Lq + 127) / 128 * 128; }

int band_of(BandArgs& a, const ix_band* s, const char* who) {
    IX_CHECK_ARG(s, "%s: null description", who);
    IX_CHECK_ARG(s->dtype >= 0 && s->dtype <= 2, "%s: dtype %d is none of 0 (f32), 1 (bf16), 2 (fp16)", who, s->dtype);
    IX_CHECK_ARG(s->hd == 32 || s->hd == 64 || s->hd == 128, "%s: head dim %d is none of 32, 64, 128", who, s->hd);
    IX_CHECK_ARG(s->batch > 0 && s->Lq > 0 && s->Lk > 0 && s->Lq < (1 << 22) && s->Lk < (1 << 22), "%s: bad sizes (batch %d, %d queries, %d keys)", who,
                 s->batch, s->Lq, s->Lk);
    IX_CHECK_ARG(s->heads > 0 && s->kv_heads > 0 && s->heads % s->kv_heads == 0, "%s: %d query heads over %d key heads", who, s->heads, s->kv_heads);
    IX_CHECK_ARG((int64_t)s->batch * s->heads < (1 << 30), "%s: too many heads", who);
    IX_CHECK_ARG(s->window >= 0 && s->sinks >= 0, "%s: negative window or sinks", who);
    IX_CHECK_ARG(s->scale == s->scale && s->scale < INFINITY && s->scale > -INFINITY, "%s: the scale is no number", who);
    IX_CHECK_ARG(s->q && s->k && s->v && ix_al16(s->q) && ix_al16(s->k) && ix_al16(s->v), "%s: null or unaligned q, k or v", who);
    const int64_t eb = s->dtype == 0 ? 4 : 2;
    for (int64_t x : {s->q_sb, s->q_sl, s->q_sh, s->k_sb, s->k_sl, s->k_sh, s->v_sb, s->v_sl, s->v_sh})
        IX_CHECK_ARG(x * eb % 16 == 0, "%s: rows that do not start on 16 bytes", who);
    a = BandArgs{};
    a.q = static_cast<const unsigned char*>(s->q);
    a.k = static_cast<const unsigned char*>(s->k);
    a.v = static_cast<const unsigned char*>(s->v);
    a.qb = s->q_sb * eb; a.ql = s->q_sl * eb; a.qh = s->q_sh * eb;
    a.kb = s->k_sb * eb; a.kl = s->k_sl * eb; a.kh = s->k_sh * eb;
    a.vb = s->v_sb * eb; a.vl = s->v_sl * eb; a.vh = s->v_sh * eb;
    a.q_lens = s->q_lens;
    a.kv_lens = s->kv_lens;
    a.B = s->batch; a.Lq = s->Lq; a.Lk = s->Lk; a.Lp = (int)lse_pitch(s); a.H = s->heads; a.kv = s->kv_heads;
    a.left = s->window > 0 ? s->window - 1 : kFar;
    if (a.left > kFar) a.left = kFar;
    a.right = s->causal ? 0 : a.left;
    a.sinks = s->sinks;
    a.causal = s->causal != 0;
    a.scale = s->scale;
    // the scores' signs go into the resident operand's bits; a scale of zero stays one that a masked score's -inf survives
    a.c2 = (s->scale < 0 ? -s->scale : s->scale) * SEQ_LOG2E;
    if (a.c2 == 0.f) a.c2 = 1e-36f;
    a.flip = s->scale < 0 ? (s->dtype == 0 ? 0x80000000u : 0x80008000u) : 0u;
    return IX_OK;
}

}  // namespace

#define BAND_HD(CALL, DT) { if (s->hd == 32) CALL(DT, 32); else if (s->hd == 64) CALL(DT, 64); else CALL(DT, 128); }
#define BAND_GO(CALL) { if (s->dtype == 0) BAND_HD(CALL, 0) else if (s->dtype == 1) BAND_HD(CALL, 1) else BAND_HD(CALL, 2) }

extern "C" int ix_band_attn_fwd(const struct ix_band* s, void* out, float* lse, void* rest, hipStream_t stream) {
    BandArgs a;
    if (int rc = band_of(a, s, "ix_band_attn_fwd")) return rc;
    IX_CHECK_ARG(out && ix_al16(out) && ix_al16(rest), "ix_band_attn_fwd: null or unaligned output");
    a.out = static_cast<unsigned char*>(out);
    a.rest = s->dtype ? static_cast<unsigned char*>(rest) : nullptr;
    a.lse = lse;
    const dim3 grid(a.B * a.H, (a.Lq + owner_rows(s->dtype) - 1) / owner_rows(s->dtype));
#define BAND_FWD(DT, D) band_fwd_kernel<DT, D, owner_blocks(DT), key_tile(DT)><<<grid, kBlock, 0, stream>>>(a)
    BAND_GO(BAND_FWD)
    IX_CHECK_LAUNCH("ix_band_attn_fwd");
    return IX_OK;
}

extern "C" int ix_band_attn_lse_pitch(int Lq, int64_t* out_host) {
    IX_CHECK_ARG(Lq > 0 && out_host, "ix_band_attn_lse_pitch: bad argument");
    ix_band s{};
    s.Lq = Lq;
    *out_host = lse_pitch(&s);
    return IX_OK;
}

extern "C" int ix_workspace_bytes_band_attn_bwd(const struct ix_band* s, size_t* out_host) {
    BandArgs a;
    if (int rc = band_of(a, s, "ix_workspace_bytes_band_attn_bwd")) return rc;
    IX_CHECK_ARG(out_host, "ix_workspace_bytes_band_attn_bwd: null output");
    *out_host = (size_t)a.B * a.H * a.Lp * 4 + part_bytes(s, key_plan(s));
    return IX_OK;
}

extern "C" int ix_band_attn_bwd(const struct ix_band* s, const void* out, const void* rest, const float* lse, const void* d_out, int64_t g_sb, int64_t g_sl,
                                int64_t g_sh, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    BandArgs a;
    if (int rc = band_of(a, s, "ix_band_attn_bwd")) return rc;
    const int64_t eb = s->dtype == 0 ? 4 : 2;
    IX_CHECK_ARG(out && (rest || s->dtype == 0) && lse && d_out && dq && dk && dv, "ix_band_attn_bwd: null pointer");
    IX_CHECK_ARG(ix_al16(out) && ix_al16(rest) && ix_al16(d_out) && ix_al16(dq) && ix_al16(dk) && ix_al16(dv), "ix_band_attn_bwd: unaligned pointer");
    for (int64_t x : {g_sb, g_sl, g_sh}) IX_CHECK_ARG(x * eb % 16 == 0, "ix_band_attn_bwd: rows that do not start on 16 bytes");
    const KeyPlan r = key_plan(s);
    const size_t parts = part_bytes(s, r), need = (size_t)a.B * a.H * a.Lp * 4 + parts;
    if (!workspace || workspace_bytes < need || !ix_al16(workspace)) {
        ix_set_error("ix_band_attn_bwd: workspace of %zu bytes (16-byte aligned), %zu needed", workspace ? workspace_bytes : (size_t)0, need);
        return IX_ERR_WORKSPACE;
    }
    a.o = static_cast<const unsigned char*>(out);
    a.o_rest = static_cast<const unsigned char*>(rest);
    a.go = static_cast<const unsigned char*>(d_out);
    a.gb = g_sb * eb; a.gl = g_sl * eb; a.gh = g_sh * eb;
    a.lse = const_cast<float*>(lse);
    a.delta = static_cast<float*>(workspace);
    a.part = a.delta + (size_t)a.B * a.H * a.Lp;
    a.dq = static_cast<unsigned char*>(dq);
    a.dk = static_cast<unsigned char*>(dk);
    a.dv = static_cast<unsigned char*>(dv);
    a.wide_blocks = r.wide;
    a.wide_splits = r.wide_splits;
    a.splits = r.splits;
    const int rows = owner_rows(s->dtype);
    const int64_t key_groups = (int64_t)a.B * a.kv * r.items, groups = key_groups + (int64_t)a.B * a.H * ((a.Lq + rows - 1) / rows);
    const int64_t delta_groups = ((int64_t)a.B * a.H * a.Lp * (s->hd * eb / 16) + kBlock - 1) / kBlock;
    IX_CHECK_ARG(groups < (1ll << 31) && delta_groups < (1ll << 31), "ix_band_attn_bwd: too many rows for one launch");
    a.key_groups = (int)key_groups;
#define BAND_DELTA(DT, D) band_delta_kernel<DT, D><<<(unsigned)delta_groups, kBlock, 0, stream>>>(a)
    BAND_GO(BAND_DELTA)
    IX_CHECK_LAUNCH("ix_band_attn_bwd (delta)");
#define BAND_BWD(DT, D) band_bwd_kernel<DT, D, owner_blocks(DT)><<<(unsigned)groups, kBlock, 0, stream>>>(a)
    BAND_GO(BAND_BWD)
    IX_CHECK_LAUNCH("ix_band_attn_bwd");
    if (parts) {
        const int blocks = r.splits > 1 ? r.blocks : r.wide;
        IX_CHECK_ARG(blocks <= 65535, "ix_band_attn_bwd: too many keys for one launch");
        const dim3 sgrid(a.B * a.kv, blocks, 4);
#define BAND_SUM(DT, D) band_sum_kernel<DT, D><<<sgrid, kBlock, 0, stream>>>(a, r.items, owner_rows(DT))
        BAND_GO(BAND_SUM)
        IX_CHECK_LAUNCH("ix_band_attn_bwd (sum)");
    }
    return IX_OK;
}
