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
constexpr int64_t kMostGroups = 1 << 24;   // workgroups along x: a launch counts its threads in 32 bits

// owner rows of a workgroup: one or two blocks of 16 a wave
constexpr int owner_rows(int nb) { return 16 * nb * kWaves; }
constexpr int key_tile(int dt) { return dt == 0 ? 32 : 64; }
constexpr int query_tile(int dt, int hd) { return dt == 0 || hd == 128 ? 32 : 64; }

// ---- the LDS image of a tile of rows ------------------------------------------------------------------------------------------------
// 32-byte pairs of a row change places by the row's number, so that eight neighbouring rows' pieces lie in different banks for both ways
// of reading.  f32: also the four rows 4 apart that a transposed read takes at once.
template <int DT, int D> struct Img {
    static constexpr int EB = SeqT<DT>::bytes, ROW = D * EB, PAIRS = ROW / 32, SWEEP = ROW >= 256 ? 1 : 256 / ROW, KS = D / 32, DB = D / 16, DN = DB < 4 ? DB : 4;
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
    // Columns d = 16 db + n of rows row0 + 4 g + i and row0 + 16 + 4 g + i (row0 a multiple of 32).  The transposing reads stand in one block
    // with their wait: the compiler would let each of them wait for every request into LDS that is still on its way, those of the next tiles
    // too.  Four or eight fragments a block.
    __device__ static __forceinline__ unsigned col_at(const unsigned char* img, int row0, int db, int n, int g) {
        const int row = row0 + 4 * g + (n >> 2);
        return (unsigned)(uintptr_t)(const unsigned char __attribute__((address_space(3)))*)img + row * ROW + ((n & 3) << 3) + ((db ^ turn(row)) << 5);
    }
    __device__ static __forceinline__ Frag<DT> col_frag32(const unsigned char* img, int row0, int db, int n, int g) {   // (f32: plain reads)
        Frag<DT> f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = row0 + 16 * (i / 4) + 4 * g + i % 4;
            f.w[i] = *reinterpret_cast<const unsigned*>(img + row * ROW + (((2 * db + (n >> 3)) ^ turn(row)) << 5) + ((n & 7) << 2));
        }
        return f;
    }
};
#ifdef __HIP_DEVICE_COMPILE__   // (the host's pass does not know the registers' constraint)
#define TR_READ(O, A, OFF) "ds_read_b64_tr_b16 %" #O ", %" #A " offset:%" #OFF "\n\t"
// x[2 i], x[2 i + 1]: rows 4 g .. and 16 + 4 g .. of the column at address i
template <int HALF> __device__ __forceinline__ void tr_8(u32x2 (&x)[16], const unsigned (&a)[8]) {
    asm volatile(TR_READ(0, 16, 24) TR_READ(1, 16, 25) TR_READ(2, 17, 24) TR_READ(3, 17, 25) TR_READ(4, 18, 24) TR_READ(5, 18, 25) TR_READ(6, 19, 24)
                 TR_READ(7, 19, 25) TR_READ(8, 20, 24) TR_READ(9, 20, 25) TR_READ(10, 21, 24) TR_READ(11, 21, 25) TR_READ(12, 22, 24) TR_READ(13, 22, 25)
                 TR_READ(14, 23, 24) TR_READ(15, 23, 25) "s_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7]), "=&v"(x[8]), "=&v"(x[9]),
                   "=&v"(x[10]), "=&v"(x[11]), "=&v"(x[12]), "=&v"(x[13]), "=&v"(x[14]), "=&v"(x[15])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]), "n"(0), "n"(HALF) : "memory");
}
// the same of four addresses, and (x[8 + ..]) of the places 2 HALF behind them
template <int HALF> __device__ __forceinline__ void tr_4_twice(u32x2 (&x)[16], const unsigned (&a)[4]) {
    asm volatile(TR_READ(0, 16, 20) TR_READ(1, 16, 21) TR_READ(2, 17, 20) TR_READ(3, 17, 21) TR_READ(4, 18, 20) TR_READ(5, 18, 21) TR_READ(6, 19, 20)
                 TR_READ(7, 19, 21) TR_READ(8, 16, 22) TR_READ(9, 16, 23) TR_READ(10, 17, 22) TR_READ(11, 17, 23) TR_READ(12, 18, 22) TR_READ(13, 18, 23)
                 TR_READ(14, 19, 22) TR_READ(15, 19, 23) "s_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7]), "=&v"(x[8]), "=&v"(x[9]),
                   "=&v"(x[10]), "=&v"(x[11]), "=&v"(x[12]), "=&v"(x[13]), "=&v"(x[14]), "=&v"(x[15])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(0), "n"(HALF), "n"(2 * HALF), "n"(3 * HALF) : "memory");
}
template <int HALF> __device__ __forceinline__ void tr_4(u32x2 (&x)[8], const unsigned (&a)[4]) {
    asm volatile(TR_READ(0, 8, 12) TR_READ(1, 8, 13) TR_READ(2, 9, 12) TR_READ(3, 9, 13) TR_READ(4, 10, 12) TR_READ(5, 10, 13) TR_READ(6, 11, 12)
                 TR_READ(7, 11, 13) "s_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(0), "n"(HALF) : "memory");
}
#undef TR_READ
#else
template <int HALF> __device__ void tr_8(u32x2 (&x)[16], const unsigned (&a)[8]);
template <int HALF> __device__ void tr_4_twice(u32x2 (&x)[16], const unsigned (&a)[4]);
template <int HALF> __device__ void tr_4(u32x2 (&x)[8], const unsigned (&a)[4]);
#endif
template <int DT> __device__ __forceinline__ Frag<DT> frag_of(const u32x2& a, const u32x2& b) {
    Frag<DT> f;
    f.w[0] = a.x; f.w[1] = a.y; f.w[2] = b.x; f.w[3] = b.y;
    return f;
}
// f[i]: column block db0 + i of image A (rows row0 ..), f[4 + i]: of image B, DN <= 4 of each
template <int DT, int D, int DN>
__device__ __forceinline__ void two_images(Frag<DT> (&f)[2][DN], const unsigned char* A, const unsigned char* B, int row0, int db0, int n, int g) {
    typedef Img<DT, D> I;
    if constexpr (DT == 0) {
#pragma unroll
        for (int i = 0; i < DN; ++i) { f[0][i] = I::col_frag32(A, row0, db0 + i, n, g); f[1][i] = I::col_frag32(B, row0, db0 + i, n, g); }
    } else if constexpr (DN == 4) {
        u32x2 x[16];
        const unsigned a[8] = {I::col_at(A, row0, db0, n, g), I::col_at(A, row0, db0 + 1, n, g), I::col_at(A, row0, db0 + 2, n, g), I::col_at(A, row0, db0 + 3, n, g),
                               I::col_at(B, row0, db0, n, g), I::col_at(B, row0, db0 + 1, n, g), I::col_at(B, row0, db0 + 2, n, g), I::col_at(B, row0, db0 + 3, n, g)};
        tr_8<16 * I::ROW>(x, a);
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[0][i] = frag_of<DT>(x[2 * i], x[2 * i + 1]); f[1][i] = frag_of<DT>(x[8 + 2 * i], x[8 + 2 * i + 1]); }
    } else {
        u32x2 x[8];
        const unsigned a[4] = {I::col_at(A, row0, db0, n, g), I::col_at(A, row0, db0 + 1, n, g), I::col_at(B, row0, db0, n, g), I::col_at(B, row0, db0 + 1, n, g)};
        tr_4<16 * I::ROW>(x, a);
#pragma unroll
        for (int i = 0; i < 2; ++i) { f[0][i] = frag_of<DT>(x[2 * i], x[2 * i + 1]); f[1][i] = frag_of<DT>(x[4 + 2 * i], x[4 + 2 * i + 1]); }
    }
}
// f[kk][i]: column block db0 + i of rows row0 + 32 kk ..
template <int DT, int D, int KK, int DN>
__device__ __forceinline__ void one_image(Frag<DT> (&f)[KK][DN], const unsigned char* A, int row0, int db0, int n, int g) {
    typedef Img<DT, D> I;
    if constexpr (DT == 0) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int i = 0; i < DN; ++i) f[kk][i] = I::col_frag32(A, row0 + 32 * kk, db0 + i, n, g);
    } else if constexpr (DN == 4 && KK == 2) {
        u32x2 x[16];
        unsigned a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = I::col_at(A, row0, db0 + i, n, g);
        tr_4_twice<16 * I::ROW>(x, a);
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[0][i] = frag_of<DT>(x[2 * i], x[2 * i + 1]); f[1][i] = frag_of<DT>(x[8 + 2 * i], x[8 + 2 * i + 1]); }
    } else if constexpr (DN == 4) {
        u32x2 x[8];
        const unsigned a[4] = {I::col_at(A, row0, db0, n, g), I::col_at(A, row0, db0 + 1, n, g), I::col_at(A, row0, db0 + 2, n, g), I::col_at(A, row0, db0 + 3, n, g)};
        tr_4<16 * I::ROW>(x, a);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[0][i] = frag_of<DT>(x[2 * i], x[2 * i + 1]);
    } else {   // head dim 32: two column blocks
        static_assert(DN == 2 && KK <= 2, "");
        u32x2 x[8];
        const unsigned a[4] = {I::col_at(A, row0, 0, n, g), I::col_at(A, row0, 1, n, g), I::col_at(A, row0 + 32 * (KK - 1), 0, n, g), I::col_at(A, row0 + 32 * (KK - 1), 1, n, g)};
        tr_4<16 * I::ROW>(x, a);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int i = 0; i < 2; ++i) f[kk][i] = frag_of<DT>(x[4 * kk + 2 * i], x[4 * kk + 2 * i + 1]);
    }
}
static_assert(Img<1, 128>::PAIRS == 8 && Img<1, 32>::SWEEP == 4, "image geometry");

// A tile of ROWS rows from memory to LDS without registers: every lane names the 16 bytes that belong at its place of the image
// (the image's order is the lanes'), rows from `rows` on read as zeros (they lie behind the descriptor's end).
typedef void __attribute__((address_space(3))) lds_void;
template <int DT, int D, int ROWS> struct Dma {
    static constexpr int CH = Img<DT, D>::ROW / 16, N = ROWS * CH / kBlock;   // requests of a wave
    static_assert(ROWS * CH % kBlock == 0, "a tile is whole passes of the workgroup");
    int at[N];
    const unsigned char* base;
    int64_t stride;
    __device__ __forceinline__ Dma(const unsigned char* base_, int64_t stride_, int wave, int lane) : base(base_), stride(stride_) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int place = (wave * N + u) * 64 + lane, row = place / CH, c = place % CH;
            at[u] = row * (int)stride + ((((c >> 1) ^ Img<DT, D>::turn(row)) << 1 | (c & 1)) << 4);
        }
    }
    __device__ __forceinline__ void issue(unsigned char* img, int wave, int row0, int rows) const {
        const int64_t end = row0 < rows ? (int64_t)(rows - row0 - 1) * stride + Img<DT, D>::ROW : 0;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(base + row0 * stride), 0, (int)min(end, (int64_t)0x7ffffff0), 0x00020000);
#pragma unroll
        for (int u = 0; u < N; ++u) __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(img + (wave * N + u) * 1024), 16, at[u], 0, 0, 0);
    }
};
// this wave's requests but the newest N have landed, and it has read what it wanted of the other stages; then everybody's and everybody
template <int N> __device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// stages of the ring: three (requests two tiles ahead) where a workgroup's LDS stays within the limit, else two.  Gradients 48 KB; forward 32,
// where one more workgroup fits on a compute unit instead (48 / 32 KB: f32 of 8 heads of 64, 8 192 with window 1 000 167 / 153 us; bf16, 12 755
// with window 2 551 128 / 130, 2 x 2 060 with window 412 24.2 / 24.0, 2 x 4 096 in full 69 / 70).
constexpr int stages(int bytes, int limit) { return 3 * bytes <= limit ? 3 : 2; }
constexpr int kFwdRing = 32768, kBwdRing = 49152;

struct BandArgs {
    const unsigned char *q, *k, *v, *go, *o, *o_rest;
    int64_t qb, ql, qh, kb, kl, kh, vb, vl, vh, gb, gl, gh;   // bytes
    unsigned char *out, *rest, *dq, *dk, *dv;                 // dense; rest: what rounding the output to 16 bits took away, in 16 bits
    float *lse, *delta, *part, *part_ml, *part_q;             // [B][H][Lp] base-2 normalisers (+inf: nothing visible) and delta; partial sums
    const int *q_lens, *kv_lens;
    int B, Lq, Lk, Lp, H, kv, left, right, sinks, causal;
    int wide_blocks, wide_splits, splits, key_groups, cut;    // dk / dv: see the host side; workgroups of theirs; of a (batch, key head) cut blocks have
    int q_splits;                                             // dq: pieces of a block's key tiles
    int fwd_splits;                                           // forward: pieces of a block's key tiles
    float c2, scale;                                          // |scale| log2(e), scale
    unsigned flip;                                            // sign bits of a fragment's register where scale < 0
    __device__ __forceinline__ int m(int b) const { return q_lens ? min(max(q_lens[b], 0), Lq) : Lq; }
    __device__ __forceinline__ int n(int b) const { return kv_lens ? min(max(kv_lens[b], 0), Lk) : Lk; }
    // every pair of p0 .. p1 and j0 .. j1 sees each other (apart from j < n)
    __device__ __forceinline__ bool all_see(int p0, int p1, int j0, int j1) const {
        return (j0 >= p1 - left && j1 <= p0 + right) || (j1 < sinks && (!causal || j1 <= p0));
    }
    __device__ __forceinline__ bool none_sees(int p0, int p1, int j0, int j1) const {
        return (j1 < p0 - left || j0 > p1 + right) && (j0 >= sinks || (causal && j0 > p1));
    }
};

// The streamed rows x that go with one owner row: lo <= x <= lo + width, or x < first.
struct Range {
    int lo, first;
    unsigned width;
    __device__ __forceinline__ bool in(int x) const { return (unsigned)(x - lo) <= width; }
};
// the keys that a query at p sees among n
__device__ __forceinline__ Range keys_of(const BandArgs& a, int p, int n) {
    const int hi = min(n - 1, p + a.right), lo = p - a.left;
    const bool some = lo <= hi;
    return Range{some ? lo : kFar, max(0, min(n, a.causal ? min(a.sinks, p + 1) : a.sinks)), some ? (unsigned)(hi - lo) : 0u};
}
// the positions of the queries that see key j
__device__ __forceinline__ Range queries_of(const BandArgs& a, int j) {
    const bool to_all = j < a.sinks;
    const int lo = to_all ? (a.causal ? j : -kFar) : j - a.right;
    return Range{lo, 0, to_all ? 2u * kFar : (unsigned)a.left + (unsigned)a.right};
}

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

// ... and the operand of what that rounding took away.  Weights (into the outputs and dv) and score gradients (into dq and dk) are carried as
// these two terms: outputs and gradients are then as good as from 32-bit ones.  With one term the error against 64 bits is 1.4 (outputs, dv)
// and 1.45 to 1.7 times (dq, dk) that of the result's own rounding, with two 1.0 times.  The second terms of the weights cost 58 of 446 us
// (forward and gradients, bf16, 12 755 queries and keys of 8 heads of 64, window 2 551) and 67 of 347 us (forward, fp16, 8 192 of 32 heads
// over 8 of 128, window 2 048), those of the score gradients 60 us of the former.
template <int DT> __device__ __forceinline__ Frag<DT> rest_frag(const f32x4& a, const f32x4& b, const Frag<DT>& f) {
    Frag<DT> r;
    r.w[0] = seq_pack<DT>(seq_less_lo<DT>(a[0], f.w[0]), seq_less_hi<DT>(a[1], f.w[0]));
    r.w[1] = seq_pack<DT>(seq_less_lo<DT>(a[2], f.w[1]), seq_less_hi<DT>(a[3], f.w[1]));
    r.w[2] = seq_pack<DT>(seq_less_lo<DT>(b[0], f.w[2]), seq_less_hi<DT>(b[1], f.w[2]));
    r.w[3] = seq_pack<DT>(seq_less_lo<DT>(b[2], f.w[3]), seq_less_hi<DT>(b[3], f.w[3]));
    return r;
}

// four neighbouring values of a row
template <int DT> __device__ __forceinline__ void store4(unsigned char* p, const f32x4& x) {
    if constexpr (DT == 0) *reinterpret_cast<f32x4*>(p) = x;
    else *reinterpret_cast<u32x2*>(p) = u32x2{seq_pack<DT>(x[0], x[1]), seq_pack<DT>(x[2], x[3])};
}

// four values of the output, and of what rounding takes from them
template <int DT> __device__ __forceinline__ void store_out(const BandArgs& a, int64_t at, const f32x4& x) {
    store4<DT>(a.out + at, x);
    if constexpr (DT != 0) {
        if (a.rest) {
            f32x4 y;
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                const unsigned w = seq_pack<DT>(x[r], x[r + 1]);
                y[r] = x[r] - seq_lo<DT>(w);
                y[r + 1] = x[r + 1] - seq_hi<DT>(w);
            }
            store4<DT>(a.rest + at, y);
        }
    }
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
// most tiles leave the accumulators alone.  16-bit types: a weight goes into the second product as two terms (rest_frag), into the sum unrounded.
// 16-bit types are bound by matrix and vector instructions together (matrix pipe 54 % and vector instructions 54 % of busy cycles at hd 128, 37 and
// 70 % at hd 64, no LDS conflicts): fp16, 8 192 queries and keys of 32 / 8 heads of 128, window 2 048: 342-358 us = 1 070-1 115 TFLOP/s over
// three products, 0.92-0.96 of what a plain product of 8 192^3 reaches; bf16, 12 755 of 8 heads of 64, window 2 551: 119-130 us = 730-795 TFLOP/s
// (a score costs as much exponential for half the product); 2 060 of 16 heads of 64, window 412: 24 us, its 528 workgroups' first and last
// tiles.  f32, 16 x 361 of 8 heads of 32, window 64: 20 us = 52 of 154 TFLOP/s, matrix pipe 40 %, vector instructions 23 %, and of the LDS cycles
// a quarter bank conflicts: six short tiles a workgroup do not cover their waits.
constexpr float kSlack = 8.f;
// fp16: weights are carried 2^7 and, for dv, 2^10 times as large (the largest forward weight, 2^8 by the slack, is then 2^15; the type ends at
// 65 504), so that its smallest step, 2^-24, is 2^-31 of the row's largest weight and 2^-34: a row whose first key takes nearly all the weight
// keeps what the others have.  Where exponents are so large that a float32 does not hold them to less than a step (kWide), a weight can come
// out beyond 2^15: it is cut there (a select, which a NaN passes), in a branch that other rows do not take.
template <int DT> constexpr float kUp = DT == 2 ? 7.f : 0.f;
template <int DT> constexpr float kUpFactor = DT == 2 ? 128.f : 1.f;
template <int DT> constexpr float kUpDv = DT == 2 ? 1024.f : 1.f;
constexpr float kWide = 1048576.f;   // 2^20: steps of 2^-3

template <int DT, int D, int NB, int TB>
__device__ __forceinline__ void band_fwd(const BandArgs& a, unsigned char* mem) {
    typedef Img<DT, D> I;
    constexpr int ROWS = 16 * NB * kWaves, SB = TB / 16, BYTES = TB * I::ROW, STG = stages(2 * BYTES, kFwdRing);
    auto lds = reinterpret_cast<unsigned char (*)[2][BYTES]>(mem);
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
        const Dma<DT, D, TB> dk(kp, a.kl, wave, lane), dv(vp, a.vl, wave, lane);
        auto issue = [&](int t) {
            const int row0 = kt.tile(t) * TB, st = t % STG;
            dk.issue(lds[st][0], wave, row0, n);
            dv.issue(lds[st][1], wave, row0, n);
        };
        const int t0 = kt.count * blockIdx.z / a.fwd_splits, t1 = kt.count * (blockIdx.z + 1) / a.fwd_splits;
#pragma unroll
        for (int t = 0; t < STG - 1; ++t)
            if (t0 + t < t1) issue(t0 + t);
        for (int t = t0; t < t1; ++t) {
            const unsigned char *ki = lds[t % STG][0], *vi = lds[t % STG][1];
            const int j0 = kt.tile(t) * TB;
            if (STG == 3 && t + 1 < t1) landed<2 * Dma<DT, D, TB>::N>();
            else landed<0>();
            if (t + STG - 1 < t1) issue(t + STG - 1);
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
                    const bool firsts = j0 < a.sinks;   // (uniform: most masked tiles have no first keys)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const Range r = keys_of(a, iw + 16 * nb + n16 + shift, n);
                        if (firsts) {
#pragma unroll
                            for (int sb = 0; sb < SB; ++sb)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int j = j0 + 4 * g + 16 * sb + e;
                                    s[nb][sb][e] = r.in(j) | (j < r.first) ? s[nb][sb][e] : -INFINITY;
                                }
                        } else {
#pragma unroll
                            for (int sb = 0; sb < SB; ++sb)
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[nb][sb][e] = r.in(j0 + 4 * g + 16 * sb + e) ? s[nb][sb][e] : -INFINITY;
                        }
                    }
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int sb = 0; sb < SB; ++sb)
#pragma unroll
                        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[nb][sb][r]);
                    mx *= a.c2;
                    if (__builtin_amdgcn_ballot_w64(mx > top[nb] + kSlack)) {   // (each lane by its own keys: no exchange where nobody exceeds)
                        mx = seq_max_g(mx);
                        const float up = fmaxf(top[nb], mx), down = up == -INFINITY ? 1.f : seq_exp2(top[nb] - up);
                        top[nb] = up;
                        sum[nb] *= down;
#pragma unroll
                        for (int db = 0; db < I::DB; ++db) o[nb][db] *= down;
                    }
                    const float ref = (top[nb] == -INFINITY ? 0.f : top[nb]) - kUp<DT>;
#pragma unroll
                    for (int sb = 0; sb < SB; ++sb)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[nb][sb][r] = seq_exp2(fmaf(s[nb][sb][r], a.c2, -ref));
                    if constexpr (DT == 2) {
                        if (__builtin_amdgcn_ballot_w64(fabsf(ref) > kWide)) {
#pragma unroll
                            for (int sb = 0; sb < SB; ++sb)
#pragma unroll
                                for (int r = 0; r < 4; ++r) s[nb][sb][r] = s[nb][sb][r] > 32768.f ? 32768.f : s[nb][sb][r];
                        }
                    }
#pragma unroll
                    for (int sb = 0; sb < SB; ++sb)
#pragma unroll
                        for (int r = 0; r < 4; ++r) sum[nb] += s[nb][sb][r];
                }
                // 32-row steps whose columns come in one block of reads (head dim 128: four column blocks of one step; more at once was no faster)
                constexpr int KK = SB / 2, TOGETHER = I::DB == 8 ? 1 : KK;
#pragma unroll
                for (int k0 = 0; k0 < KK; k0 += TOGETHER) {
                    Frag<DT> pf[TOGETHER][NB], pr[TOGETHER][NB];
#pragma unroll
                    for (int kk = 0; kk < TOGETHER; ++kk)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const f32x4 &x = s[nb][2 * (k0 + kk)], &y = s[nb][2 * (k0 + kk) + 1];
                            pf[kk][nb] = as_frag<DT>(x, y);
                            if constexpr (DT != 0) pr[kk][nb] = rest_frag<DT>(x, y, pf[kk][nb]);
                        }
#pragma unroll
                    for (int d0 = 0; d0 < I::DB; d0 += I::DN) {
                        Frag<DT> vf[TOGETHER][I::DN];
                        one_image<DT, D>(vf, vi, 32 * k0, d0, n16, g);
#pragma unroll
                        for (int kk = 0; kk < TOGETHER; ++kk)
#pragma unroll
                            for (int db = 0; db < I::DN; ++db)
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb) {
                                    if constexpr (DT != 0) o[nb][d0 + db] = seq_mma<DT>(vf[kk][db], pr[kk][nb], o[nb][d0 + db]);
                                    o[nb][d0 + db] = seq_mma<DT>(vf[kk][db], pf[kk][nb], o[nb][d0 + db]);
                                }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int i = iw + 16 * nb + n16;
        const float total = seq_sum_g(sum[nb]);
        if (a.fwd_splits > 1) {   // what this piece has, for band_join_kernel
            if (i >= a.Lq) continue;
            const int64_t at = ((int64_t)bh * a.Lq + i) * a.fwd_splits + blockIdx.z;
            if (g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = float2{top[nb], total / kUpFactor<DT>};
#pragma unroll
            for (int db = 0; db < I::DB; ++db) *reinterpret_cast<f32x4*>(a.part + at * D + 16 * db + 4 * g) = o[nb][db] * (1.f / kUpFactor<DT>);
            continue;
        }
        const bool none = i >= m || total == 0.f;
        const float inv = 1.f / total;
        if (a.lse && g == 0 && i < a.Lp) a.lse[(int64_t)bh * a.Lp + i] = none ? INFINITY : top[nb] - kUp<DT> + __log2f(total);
        if (i >= a.Lq) continue;
        const int64_t at = (((int64_t)b * a.Lq + i) * a.H + h) * I::ROW;
#pragma unroll
        for (int db = 0; db < I::DB; ++db) store_out<DT>(a, at + (16 * db + 4 * g) * I::EB, none ? f32x4{0.f, 0.f, 0.f, 0.f} : o[nb][db] * inv);
    }
}

// (the body is a device function: with it in the kernel, ROCm 7.2's host pass left the stubs of two blocks a wave undefined)
template <int DT, int D, int NB>
__global__ __launch_bounds__(kBlock, 2) void band_fwd_kernel(BandArgs a) {
    constexpr int STAGE = 2 * key_tile(DT) * Img<DT, D>::ROW;
    __shared__ __attribute__((aligned(256))) unsigned char mem[stages(STAGE, kFwdRing) * STAGE];
    band_fwd<DT, D, NB, key_tile(DT)>(a, mem);
}

// The pieces of every row joined, in their order, four values a lane: 5 us for 640 rows of 128 in 23 pieces (7.6 MB), 12 with one piece at a time.
template <int DT, int D>
__global__ __launch_bounds__(kBlock) void band_join_kernel(BandArgs a) {
    constexpr int LANES = D / 4;
    const int64_t row = ((int64_t)blockIdx.x * kBlock + threadIdx.x) / LANES;   // (batch, head, query up to the pitch)
    const int c = threadIdx.x % LANES, i = (int)(row % a.Lp);
    const int64_t bh = row / a.Lp;
    if (bh >= (int64_t)a.B * a.H) return;
    const int b = (int)(bh / a.H), h = (int)(bh % a.H);
    float top = -INFINITY, sum = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (i < a.m(b)) {
        const int64_t at = (bh * a.Lq + i) * a.fwd_splits;
        for (int s0 = 0; s0 < a.fwd_splits; s0 += 8) {   // eight pieces' loads in flight
            float2 ml[8];
            f32x4 o[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int s = min(s0 + u, a.fwd_splits - 1);
                ml[u] = *reinterpret_cast<const float2*>(a.part_ml + 2 * (at + s));
                o[u] = *reinterpret_cast<const f32x4*>(a.part + (at + s) * D + 4 * c);
            }
            float up = top;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                ml[u].x = s0 + u < a.fwd_splits ? ml[u].x : -INFINITY;
                up = fmaxf(up, ml[u].x);
            }
            const float ref = up == -INFINITY ? 0.f : up, down = seq_exp2(top - ref);
            sum *= down;
            x *= down;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float f = seq_exp2(ml[u].x - ref);
                sum += ml[u].y * f;
                x += o[u] * f;
            }
            top = up;
        }
    }
    if (c == 0 && a.lse) a.lse[row] = sum == 0.f ? INFINITY : top + __log2f(sum);
    if (i < a.Lq) store_out<DT>(a, (((int64_t)b * a.Lq + i) * a.H + h) * Img<DT, D>::ROW + c * 4 * SeqT<DT>::bytes, sum == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : x * (1.f / sum));
}

// ====================================================================================================================================
// gradients
// ====================================================================================================================================
// -delta_i = -do_i o_i (where the sums of do_i v_j start), a row by the lanes that hold 16 bytes of it each.  16-bit: o is the stored output and
// the rest its rounding took, so that delta -- which is subtracted from every do_i v_j of the row -- is as good as from the 32-bit output.
// HBM-bound, with a launch's few microseconds before it: 102 040 rows of 64 in bf16 8 us, 4.9 TB/s.
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
    if (c == 0) a.delta[((int64_t)b * a.H + h) * a.Lp + i] = -d;
}

// dq: query-owning, streams k (both ways) and v (rows).  Tiles are taken 32 keys at a time.  Pieces of a block's tiles leave f32 partial sums
// [ROWS][D]; band_sum_kernel adds them in order.
template <int DT, int D, int NB, int TB>
__device__ __forceinline__ void band_dq(const BandArgs& a, unsigned char* mem, int group) {
    typedef Img<DT, D> I;
    constexpr int ROWS = 16 * NB * kWaves, BYTES = TB * I::ROW, STG = stages(2 * BYTES, kBwdRing);
    auto lds = reinterpret_cast<unsigned char (*)[2][BYTES]>(mem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g = lane >> 4;
    const int bh = spread_heads(group % (a.B * a.H), a.B * a.H), b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.kv);
    const int piece = group / (a.B * a.H), split = piece % a.q_splits, y = piece / a.q_splits;
    const int blocks = (a.Lq + ROWS - 1) / ROWS, blk = a.causal ? blocks - 1 - y : y, i0 = blk * ROWS;
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
        const Dma<DT, D, TB> dk(kp, a.kl, wave, lane), dv(vp, a.vl, wave, lane);
        auto issue = [&](int t) {
            const int row0 = kt.tile(t) * TB, st = t % STG;
            dk.issue(lds[st][0], wave, row0, n);
            dv.issue(lds[st][1], wave, row0, n);
        };
        const int t0 = kt.count * split / a.q_splits, t1 = kt.count * (split + 1) / a.q_splits;
#pragma unroll
        for (int t = 0; t < STG - 1; ++t)
            if (t0 + t < t1) issue(t0 + t);
        for (int t = t0; t < t1; ++t) {
            const unsigned char *ki = lds[t % STG][0], *vi = lds[t % STG][1];
            const int j0 = kt.tile(t) * TB;
            if (STG == 3 && t + 1 < t1) landed<2 * Dma<DT, D, TB>::N>();
            else landed<0>();
            if (t + STG - 1 < t1) issue(t + STG - 1);
            if (iw < m && !a.none_sees(pw0, pw1, j0, j0 + TB - 1)) {
                const bool part = j0 + TB > n || !a.all_see(pw0, pw1, j0, j0 + TB - 1);
#pragma unroll
                for (int kk = 0; kk < TB / 32; ++kk) {
                    f32x4 s[NB][2], z[NB][2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {   // (the second product's sum starts at -delta)
                            s[nb][u] = f32x4{0.f, 0.f, 0.f, 0.f};
                            z[nb][u] = f32x4{delta[nb], delta[nb], delta[nb], delta[nb]};
                        }
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
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) s[nb][u][r] = seq_exp2(fmaf(s[nb][u][r], a.c2, -lse[nb]));
                    if (part) {
                        const bool firsts = j0 < a.sinks;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const Range r = keys_of(a, iw + 16 * nb + n16 + shift, n);
#pragma unroll
                            for (int u = 0; u < 2; ++u)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int j = j0 + 4 * g + 32 * kk + 16 * u + e;
                                    s[nb][u][e] = r.in(j) | (firsts & (j < r.first)) ? s[nb][u][e] : 0.f;
                                }
                        }
                    }
                    Frag<DT> zf[NB], zr[NB];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) z[nb][u][r] *= s[nb][u][r];
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
                        if constexpr (DT != 0) zr[nb] = rest_frag<DT>(z[nb][0], z[nb][1], zf[nb]);
                    }
#pragma unroll
                    for (int d0 = 0; d0 < I::DB; d0 += I::DN) {
                        Frag<DT> kc[1][I::DN];
                        one_image<DT, D>(kc, ki, 32 * kk, d0, n16, g);
#pragma unroll
                        for (int db = 0; db < I::DN; ++db)
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                if constexpr (DT != 0) acc[nb][d0 + db] = seq_mma<DT>(kc[0][db], zr[nb], acc[nb][d0 + db]);
                                acc[nb][d0 + db] = seq_mma<DT>(kc[0][db], zf[nb], acc[nb][d0 + db]);
                            }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int i = iw + 16 * nb + n16;
        const float f = DT == 2 ? a.scale / F[nb] : a.scale;
        if (a.q_splits > 1) {
            float* dst = a.part_q + ((((int64_t)bh * blocks + blk) * a.q_splits + split) * ROWS + i - i0) * D;
#pragma unroll
            for (int db = 0; db < I::DB; ++db) *reinterpret_cast<f32x4*>(dst + 16 * db + 4 * g) = acc[nb][db] * f;
            continue;
        }
        if (i >= a.Lq) continue;
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
    constexpr int ROWS = 16 * NB * kWaves, BYTES = TB * I::ROW, STG = stages(2 * BYTES, kBwdRing);
    auto lds = reinterpret_cast<unsigned char (*)[2][BYTES]>(mem);
    auto row_c = reinterpret_cast<float (*)[4][64]>(mem + STG * 2 * BYTES);   // lse, -delta of the tile's queries (and what waves 2, 3 fetch)
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
        const int jw1 = min(jw + 16 * NB, n) - 1, h0 = hk * G;
        Dma<DT, D, TB> dq(a.q + b * a.qb + h0 * a.qh, a.ql, wave, lane), dg(a.go + b * a.gb + h0 * a.gh, a.gl, wave, lane);
        int ahead_h = u0 / tiles, ahead = u0 % tiles, now = ahead;   // head and tile of the next request, tile being worked on
        const float* consts = (wave & 1 ? a.delta : a.lse) + ((int64_t)b * a.H + h0) * a.Lp;
        const unsigned char *q0 = dq.base, *g0 = dg.base;
        auto issue = [&](int st) {
            const int i0 = (first + ahead) * TB;
            dq.base = q0 + ahead_h * a.qh;
            dg.base = g0 + ahead_h * a.gh;
            dq.issue(lds[st][0], wave, i0, m);
            dg.issue(lds[st][1], wave, i0, m);
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(consts + (int64_t)ahead_h * a.Lp + i0), 0, (a.Lp - i0) * 4, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(&row_c[st][wave][0]), 4, lane * 4, 0, 0, 0);
            if (++ahead == tiles) { ahead = 0; ++ahead_h; }
        };
        const int count = u1 - u0;
#pragma unroll
        for (int t = 0; t < STG - 1; ++t)
            if (t < count) issue(t);
        for (int t = 0; t < count; ++t) {
            const int buf = t % STG;
            const unsigned char *qi = lds[buf][0], *gi = lds[buf][1];
            const int p0 = (first + now) * TB + shift, p1 = p0 + TB - 1;   // (queries behind m: do = 0 and P = 0)
            if (++now == tiles) now = 0;
            if (STG == 3 && t + 1 < count) landed<2 * Dma<DT, D, TB>::N + 1>();
            else landed<0>();
            if (t + STG - 1 < count) issue((t + STG - 1) % STG);
            if (jw < n && !a.none_sees(p0, p1, jw, jw1)) {
                const bool part = !a.all_see(p0, p1, jw, jw1);
#pragma unroll
                for (int kk = 0; kk < TB / 32; ++kk) {
                    f32x4 s[NB][2], z[NB][2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const f32x4 del = *reinterpret_cast<const f32x4*>(&row_c[buf][1][32 * kk + 16 * x + 4 * g]);   // (-delta)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            s[nb][x] = f32x4{0.f, 0.f, 0.f, 0.f};
                            z[nb][x] = del;
                        }
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
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const f32x4 lse = *reinterpret_cast<const f32x4*>(&row_c[buf][0][32 * kk + 16 * x + 4 * g]);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int r = 0; r < 4; ++r) s[nb][x][r] = seq_exp2(fmaf(s[nb][x][r], a.c2, -lse[r]));
                    }
                    if (part) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const Range r = queries_of(a, jw + 16 * nb + n16);
#pragma unroll
                            for (int x = 0; x < 2; ++x)
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[nb][x][e] = r.in(p0 + 4 * g + 32 * kk + 16 * x + e) ? s[nb][x][e] : 0.f;
                        }
                    }
                    Frag<DT> pf[NB], pr[NB], zf[NB], zr[NB];
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) z[nb][x] *= s[nb][x];
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
                            s[nb][0] *= kUpDv<DT>;
                            s[nb][1] *= kUpDv<DT>;
                        }
                        pf[nb] = as_frag<DT>(s[nb][0], s[nb][1]);
                        zf[nb] = as_frag<DT>(z[nb][0], z[nb][1]);
                        if constexpr (DT != 0) {
                            pr[nb] = rest_frag<DT>(s[nb][0], s[nb][1], pf[nb]);
                            zr[nb] = rest_frag<DT>(z[nb][0], z[nb][1], zf[nb]);
                        }
                    }
#pragma unroll
                    for (int d0 = 0; d0 < I::DB; d0 += I::DN) {
                        Frag<DT> gq[2][I::DN];   // columns of do, of q
                        two_images<DT, D, I::DN>(gq, gi, qi, 32 * kk, d0, n16, g);
#pragma unroll
                        for (int db = 0; db < I::DN; ++db)
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                if constexpr (DT != 0) av[nb][d0 + db] = seq_mma<DT>(gq[0][db], pr[nb], av[nb][d0 + db]);
                                av[nb][d0 + db] = seq_mma<DT>(gq[0][db], pf[nb], av[nb][d0 + db]);
                                if constexpr (DT != 0) ak[nb][d0 + db] = seq_mma<DT>(gq[1][db], zr[nb], ak[nb][d0 + db]);
                                ak[nb][d0 + db] = seq_mma<DT>(gq[1][db], zf[nb], ak[nb][d0 + db]);
                            }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int row = wave * 16 * NB + 16 * nb + n16, j = j0 + row;
        const float fk = DT == 2 ? a.scale / F[nb] : a.scale, fv = 1.f / kUpDv<DT>;
        if (j >= n) {   // (padding: columns beside the valid ones of this block)
#pragma unroll
            for (int db = 0; db < I::DB; ++db) ak[nb][db] = av[nb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (it.splits > 1) {
            float* dst = a.part + (((int64_t)bk * a.cut + item) * 2 * ROWS + row) * D;
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
// Ten products of 2 hd operations a pair (four of the formulas, q k^T and do v^T twice, the second terms of P and dz): 12 755 queries and keys of 8
// heads of 64, window 2 551, bf16: 300 us (353 under a profiler) = 1 050 TFLOP/s, matrix pipe 44 % and vector instructions 58 % of busy cycles;
// 2 x 2 060, window 412: 57-64 us = 460-520 TFLOP/s, 1 056 workgroups in 768 places; head dim 128 at 8 192 of 32 / 8 heads, window 2 048: 1 200
// us; f32 (seven products), 16 x 361 of 8 heads of 32, window 64: 48 us = 72 TFLOP/s, matrix pipe 55 %, vector instructions 20 %.  Scores of
// the next 32 rows ahead of this one's exponentials gained nothing (350 / 350 us before the weights had a second term).
template <int DT, int D> constexpr int bwd_bytes() {
    constexpr int qs = 2 * key_tile(DT) * Img<DT, D>::ROW, ks = 2 * query_tile(DT, D) * Img<DT, D>::ROW;
    constexpr int q = stages(qs, kBwdRing) * qs, k = stages(ks, kBwdRing) * (ks + 1024);
    return q > k ? q : k;
}
template <int DT, int D, int NB>
__global__ __launch_bounds__(kBlock, 2) void band_bwd_kernel(BandArgs a) {
    __shared__ __attribute__((aligned(256))) unsigned char mem[bwd_bytes<DT, D>()];
    if ((int)blockIdx.x < a.key_groups) band_dkv<DT, D, NB, query_tile(DT, D)>(a, mem, blockIdx.x);
    else band_dq<DT, D, NB, key_tile(DT)>(a, mem, blockIdx.x - a.key_groups);
}

// dk, dv (and, with pieces of dq, then dq) of the blocks that were cut: the partial sums in their order, four values a thread
template <int DT, int D>
__global__ __launch_bounds__(kBlock) void band_sum_kernel(BandArgs a, int rows) {
    typedef Img<DT, D> I;
    const int block = blockIdx.y;
    if ((int)blockIdx.x >= a.B * a.kv) {
        const int bh = blockIdx.x - a.B * a.kv, b = bh / a.H, h = bh % a.H, blocks = (a.Lq + rows - 1) / rows;
        if (block >= blocks) return;
        for (int e = (blockIdx.z * kBlock + threadIdx.x) * 4; e < rows * D; e += gridDim.z * kBlock * 4) {
            const int i = block * rows + e / D;
            if (i >= a.Lq) continue;
            const float* src = a.part_q + ((int64_t)bh * blocks + block) * a.q_splits * rows * D + e;
            f32x4 x = *reinterpret_cast<const f32x4*>(src);
#pragma unroll 8
            for (int s = 1; s < a.q_splits; ++s) x += *reinterpret_cast<const f32x4*>(src + (int64_t)s * rows * D);
            store4<DT>(a.dq + (((int64_t)b * a.Lq + i) * a.H + h) * I::ROW + e % D * I::EB, x);
        }
        return;
    }
    const int bk = blockIdx.x, b = bk / a.kv, hk = bk % a.kv;
    const bool wide = block < a.wide_blocks;
    const int splits = wide ? a.wide_splits : a.splits;
    if (splits == 1 || (int64_t)block * rows >= a.Lk) return;
    const int item = wide ? block * splits : a.wide_blocks * a.wide_splits + (block - a.wide_blocks) * splits;
    for (int e = (blockIdx.z * kBlock + threadIdx.x) * 4; e < 2 * rows * D; e += gridDim.z * kBlock * 4) {
        const int which = e / (rows * D), row = e / D % rows, d = e % D, j = block * rows + row;
        if (j >= a.Lk) continue;
        const float* src = a.part + ((int64_t)bk * a.cut + item) * 2 * rows * D + e;
        f32x4 x = *reinterpret_cast<const f32x4*>(src);
#pragma unroll 8
        for (int s = 1; s < splits; ++s) x += *reinterpret_cast<const f32x4*>(src + (int64_t)s * 2 * rows * D);
        store4<DT>((which ? a.dv : a.dk) + (((int64_t)b * a.Lk + j) * a.kv + hk) * I::ROW + d * I::EB, x);
    }
}

// ====================================================================================================================================
// host side
// ====================================================================================================================================
int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t reach(const ix_band* s) {   // rows on both sides that a band takes from a row's place
    const int64_t far = s->window > 0 ? s->window - 1 : (int64_t)s->Lq + s->Lk;
    return s->causal ? far : 2 * far;
}

// Owner rows: 64 or 128 a workgroup (one or two blocks of 16 for every wave).  Two blocks read LDS half as often for the same products, one
// gives twice as many workgroups and waves, and evens out the lengths of causal rows.  Measured, bf16 (us, one / two, by the number of
// workgroups of 128 rows): forward head dim 64, 64: 15 / 25, 272: 34 / 48, 800: 122 / 119 (12 755 rows) and, of 800-row sequences, 28 / 33;
// head dim 32, 576: 21 / 25, 1 024: 50 / 49, 800: 92 / 101 (12 755 rows); head dim 128, where LDS counts double, 64: 23 / 33, 256: 26 / 34
// causal and 33 / 35 not, 384: 39 / 51 causal but 72 / 68 not and 31 / 30 with a window, 448: 61 / 66, 111 / 92 and 35 / 35, 512: 66 / 68, 114 / 96
// and 38 / 35, 2 048: 392 / 331.  Gradients (with the forward) head dim 64, 192: 44 / 48, 576: 68 / 75, 1 152: 162 / 161, 1 600: 444 / 427; head
// dim 128 only one (two take the registers of a second wave).  f32 has room for one.
int fwd_nb(const ix_band* s) {
    if (s->dtype == 0) return 1;
    const int few = s->hd < 128 ? 600 : s->causal && s->window == 0 ? 512 : 384;
    return (int64_t)s->batch * s->heads * div_up(s->Lq, 128) < few ? 1 : 2;
}
int bwd_nb(const ix_band* s) {
    if (s->dtype == 0 || s->hd == 128) return 1;
    return (int64_t)s->batch * (s->heads * div_up(s->Lq, 128) + s->kv_heads * div_up(s->Lk, 128)) < 600 ? 1 : 2;
}

// Pieces of the forward's key tiles: where the blocks of queries are fewer than two a compute unit, about 512 in all, up to 32 of a block and
// at least four tiles each (eight where more than half of the units have a block: the join costs 4 to 5 us).  One piece / these: bf16, 40
// queries of 16 heads of 128 over 6 000 keys 119 / 21 us, 6 000 of 2 heads of 64 83 / 42, 3 000 of 4 heads 44 / 27, 4 x 512 of 8 heads of 128
// over 8 192 keys 160 / 123; fp16, 8 192 of 2 heads of 128 153 / 113; f32, 4 096 of 4 heads of 64 185 / 145.  No gain: sixteen tiles (2 060 of 8
// heads of 64) 31.4 / 30.6.  About 768 pieces: 88 us for the 8 192 of 2 heads, but 128 for the 4 x 512.  Blocks of 128 rows, of which a compute
// unit holds half as many, stay whole (384 of them with 1 536 keys of hd 128 54 / 57).
int fwd_splits(const ix_band* s) {
    const int64_t groups = (int64_t)s->batch * s->heads * div_up(s->Lq, owner_rows(fwd_nb(s)));
    if (groups >= 512 || fwd_nb(s) == 2) return 1;
    const int tb = key_tile(s->dtype);
    const int64_t all = div_up(s->Lk, tb), some = div_up(reach(s) + 64, tb) + 1 + div_up(s->sinks, tb), tiles = some < all ? some : all;
    const int64_t most = tiles / (groups > 128 ? 8 : 4);
    int64_t r = div_up(512, groups);
    if (r > most) r = most;
    return (int)(r < 2 ? 1 : r > 32 ? 32 : r);
}
size_t fwd_part(const ix_band* s) {   // partial rows
    const int r = fwd_splits(s);
    return r == 1 ? 0 : (size_t)s->batch * s->heads * s->Lq * r;
}

struct KeyPlan { int blocks, wide, wide_splits, splits, items, cut; };   // cut: how many of the items leave partial sums (they come first)

// Pieces of every block in the backward pass, of `wgs` blocks (of keys for dk / dv, of queries for dq) that stream `tiles` tiles of `tb` rows.
// Fewer blocks than compute units (few heads, or few key heads): about 384 pieces, no more than one for every four tiles begun (five tiles
// may become a piece of two and one of three).  Fewer than two a unit: two pieces of at least 1 536 rows.  Forward and gradients, us: uncut /
// with 256 / 384 / 512 pieces, f32, 2 x 2 041 of 2 heads of 64 207 / 178 / 141 / 136, 6 000 of one head of 128 933 / 556 / 413 / 429; bf16, the same
// 73 / 60 / 57 / 52 and 272 / 135 / 113 / 113, 40 queries of 16 heads over 6 000 keys of 4 of 128 167 / 63 / 60 / 60.  256 to 511 blocks, one piece /
// two: 8 192 of 2 heads of 128 459 / 329, 4 096 of 4 heads of 64 in f32 621 / 457, 4 x 512 of 8 heads over 8 192 keys 572 / 495; shorter rows stay
// whole: of 12 heads of 2 060, window 800, 59 / 66, though of 8 heads in full 85 / 76.
int64_t bwd_pieces(int64_t wgs, int64_t tiles, int tb) {
    int64_t r = wgs < 256 ? div_up(384, wgs) : wgs < 512 ? 2 : 1;
    const int64_t most = wgs < 256 ? div_up(tiles, 4) : tiles * tb / 1536;
    if (r > most) r = most;
    return r < 1 ? 1 : r;
}

// Splits of dk / dv.  A block of keys streams the queries of its band; a block with some of the first `sinks` keys streams all of them, and
// where these are more than two and a half times the others' it would run on alone: it is cut into pieces of up to twice the others'
// length.
KeyPlan key_plan(const ix_band* s) {
    KeyPlan r;
    const int rows = owner_rows(bwd_nb(s)), group = s->heads / s->kv_heads, tb = query_tile(s->dtype, s->hd);
    r.blocks = (int)div_up(s->Lk, rows);
    r.wide = s->sinks > 0 ? (s->sinks < s->Lk ? (int)div_up(s->sinks, rows) : r.blocks) : 0;
    const int64_t all = div_up(s->Lq, tb), band = div_up(reach(s) + rows, tb) + 1, each = (band < all ? band : all) * group;
    const int64_t wgs = (int64_t)s->batch * s->kv_heads * r.blocks;
    r.splits = (int)bwd_pieces(wgs, each, tb);
    const int64_t piece = div_up(each, r.splits);
    int64_t ws = 2 * all * group <= 5 * piece ? 1 : div_up(all * group, 2 * piece);
    const int64_t wide = (int64_t)s->batch * s->kv_heads * r.wide;
    if (wide && ws > div_up(1024, wide)) ws = div_up(1024, wide);   // (many such blocks fill the compute units by themselves)
    if (ws < r.splits) ws = r.splits;
    r.wide_splits = (int)(ws > 64 ? 64 : ws);
    r.items = r.wide * r.wide_splits + (r.blocks - r.wide) * r.splits;
    r.cut = r.splits > 1 ? r.items : r.wide_splits > 1 ? r.wide * r.wide_splits : 0;
    return r;
}

int dq_splits(const ix_band* s) {
    const int rows = owner_rows(bwd_nb(s)), tb = key_tile(s->dtype);
    const int64_t all = div_up(s->Lk, tb), some = div_up(reach(s) + rows, tb) + 1 + div_up(s->sinks, tb);
    const int64_t r = bwd_pieces((int64_t)s->batch * s->heads * div_up(s->Lq, rows), some < all ? some : all, tb);
    return (int)(r > 32 ? 32 : r);
}
size_t dq_part_bytes(const ix_band* s) {
    const int r = dq_splits(s), rows = owner_rows(bwd_nb(s));
    return r == 1 ? 0 : (size_t)s->batch * s->heads * div_up(s->Lq, rows) * r * rows * s->hd * 4;
}

size_t part_bytes(const ix_band* s, const KeyPlan& r) { return (size_t)s->batch * s->kv_heads * r.cut * 2 * owner_rows(bwd_nb(s)) * s->hd * 4; }

int64_t lse_pitch(const ix_band* s) { return ((int64_t)s->Lq + 127) / 128 * 128; }

int band_of(BandArgs& a, const ix_band* s, const char* who) {
    IX_CHECK_ARG(s, "%s: null description", who);
    IX_CHECK_ARG(s->dtype >= 0 && s->dtype <= 2, "%s: dtype %d is none of 0 (f32), 1 (bf16), 2 (fp16)", who, s->dtype);
    IX_CHECK_ARG(s->hd == 32 || s->hd == 64 || s->hd == 128, "%s: head dim %d is none of 32, 64, 128", who, s->hd);
    IX_CHECK_ARG(s->batch > 0 && s->Lq > 0 && s->Lk > 0 && s->Lq <= 65535 * 64 && s->Lk <= 65535 * 64, "%s: bad sizes (batch %d, %d queries, %d keys)", who,
                 s->batch, s->Lq, s->Lk);
    IX_CHECK_ARG(s->heads > 0 && s->kv_heads > 0 && s->heads % s->kv_heads == 0, "%s: %d query heads over %d key heads", who, s->heads, s->kv_heads);
    IX_CHECK_ARG((int64_t)s->batch * s->heads < kMostGroups, "%s: too many heads", who);
    IX_CHECK_ARG(s->window >= 0 && s->sinks >= 0, "%s: negative window or sinks", who);
    IX_CHECK_ARG(seq_scale_ok(s->scale), "%s: the scale is no number, or too large", who);
    IX_CHECK_ARG(s->q && s->k && s->v && ix_al16(s->q) && ix_al16(s->k) && ix_al16(s->v), "%s: null or unaligned q, k or v", who);
    const int64_t eb = s->dtype == 0 ? 4 : 2;
    for (int64_t x : {s->q_sb, s->q_sl, s->q_sh, s->k_sb, s->k_sl, s->k_sh, s->v_sb, s->v_sl, s->v_sh})
        IX_CHECK_ARG(x * eb % 16 == 0, "%s: rows that do not start on 16 bytes", who);
    for (int64_t x : {s->q_sl, s->k_sl, s->v_sl}) IX_CHECK_ARG(x >= 0 && x * eb < (1 << 24), "%s: rows 2^24 bytes apart or more", who);
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

template <int DT, int D> void launch_fwd(const BandArgs& a, int nb, dim3 grid, hipStream_t stream) {
    if constexpr (DT == 0) band_fwd_kernel<DT, D, 1><<<grid, kBlock, 0, stream>>>(a);
    else if (nb == 1) band_fwd_kernel<DT, D, 1><<<grid, kBlock, 0, stream>>>(a);
    else band_fwd_kernel<DT, D, 2><<<grid, kBlock, 0, stream>>>(a);
}
template <int DT, int D> void launch_bwd(const BandArgs& a, int nb, unsigned groups, hipStream_t stream) {
    if constexpr (DT == 0) band_bwd_kernel<DT, D, 1><<<groups, kBlock, 0, stream>>>(a);
    else if constexpr (D == 128) band_bwd_kernel<DT, D, 1><<<groups, kBlock, 0, stream>>>(a);
    else if (nb == 1) band_bwd_kernel<DT, D, 1><<<groups, kBlock, 0, stream>>>(a);
    else band_bwd_kernel<DT, D, 2><<<groups, kBlock, 0, stream>>>(a);
}

}  // namespace

#define BAND_HD(CALL, DT) { if (s->hd == 32) { CALL(DT, 32); } else if (s->hd == 64) { CALL(DT, 64); } else { CALL(DT, 128); } }
#define BAND_GO(CALL) { if (s->dtype == 0) BAND_HD(CALL, 0) else if (s->dtype == 1) BAND_HD(CALL, 1) else BAND_HD(CALL, 2) }

extern "C" int ix_workspace_bytes_band_attn_fwd(const struct ix_band* s, size_t* out_host) {
    BandArgs a;
    if (int rc = band_of(a, s, "ix_workspace_bytes_band_attn_fwd")) return rc;
    IX_CHECK_ARG(out_host, "ix_workspace_bytes_band_attn_fwd: null output");
    *out_host = fwd_part(s) * (s->hd + 2) * 4;
    return IX_OK;
}

extern "C" int ix_band_attn_fwd(const struct ix_band* s, void* out, float* lse, void* rest, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    BandArgs a;
    if (int rc = band_of(a, s, "ix_band_attn_fwd")) return rc;
    IX_CHECK_ARG(out && ix_al16(out) && ix_al16(rest), "ix_band_attn_fwd: null or unaligned output");
    const size_t parts = fwd_part(s), need = parts * (s->hd + 2) * 4;
    if (need && (!workspace || workspace_bytes < need || !ix_al16(workspace))) {
        ix_set_error("ix_band_attn_fwd: workspace of %zu bytes (16-byte aligned), %zu needed", workspace ? workspace_bytes : (size_t)0, need);
        return IX_ERR_WORKSPACE;
    }
    a.out = static_cast<unsigned char*>(out);
    a.rest = s->dtype ? static_cast<unsigned char*>(rest) : nullptr;
    a.lse = lse;
    a.fwd_splits = fwd_splits(s);
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + parts * s->hd;
    const int nb = fwd_nb(s), rows = owner_rows(nb);
    const dim3 grid(a.B * a.H, (a.Lq + rows - 1) / rows, a.fwd_splits);
#define BAND_FWD(DT, D) launch_fwd<DT, D>(a, nb, grid, stream)
    BAND_GO(BAND_FWD)
    IX_CHECK_LAUNCH("ix_band_attn_fwd");
    if (a.fwd_splits > 1) {
        const unsigned groups = (unsigned)div_up((int64_t)a.B * a.H * a.Lp * (s->hd / 4), kBlock);
#define BAND_JOIN(DT, D) band_join_kernel<DT, D><<<groups, kBlock, 0, stream>>>(a)
        BAND_GO(BAND_JOIN)
        IX_CHECK_LAUNCH("ix_band_attn_fwd (join)");
    }
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
    *out_host = (size_t)a.B * a.H * a.Lp * 4 + part_bytes(s, key_plan(s)) + dq_part_bytes(s);
    return IX_OK;
}

extern "C" int ix_band_attn_bwd_some(const struct ix_band* s, int want, const void* out, const void* rest, const float* lse, const void* d_out, int64_t g_sb,
                                     int64_t g_sl, int64_t g_sh, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                     hipStream_t stream) {
    BandArgs a;
    if (int rc = band_of(a, s, "ix_band_attn_bwd")) return rc;
    IX_CHECK_ARG(want >= 1 && want <= 3, "ix_band_attn_bwd: want %d is none of 1 (dq), 2 (dk and dv), 3", want);
    const bool to_q = want & 1, to_k = want & 2;
    if (!to_q) dq = nullptr;
    if (!to_k) dk = dv = nullptr;
    const int64_t eb = s->dtype == 0 ? 4 : 2;
    IX_CHECK_ARG(out && (rest || s->dtype == 0) && lse && d_out && (dq || !to_q) && ((dk && dv) || !to_k), "ix_band_attn_bwd: null pointer");
    IX_CHECK_ARG(ix_al16(out) && ix_al16(rest) && ix_al16(d_out) && ix_al16(dq) && ix_al16(dk) && ix_al16(dv), "ix_band_attn_bwd: unaligned pointer");
    for (int64_t x : {g_sb, g_sl, g_sh}) IX_CHECK_ARG(x * eb % 16 == 0, "ix_band_attn_bwd: rows that do not start on 16 bytes");
    IX_CHECK_ARG(g_sl >= 0 && g_sl * eb < (1 << 24), "ix_band_attn_bwd: rows 2^24 bytes apart or more");
    const KeyPlan r = to_k ? key_plan(s) : KeyPlan{0, 0, 1, 1, 0, 0};   // (no blocks of keys: none of them cut)
    const size_t parts = part_bytes(s, r), parts_q = to_q ? dq_part_bytes(s) : 0, need = (size_t)a.B * a.H * a.Lp * 4 + parts + parts_q;
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
    a.part_q = a.part + parts / 4;
    a.q_splits = dq_splits(s);
    a.dq = static_cast<unsigned char*>(dq);
    a.dk = static_cast<unsigned char*>(dk);
    a.dv = static_cast<unsigned char*>(dv);
    a.wide_blocks = r.wide;
    a.wide_splits = r.wide_splits;
    a.splits = r.splits;
    a.cut = r.cut;
    const int nb = bwd_nb(s), rows = owner_rows(nb);
    const int64_t key_groups = (int64_t)a.B * a.kv * r.items, groups = key_groups + (to_q ? (int64_t)a.B * a.H * ((a.Lq + rows - 1) / rows) * a.q_splits : 0);
    const int64_t delta_groups = ((int64_t)a.B * a.H * a.Lp * (s->hd * eb / 16) + kBlock - 1) / kBlock;
    IX_CHECK_ARG(groups < kMostGroups && delta_groups < kMostGroups, "ix_band_attn_bwd: too many rows for one launch");
    a.key_groups = (int)key_groups;
#define BAND_DELTA(DT, D) band_delta_kernel<DT, D><<<(unsigned)delta_groups, kBlock, 0, stream>>>(a)
    BAND_GO(BAND_DELTA)
    IX_CHECK_LAUNCH("ix_band_attn_bwd (delta)");
#define BAND_BWD(DT, D) launch_bwd<DT, D>(a, nb, (unsigned)groups, stream)
    BAND_GO(BAND_BWD)
    IX_CHECK_LAUNCH("ix_band_attn_bwd");
    if (parts || parts_q) {
        const int k_blocks = r.splits > 1 ? r.blocks : parts ? r.wide : 0, q_blocks = parts_q ? (a.Lq + rows - 1) / rows : 0;   // (both under 65 536)
        const dim3 sgrid(a.B * (a.kv + (parts_q ? a.H : 0)), k_blocks > q_blocks ? k_blocks : q_blocks, 4);
#define BAND_SUM(DT, D) band_sum_kernel<DT, D><<<sgrid, kBlock, 0, stream>>>(a, rows)
        BAND_GO(BAND_SUM)
        IX_CHECK_LAUNCH("ix_band_attn_bwd (sum)");
    }
    return IX_OK;
}

extern "C" int ix_band_attn_bwd(const struct ix_band* s, const void* out, const void* rest, const float* lse, const void* d_out, int64_t g_sb, int64_t g_sl,
                                int64_t g_sh, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    return ix_band_attn_bwd_some(s, 3, out, rest, lse, d_out, g_sb, g_sl, g_sh, dq, dk, dv, workspace, workspace_bytes, stream);
}
