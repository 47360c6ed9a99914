// mocha_kv_prefill: attention of ragged prompt pieces over a paged cache (mocha_kv.h).
//
// A unit is a block of a sequence's query rows with all the query heads of one kv head:
// row r of the unit is token r / group, head r % group, so the heads of a group share the
// key and value tiles and a short piece still fills a tile.  Its key tiles are shared out
// over the CTAs (kv_common.cuh).
#include "kv_common.cuh"

namespace {

using namespace kv;

// A sequence's rows and keys.
struct Piece {
    int q0, nq, len, pre, blocks;
    MB_DEV void load(const Args &a, int s, int tokens)
    {
        q0 = min(max(__ldg(a.q_start + s), 0), a.rows);
        nq = min(max(__ldg(a.q_start + s + 1), q0), a.rows) - q0;
        len = seq_len(a, s);
        pre = seq_prefix(a, s, len);
        blocks = (nq + tokens - 1) / tokens;
    }
    MB_DEV int pos(int token) const { return len - nq + token; }
};

template <int T>
MB_DEV Tiles<T> block_tiles(const Args &a, const Piece &s, int block, int tokens)
{
    Tiles<T> t;
    const int pa = s.pos(block * tokens);
    t.set(a, s.len, s.pre, pa, min(pa + tokens, s.len) - 1);
    return t;
}

constexpr int kScan = 256;  // sequences whose tile counts a CTA keeps; past them it walks one by one (512: 169 us for 50)

struct Share {
    long long start, end, per;
    int seq, kvh, block, i;
};

struct ShareSmem {
    long long tot[kScan], warp[32], rem;
    Share out;
};

// What a unit's end counts for in a share, in tiles: outputs, and the next unit's start.  With 0,
// 1 and 3 the prompt of 8192 takes 528, 493 and 467 us for 464, that of 1024 25.1, 24.6 and 24.9
// for 23.9; the pieces after long texts 42.8, 41.6 and 39.9 for 40.8; every option 222, 219 and
// 218 for 219.
constexpr int kUnitEnd = 2;

// Tiles of sequence s per kv head with its units' ends, by a warp.
template <int T>
MB_DEV long long seq_tiles(const Args &a, int s, int tokens)
{
    Piece p;
    p.load(a, s, tokens);
    long long n = 0;
    for (int b = threadIdx.x & 31; b < p.blocks; b += 32) n += block_tiles<T>(a, p, b, tokens).n + kUnitEnd;
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}

// A walk along the units of a CTA's share.
template <int T>
struct Units {
    int seq, kvh, block;
    Piece p;
    Tiles<T> t;
    MB_DEV void start(const Args &a, const Share &h, int tokens)
    {
        seq = h.seq;
        kvh = h.kvh;
        block = h.block;
        p.load(a, seq, tokens);
        t = block_tiles<T>(a, p, block, tokens);
    }
    MB_DEV void next(const Args &a, int tokens)
    {
        if (++block == p.blocks) {
            block = 0;
            if (++kvh == a.kv_heads) {
                kvh = 0;
                do {
                    seq++;
                    p.load(a, seq, tokens);
                } while (p.blocks == 0);
            }
        }
        t = block_tiles<T>(a, p, block, tokens);
    }
};

// This CTA's share; false when it has none.  Called by all threads.
template <int T, int THREADS>
MB_DEV bool find_share(const Args &a, int tokens, int min_tiles, ShareSmem &sm)
{
    constexpr int W = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long mine = 0;
    for (int s = warp; s < a.seqs; s += W) {
        const long long n = seq_tiles<T>(a, s, tokens);
        if (s < kScan && lane == 0) sm.tot[s] = n;
        mine += n;
    }
    if (lane == 0) sm.warp[warp] = mine;
    __syncthreads();
    if (warp == 0) {
        long long total = 0;
        for (int w = 0; w < W; w++) total += sm.warp[w];
        total *= a.kv_heads;
        Share h{};
        h.per = max(div64(total + gridDim.x - 1, gridDim.x), (long long)min_tiles);
        h.start = h.per * blockIdx.x;
        h.end = min(h.start + h.per, total);
        if (h.start < total) {
            long long at = 0, n;
            int s = 0;
            for (;; s++) {
                n = s < kScan ? sm.tot[s] : seq_tiles<T>(a, s, tokens);
                if (h.start < at + n * a.kv_heads) break;
                at += n * a.kv_heads;
            }
            h.seq = s;
            long long rem = h.start - at;
            h.kvh = (int)div64(rem, n);
            rem -= h.kvh * n;
            Piece p;
            p.load(a, s, tokens);
            for (int b = 0;; b += 32) {
                const int x = b + lane < p.blocks ? block_tiles<T>(a, p, b + lane, tokens).n + kUnitEnd : 0;
                int incl = x;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += y;
                }
                const unsigned in = __ballot_sync(0xffffffffu, rem < incl);
                if (in) {
                    const int f = __ffs(in) - 1;
                    h.block = b + f;
                    h.i = (int)rem - (__shfl_sync(0xffffffffu, incl, f) - __shfl_sync(0xffffffffu, x, f));
                    break;
                }
                rem -= __shfl_sync(0xffffffffu, incl, 31);
            }
            Units<T> u;
            u.start(a, h, tokens);
            if (h.i >= u.t.n) {  // within a unit's end: the next unit is the first
                h.start += u.t.n + kUnitEnd - h.i;
                if (h.start < h.end) {
                    u.next(a, tokens);
                    h.seq = u.seq;
                    h.kvh = u.kvh;
                    h.block = u.block;
                    h.i = 0;
                }
            }
        }
        if (lane == 0) sm.out = h;
    }
    __syncthreads();
    return sm.out.start < sm.out.end;
}

// ---- fp32 ------------------------------------------------------------------------------
// Products on the FMA units: 64 rows x 64 keys, 256 threads of 4 x 4 scores and 4 rows x
// dim / 16 outputs.  Bound by their operands' way out of shared memory, which four barriers a
// tile leave idle at times: the FMA units run at 28 %.  Five pieces of up to 70 tokens after up
// to 600: 31 us, of which 2 find the shares, 2.5 are the first keys' way, two tiles in line take 6
// to 8 each, the unit's end 1.6 and the join 5.
constexpr int kRows = 64, kKeys = 64, kThreads = 256;

template <int DP>
struct Smem32 {
    static constexpr int kRow = DP + 4;  // floats; 16 bytes on from line to line: no bank conflicts down a column
    static constexpr int kPRow = kKeys + 4;
    static constexpr int kTotal = (kRows + 2 * kKeys) * kRow * 4 + kRows * kPRow * 4;
    static constexpr int kCtas = DP == 64 ? 2 : 1;  // of an SM
};

template <int DP>
__global__ void __launch_bounds__(kThreads, Smem32<DP>::kCtas) k_prefill(const __grid_constant__ Args a, int tokens, int min_tiles)
{
    using S = Smem32<DP>;
    extern __shared__ __align__(16) float sm[];
    constexpr int kCopies = kKeys * (DP / 4) / kThreads;  // 16-byte copies of a thread for a tile
    float *sq = sm, *sk = sq + kRows * S::kRow, *sv = sk + kKeys * S::kRow, *sp = sv + kKeys * S::kRow;
    __shared__ ShareSmem share;
    __shared__ unsigned char s_bad[kRows];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, warp = tid >> 5;
    mb::as::griddep_launch();
    mb::as::griddep_wait();
    if (!find_share<kKeys, kThreads>(a, tokens, min_tiles, share)) {
        if (tid == 0) a.note[blockIdx.x] = make_int2(-1, 0);
        return;
    }
    const Share h = share.out;
    const bool extra = a.cap > 0.f || a.slopes;
    Units<kKeys> u;
    u.start(a, h, tokens);
    int i = h.i;
    for (long long left = h.end - h.start; left > 0;) {
        const int tok0 = u.block * tokens, ntok = min(tokens, u.p.nq - tok0), nrow = ntok * a.group;
        const int pa = u.p.pos(tok0), pb = pa + ntok - 1;
        const int first = i, stop = (int)min((long long)u.t.n, i + left);
        const int low = a.window ? pa - a.window + 1 : 0;
        for (int e = tid; e < kRows * (DP / 4); e += kThreads) {
            const int r = e / (DP / 4), c = e % (DP / 4);
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < nrow && c * 4 < a.d) {
                const int t = div(a.group_div, r), head = u.kvh * a.group + r - t * a.group;
                x = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(a.q) + (u.p.q0 + tok0 + t) * a.q_row + head * a.q_head + c * 4);
            }
            *reinterpret_cast<float4 *>(sq + r * S::kRow + c * 4) = x;
        }
        float m[4], l[4], slope[4], acc[4][DP / 16];
        int rp[4];
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const int r = ty + 16 * y, t = div(a.group_div, r);
            rp[y] = r < nrow ? pa + t : INT_MIN / 2;
            slope[y] = a.slopes && r < nrow ? a.slopes[u.kvh * a.group + r - t * a.group] : 0.f;
            m[y] = -INFINITY;
            l[y] = 0.f;
#pragma unroll
            for (int c = 0; c < DP / 16; c++) acc[y][c] = 0.f;
        }
        // keys and values on their way by asynchronous copies: the next keys while the weights
        // and outputs of a tile are made, its values while the next scores are
        auto offsets = [&](int j0, long long (&at)[kCopies]) {
#pragma unroll
            for (int y = 0; y < kCopies; y++) {
                const int j = j0 + (tid + kThreads * y) / (DP / 4);
                at[y] = -1;
                if (j < u.p.len && (j < u.p.pre || (j >= low && j <= pb))) {
                    const int id = page_of(a, u.seq, j);
                    if (id >= 0) at[y] = (id * a.ps + u.kvh * a.hs + (long long)(j - div(a.page, j) * a.page.d) * a.ts) * 4;
                }
            }
        };
        auto copy = [&](float *to, const char *from, const long long (&at)[kCopies]) {
#pragma unroll
            for (int y = 0; y < kCopies; y++) {
                const int e = tid + kThreads * y, r = e / (DP / 4), c = e % (DP / 4);
                const bool use = at[y] >= 0 && c * 4 < a.d;
                cp_async16(mb::as::smem_u32(to + r * S::kRow + c * 4), use ? from + at[y] + c * 16 : from, use);
            }
            cp_commit();
        };
        long long at[kCopies], at_next[kCopies];
        offsets(u.t.key(i), at);
        copy(sk, a.k, at);
        copy(sv, a.v, at);
        for (; i < stop; i++) {
            const int j0 = u.t.key(i);
            const bool more = i + 1 < stop;
            cp_wait<1>();
            __syncthreads();  // the keys and the queries are there
            float s[4][4];
#pragma unroll
            for (int y = 0; y < 4; y++)
#pragma unroll
                for (int x = 0; x < 4; x++) s[y][x] = 0.f;
#pragma unroll 4
            for (int c = 0; c < DP / 4; c++) {
                float4 q[4], k[4];
#pragma unroll
                for (int y = 0; y < 4; y++) q[y] = *reinterpret_cast<const float4 *>(sq + (ty + 16 * y) * S::kRow + c * 4);
#pragma unroll
                for (int x = 0; x < 4; x++) k[x] = *reinterpret_cast<const float4 *>(sk + (tx + 16 * x) * S::kRow + c * 4);
#pragma unroll
                for (int y = 0; y < 4; y++)
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        s[y][x] = fmaf(q[y].x, k[x].x, s[y][x]);
                        s[y][x] = fmaf(q[y].y, k[x].y, s[y][x]);
                        s[y][x] = fmaf(q[y].z, k[x].z, s[y][x]);
                        s[y][x] = fmaf(q[y].w, k[x].w, s[y][x]);
                    }
            }
            if (more) offsets(u.t.key(i + 1), at_next);
            __syncthreads();  // the keys have been read
            if (more) copy(sk, a.k, at_next);
            else cp_commit();
            const bool full = (j0 + kKeys <= min(pa + 1, u.p.len) && (a.window == 0 || pb - j0 < a.window)) || j0 + kKeys <= u.p.pre;
#pragma unroll
            for (int y = 0; y < 4; y++) {
                float mx = -INFINITY;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int j = j0 + tx + 16 * x;
                    s[y][x] = extra ? score2(a, s[y][x], slope[y], rp[y], j) : s[y][x] * a.scale * kLog2e;
                    if (!full && !visible(j, rp[y], u.p.len, u.p.pre, a.window)) s[y][x] = -INFINITY;
                    mx = fmaxf(mx, s[y][x]);
                }
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const float mn = fmaxf(m[y], mx), ms = mn == -INFINITY ? 0.f : mn, f = exp2f(m[y] - ms);
                m[y] = mn;
                l[y] *= f;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const float e = exp2f(s[y][x] - ms);
                    l[y] += e;
                    sp[(ty + 16 * y) * S::kPRow + tx + 16 * x] = e;
                }
#pragma unroll
                for (int c = 0; c < DP / 16; c++) acc[y][c] *= f;
            }
            cp_wait<1>();
            __syncthreads();  // the values are there, and the weights
#pragma unroll 4
            for (int k = 0; k < kKeys; k += 4) {
                float4 e[4];
#pragma unroll
                for (int y = 0; y < 4; y++) e[y] = *reinterpret_cast<const float4 *>(sp + (ty + 16 * y) * S::kPRow + k);
#pragma unroll
                for (int kk = 0; kk < 4; kk++)
#pragma unroll
                    for (int c = 0; c < DP / 64; c++) {
                        const float4 v = *reinterpret_cast<const float4 *>(sv + (k + kk) * S::kRow + tx * 4 + 64 * c);
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            const float w = kk == 0 ? e[y].x : kk == 1 ? e[y].y : kk == 2 ? e[y].z : e[y].w;
                            acc[y][4 * c] = fmaf(w, v.x, acc[y][4 * c]);
                            acc[y][4 * c + 1] = fmaf(w, v.y, acc[y][4 * c + 1]);
                            acc[y][4 * c + 2] = fmaf(w, v.z, acc[y][4 * c + 2]);
                            acc[y][4 * c + 3] = fmaf(w, v.w, acc[y][4 * c + 3]);
                        }
                    }
            }
            __syncthreads();  // the values have been read
            if (more) copy(sv, a.v, at_next);
            else cp_commit();
        }
        left -= stop - first + (stop == u.t.n ? kUnitEnd : 0);
        const bool whole = first == 0 && stop == u.t.n;
        float *part = a.part + ((size_t)blockIdx.x * 2 + (first == 0 ? 1 : 0)) * ((size_t)kRows * (DP + 2));
        if (tid < kRows) s_bad[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const int r = ty + 16 * y, t = div(a.group_div, r), head = u.kvh * a.group + r - t * a.group;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) l[y] += __shfl_xor_sync(0xffffffffu, l[y], o);
            bool bad = false;
            const float inv = !whole ? 1.f : 1.f / l[y];
#pragma unroll
            for (int c = 0; c < DP / 16; c++) {
                acc[y][c] = whole && l[y] == 0.f ? 0.f : acc[y][c] * inv;
                bad |= !isfinite(acc[y][c]);
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
            if (r >= nrow) continue;
            const long long row = u.p.q0 + tok0 + t;
            if (whole && bad && tx == 0) s_bad[r] = 1;
#pragma unroll
            for (int c = 0; c < DP / 64; c++) {
                const int at = tx * 4 + 64 * c;
                const float4 x = make_float4(acc[y][4 * c], acc[y][4 * c + 1], acc[y][4 * c + 2], acc[y][4 * c + 3]);
                if (!whole) *reinterpret_cast<float4 *>(part + (size_t)r * DP + at) = x;
                else if (at < a.d) store4(reinterpret_cast<float *>(a.out) + row * a.o_row + head * a.o_head + at, x);
            }
            if (tx == 0) {
                if (!whole) {
                    part[(size_t)kRows * DP + 2 * r] = m[y];
                    part[(size_t)kRows * DP + 2 * r + 1] = l[y];
                } else if (a.lse)
                    a.lse[row * a.heads + head] = l[y] == 0.f ? -INFINITY : (m[y] + log2f(l[y])) * kLn2;
            }
        }
        if (whole) {
            __syncthreads();
            for (int r = warp; r < nrow; r += kThreads / 32)
                if (s_bad[r]) {
                    const int t = div(a.group_div, r), head = u.kvh * a.group + r - t * a.group;
                    if (unseen_values<float, kKeys>(a, u.seq, pa + t, head, pa, pb))
                        lone_row<float>(a, u.seq, pa + t, head, u.p.q0 + tok0 + t);
                }
        }
        if (left <= 0 && tid == 0) {
            a.note[blockIdx.x] = make_int2(first == 0 && !whole ? (int)div64(h.end - 1 + (u.t.n - stop), h.per) : -1, nrow);
            a.meta[blockIdx.x] = Meta{u.p.q0 + tok0, u.kvh * a.group, a.group, u.seq, pa};
        }
        if (left > 0) u.next(a, tokens);
        i = 0;
    }
}


// ---- 16-bit types: the tensor cores ----------------------------------------------------
// One CTA per SM with two tiles of 128 query rows (a unit of one tile, as of a few tokens
// over a long cache, has its keys dealt to both in turn and the outputs added at its end:
// 4 tokens of 32 sequences over up to 4000 keys: 71 -> 62 us).  A warp copies queries, keys and
// values into shared memory by TMA (a page or a part of one per copy, 128-byte swizzle), one
// issues the products, and four per tile, a row per thread, turn scores into
// weights.  Scores S = Q K^T and outputs O += P V are accumulated in TMEM; P goes back to
// TMEM over the scores it came from and is the second product's first operand there.  While
// the warps of one tile work on its weights the tensor core has the other tile's products,
// so the products (4 * 128 * 128 * dim operations per tile and key tile) are the floor.  The
// two chains, products and weights, still wait for one another: at 8192 tokens the tensor pipe is
// busy for 57 % of the time and the exponential unit for 60 %.
//
// The maximum that a row's weights are taken from is renewed only when it is exceeded by
// 2^8, so outputs are rescaled a few times per row and not per tile.  Weights are rounded to 16
// bits once (kLift in kv_common.cuh has the reason), after their sums, which are fp32.
//
// Measured: a prompt of 8192, 32 heads of 128, causal: 465 us, 1.18 PFLOP/s; after a second of
// it the card is at its power limit and it takes 540.  A prompt of 1024, 14 heads of 64: 24 us, of
// which the products are 2: a start of 4 to 5 us, two to three tiles in line, and the join's 5.
// Two pieces of 16 tokens after 65,521, 134 MB: 41 us; the tiles come at memory's rate, the start
// and the ends of units are the rest.  Two threads per row (750 us) and a thread per tile for
// the products (650 us) were worse; exponentials on the FMA units, an eighth to a half of them,
// measured from 1 % better to 5 % worse.  With a cap or a bias the warps of weights, which then
// spill 36 to 48 bytes a thread, are what a step waits for: six prompts with every option, 212 us,
// have the tensor pipe busy for 21 % of the time, the exponential unit for 24 %, and 38 % of the
// issue slots used.
constexpr int kTcThreads = 384;  // warps 0-3 and 4-7: weights of the two tiles; 8: products; 9: copies; 10, 11: none
constexpr int kTcUnits = 4;      // units that the copies may be ahead
constexpr int kTcKeys = 128;
constexpr int kWaitPolls = 1 << 18;  // of 3.9 us each: a second

struct Maps {
    CUtensorMap q, k, v;
};

template <int DP>
struct SmemTc {
    static constexpr int kTile = 128 * DP * 2;           // bytes of a tile of 128 rows
    static constexpr int kStages = DP == 128 ? 5 : 10;   // key and value tiles in flight
    static constexpr int kTiles = (2 + kStages) * kTile;
};

// A unit as the warps see it: the copying warp walks along the share and passes units on.
struct TcUnit {
    int ntok;           // tokens of the unit; 0 after the last unit
    int row0, pos0;     // first token's row and position
    int kvh, seq, len, pre;
    int pre_t, lo_t;    // tiles, as in Tiles
    int first, stop, n; // tiles of this share, and of the unit
    MB_DEV int key(int i) const { return (i < pre_t ? i : i - pre_t + lo_t) * kTcKeys; }
    MB_DEV bool whole() const { return first == 0 && stop == n; }
    // one tile of rows: the tiles' warps take its key tiles in turn
    MB_DEV bool lone(int tok) const { return ntok <= tok; }
};

struct TcBars {
    uint64_t q_full[2], q_empty[2], s_full[2], p_full[2][2], o_full[2], kv_full[10], kv_empty[10], unit_full[kTcUnits],
        unit_empty[kTcUnits], pair_full, pair_done, edge, drain;
    TcUnit unit[kTcUnits];
    Share share;
    float2 pair[128];         // of a lone unit: the second tile's (m, l)
    uint32_t tmem;
    volatile int abort, bad;  // a wait ran out; an output is not finite
};

MB_DEV void tma_load_4d(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, int c3, uint64_t *bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(mb::as::smem_u32(bar))
        : "memory");
}

// Descriptor of a value tile as the second operand: its rows (keys) are the summed
// dimension, so the operand is "MN-major": 64 dims in a 128-byte row, `block` bytes on to the
// next 64 dims, 1024 bytes to the next 8 keys.
MB_DEV uint64_t mn_desc(uint32_t addr, int block)
{
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(block >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// D[tmem] (+)= A[tmem] * B[smem], issued by one thread.
MB_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, bool accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

// Waits for phase `parity` of `bar`; false when *abort is set (another role of the CTA gave
// up) or after the call's number of polls.  Polls and not cycles, for the clock runs on while
// another process has the GPU, and what is awaited does not.
MB_DEV bool wait_for(const Args &a, uint64_t *bar, uint32_t parity, const volatile int *abort)
{
    if (mb::as::mbar_test(bar, parity)) return true;
    for (int n = 0;;) {
        if (mb::as::mbar_test(bar, parity)) return true;
        if (*abort || ++n > a.wait_polls) return false;
    }
}

// The share of a CTA that gave up: its finished units' rows, and a note for the join.  Called
// by all threads.
template <int T, typename E>
MB_DEV void lost_share(const Args &a, const Share &h, int tokens)
{
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int2 note = make_int2(-1, -1);
    Units<T> u;
    u.start(a, h, tokens);
    int i = h.i;
    for (long long left = h.end - h.start; left > 0; i = 0) {
        const int tok0 = u.block * tokens, ntok = min(tokens, u.p.nq - tok0), stop = (int)min((long long)u.t.n, i + left);
        if (i == 0 && stop < u.t.n) {
            note = make_int2((int)div64(h.end - 1 + (u.t.n - stop), h.per), -1 - ntok * a.group);
            if (threadIdx.x == 0) a.meta[blockIdx.x] = Meta{u.p.q0 + tok0, u.kvh * a.group, a.group, u.seq, u.p.pos(tok0)};
        } else if (i == 0) {
            for (int r = warp; r < ntok * a.group; r += warps) {
                const int t = div(a.group_div, r);
                lost_row<E>(a, u.p.q0 + tok0 + t, u.kvh * a.group + r - t * a.group);
            }
        }
        left -= stop - i + (stop == u.t.n ? kUnitEnd : 0);
        if (left > 0) u.next(a, tokens);
    }
    if (threadIdx.x == 0) {
        a.note[blockIdx.x] = note;
        if (a.status) atomicMax(a.status, 2);
    }
}

MB_DEV bool elect_one()
{
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

#define KV_O8(x, i) "=f"(x[i]), "=f"(x[i + 1]), "=f"(x[i + 2]), "=f"(x[i + 3]), "=f"(x[i + 4]), "=f"(x[i + 5]), "=f"(x[i + 6]), "=f"(x[i + 7])
#define KV_F8(x, i) "f"(x[i]), "f"(x[i + 1]), "f"(x[i + 2]), "f"(x[i + 3]), "f"(x[i + 4]), "f"(x[i + 5]), "f"(x[i + 6]), "f"(x[i + 7])
#define KV_I8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])

// 32 TMEM columns of this thread's row, to x[I..I + 31].
template <int I, int N>
MB_DEV void tmem_ld32(uint32_t addr, float (&x)[N])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : KV_O8(x, I), KV_O8(x, I + 8), KV_O8(x, I + 16), KV_O8(x, I + 24)
        : "r"(addr));
}
// 16 TMEM columns.
MB_DEV void tmem_st16(uint32_t addr, const uint32_t (&x)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::KV_I8(x, 0),
                 KV_I8(x, 8), "r"(addr));
}
MB_DEV void tmem_ld16f(uint32_t addr, float (&x)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : KV_O8(x, 0), KV_O8(x, 8)
                 : "r"(addr));
}
MB_DEV void tmem_st16f(uint32_t addr, const float (&x)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::KV_F8(x, 0),
                 KV_F8(x, 8), "r"(addr));
}
MB_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Pairs of fp32 operations in one instruction, each rounded to nearest.
MB_DEV void fma2(float &d0, float &d1, float a0, float a1, float b0, float b1, float c0, float c1)
{
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
MB_DEV void add2(float &d0, float &d1, float a0, float a1)
{
    asm("{\n\t.reg .b64 a, d;\n\tmov.b64 d, {%0, %1};\n\tmov.b64 a, {%2, %3};\n\tadd.rn.f32x2 d, d, a;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "+f"(d0), "+f"(d1)
        : "f"(a0), "f"(a1));
}

// cap tanh(k s) + bias of a row of scores, bias = base - slope c for column c, where cap is in
// log2.  Where all of a warp's |k s| are within tanh_of's polynomial, as those of ordinary
// scores under an ordinary cap are, on the FMA units alone: its coefficients take up k and cap.
// The other way rounds such scores alike, bit by bit, for what the vote sees are also scores of
// keys that no row sees and that anything may lie in.  Rows that do not exist have no say.
MB_DEV void cap_scores(float (&s)[128], float cap, float k, float slope, float base, bool there)
{
    float big = 0.f;
#pragma unroll
    for (int c = 0; c < 128; c += 2) big = fmaxf(big, fmaxf(fabsf(s[c]), fabsf(s[c + 1])));
    const float kk = k * k;
    float c0 = kTanh0 * cap * k, c1 = kTanh1 * cap * k * kk, c2 = kTanh2 * cap * k * kk * kk,
          c3 = kTanh3 * cap * k * kk * kk * kk, c4 = kTanh4 * cap * k * kk * kk * kk * kk;
    // the coefficients and the scores' squares have to be normal numbers: c4 within these bounds
    // holds |k| between 2^-18 and 2^17.  Elsewhere the polynomial takes k s.
    const bool normal = fabsf(c4) >= 0x1p-120f && fabsf(c4) <= 0x1p100f;
    if (!normal || __any_sync(0xffffffffu, there && big * fabsf(k) > kTanhPart)) {
        const float f = normal ? 1.f : k;
        if (!normal) c0 = kTanh0 * cap, c1 = kTanh1 * cap, c2 = kTanh2 * cap, c3 = kTanh3 * cap, c4 = kTanh4 * cap;
#pragma unroll
        for (int c = 0; c < 128; c++) {
            const float x = s[c] * k, a = s[c] * f, t = fmaf(a, a, 0.f), bias = fmaf(-slope, (float)c, base);
            const float y = fmaf(fmaf(fmaf(fmaf(c4, t, c3), t, c2), t, c1), t, c0);
            s[c] = fabsf(x) <= kTanhPart ? fmaf(a, y, bias) : fmaf(cap, tanh_large(x), bias);
        }
    } else {
#pragma unroll
        for (int c = 0; c < 128; c += 2) {
            float t0, t1, y0, y1;
            fma2(t0, t1, s[c], s[c + 1], s[c], s[c + 1], 0.f, 0.f);
            fma2(y0, y1, t0, t1, c4, c4, c3, c3);
            fma2(y0, y1, y0, y1, t0, t1, c2, c2);
            fma2(y0, y1, y0, y1, t0, t1, c1, c1);
            fma2(y0, y1, y0, y1, t0, t1, c0, c0);
            fma2(s[c], s[c + 1], s[c], s[c + 1], y0, y1, fmaf(-slope, (float)c, base), fmaf(-slope, (float)(c + 1), base));
        }
    }
}

// The n lowest bits.
MB_DEV uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; }

// Four lanes with four units of eight words each (their rows' next 128 bytes) exchange them:
// lane q of the four then holds unit q of the four rows, so that a store writes whole lines.
MB_DEV void exchange4(uint32_t (&r)[32])
{
    const int q = threadIdx.x & 3;
#pragma unroll
    for (int step = 1; step <= 2; step <<= 1) {
        const bool up = q & step;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (u & step) continue;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                uint32_t &lo = r[8 * u + e], &hi = r[8 * (u + step) + e];
                const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, step);
                if (up) lo = got;
                else hi = got;
            }
        }
    }
}

template <typename T, int DP, bool EXTRA>
__global__ void __launch_bounds__(kTcThreads, 1)
    k_prefill_tc(const __grid_constant__ Args a, const __grid_constant__ Maps maps, int tok, int box, int min_tiles)
{
    using namespace mb::as;
    using S = SmemTc<DP>;
    extern __shared__ __align__(1024) unsigned char smem[];
    TcBars &bar = *reinterpret_cast<TcBars *>(smem + S::kTiles);
    ShareSmem &share = *reinterpret_cast<ShareSmem *>(smem);  // before the tiles
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tokens = 2 * tok;
    griddep_launch();
    if (tid == 32) {
        prefetch_map(&maps.q);
        prefetch_map(&maps.k);
        prefetch_map(&maps.v);
    }
    if (tid == 0) {
        for (int x = 0; x < 2; x++) {
            mbar_init(&bar.q_full[x], 1);
            mbar_init(&bar.q_empty[x], 1);
            mbar_init(&bar.s_full[x], 1);
            mbar_init(&bar.p_full[x][0], 128);
            mbar_init(&bar.p_full[x][1], 128);
            mbar_init(&bar.o_full[x], 1);
        }
        for (int i = 0; i < S::kStages; i++) {
            mbar_init(&bar.kv_full[i], 1);
            mbar_init(&bar.kv_empty[i], 1);
        }
        for (int i = 0; i < kTcUnits; i++) {
            mbar_init(&bar.unit_full[i], 1);
            mbar_init(&bar.unit_empty[i], 9);  // eight warps of weights and the thread of products
        }
        mbar_init(&bar.pair_full, 128);
        mbar_init(&bar.pair_done, 128);
        mbar_init(&bar.edge, 1);
        mbar_init(&bar.drain, 1);
        bar.abort = bar.bad = 0;
        fence_barrier_init();
    }
    griddep_wait();
    // swizzled tiles are laid out by address: their base has to be a multiple of 1024
    const bool any = find_share<kTcKeys, kTcThreads>(a, tokens, min_tiles, share), placed = (smem_u32(smem) & 1023) == 0;
    if (!any || !placed) {
        if (any) lost_share<kTcKeys, T>(a, share.out, tokens);
        else if (tid == 0) a.note[blockIdx.x] = make_int2(-1, 0);
        return;
    }
    if (tid == 0) bar.share = share.out;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // queries are copied to where the search kept its sums
    if (warp == 8) tmem_alloc(&bar.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar.tmem;
    const uint32_t sq = smem_u32(smem), skv = sq + 2 * S::kTile;
    bool ok = true;

    // 12 warps of 168 registers at launch: 128 threads of 88 and 256 of 208 fit in those
    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 9) {
        // copies
        Units<kTcKeys> u;
        u.start(a, bar.share, tokens);
        int i = bar.share.i, it = 0, edges = 0, units = 0, asked[2] = {0, 0};
        long long left = bar.share.end - bar.share.start;
        // together, for lanes that part here meet the warp's next barrier apart
        auto wait = [&](uint64_t *b, uint32_t parity) { return ok = __all_sync(0xffffffffu, wait_for(a, b, parity, &bar.abort)); };
        for (;; units++) {
            const bool more = left > 0;
            const int stop = more ? (int)min((long long)u.t.n, i + left) : 0, begin = i;
            const int tok0 = u.block * tokens, ntok = min(tokens, u.p.nq - tok0), pa = u.p.pos(tok0), pb = pa + ntok - 1;
            if (!wait(&bar.unit_empty[units % kTcUnits], ((units / kTcUnits) & 1) ^ 1)) break;
            if (lane == 0) {
                TcUnit &d = bar.unit[units % kTcUnits];
                d.ntok = more ? ntok : 0;
                d.row0 = u.p.q0 + tok0;
                d.pos0 = pa;
                d.kvh = u.kvh;
                d.seq = u.seq;
                d.len = u.p.len;
                d.pre = u.p.pre;
                d.pre_t = u.t.pre_t;
                d.lo_t = u.t.lo_t;
                d.first = i;
                d.stop = stop;
                d.n = u.t.n;
                mbar_arrive(&bar.unit_full[units % kTcUnits]);
            }
            if (!more) break;
            left -= stop - i + (stop == u.t.n ? kUnitEnd : 0);
            // lane b has the page of the tile's keys b * box ..; the next tile's is asked for a tile ahead
            auto page_at = [&](int tile) {
                const int j = u.t.key(tile) + lane * box;
                return tile < stop && lane * box < kTcKeys && j < u.p.len ? __ldg(a.table + u.seq * a.table_stride + div(a.page, j)) : 0;
            };
            int id = page_at(i);
            for (; i < stop && ok; i++) {
                const int j0 = u.t.key(i), j = j0 + lane * box;
                const int keys = min(kTcKeys, u.p.len - j0);           // keys there are (not positive: none)
                const int boxes = keys > 0 ? (keys + box - 1) / box : 0;
                const bool edge = keys < kTcKeys;
                const int row = lane < boxes ? j - (int)(div(a.page, j) * a.page.d) : 0;
                const int id_next = page_at(i + 1);
                if (lane < boxes && (unsigned)id >= (unsigned)a.pages && a.status) {
                    bool seen = false;
                    for (int y = 0; y < box && j + y < u.p.len; y++)
                        seen |= (j + y <= pb && (a.window == 0 || pa - (j + y) < a.window)) || j + y < u.p.pre;
                    if (seen) atomicMax(a.status, 1);
                }
                for (int v = 0; v < 2 && ok; v++, it++) {
                    const int st = it % S::kStages;
                    if (!wait(&bar.kv_empty[st], ((it / S::kStages) & 1) ^ 1)) break;
                    if (v && a.drop && it / 2 == blockIdx.x % a.drop) continue;
                    const uint32_t dst = skv + st * S::kTile;
                    uint64_t *full = v && edge ? &bar.edge : &bar.kv_full[st];
                    if (lane == 0) mbar_expect_tx(full, (uint32_t)(boxes * box * DP * 2));
                    __syncwarp();
                    if (lane < boxes)
                        for (int c = 0; c < DP / 64; c++)
                            tma_load_4d(dst + c * (128 * 128) + lane * box * 128, v ? &maps.v : &maps.k, 64 * c, row, u.kvh, id, full);
                    if (!v && i == begin) {
                        // the queries, behind the first keys: once the unit before no longer reads its own
                        for (int x = 0; x < 2 && x * tok < ntok; x++) {
                            if (!wait(&bar.q_empty[x], (asked[x]++ & 1) ^ 1)) break;
                            if (lane == 0) {
                                mbar_expect_tx(&bar.q_full[x], (uint32_t)(DP * 2 * tok * a.group));
                                for (int b = 0; b < DP / 64; b++)
                                    tma_load_4d(sq + x * S::kTile + b * (128 * 128), &maps.q, 64 * b, 0, u.kvh, u.p.q0 + tok0 + x * tok, &bar.q_full[x]);
                            }
                        }
                    }
                    if (v && edge) {
                        // rows past the sequence's end hold anything: 0 * NaN must not reach the sums
                        if (!wait(&bar.edge, edges++ & 1)) break;
                        const int r0 = max(keys, 0);
                        for (int e = lane; e < (128 - r0) * (DP / 8); e += 32) {
                            const int r = r0 + e / (DP / 8), c = e % (DP / 8);
                            *reinterpret_cast<uint4 *>(smem + 2 * S::kTile + st * S::kTile + (c / 8) * (128 * 128) + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.kv_full[st]);
                    }
                }
                id = id_next;
            }
            if (!ok) break;
            if (left > 0) u.next(a, tokens);
            i = 0;
        }
        if (!ok) bar.abort = 1;
    } else if (warp == 8) {
        // products: the warp goes along together, one elected lane issues
        constexpr int fmt = std::is_same<T, __half>::value ? 0 : 1;
        constexpr uint32_t base = (1u << 4) | (fmt << 7) | (fmt << 10) | (8u << 24);
        constexpr uint32_t id_qk = base | ((128u >> 3) << 17), id_pv = base | (1u << 16) | ((uint32_t)(DP >> 3) << 17);
        int it = 0, steps[2] = {0, 0}, asked[2] = {0, 0};  // steps: weights taken; asked: queries taken
        auto wait = [&](uint64_t *b, uint32_t parity) {
            ok = ok && __all_sync(0xffffffffu, wait_for(a, b, parity, &bar.abort));
            tc_fence_after();
            return ok;
        };
        auto full = [&](int n) { return wait(&bar.kv_full[n % S::kStages], (n / S::kStages) & 1); };
        // keys of stage st; last: the unit's last keys for these queries; both: the stage is done with
        auto qk = [&](int x, int st, bool lone, bool last, bool both) {
            const uint64_t q = sw128_desc(sq + (lone ? 0 : x * S::kTile)), k = sw128_desc(skv + st * S::kTile);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; kk++) {
                    const uint32_t off = ((kk / 4) * (128 * 128) + (kk % 4) * 32) >> 4;
                    mma_bf16(tmem + x * 128, q + off, k + off, id_qk, kk > 0);
                }
                mma_commit(&bar.s_full[x]);
                if (last) mma_commit(&bar.q_empty[lone ? 0 : x]);
                if (both) mma_commit(&bar.kv_empty[st]);
            }
            __syncwarp();
        };
        // weights of tile x with the values of stage st; the first 64 keys' are used while the others' are made
        auto pv = [&](int x, int st, bool accumulate, bool both) {
            const uint64_t v = mn_desc(skv + st * S::kTile, 128 * 128);
            const uint32_t step = steps[x]++ & 1;
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                if (!wait(&bar.p_full[x][hf], step)) return false;
                if (elect_one()) {
#pragma unroll
                    for (int kk = 4 * hf; kk < 4 * hf + 4; kk++)
                        mma_ts(tmem + 256 + x * 128, tmem + x * 128 + kk * 8, v + (kk * 2048 >> 4), id_pv, accumulate || kk > 0);
                    if (hf) mma_commit(&bar.o_full[x]);
                    if (hf && both) mma_commit(&bar.kv_empty[st]);
                }
                __syncwarp();
            }
            return true;
        };
        for (int units = 0; wait(&bar.unit_full[units % kTcUnits], (units / kTcUnits) & 1); units++) {
            const TcUnit &d = bar.unit[units % kTcUnits];
            const int n = d.stop - d.first, tiles = d.ntok > tok ? 2 : 1;
            const bool done = d.ntok == 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.unit_empty[units % kTcUnits]);
            if (done || !full(it)) break;
            if (tiles == 1) {
                // key tile j is tile j % 2's: K 0, K 1, then V j and K j + 2 in turn
                if (!wait(&bar.q_full[0], asked[0]++ & 1)) break;
                qk(0, it % S::kStages, true, n == 1, true);
                if (n > 1) {
                    if (!full(it + 2)) break;
                    qk(1, (it + 2) % S::kStages, true, n == 2, true);
                }
                for (int j = 0; j < n; j++, it += 2) {
                    if (!full(it + 1) || !pv(j & 1, (it + 1) % S::kStages, j > 1, true)) break;
                    if (j + 2 < n) {
                        if (!full(it + 4)) break;
                        qk(j & 1, (it + 4) % S::kStages, true, j + 3 == n, true);
                    }
                }
                continue;
            }
            for (int x = 0; x < 2 && wait(&bar.q_full[x], asked[x]++ & 1); x++) qk(x, it % S::kStages, false, n == 1, x == 1);
            for (int j = 0; j < n && ok; j++, it += 2) {
                // copies are ahead: asked for before the weights, they hold nothing up after
                if (!full(it + 1) || (j + 1 < n && !full(it + 2))) break;
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    if (!pv(x, (it + 1) % S::kStages, j > 0, x == 1)) break;
                    if (j + 1 < n) qk(x, (it + 2) % S::kStages, false, j + 2 == n, x == 1);
                }
            }
        }
        if (!ok) bar.abort = 1;
        if (elect_one()) mma_commit(&bar.drain);
        int never = 0;
        mbar_wait(&bar.drain, 0, &never);
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // weights: thread = row of tile x
        const int x = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t ts = tmem + x * 128 + ((uint32_t)((warp & 3) * 32) << 16), to = ts + 256;
        const float k2 = EXTRA ? 1.f : a.scale * kLog2e;
        uint32_t step = 0, pairs = 0;
        // false when a wait has run out, here or elsewhere in the CTA
        auto wait = [&](uint64_t *b, uint32_t parity) {
            ok = __all_sync(0xffffffffu, wait_for(a, b, parity, &bar.abort));
            tc_fence_after();
            return ok;
        };
        for (int units = 0; wait(&bar.unit_full[units % kTcUnits], (units / kTcUnits) & 1); units++) {
            const TcUnit &d = bar.unit[units % kTcUnits];
            if (d.ntok == 0) break;
            const bool lone = d.lone(tok);
            const int xt = lone ? 0 : x * tok;  // first token of this tile's rows
            if (lone ? x < d.stop - d.first : xt < d.ntok) {
                const int t = div(a.group_div, r);
                float m = -INFINITY, l = 0.f;
                {
                    const int p0 = d.pos0 + xt, p1 = p0 + min(tok, d.ntok - xt) - 1, p = p0 + t, pre = d.pre;
                    const int hi = min(p + 1, d.len), lo = a.window ? max(p - a.window + 1, 0) : 0;
                    const int full_hi = min(p0 + 1, d.len) - kTcKeys, full_lo = a.window ? p1 - a.window + 1 : 0;
                    const int first = d.first + (lone ? x : 0), stop = d.stop, stride = lone ? 2 : 1;
                    const float slope = EXTRA && a.slopes && t < tok ? -kLog2e * __ldg(a.slopes + d.kvh * a.group + r - t * a.group) : 0.f;
                    for (int i = first; i < stop; i += stride, step++) {
                        const int j0 = d.key(i);
                        const bool full = (j0 <= full_hi && j0 >= full_lo) || j0 + kTcKeys <= pre;
                        if (!wait(&bar.s_full[x], step & 1)) break;
                        float s[128];
                        tmem_ld32<0>(ts, s);
                        tmem_ld32<32>(ts + 32, s);
                        tmem_ld32<64>(ts + 64, s);
                        tmem_ld32<96>(ts + 96, s);
                        tmem_wait_ld();
                        if (EXTRA) {
                            // the cap, the bias by distance, and to powers of two.  No key is after
                            // the row but in a prefix; there the distance changes its sign.
                            const bool ahead = a.slopes && j0 < pre && j0 + kTcKeys > p0 + 1;
                            const float by = ahead ? 0.f : slope, base = by * (float)(p - j0);
                            if (a.cap > 0.f) {
                                cap_scores(s, a.cap * kLog2e, a.scale / a.cap, by, base, t < tok && xt + t < d.ntok);
                            } else {
#pragma unroll
                                for (int c = 0; c < 128; c++) s[c] = fmaf(s[c], a.scale * kLog2e, fmaf(-by, (float)c, base));
                            }
                            if (ahead) {
#pragma unroll
                                for (int c = 0; c < 128; c++) s[c] = fmaf(slope, fabsf((float)(p - j0) - c), s[c]);
                            }
                        }
                        if (!full) {
#pragma unroll
                            for (int b = 0; b < 4; b++) {
                                const int j = j0 + 32 * b;
                                const uint32_t vis = (low_bits(hi - j) & ~low_bits(lo - j)) | low_bits(pre - j);
#pragma unroll
                                for (int c = 0; c < 32; c++)
                                    if (!(vis >> c & 1)) s[32 * b + c] = -INFINITY;
                            }
                        }
                        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 0; c < 128; c += 2) mx[(c / 2) & 3] = fmaxf(mx[(c / 2) & 3], fmaxf(s[c], s[c + 1]));
                        const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                        // a new maximum, and the output so far to its scale
                        const bool grown = (mn - m) * k2 > 8.f;
                        if (__any_sync(0xffffffffu, grown)) {
                            const float f = grown ? ex2((m - mn) * k2) : 1.f;
                            if (grown) m = mn;
                            l *= f;
                            if (i > first) {
                                if (!wait(&bar.o_full[x], (step & 1) ^ 1)) break;
#pragma unroll
                                for (int c = 0; c < DP; c += 16) {
                                    float o[16];
                                    tmem_ld16f(to + c, o);
                                    tmem_wait_ld();
#pragma unroll
                                    for (int e = 0; e < 16; e++) o[e] *= f;
                                    tmem_st16f(to + c, o);
                                }
                            }
                        }
                        const float sub = m == -INFINITY ? 0.f : fmaf(-m, k2, kLift<T>);
                        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int b = 0; b < 4; b++) {
                            uint32_t w[16];  // over scores that have been read
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                float e0, e1;
                                fma2(e0, e1, s[32 * b + 2 * e], s[32 * b + 2 * e + 1], k2, k2, sub, sub);
                                e0 = ex2(e0);
                                e1 = ex2(e1);
                                add2(sum[(2 * e) & 3], sum[(2 * e + 1) & 3], e0, e1);
                                w[e] = pack2<T>(e0, e1);
                            }
                            tmem_st16(ts + 16 * b, w);
                            if (b & 1) {
                                tmem_wait_st();
                                tc_fence_before();
                                mbar_arrive(&bar.p_full[x][b / 2]);
                            }
                        }
                        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    }
                }
                if (!ok || !wait(&bar.o_full[x], (step & 1) ^ 1)) break;
                // a lone unit's outputs: both tiles' rows are the same, the first's warps add them
                float fa = 1.f, fb = 0.f;
                const bool two = lone && d.stop - d.first > 1;
                if (two) {
                    if (x == 1) {
                        bar.pair[r] = make_float2(m, l);
                        tc_fence_before();
                        mbar_arrive(&bar.pair_full);
                        if (!wait(&bar.pair_done, pairs++ & 1)) break;  // the outputs have been read
                    } else {
                        if (!wait(&bar.pair_full, pairs++ & 1)) break;
                        const float2 other = bar.pair[r];
                        const float mm = fmaxf(m, other.x), ms = mm == -INFINITY ? 0.f : mm;
                        fa = ex2((m - ms) * k2);
                        fb = ex2((other.x - ms) * k2);
                        l = l * fa + other.y * fb;
                        m = mm;
                    }
                }
                const bool mine = t < tok && xt + t < d.ntok && !(lone && x), whole = d.whole();
                const int g = r - t * a.group, head = d.kvh * a.group + g;
                const int at = (xt + t) * a.group + g;
                const long long row = d.row0 + xt + t;
                float *part = a.part + ((size_t)blockIdx.x * 2 + (d.first == 0 ? 1 : 0)) * ((size_t)256 * (DP + 2));
                const bool none = whole && l == 0.f;  // has seen nothing, or scores of -infinity alone
                const float inv = !whole ? 1.f : 1.f / l;
                bool bad = false;
                // 128 bytes of a row at a time; the four lanes of a quad write their rows' lines together
                unsigned char *base = whole ? reinterpret_cast<unsigned char *>(a.out) + (row * a.o_row + head * a.o_head) * 2
                                            : reinterpret_cast<unsigned char *>(part + (size_t)at * DP);
                const unsigned ours = __ballot_sync(0xffffffffu, mine);
#pragma unroll 1
                for (int line = 0; line < (lone && x ? 0 : whole ? DP / 64 : DP / 32); line++) {
                    uint32_t w[32];
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float o[32];
                        const int col = whole ? 64 * line + 32 * c : 32 * line;
                        tmem_ld32<0>(to + col, o);
                        tmem_wait_ld();
                        if (two) {
                            float o2[32];
                            tmem_ld32<0>(to + 128 + col, o2);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = fmaf(o2[e], fb, o[e] * fa);
                        }
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            o[e] = none ? 0.f : o[e] * inv;
                            bad |= !isfinite(o[e]);
                        }
                        if (whole) {
#pragma unroll
                            for (int e = 0; e < 16; e++) w[16 * c + e] = pack2<T>(o[2 * e], o[2 * e + 1]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; e++) w[e] = __float_as_uint(o[e]);
                            break;
                        }
                    }
                    exchange4(w);
                    const int byte = line * 128 + (lane & 3) * 32;
#pragma unroll
                    for (int f = 0; f < 4; f++) {
                        const int from = (lane & ~3) + f;
                        unsigned char *dst = reinterpret_cast<unsigned char *>(__shfl_sync(0xffffffffu, (unsigned long long)base, from)) + byte;
                        if ((ours >> from & 1) && (!whole || byte < a.d * 2)) {
                            *reinterpret_cast<uint4 *>(dst) = make_uint4(w[8 * f], w[8 * f + 1], w[8 * f + 2], w[8 * f + 3]);
                            *reinterpret_cast<uint4 *>(dst + 16) = make_uint4(w[8 * f + 4], w[8 * f + 5], w[8 * f + 6], w[8 * f + 7]);
                        }
                    }
                }
                if (mine) {
                    if (!whole) {
                        part[(size_t)256 * DP + 2 * at] = m == -INFINITY ? m : fmaf(m, k2, -kLift<T>);
                        part[(size_t)256 * DP + 2 * at + 1] = l;
                    } else {
                        if (a.lse) a.lse[row * a.heads + head] = none ? -INFINITY : ((m == -INFINITY ? 0.f : fmaf(m, k2, -kLift<T>)) + log2f(l)) * kLn2;
                        if (bad) bar.bad = 1;
                    }
                }
                tc_fence_before();
                if (two && x == 0) mbar_arrive(&bar.pair_done);
            }
            if (tid == 0) {
                // the share's last unit leaves the last note
                const bool cut = d.first == 0 && d.stop < d.n;
                a.note[blockIdx.x] = make_int2(cut ? (int)div64(bar.share.end - 1 + (d.n - d.stop), bar.share.per) : -1, d.ntok * a.group);
                a.meta[blockIdx.x] = Meta{d.row0, d.kvh * a.group, a.group, d.seq, d.pos0};
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.unit_empty[units % kTcUnits]);
        }
        if (!ok) bar.abort = 1;
    }
    __syncthreads();
    if (bar.abort) {
        // a wait ran out: the copies in flight land first
        if (tid == 0) {
            const long long t0 = clock64();
            while (clock64() - t0 < kWaitCycles / 64) {
            }
        }
        __syncthreads();
    }
    if (warp == 8) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
    if (bar.abort) {
        lost_share<kTcKeys, T>(a, bar.share, tokens);
        return;
    }
    if (!bar.bad) return;
    // rows of whole units that are not finite, once more without the keys that they do not see
    Units<kTcKeys> u;
    u.start(a, bar.share, tokens);
    int i = bar.share.i;
    for (long long left = bar.share.end - bar.share.start; left > 0; i = 0) {
        const int tok0 = u.block * tokens, ntok = min(tokens, u.p.nq - tok0);
        if (i == 0 && left >= u.t.n)
            for (int r = warp; r < ntok * a.group; r += kTcThreads / 32) {
                const int t = div(a.group_div, r), head = u.kvh * a.group + r - t * a.group, row = u.p.q0 + tok0 + t;
                const T *o = reinterpret_cast<const T *>(a.out) + row * a.o_row + head * a.o_head;
                bool bad = false;
                for (int e = lane; e < a.d; e += 32) bad |= !isfinite(to_f32(o[e]));
                const int p0 = u.p.pos(tok0);
                if (__any_sync(0xffffffffu, bad) && unseen_values<T, kTcKeys>(a, u.seq, p0 + t, head, p0, p0 + ntok - 1))
                    lone_row<T>(a, u.seq, p0 + t, head, row);
            }
        left -= u.t.n - i + kUnitEnd;
        if (left > 0) u.next(a, tokens);
    }
}

template <int DP>
int run(Args &a, void *space, int device, cudaStream_t s)
{
    const char *who = "mocha_kv_prefill";
    const int tokens = kRows / a.group, ctas = mb::kSMs * Smem32<DP>::kCtas;
    lay_out(a, space, ctas);
    static std::atomic<unsigned long long> allowed{0};
    if (allow_smem(who, k_prefill<DP>, Smem32<DP>::kTotal, device, allowed) ||
        launch(who, k_prefill<DP>, dim3(ctas), kThreads, Smem32<DP>::kTotal, s, a, tokens, 1))
        return 1;
    return launch(who, k_join<float, true>, dim3(kJoinBlocks), 32 * kJoinWarps, 0, s, a, ctas, kRows, DP);
}

// ---- tensor maps -----------------------------------------------------------------------

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                             const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn()
{
    static const EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return (EncodeFn)p;
    }();
    return fn;
}

// A map of [n3][n2][n1][dim] 16-bit values with byte strides s1..s3 and a box of 64 x b1 x 1 x b3;
// what lies past an extent reads as zeros.
int encode(CUtensorMap *map, int type, const void *base, const long long (&n)[4], const long long (&s)[3], int b1, int b3)
{
    const cuuint64_t dims[4] = {(cuuint64_t)n[0], (cuuint64_t)n[1], (cuuint64_t)n[2], (cuuint64_t)n[3]};
    cuuint64_t strides[3];
    for (int i = 0; i < 3; i++) strides[i] = n[i + 1] > 1 ? (cuuint64_t)s[i] : 16;  // of one line: any valid one
    const cuuint32_t box[4] = {64, (cuuint32_t)b1, 1, (cuuint32_t)b3}, one[4] = {1, 1, 1, 1};
    const EncodeFn fn = encode_fn();
    return fn && fn(map, type == MOCHA_KV_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                    const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
int run_tc(Args &a, const mocha_kv_pages *p, void *space, int device, cudaStream_t s)
{
    const char *who = "mocha_kv_prefill";
    const int tok = 128 / a.group, d = a.d;
    int box = 128;
    while (p->page_size % box) box /= 2;
    Maps maps;
    if (!encode(&maps.q, p->type, a.q, {d, a.group, a.kv_heads, a.rows}, {a.q_head * 2, a.q_head * 2 * a.group, a.q_row * 2}, a.group, tok) ||
        !encode(&maps.k, p->type, a.k, {d, p->page_size, a.kv_heads, a.pages}, {a.ts * 2, a.hs * 2, a.ps * 2}, box, 1) ||
        !encode(&maps.v, p->type, a.v, {d, p->page_size, a.kv_heads, a.pages}, {a.ts * 2, a.hs * 2, a.ps * 2}, box, 1))
        return fail(who, "the tensor maps cannot be encoded");
    constexpr int ctas = mb::kSMs;
    lay_out(a, space, ctas);
    const auto go = [&](auto kernel, std::atomic<unsigned long long> &allowed) {
        constexpr size_t smem = SmemTc<DP>::kTiles + sizeof(TcBars);
        return allow_smem(who, kernel, smem, device, allowed) || launch(who, kernel, dim3(ctas), kTcThreads, smem, s, a, maps, tok, box, 2);
    };
    static std::atomic<unsigned long long> allowed[2] = {};
    if (a.cap > 0.f || a.slopes || !(a.scale > 0.f) ? go(k_prefill_tc<T, DP, true>, allowed[1]) : go(k_prefill_tc<T, DP, false>, allowed[0])) return 1;
    return launch(who, k_join<T, true>, dim3(kJoinBlocks), 32 * kJoinWarps, 0, s, a, ctas, 256, DP);
}

}  // namespace

namespace kv {
size_t decode_workspace(int type, int group, int d);

static size_t prefill_workspace(int type, int d)
{
    const int dp = padded_dim(d), f32 = type == MOCHA_KV_F32, n = mb::kSMs * (!f32 ? 1 : dp == 64 ? Smem32<64>::kCtas : Smem32<128>::kCtas);
    return meta_bytes(n) + part_bytes(n, f32 ? kRows : 256, dp);
}
}  // namespace kv

extern "C" int mocha_kv_workspace(const mocha_kv_pages *pages, int heads, int prefill, unsigned long long *bytes)
{
    const char *who = "mocha_kv_workspace";
    if (check_pages(who, pages)) return 1;
    if (!bytes) return fail(who, "null bytes");
    if (heads < 1 || heads % pages->kv_heads || heads / pages->kv_heads > kMaxGroup)
        return fail(who, "heads must be a multiple of kv_heads, at most 64 times as many");
    *bytes = prefill ? kv::prefill_workspace(pages->type, pages->head_dim)
                     : kv::decode_workspace(pages->type, heads / pages->kv_heads, pages->head_dim);
    return 0;
}

namespace {

int prefill(const char *who, const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, const mocha_kv_scores *scores, int rows,
            const int *q_start, const mocha_kv_rows *q, const mocha_kv_rows *out, float *lse, void *workspace,
            unsigned long long workspace_bytes, void *stream, int wait_polls, int drop)
{
    if (check_pages(who, pages) || check_seqs(who, seqs) || check_scores(who, pages, scores)) return 1;
    const int b = type_bytes(pages->type), d = pages->head_dim;
    if (rows < 0 || rows > kMostPositions) return fail(who, "rows must not be negative, nor more than 2^30");
    if (check_rows(who, "q", q, b, d, rows) || check_rows(who, "out", out, b, d, rows)) return 1;
    if (seqs->seqs && (!seqs->kv_len || !q_start)) return fail(who, "null kv_len or q_start");
    DeviceGuard guard;
    if (guard.enter(who, pages->device)) return 1;
    if (!seqs->seqs || !rows) return 0;
    Args a = make_args(pages, seqs, scores, q, out, lse);
    a.q_start = q_start;
    a.rows = rows;
    a.wait_polls = wait_polls;
    a.drop = drop;
    if (!workspace || !aligned(workspace) || workspace_bytes < kv::prefill_workspace(pages->type, d))
        return fail(who, "workspace missing, not 16-byte aligned or smaller than mocha_kv_workspace says");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int dev = guard.device();
    const bool narrow = padded_dim(d) == 64;
    switch (pages->type) {
    case MOCHA_KV_F32: return narrow ? run<64>(a, workspace, dev, s) : run<128>(a, workspace, dev, s);
    case MOCHA_KV_F16: return narrow ? run_tc<__half, 64>(a, pages, workspace, dev, s) : run_tc<__half, 128>(a, pages, workspace, dev, s);
    default: return narrow ? run_tc<__nv_bfloat16, 64>(a, pages, workspace, dev, s) : run_tc<__nv_bfloat16, 128>(a, pages, workspace, dev, s);
    }
}

}  // namespace

extern "C" int mocha_kv_prefill(const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, const mocha_kv_scores *scores,
                                int rows, const int *q_start, const mocha_kv_rows *q, const mocha_kv_rows *out,
                                float *lse, void *workspace, unsigned long long workspace_bytes, void *stream)
{
    return prefill("mocha_kv_prefill", pages, seqs, scores, rows, q_start, q, out, lse, workspace, workspace_bytes, stream,
                   kWaitPolls, 0);
}

extern "C" int mocha_kv_prefill_check(const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, const mocha_kv_scores *scores,
                                      int rows, const int *q_start, const mocha_kv_rows *q, const mocha_kv_rows *out,
                                      float *lse, void *workspace, unsigned long long workspace_bytes, void *stream,
                                      int wait_polls, int drop)
{
    const char *who = "mocha_kv_prefill_check";
    if (wait_polls < 0 || drop < 0) return fail(who, "wait_polls and drop must not be negative");
    return prefill(who, pages, seqs, scores, rows, q_start, q, out, lse, workspace, workspace_bytes, stream, wait_polls, drop);
}
