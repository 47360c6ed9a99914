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
    template <int TOKENS_DIV = 0>
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

constexpr int kScan = 256;  // sequences whose tile counts a CTA keeps

struct Share {
    long long start, end, per;
    int seq, kvh, block, i;
};

struct ShareSmem {
    long long tot[kScan], warp[32], rem;
    Share out;
};

// Tiles of sequence s per kv head, by a warp.
template <int T>
MB_DEV long long seq_tiles(const Args &a, int s, int tokens)
{
    Piece p;
    p.load(a, s, tokens);
    long long n = 0;
    for (int b = threadIdx.x & 31; b < p.blocks; b += 32) n += block_tiles<T>(a, p, b, tokens).n;
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}

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
        h.per = max((total + gridDim.x - 1) / gridDim.x, (long long)min_tiles);
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
            h.kvh = (int)(rem / n);
            rem -= h.kvh * n;
            Piece p;
            p.load(a, s, tokens);
            for (int b = 0;; b += 32) {
                const int x = b + lane < p.blocks ? block_tiles<T>(a, p, b + lane, tokens).n : 0;
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
        }
        if (lane == 0) sm.out = h;
    }
    __syncthreads();
    return sm.out.start < sm.out.end;
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

// ---- fp32 ------------------------------------------------------------------------------
// Products on the FMA units: 64 rows x 64 keys, 256 threads of 4 x 4 scores and 4 rows x
// dim / 16 outputs.
constexpr int kRows = 64, kKeys = 64, kThreads = 256;

template <int DP>
struct Smem32 {
    static constexpr int kRow = DP + 4;  // floats; 16 bytes on from line to line: no bank conflicts down a column
    static constexpr int kPRow = kKeys + 4;
    static constexpr int kTotal = (kRows + 2 * kKeys) * kRow * 4 + kRows * kPRow * 4;
};

template <typename T>
MB_DEV float4 load4(const T *p)
{
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float4 *>(p);
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const T *t = reinterpret_cast<const T *>(&u);
    return make_float4(to_f32(t[0]), to_f32(t[1]), to_f32(t[2]), to_f32(t[3]));
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) k_prefill(const __grid_constant__ Args a, int tokens, int min_tiles)
{
    using S = Smem32<DP>;
    extern __shared__ __align__(16) float sm[];
    float *sq = sm, *sk = sq + kRows * S::kRow, *sv = sk + kKeys * S::kRow, *sp = sv + kKeys * S::kRow;
    __shared__ ShareSmem share;
    __shared__ unsigned char s_bad[kRows];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, warp = tid >> 5;
    mb::as::griddep_launch();
    if (!find_share<kKeys, kThreads>(a, tokens, min_tiles, share)) {
        if (tid == 0) a.meta[blockIdx.x].c_end = -1;
        return;
    }
    const Share h = share.out;
    Units<kKeys> u;
    u.start(a, h, tokens);
    int i = h.i;
    for (long long left = h.end - h.start; left > 0;) {
        const int tok0 = u.block * tokens, ntok = min(tokens, u.p.nq - tok0), nrow = ntok * a.group;
        const int pa = u.p.pos(tok0), pb = pa + ntok - 1;
        const int first = i, stop = (int)min((long long)u.t.n, i + left);
        const int low = a.window ? pa - a.window + 1 : 0;
        __syncthreads();  // the last unit's tiles have been read
        for (int e = tid; e < kRows * (DP / 4); e += kThreads) {
            const int r = e / (DP / 4), c = e % (DP / 4);
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < nrow && c * 4 < a.d) {
                const int t = div(a.group_div, r), head = u.kvh * a.group + r - t * a.group;
                x = load4(reinterpret_cast<const T *>(a.q) + (u.p.q0 + tok0 + t) * a.q_row + head * a.q_head + c * 4);
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
        for (; i < stop; i++) {
            const int j0 = u.t.key(i);
            __syncthreads();  // the tile before has been used, the queries are there
            for (int e = tid; e < kKeys * (DP / 4); e += kThreads) {
                const int r = e / (DP / 4), c = e % (DP / 4), j = j0 + r;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
                if (c * 4 < a.d && j < u.p.len && (j < u.p.pre || (j >= low && j <= pb))) {
                    const int id = page_of(a, u.seq, j);
                    if (id >= 0) {
                        const long long at = id * a.ps + u.kvh * a.hs + (long long)(j - div(a.page, j) * a.page.d) * a.ts + c * 4;
                        x = load4(reinterpret_cast<const T *>(a.k) + at);
                        y = load4(reinterpret_cast<const T *>(a.v) + at);
                    }
                }
                *reinterpret_cast<float4 *>(sk + r * S::kRow + c * 4) = x;
                *reinterpret_cast<float4 *>(sv + r * S::kRow + c * 4) = y;
            }
            __syncthreads();
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
#pragma unroll
            for (int y = 0; y < 4; y++) {
                float mx = -INFINITY;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int j = j0 + tx + 16 * x;
                    s[y][x] = visible(j, rp[y], u.p.len, u.p.pre, a.window) ? score2(a, s[y][x], slope[y], rp[y], j) : -INFINITY;
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
            __syncwarp();  // a warp reads the rows that it wrote
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
        }
        left -= stop - first;
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
            const float inv = !whole ? 1.f : l[y] == 0.f ? 0.f : 1.f / l[y];
#pragma unroll
            for (int c = 0; c < DP / 16; c++) {
                acc[y][c] *= inv;
                bad |= !isfinite(acc[y][c]);
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
            if (r >= nrow) continue;
            const long long row = u.p.q0 + tok0 + t;
            if (whole && bad) {
                if (tx == 0) s_bad[r] = 1;
                continue;
            }
#pragma unroll
            for (int c = 0; c < DP / 64; c++) {
                const int at = tx * 4 + 64 * c;
                const float4 x = make_float4(acc[y][4 * c], acc[y][4 * c + 1], acc[y][4 * c + 2], acc[y][4 * c + 3]);
                if (!whole) *reinterpret_cast<float4 *>(part + (size_t)r * DP + at) = x;
                else if (at < a.d) store4(reinterpret_cast<T *>(a.out) + row * a.o_row + head * a.o_head + at, x);
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
                    const int t = div(a.group_div, r);
                    lone_row<T>(a, u.seq, pa + t, u.kvh * a.group + r - t * a.group, u.p.q0 + tok0 + t);
                }
        }
        if (left <= 0 && tid == 0) {
            Meta mt{};
            mt.c_end = -1;
            if (first == 0 && !whole) {
                mt.c_end = (int)((h.end - 1 + (u.t.n - stop)) / h.per);
                mt.row0 = u.p.q0 + tok0;
                mt.ntok = ntok;
                mt.head0 = u.kvh * a.group;
                mt.ng = a.group;
                mt.seq = u.seq;
                mt.pos0 = pa;
            }
            a.meta[blockIdx.x] = mt;
        }
        if (left > 0) u.next(a, tokens);
        i = 0;
    }
}

template <typename T, int DP>
int run(Args &a, int ctas, cudaStream_t s)
{
    const char *who = "mocha_kv_prefill";
    const int tokens = kRows / a.group;
    if (launch(who, k_prefill<T, DP>, dim3(ctas), kThreads, Smem32<DP>::kTotal, s, false, a, tokens, 2)) return 1;
    return launch(who, k_join<T, true>, dim3(ctas, 8), 32 * kJoinWarps, 0, s, true, a, kRows, DP);
}

}  // namespace

namespace kv {
size_t decode_workspace(int type, int group, int d);

static size_t prefill_workspace(int type, int d)
{
    (void)type;
    return meta_bytes(2 * mb::kSMs) + part_bytes(2 * mb::kSMs, kRows, padded_dim(d));
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

extern "C" int mocha_kv_prefill(const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, const mocha_kv_scores *scores,
                                int rows, const int *q_start, const mocha_kv_rows *q, const mocha_kv_rows *out,
                                float *lse, void *workspace, unsigned long long workspace_bytes, void *stream)
{
    const char *who = "mocha_kv_prefill";
    if (check_pages(who, pages) || check_seqs(who, seqs) || check_scores(who, pages, scores)) return 1;
    const int b = type_bytes(pages->type), d = pages->head_dim;
    if (rows < 0) return fail(who, "rows must not be negative");
    if (check_rows(who, "q", q, b, d, rows) || check_rows(who, "out", out, b, d, rows)) return 1;
    if (seqs->seqs && (!seqs->kv_len || !q_start)) return fail(who, "null kv_len or q_start");
    DeviceGuard guard;
    if (guard.enter(who, pages->device)) return 1;
    if (!seqs->seqs || !rows) return 0;
    Args a = make_args(pages, seqs, scores, q, out, lse);
    a.q_start = q_start;
    a.rows = rows;
    if (!workspace || !aligned(workspace) || workspace_bytes < kv::prefill_workspace(pages->type, d))
        return fail(who, "workspace missing, not 16-byte aligned or smaller than mocha_kv_workspace says");
    const int ctas = 2 * mb::kSMs;
    a.meta = static_cast<Meta *>(workspace);
    a.part = reinterpret_cast<float *>(static_cast<char *>(workspace) + meta_bytes(ctas));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool narrow = padded_dim(d) == 64;
    switch (pages->type) {
    case MOCHA_KV_F32: return narrow ? run<float, 64>(a, ctas, s) : run<float, 128>(a, ctas, s);
    case MOCHA_KV_F16: return narrow ? run<__half, 64>(a, ctas, s) : run<__half, 128>(a, ctas, s);
    default: return narrow ? run<__nv_bfloat16, 64>(a, ctas, s) : run<__nv_bfloat16, 128>(a, ctas, s);
    }
}
