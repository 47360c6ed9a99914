// mocha_kv_decode: attention of one new token per sequence over a paged cache (mocha_kv.h).
//
// Each cached value is used by heads / kv heads queries only (4 flops per element and
// head), so the kernel is bound by reading the visible keys and values once.  A unit is a
// sequence and one kv head with up to 8 NG of its query heads; its key tiles are shared out
// over the CTAs (kv_common.cuh).  The four warps of a CTA take a quarter of every tile's
// keys each and run on their own: each keeps a ring of tiles in flight in its own part of
// shared memory (16-byte asynchronous copies, which also fill the rows of keys that are not
// visible with zeros, so nothing of them can reach a sum), and softmax statistics and an
// output in registers; they meet when a unit ends.
//
// 16-bit types: scores are K q^T and outputs V^T p^T by m16n8k16 products, so the heads of
// the group are the narrow side of 8 and no lane computes on padding when a group has 8.
// For the second product a weight is the sum of two values of the cache's type, so that it
// keeps twice its bits: the outputs are off by their own rounding alone, where weights of one
// value each added up to 40 % to the error.  Memory bounds the kernel up to groups of 8, whose
// time grows by 1 % (64 and 128 sequences) or 2 % (windows); 16 heads a kv head take 5 % longer,
// 32 and 64 take 7 to 11 %.  fp32: the same tiles on the FMA units, a lane holding half a key's
// products with 8 heads.  Either way the value that weights are taken from is renewed only
// when a score passes it by 2^8, which a vote finds: no shuffles and no rescaling on most
// tiles.
//
// Measured: 128 sequences up to 8192 long, 8 kv heads of 128, 2.41 GB: 380 us, 6.3 TB/s, with
// the card at its power limit; two of 40,001 and 131,071, 0.18 GB: 37 us, 4.8 TB/s; 64 up to
// 2047 of 64 dims, 0.14 GB: 32 us, 4.5 TB/s, of which some 9 us are the start (lengths, pages,
// first keys) and the join.  One sequence of 777 in fp32: 10.4 us, all of it latency.  A
// prefetch of the next tile into L2 cost 10 % at the power limit; halves of a tile as copy
// groups of their own changed nothing.
#include "kv_common.cuh"

namespace {

using namespace kv;

// CTAs of an SM, warps of a CTA, keys of a warp's tile, and the stages of its ring (keys
// then values): 192 KB of rings and eight warps per SM, three stages of 8 KB a warp, so
// that two are in flight while one is computed.  16-bit: two CTAs of four warps overlap
// one's unit ends with the other's tiles (wide groups, for their registers, leave room for
// one, with longer rings); fp32: one of eight, as the FMA units need the warps at once.
// A unit has H query heads at most: 8 NG, or 4 for NG = 0 (fp32 alone).
template <typename T, int DP, int NG>
struct Ring {
    static constexpr bool kF32 = sizeof(T) == 4;
    static constexpr int kWarps = kF32 ? 8 : 4, kThreads = 32 * kWarps;
    static constexpr int kH = NG ? 8 * NG : 4, kHB = kF32 ? 4 : 8;  // heads; heads met at a time
    static constexpr int kKeys = (kF32 ? 1024 : 2048) / DP, kTile = kWarps * kKeys;
    static constexpr int kHalf = kKeys * DP * (int)sizeof(T), kStage = 2 * kHalf;
    static constexpr int kCtas = kF32 || NG > 1 ? 1 : 2;
    static constexpr int kStages = 192 * 1024 / kCtas / kWarps / kStage;
    static constexpr int kRings = kWarps * kStages * kStage;
    static constexpr int kPad = DP + 4;  // floats of a head's row in the merge buffers
    static constexpr int kMerge = kWarps * kHB * kPad * 4;
    static constexpr int kStat = kWarps * kH * 8;                   // (m, l)
    static constexpr int kQ = kF32 ? kH * DP * 4 : 0;              // fp32: the unit's queries,
    static constexpr int kW = kF32 ? kWarps * kH * kKeys * 4 : 0;  // and a tile's weights
    static constexpr int kShare = 8 * (kWarps + 2);
    static constexpr int kTotal = kRings + kMerge + kStat + kQ + kW + kShare;
};

struct Work {
    Args a;
    int hgroups, unit_heads;  // units per kv head, and query heads of a unit (the last may have fewer)
    int min_tiles;            // of a share
    bool one_page;            // a warp's keys of a tile lie in one page
};

// What a unit's end counts for in a share, in tiles: the warps' meeting and the next unit's
// start.  Without it the CTAs with the shortest sequences were last (64 sequences up to
// 2047: 39.3 us for 32.1; windows 45.2 for 37.5).  2 is the same for 16-bit pages and worse for
// 64 fp32 sequences (33.5 for 31.1).
constexpr int kUnitEnd = 1;

// A walk along a CTA's tiles; j is the tile's first key.
template <int TILE>
struct Walk {
    int seq, hh, i, j;
    int len, pre, lo;  // lo: first key of the window
    Tiles<TILE> t;
    MB_DEV void load(const Args &a)
    {
        len = pre = 0;
        if (seq < a.seqs) {
            len = seq_len(a, seq);
            pre = seq_prefix(a, seq, len);
        }
        lo = a.window ? max(len - a.window, 0) : 0;
        t.set(a, len, pre, len - 1, len - 1);
    }
    MB_DEV void at(int tile)
    {
        i = tile;
        j = t.key(tile);
    }
    // On to the next tile; returns what the tile left behind counts for in a share.
    MB_DEV int next(const Args &a, int hh_n)
    {
        if (++i < t.n) {
            j = i == t.pre_t ? t.lo_t * TILE : j + TILE;
            return 1;
        }
        if (++hh == hh_n) {
            hh = 0;
            seq++;
            load(a);
        }
        at(0);
        return 1 + kUnitEnd;
    }
    // whether all of n keys from k on are visible; whether key k is
    MB_DEV bool all_visible(int k, int n) const { return k + n <= len && (k >= lo || k + n <= pre); }
    MB_DEV bool sees(int k) const { return k < len && (k >= lo || k < pre); }
};

MB_DEV void ldsm4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
MB_DEV void ldsm4_t(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
MB_DEV uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <typename T>
MB_DEV void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A weight as the sum of two values: what its leading bits hold, and the rest.  The rest is
// at least 2^-16 of the weight, so that neither is zero or negative and an infinite value that
// a row sees stays infinite (fp16: under weights down to 2^-15 of the largest).
template <typename T>
MB_DEV uint32_t cut2(float x, float y)
{
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value)
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    else
        asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
MB_DEV float rest(float x, float cut) { return fmaxf(x - cut, x * 0x1p-16f); }

// The share of this CTA: its first tile as (sequence, tile within the sequence) in *s_seq
// and *s_rem, and [start, end) in tiles of the whole call.
template <int TILE, int kWarps>
MB_DEV bool find_share(const Work &w, int hh_n, long long *s_warp, int *s_seq, long long *s_rem, long long *start,
                       long long *end, long long *per)
{
    const Args &a = w.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kThreads = 32 * kWarps;
    const int chunk = (a.seqs + kThreads - 1) / kThreads, b0 = min(tid * chunk, a.seqs), b1 = min(b0 + chunk, a.seqs);
    Walk<TILE> k;
    long long sum = 0;
    for (k.seq = b0; k.seq < b1; k.seq++) {
        k.load(a);
        sum += (long long)(k.t.n + kUnitEnd) * hh_n;
    }
    long long incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; i++) {
        if (i < warp) incl += s_warp[i];
        total += s_warp[i];
    }
    *per = max(div64(total + gridDim.x - 1, gridDim.x), (long long)w.min_tiles);
    *start = *per * blockIdx.x;
    *end = min(*start + *per, total);
    long long at = incl - sum;
    if (*start < total && at <= *start && *start < incl) {
        for (k.seq = b0;; k.seq++) {
            k.load(a);
            const long long n = (long long)(k.t.n + kUnitEnd) * hh_n;
            if (*start < at + n) break;
            at += n;
        }
        *s_seq = k.seq;
        *s_rem = *start - at;
    }
    __syncthreads();
    return *start < total;
}

template <typename T, int DP, int NG>
__global__ void __launch_bounds__(Ring<T, DP, NG>::kThreads, Ring<T, DP, NG>::kCtas) k_decode(const __grid_constant__ Work w)
{
    using R = Ring<T, DP, NG>;
    constexpr bool F32 = R::kF32;
    constexpr int KEYS = R::kKeys, H = R::kH, HB = R::kHB, kWarps = R::kWarps, kThreads = R::kThreads;
    constexpr int CH = DP * (int)sizeof(T) / 16;     // 16-byte pieces of a row
    constexpr int RPI = 32 / CH;                     // rows of a warp's copy
    constexpr int GROUPS = KEYS / 8;                 // of 8 keys, which lie in one page
    constexpr int ROW = DP * (int)sizeof(T);
    constexpr int NM = F32 ? H : 2 * NG, NACC = F32 ? H : NG * DP / 16;
    constexpr int PARTS = 32 / KEYS;                 // fp32: lanes that share a key's products
    // All shared memory is dynamic, so that the rings start on a 128-byte line: behind 48 bytes of
    // static variables each copy of a line was four requests to L2 and twice its bytes (442 us
    // for 128 sequences that take 382).
    extern __shared__ __align__(128) unsigned char smem[];
    float *merge = reinterpret_cast<float *>(smem + R::kRings);
    float2 *stat = reinterpret_cast<float2 *>(smem + R::kRings + R::kMerge);
    float *sq = reinterpret_cast<float *>(smem + R::kRings + R::kMerge + R::kStat);
    float *sw = sq + R::kQ / 4;
    long long *s_warp = reinterpret_cast<long long *>(sw + R::kW / 4), &s_rem = s_warp[kWarps];
    int &s_seq = *reinterpret_cast<int *>(s_warp + kWarps + 1);
    const Args &a = w.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int hh_n = a.kv_heads * w.hgroups;
    mb::as::griddep_launch();
    mb::as::griddep_wait();
    long long start, end, per;
    if (!find_share<R::kTile, kWarps>(w, hh_n, s_warp, &s_seq, &s_rem, &start, &end, &per)) {
        if (tid == 0) a.note[blockIdx.x] = make_int2(-1, 0);
        return;
    }
    Walk<R::kTile> in;  // the next tile to load
    in.seq = s_seq;
    in.load(a);
    in.hh = (int)div64(s_rem, in.t.n + kUnitEnd);
    in.at((int)(s_rem - (long long)in.hh * (in.t.n + kUnitEnd)));
    int left = (int)(end - start);  // of the share, from tile `it` on
    if (in.i >= in.t.n) {           // within a unit's end: the next unit is the first
        left -= in.t.n + kUnitEnd - in.i;
        in.i = in.t.n - 1;
        in.next(a, hh_n);
    }
    if (left <= 0) {
        if (tid == 0) a.note[blockIdx.x] = make_int2(-1, 0);
        return;
    }
    int left_in = left;  // from tile `in` on
    Walk<R::kTile> it = in;  // the tile to compute
    const uint32_t wring = mb::as::smem_u32(smem) + warp * R::kStages * R::kStage;

    // a lane copies piece c of rows r0, r0 + RPI, ...; pieces of a row are spread by its
    // number so that eight rows' equal pieces lie in different banks
    const int r0 = lane / CH, c = lane % CH;
    const bool dims = c * 16 < a.d * (int)sizeof(T);
    const char *k_lane0 = a.k + (r0 * a.ts + c * (16 / (int)sizeof(T))) * (long long)sizeof(T);
    const long long row_step = RPI * a.ts * (long long)sizeof(T), v_off = a.v - a.k;
    uint32_t to_lane[8 / RPI];
#pragma unroll
    for (int y = 0; y < 8 / RPI; y++) to_lane[y] = wring + (r0 + RPI * y) * ROW + ((c ^ r0 ^ (RPI * y)) & (CH - 1)) * 16;

    // pages of the groups of this warp's keys of tile `in`; one when pages hold whole tiles
    int pages[GROUPS];
    auto look_up = [&](const Walk<R::kTile> &at, int (&to)[GROUPS]) {
        const int j = at.j + warp * KEYS;
        const int *row = a.table + at.seq * a.table_stride;
#pragma unroll
        for (int g = 0; g < GROUPS; g++)
            if (g == 0 || !w.one_page) to[g] = j + 8 * g < at.len ? __ldg(row + div(a.page, j + 8 * g)) : 0;
    };
    auto issue = [&](uint32_t slot) {
        const int j = in.j + warp * KEYS;
        const int kvh = w.hgroups == 1 ? in.hh : in.hh / w.hgroups;
        const bool full = in.all_visible(j, KEYS);
        long long head = kvh * a.hs;
        const char *from = nullptr;
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            const int jg = j + 8 * g;
            bool good = true;
            if (g == 0 || !w.one_page) {
                const int id = pages[g];
                good = (unsigned)id < (unsigned)a.pages;
                const int row = jg - (int)(div(a.page, jg) * a.page.d);
                from = k_lane0 + (id * a.ps + head + row * a.ts) * (long long)sizeof(T);
            }
            if (w.one_page) good = (unsigned)pages[0] < (unsigned)a.pages;
            const uint32_t group = slot + g * 8 * ROW;
            if (full && good && dims) {
#pragma unroll
                for (int y = 0; y < 8 / RPI; y++, from += row_step) {
                    cp_async16(group + to_lane[y], from);
                    cp_async16(group + to_lane[y] + R::kHalf, from + v_off);
                }
            } else {
                if (!good && jg < in.len && a.status && (in.sees(jg) || in.sees(min(jg + 7, in.len - 1)))) atomicMax(a.status, 1);
#pragma unroll
                for (int y = 0; y < 8 / RPI; y++, from += row_step) {
                    const bool use = good && dims && in.sees(jg + r0 + RPI * y);
                    cp_async16(group + to_lane[y], use ? from : a.k, use);
                    cp_async16(group + to_lane[y] + R::kHalf, use ? from + v_off : a.v, use);
                }
            }
        }
    };

    {
        // the first tiles' pages are asked for together
        int first[R::kStages][GROUPS], left_at = left;
        Walk<R::kTile> at = in;
#pragma unroll
        for (int x = 0; x < R::kStages; x++)
            if (left_at > 0) {
                look_up(at, first[x]);
                left_at -= at.next(a, hh_n);
            }
#pragma unroll
        for (int x = 0; x < R::kStages; x++) {
#pragma unroll
            for (int g = 0; g < GROUPS; g++) pages[g] = first[x][g];
            if (x == R::kStages - 1) break;
            if (left_in > 0) {
                issue(x * R::kStage);
                left_in -= in.next(a, hh_n);
            }
            cp_commit();
        }
    }

    // the unit's heads and queries: 16-bit, the products' narrow operand in registers
    int head0 = 0, ng = 0;
    uint32_t q[F32 ? 1 : NG][F32 ? 1 : DP / 16][2];
    auto queries = [&]() {
        const int kvh = w.hgroups == 1 ? it.hh : it.hh / w.hgroups, hg = it.hh - kvh * w.hgroups;
        head0 = kvh * a.group + hg * w.unit_heads;
        ng = min(w.unit_heads, a.group - hg * w.unit_heads);
        if constexpr (!F32) {
#pragma unroll
            for (int n = 0; n < NG; n++) {
                const int h = n * 8 + (lane >> 2);
                const T *row = reinterpret_cast<const T *>(a.q) + it.seq * a.q_row + (head0 + h) * a.q_head + 2 * (lane & 3);
#pragma unroll
                for (int k = 0; k < DP / 16; k++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        q[n][k][e] = h < ng && 16 * k < a.d ? __ldg(reinterpret_cast<const uint32_t *>(row + 16 * k + 8 * e)) : 0;
            }
        }
    };
    queries();

    const bool extra = a.cap > 0.f || a.slopes || !(a.scale > 0.f);  // scores are more than a positive multiple of products
    const float k2 = extra && !F32 ? 1.f : a.scale * kLog2e, kcap = a.cap > 0.f ? a.scale / a.cap : 0.f;
    // where a lane's matrices of the products lie in a stage
    uint32_t k_at[F32 ? 1 : DP / 16], v_at[F32 ? 1 : DP / 16];
    if constexpr (!F32) {
#pragma unroll
        for (int i = 0; i < DP / 16; i++) {
            k_at[i] = wring + (lane & 15) * ROW + ((((lane >> 4) ^ (lane & 7)) * 16) ^ i * 32);
            v_at[i] = wring + R::kHalf + ((lane & 7) + ((lane >> 4) << 3)) * ROW + (((((lane >> 3) & 1) ^ (lane & 7)) * 16) ^ i * 32);
        }
    }
    uint32_t slot = 0, slot_in = (R::kStages - 1) * R::kStage;  // of the tile to compute and to load
    bool began = it.i == 0;  // the unit's first tile lies in this share
    bool fresh = true;
    float m[NM], l[NM];  // value that weights are taken from (log2), sums of this lane's weights
    uint32_t seen = 0;   // heads that have such a value
    float acc[NACC][4];
    while (left > 0) {
        if (fresh) {
            if constexpr (F32) {
                // the last unit's queries are no longer read: its end was met
                for (int e = tid; e < H * CH; e += kThreads) {
                    const int h = e / CH, cc = e % CH;
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (h < ng && cc * 4 < a.d) y = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(a.q) + it.seq * a.q_row + (head0 + h) * a.q_head + cc * 4);
                    *reinterpret_cast<float4 *>(sq + h * DP + cc * 4) = y;
                }
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < NM; i++) m[i] = F32 ? -INFINITY : 0.f, l[i] = 0.f;
            seen = 0;
#pragma unroll
            for (int i = 0; i < NACC; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][e] = 0.f;
            fresh = false;
        }
        cp_wait<R::kStages - 2>();
        __syncwarp();
        if (left_in > 0) {
            issue(slot_in);
            left_in -= in.next(a, hh_n);
            look_up(in, pages);
        }
        cp_commit();
        const int j = it.j + warp * KEYS, p = it.len - 1;
        const bool full = it.all_visible(j, KEYS);
        if constexpr (!F32) {
            constexpr int MT = KEYS / 16;
            float s[MT][NG][4];
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int n = 0; n < NG; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[t][n][e] = 0.f;
#pragma unroll
            for (int k = 0; k < DP / 16; k++)
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    uint32_t kf[4];
                    ldsm4(slot + t * 16 * ROW + k_at[k], kf);
#pragma unroll
                    for (int n = 0; n < NG; n++) mma<T>(s[t][n], kf, q[n][k][0], q[n][k][1]);
                }
            // element e of tile t: key 16 t + lane / 4 (+ 8 for e > 1), head 2 (lane % 4) + e % 2
            if (a.cap > 0.f) {
                float big = 0.f;
#pragma unroll
                for (int t = 0; t < MT; t++)
#pragma unroll
                    for (int n = 0; n < NG; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) big = fmaxf(big, fabsf(s[t][n][e] *= kcap));
                const bool far = __any_sync(0xffffffffu, big > kTanhPart);
#pragma unroll
                for (int t = 0; t < MT; t++)
#pragma unroll
                    for (int n = 0; n < NG; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) s[t][n][e] = far ? tanh_of(s[t][n][e]) : tanh_small(s[t][n][e]);
            }
            if (extra || !full) {
#pragma unroll
                for (int t = 0; t < MT; t++)
#pragma unroll
                    for (int n = 0; n < NG; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int jj = j + 16 * t + (lane >> 2) + (e >> 1) * 8;
                            float z = s[t][n][e];
                            if (extra) {
                                const int h = n * 8 + 2 * (lane & 3) + (e & 1);
                                z *= a.cap > 0.f ? a.cap : a.scale;
                                if (a.slopes && h < ng) z -= __ldg(a.slopes + head0 + h) * (float)(p - jj);
                                z *= kLog2e;
                            }
                            if (!full && !it.sees(jj)) z = -INFINITY;
                            s[t][n][e] = z;
                        }
            }
            // exponents: scores in log2 less the value that weights are taken from
            bool past = seen != (1u << NM) - 1;
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int n = 0; n < NG; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        s[t][n][e] = fmaf(s[t][n][e], k2, -m[2 * n + (e & 1)]);
                        past |= s[t][n][e] > 8.f + kLift<T>;
                    }
            if (__any_sync(0xffffffffu, past)) {
#pragma unroll
                for (int i = 0; i < NM; i++) {
                    const int n = i / 2, e = i & 1;
                    float by = -INFINITY;  // how far the largest score passes m
#pragma unroll
                    for (int t = 0; t < MT; t++) by = fmaxf(by, fmaxf(s[t][n][e], s[t][n][e + 2]));
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) by = fmaxf(by, __shfl_xor_sync(0xffffffffu, by, o));
                    const bool first = !(seen >> i & 1);
                    if (first ? by > -INFINITY : by > kLift<T>) {
                        by -= kLift<T>;
                        const float f = first ? 0.f : ex2(-by);
                        seen |= 1u << i;
                        m[i] += by;
                        l[i] *= f;
#pragma unroll
                        for (int d = 0; d < DP / 16; d++) {
                            acc[n * (DP / 16) + d][e] *= f;
                            acc[n * (DP / 16) + d][e + 2] *= f;
                        }
#pragma unroll
                        for (int t = 0; t < MT; t++) {
                            s[t][n][e] -= by;
                            s[t][n][e + 2] -= by;
                        }
                    }
                }
            }
            uint32_t ph[MT][NG][2], pl[MT][NG][2];  // weights to the type, and what that leaves of them
#pragma unroll
            for (int n = 0; n < NG; n++) {
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    float(&z)[4] = s[t][n];
#pragma unroll
                    for (int e = 0; e < 4; e++) z[e] = ex2(z[e]);
                    l[2 * n] += z[0] + z[2];
                    l[2 * n + 1] += z[1] + z[3];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float x = z[2 * e], y = z[2 * e + 1];
                        const uint32_t hi = cut2<T>(x, y);
                        const T *h = reinterpret_cast<const T *>(&hi);
                        ph[t][n][e] = transpose8(hi);
                        pl[t][n][e] = transpose8(pack2<T>(rest(x, to_f32(h[0])), rest(y, to_f32(h[1]))));
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < DP / 16; d++)
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    uint32_t vf[4];
                    ldsm4_t(slot + t * 16 * ROW + v_at[d], vf);
#pragma unroll
                    for (int n = 0; n < NG; n++) {
                        mma<T>(acc[n * (DP / 16) + d], vf, ph[t][n][0], ph[t][n][1]);
                        mma<T>(acc[n * (DP / 16) + d], vf, pl[t][n][0], pl[t][n][1]);
                    }
                }
        } else {
            // scores: lane = key x part of the dims (32 of them), all heads.  The parts start
            // two pieces apart, so that their queries lie in different banks.
            const int r = lane % KEYS, pt = lane / KEYS;
            float s[H];
#pragma unroll
            for (int h = 0; h < H; h++) s[h] = 0.f;
            const float *kr = reinterpret_cast<const float *>(smem + warp * R::kStages * R::kStage + slot);
#pragma unroll 4
            for (int i = 0; i < 8; i++) {
                const int cc = pt * 8 + ((i + 2 * pt) & 7);
                const float4 kx = *reinterpret_cast<const float4 *>(kr + r * DP + ((cc ^ (r & 7)) * 4));
#pragma unroll
                for (int h = 0; h < H; h++) {
                    const float4 qx = *reinterpret_cast<const float4 *>(sq + h * DP + cc * 4);
                    s[h] = fmaf(kx.x, qx.x, s[h]);
                    s[h] = fmaf(kx.y, qx.y, s[h]);
                    s[h] = fmaf(kx.z, qx.z, s[h]);
                    s[h] = fmaf(kx.w, qx.w, s[h]);
                }
            }
            const bool see = full || it.sees(j + r);
            float *wt = sw + warp * H * KEYS;
            bool past = false;
#pragma unroll
            for (int h = 0; h < H; h++) {
#pragma unroll
                for (int o = KEYS; o < 32; o <<= 1) s[h] += __shfl_xor_sync(0xffffffffu, s[h], o);
                const float slope = a.slopes && h < ng ? __ldg(a.slopes + head0 + h) : 0.f;
                s[h] = !see ? -INFINITY : extra ? score2(a, s[h], slope, p, j + r) : s[h] * k2;
                past |= s[h] > m[h] + 8.f;
            }
            if (__any_sync(0xffffffffu, past)) {
#pragma unroll
                for (int h = 0; h < H; h++) {
                    const float mx = fmaxf(m[h], mb::warp_max(s[h])), f = mx == -INFINITY ? 1.f : exp2f(m[h] - mx);
                    m[h] = mx;
                    l[h] *= f;
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[h][i] *= f;
                }
            }
#pragma unroll
            for (int h = 0; h < H; h++) {
                const float e = exp2f(s[h] - (m[h] == -INFINITY ? 0.f : m[h]));
                l[h] += e;  // every key counts in PARTS lanes
                if (pt == 0) wt[h * KEYS + r] = e;
            }
            __syncwarp();
            // outputs: a lane holds 4 dims; with 64 dims the half-warps take 8 keys each
            const float *vr = kr + R::kHalf / 4;
            const int cv = lane % CH, k0 = lane / CH * 8;
#pragma unroll
            for (int g = 0; g < 2; g++) {
                float4 v[4];
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = *reinterpret_cast<const float4 *>(vr + (k0 + 4 * g + i) * DP + ((cv ^ (4 * g + i)) * 4));
#pragma unroll
                for (int h = 0; h < H; h++) {
                    const float4 e = *reinterpret_cast<const float4 *>(wt + h * KEYS + k0 + 4 * g);
                    const float ew[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        acc[h][0] = fmaf(ew[i], v[i].x, acc[h][0]);
                        acc[h][1] = fmaf(ew[i], v[i].y, acc[h][1]);
                        acc[h][2] = fmaf(ew[i], v[i].z, acc[h][2]);
                        acc[h][3] = fmaf(ew[i], v[i].w, acc[h][3]);
                    }
                }
            }
            __syncwarp();
        }

        slot = slot == (R::kStages - 1) * R::kStage ? 0 : slot + R::kStage;
        slot_in = slot_in == (R::kStages - 1) * R::kStage ? 0 : slot_in + R::kStage;
        const bool last = it.i == it.t.n - 1;
        if (last || left == 1) {
            const int seq = it.seq, h0 = head0, hn = ng, rest = it.t.n - 1 - it.i;
            const bool whole = began && last, noted = began && !last;
            left -= it.next(a, hh_n);
            if (left > 0) queries();  // the next unit's, on their way while this one ends
            // the four warps' (m, l, output) into one, in the order of the warps
            if constexpr (!F32) {
#pragma unroll
                for (int i = 0; i < NM; i++) {
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
                    if (lane < 4) stat[warp * H + (i / 2) * 8 + 2 * lane + (i & 1)] = make_float2(seen >> i & 1 ? m[i] : -INFINITY, l[i]);
                }
            } else {
#pragma unroll
                for (int h = 0; h < H; h++) {
                    l[h] = mb::warp_sum(l[h]) * (1.f / PARTS);
                    if (DP == 64) {
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[h][i] += __shfl_xor_sync(0xffffffffu, acc[h][i], 16);
                    }
                    if (lane == h) stat[warp * H + h] = make_float2(m[h], l[h]);
                }
            }
            float *part = a.part + ((size_t)blockIdx.x * 2 + (began ? 1 : 0)) * ((size_t)H * (DP + 2));
            float *mine = merge + warp * HB * R::kPad;
#pragma unroll
            for (int n = 0; n < H / HB; n++) {
                if constexpr (!F32) {
#pragma unroll
                    for (int d = 0; d < DP / 16; d++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            mine[(2 * (lane & 3) + (e & 1)) * R::kPad + d * 16 + (lane >> 2) + (e >> 1) * 8] = acc[n * (DP / 16) + d][e];
                } else if (lane * 4 < DP) {
#pragma unroll
                    for (int h = 0; h < HB; h++) {
                        const float(&y)[4] = acc[n * HB + h];
                        *reinterpret_cast<float4 *>(mine + h * R::kPad + lane * 4) = make_float4(y[0], y[1], y[2], y[3]);
                    }
                }
                __syncthreads();
                for (int e = tid; e < HB * (DP / 4); e += kThreads) {
                    const int hl = e / (DP / 4), cc = e % (DP / 4), h = n * HB + hl;
                    if (h >= hn) break;
                    float M = -INFINITY, L = 0.f;
                    float2 ml[kWarps];
#pragma unroll
                    for (int i = 0; i < kWarps; i++) {
                        ml[i] = stat[i * H + h];
                        M = fmaxf(M, ml[i].x);
                    }
                    const float ms = M == -INFINITY ? 0.f : M;
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < kWarps; i++) {
                        const float f = exp2f(ml[i].x - ms);
                        const float4 z = *reinterpret_cast<const float4 *>(merge + (i * HB + hl) * R::kPad + cc * 4);
                        L = fmaf(ml[i].y, f, L);
                        y.x = fmaf(z.x, f, y.x);
                        y.y = fmaf(z.y, f, y.y);
                        y.z = fmaf(z.z, f, y.z);
                        y.w = fmaf(z.w, f, y.w);
                    }
                    if (whole) {
                        const float inv = 1.f / L;
                        if (cc * 4 < a.d)
                            store4(reinterpret_cast<T *>(a.out) + seq * a.o_row + (h0 + h) * a.o_head + cc * 4,
                                   L == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
                        if (a.lse && cc == 0) a.lse[(long long)seq * a.heads + h0 + h] = L == 0.f ? -INFINITY : (ms + log2f(L)) * kLn2;
                    } else {
                        *reinterpret_cast<float4 *>(part + (size_t)h * DP + cc * 4) = y;
                        if (cc == 0) *reinterpret_cast<float2 *>(part + (size_t)H * DP + 2 * h) = make_float2(M, L);
                    }
                }
                __syncthreads();  // the buffers are written again
            }
            if (left <= 0 && tid == 0) {
                a.note[blockIdx.x] = make_int2(noted ? (int)div64(end - 1 + rest, per) : -1, hn);
                a.meta[blockIdx.x] = Meta{seq, h0, hn, seq, p};
            }
            began = true;
            fresh = true;
        } else
            left -= it.next(a, hh_n);
    }
    cp_wait<0>();
}

template <typename T, int DP, int NG>
struct Plan {
    using R = Ring<T, DP, NG>;
    static constexpr int kCtas = mb::kSMs * R::kCtas;
    static size_t workspace() { return meta_bytes(kCtas) + part_bytes(kCtas, R::kH, DP); }
    static int run(Work &w, int page_size, char *space, int device, cudaStream_t s)
    {
        const char *who = "mocha_kv_decode";
        w.unit_heads = R::kH;
        w.hgroups = (w.a.group + R::kH - 1) / R::kH;
        w.min_tiles = 1;  // 2: one fp32 sequence of 777 in 12.1 us for 10.4, the others as they are
        w.one_page = page_size % R::kKeys == 0;
        lay_out(w.a, space, kCtas);
        static std::atomic<unsigned long long> allowed{0};
        if (allow_smem(who, k_decode<T, DP, NG>, R::kTotal, device, allowed) ||
            launch(who, k_decode<T, DP, NG>, dim3(kCtas), R::kThreads, R::kTotal, s, w))
            return 1;
        return launch(who, k_join<T, false>, dim3(kJoinBlocks), 32 * kJoinWarps, 0, s, w.a, kCtas, R::kH, DP);
    }
};

// Calls f with the plan for a type, group and dim: units of all heads of a group up to 32
// (16-bit), of 4 or 8 (fp32, where a wider group's heads read the keys again, from L2).  Units of
// 16 heads in place of 32, each reading the keys: with 128 dims, where 32 heads spill (414 bytes a
// thread), faster while a sequence's keys stay in L2 (64 sequences up to 8192, one kv head: 76 us
// for 89), slower past it (128 sequences up to 16000, two kv heads: 516 for 472); with 64 dims
// slower throughout (49 for 41).
template <typename F>
auto with_plan(int type, int group, int d, F f)
{
    const bool wide = padded_dim(d) == 128;
    auto half = [&](auto t) {
        using T = decltype(t);
        if (group <= 8) return wide ? f(Plan<T, 128, 1>{}) : f(Plan<T, 64, 1>{});
        if (group <= 16) return wide ? f(Plan<T, 128, 2>{}) : f(Plan<T, 64, 2>{});
        return wide ? f(Plan<T, 128, 4>{}) : f(Plan<T, 64, 4>{});
    };
    if (type == MOCHA_KV_F16) return half(__half{});
    if (type == MOCHA_KV_BF16) return half(__nv_bfloat16{});
    if (group <= 4) return wide ? f(Plan<float, 128, 0>{}) : f(Plan<float, 64, 0>{});
    return wide ? f(Plan<float, 128, 1>{}) : f(Plan<float, 64, 1>{});
}

}  // namespace

namespace kv {
size_t decode_workspace(int type, int group, int d)
{
    return with_plan(type, group, d, [](auto plan) { return plan.workspace(); });
}
}  // namespace kv

extern "C" int mocha_kv_decode(const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, const mocha_kv_scores *scores,
                               const mocha_kv_rows *q, const mocha_kv_rows *out, float *lse, void *workspace,
                               unsigned long long workspace_bytes, void *stream)
{
    const char *who = "mocha_kv_decode";
    if (check_pages(who, pages) || check_seqs(who, seqs) || check_scores(who, pages, scores)) return 1;
    const int b = type_bytes(pages->type), d = pages->head_dim;
    if (check_rows(who, "q", q, b, d, seqs->seqs) || check_rows(who, "out", out, b, d, seqs->seqs)) return 1;
    if (seqs->seqs && !seqs->kv_len) return fail(who, "null kv_len");
    DeviceGuard guard;
    if (guard.enter(who, pages->device)) return 1;
    if (!seqs->seqs) return 0;
    Work w{};
    w.a = make_args(pages, seqs, scores, q, out, lse);
    if (!workspace || !aligned(workspace) || workspace_bytes < decode_workspace(pages->type, w.a.group, d))
        return fail(who, "workspace missing, not 16-byte aligned or smaller than mocha_kv_workspace says");
    return with_plan(pages->type, w.a.group, d, [&](auto plan) {
        return plan.run(w, pages->page_size, static_cast<char *>(workspace), guard.device(), static_cast<cudaStream_t>(stream));
    });
}
