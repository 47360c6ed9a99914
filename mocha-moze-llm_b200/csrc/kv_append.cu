// mocha_kv_append: rotary positions on new queries and keys, and keys and values into
// their pages (mocha_kv.h).
//
// Every value is read once and written once; nothing else is to be done, so the kernel is
// bound by memory: (heads + 2 kv heads) * dim values in and out per token, and 2 * dim / 2
// angles.  A thread takes two 16-byte vectors of a head (four of fp32) that lie half the
// rotated values apart: the two ends of eight pairs (i, i + dims/2), or twice four
// interleaved pairs, or values that are only copied, likewise far apart.  Threads go along a
// token's heads, so each of a warp's accesses covers whole lines in every layout, and the
// token's slot, page and angles are L1 hits after the first thread's.  12810 rows of 32 + 16
// heads of 128, bf16: 57 us, 5.6 TB/s; from fp32 74.8 us, 6.4 TB/s; one row of 14 + 4 heads of
// 64: 2 us, a launch.
#include "kv_common.cuh"

namespace {

using namespace kv;

struct Append {
    char *k_pages, *v_pages;
    long long ps, hs, ts;
    int pages, kv_heads, chunks;  // chunks: 16-value pieces of a head
    FastDiv page, items, chunk_div;
    const int *table;
    long long table_stride;
    int max_len, seqs;
    int *status;
    const int *seq, *pos;
    const char *q, *k, *v;
    long long q_row, q_head, k_row, k_head, v_row, v_head;
    char *q_out;
    long long o_row, o_head;
    int heads;  // query heads; 0 without queries
    const float *cos, *sin;
    long long rope_stride;
    int positions, rot_chunks, half;
    int per_thread;
    long long total;
};

// Heads of a thread, which share its angles and addresses, once half as many threads still
// fill half the card: 32 + 16 heads of 128, bf16, take 4.9 us (1024 rows), 18.0 (4096) and 71.5
// (16384) with two heads, 5.5, 21.3 and 83.4 with one; at 512 rows 3.75 and 3.65.  Four and
// eight heads measured 3 to 20 % worse up to 4096 rows.  64 registers at most, for 32 warps of
// an SM: with 68 and 24 warps the 16384 rows took 79.9 us, with 48 and spills 76 to 79.  From
// fp32, where 64 registers spill 40 to 60 bytes a thread, 12810 rows take 74.8 us with them and
// 78.0 with 84, 4287 rows 27.5 and 28.4, and from fp32 to fp32 99.7 and 100.7.
constexpr int kHeads = 2;

MB_DEV void load4(const float *p, float *x)
{
    const float4 a = *reinterpret_cast<const float4 *>(p);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
}

template <typename T>
MB_DEV void store8(T *p, const float (&x)[8])
{
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint4 u;
        T *t = reinterpret_cast<T *>(&u);
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = from_f32<T>(x[i]);
        *reinterpret_cast<uint4 *>(p) = u;
    }
}

// 16 values as they are stored.
template <typename T>
struct Raw {
    uint4 v[sizeof(T)];  // 8 values take sizeof(T) / 2 vectors
    MB_DEV void load(const T *first, const T *second)
    {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            v[i] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(first) + 16 * i);
            v[sizeof(T) / 2 + i] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(second) + 16 * i);
        }
    }
    MB_DEV void values(float (&x)[8], float (&y)[8]) const
    {
        const T *t = reinterpret_cast<const T *>(v);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = to_f32(t[i]), y[i] = to_f32(t[8 + i]);
    }
};

template <typename TI, typename TO, bool INTERLEAVED, int HEADS>
__global__ void __launch_bounds__(256, 4) k_append(const __grid_constant__ Append a)
{
    mb::as::griddep_launch();
    mb::as::griddep_wait();
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.total) return;
    const long long row = a.total <= INT_MAX ? (long long)div(a.items, (uint32_t)id) : id / a.items.d;
    const int item = (int)(id - row * a.items.d);
    const int s = __ldg(a.seq + row), p = __ldg(a.pos + row);
    if (s < 0 || s >= a.seqs || p < 0) return;
    if (p >= a.max_len || (a.rot_chunks && p >= a.positions)) {
        if (a.status) atomicMax(a.status, 1);
        return;
    }
    const int h0 = div(a.chunk_div, item), c = item - h0 * a.chunks;
    const int heads = a.heads + 2 * a.kv_heads;
    const uint32_t slot = div(a.page, p);
    const int page = __ldg(a.table + s * a.table_stride + slot);
    const long long at = (p - (int)(slot * a.page.d)) * a.ts;
    // two vectors of 8 values, half the rotated (or the other) values apart, of heads h0 HEADS ..
    const bool turned = c < a.rot_chunks;
    const int first = turned ? 8 * c : 2 * a.half + 8 * (c - a.rot_chunks);
    const int second = first + (turned ? a.half : 8 * (a.chunks - a.rot_chunks));
    Raw<TI> raw[HEADS];
    float cs[8], sn[8];
    if (turned && h0 * HEADS < a.heads + a.kv_heads) {
        const float *cos = a.cos + p * a.rope_stride, *sin = a.sin + p * a.rope_stride;
        if (INTERLEAVED) {
            load4(cos + first / 2, cs), load4(cos + second / 2, cs + 4);
            load4(sin + first / 2, sn), load4(sin + second / 2, sn + 4);
        } else {
            load4(cos + first, cs), load4(cos + first + 4, cs + 4);
            load4(sin + first, sn), load4(sin + first + 4, sn + 4);
        }
    }
#pragma unroll
    for (int h = 0; h < HEADS; h++) {
        const int head = h0 * HEADS + h;
        if (head >= heads) break;
        const int kv = head - a.heads;
        const TI *src = kv < 0 ? reinterpret_cast<const TI *>(a.q) + row * a.q_row + head * a.q_head
                        : kv < a.kv_heads ? reinterpret_cast<const TI *>(a.k) + row * a.k_row + kv * a.k_head
                                          : reinterpret_cast<const TI *>(a.v) + row * a.v_row + (kv - a.kv_heads) * a.v_head;
        raw[h].load(src + first, src + second);
    }
#pragma unroll
    for (int h = 0; h < HEADS; h++) {
        const int head = h0 * HEADS + h;
        if (head >= heads) break;
        const int kv = head - a.heads;
        TO *dst;
        if (kv < 0) {
            dst = reinterpret_cast<TO *>(a.q_out) + row * a.o_row + head * a.o_head;
        } else {
            if ((unsigned)page >= (unsigned)a.pages) {
                if (a.status) atomicMax(a.status, 1);
                return;  // queries come first
            }
            dst = reinterpret_cast<TO *>(kv < a.kv_heads ? a.k_pages : a.v_pages) + page * a.ps + (kv < a.kv_heads ? kv : kv - a.kv_heads) * a.hs + at;
        }
        float x[8], y[8];
        raw[h].values(x, y);
        if (turned && head < a.heads + a.kv_heads) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float &u = INTERLEAVED ? (i < 4 ? x[2 * i] : y[2 * i - 8]) : x[i], &w = INTERLEAVED ? (i < 4 ? x[2 * i + 1] : y[2 * i - 7]) : y[i];
                const float r = u * cs[i] - w * sn[i];
                w = u * sn[i] + w * cs[i];
                u = r;
            }
        }
        store8(dst + first, x);
        store8(dst + second, y);
    }
}

template <typename TI, typename TO>
int run(const Append &a, bool interleaved, cudaStream_t s)
{
    const dim3 grid((unsigned)((a.total + 255) / 256));
    const char *who = "mocha_kv_append";
    if (a.per_thread == 1)
        return interleaved ? launch(who, k_append<TI, TO, true, 1>, grid, 256, 0, s, a) : launch(who, k_append<TI, TO, false, 1>, grid, 256, 0, s, a);
    return interleaved ? launch(who, k_append<TI, TO, true, kHeads>, grid, 256, 0, s, a) : launch(who, k_append<TI, TO, false, kHeads>, grid, 256, 0, s, a);
}

template <typename TI>
int run_to(const Append &a, int type, bool interleaved, cudaStream_t s)
{
    return type == MOCHA_KV_F32   ? run<TI, float>(a, interleaved, s)
           : type == MOCHA_KV_F16 ? run<TI, __half>(a, interleaved, s)
                                  : run<TI, __nv_bfloat16>(a, interleaved, s);
}

}  // namespace

extern "C" int mocha_kv_append(const mocha_kv_pages *pages, const mocha_kv_seqs *seqs, int rows, const int *seq,
                               const int *pos, int in_type, int heads, const mocha_kv_rows *q, const mocha_kv_rows *k,
                               const mocha_kv_rows *v, const mocha_kv_rows *q_out, const mocha_kv_rope *rope, void *stream)
{
    const char *who = "mocha_kv_append";
    if (check_pages(who, pages) || check_seqs(who, seqs)) return 1;
    const int in_bytes = type_bytes(in_type), out_bytes = type_bytes(pages->type), d = pages->head_dim;
    if (!in_bytes) return fail(who, "in_type must be MOCHA_KV_F32, MOCHA_KV_F16 or MOCHA_KV_BF16");
    if (rows < 0 || (rows && (!seq || !pos))) return fail(who, "rows must not be negative, seq and pos not null");
    if (!q != !q_out) return fail(who, "q and q_out go together");
    if (q && (heads < 1 || check_rows(who, "q", q, in_bytes, d, rows) || check_rows(who, "q_out", q_out, out_bytes, d, rows)))
        return heads < 1 ? fail(who, "heads must be positive") : 1;
    if (check_rows(who, "k", k, in_bytes, d, rows) || check_rows(who, "v", v, in_bytes, d, rows)) return 1;
    if (q && q->data == q_out->data && rows &&
        (in_type != pages->type || q->row_stride != q_out->row_stride || q->head_stride != q_out->head_stride))
        return fail(who, "q_out may be q only with the same type and strides");
    if (!rope || rope->dims < 0 || rope->dims % 16 || rope->dims > d) return fail(who, "rope dims must be a multiple of 16 up to head_dim");
    if (rope->dims && (!rope->cos || !rope->sin || !aligned(rope->cos) || !aligned(rope->sin) || rope->positions < 1 ||
                       rope->stride < rope->dims / 2 || rope->stride % 4))
        return fail(who, "cos and sin must be 16-byte aligned tables with a stride of at least dims / 2, a multiple of 4");
    const long long all_heads = (q ? heads : 0) + 2ll * pages->kv_heads;
    const int per_thread = all_heads * rows * (d / 16) >= mb::kSMs * 2048ll ? kHeads : 1;
    const long long items = (all_heads + per_thread - 1) / per_thread * (d / 16);
    if (all_heads > INT_MAX / 16 || items * rows > 256ll * INT_MAX) return fail(who, "too many rows or heads for one call");
    DeviceGuard guard;
    if (guard.enter(who, pages->device)) return 1;
    if (!rows) return 0;
    Append a{};
    a.k_pages = (char *)pages->k;
    a.v_pages = (char *)pages->v;
    a.ps = pages->page_stride;
    a.hs = pages->head_stride;
    a.ts = pages->token_stride;
    a.pages = pages->pages;
    a.kv_heads = pages->kv_heads;
    a.chunks = d / 16;
    a.page = fast_div(pages->page_size);
    a.items = fast_div((uint32_t)items);
    a.chunk_div = fast_div(d / 16);
    a.table = seqs->table;
    a.table_stride = seqs->table_stride;
    a.max_len = max_len(pages, seqs);
    a.seqs = seqs->seqs;
    a.status = seqs->status;
    a.seq = seq;
    a.pos = pos;
    if (q) {
        a.q = (const char *)q->data;
        a.q_row = q->row_stride;
        a.q_head = q->head_stride;
        a.q_out = (char *)q_out->data;
        a.o_row = q_out->row_stride;
        a.o_head = q_out->head_stride;
        a.heads = heads;
    }
    a.k = (const char *)k->data;
    a.k_row = k->row_stride;
    a.k_head = k->head_stride;
    a.v = (const char *)v->data;
    a.v_row = v->row_stride;
    a.v_head = v->head_stride;
    a.cos = rope->cos;
    a.sin = rope->sin;
    a.rope_stride = rope->stride;
    a.positions = rope->positions;
    a.rot_chunks = rope->dims / 16;
    a.half = rope->dims / 2;
    a.per_thread = per_thread;
    a.total = items * rows;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return in_type == MOCHA_KV_F32   ? run_to<float>(a, pages->type, rope->interleaved != 0, s)
           : in_type == MOCHA_KV_F16 ? run_to<__half>(a, pages->type, rope->interleaved != 0, s)
                                     : run_to<__nv_bfloat16>(a, pages->type, rope->interleaved != 0, s);
}
