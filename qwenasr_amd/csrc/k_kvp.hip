// Pages of a KV cache: forked to new sequences, compacted, written.
//
// Which pages are in use is not kept anywhere: a fork reads it off the tables, into a
// bitmap in LDS (one bit a page, 32 KiB for 2^18 pages), in the one block that then
// hands the free ones out.  The entries of the tables are few (one per 16 to 256
// positions), and there are no counts that could go out of step with them.
#include "kernels.h"
#include "gemm_common.h"
#include "qasr_hip.h"

namespace qasr {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#define KVP_THREADS 1024
#define KVP_WAVES (KVP_THREADS / 64)
#define KVP_SEQS QASR_KVP_MAX_SEQ
#define KVP_PAGES QASR_KVP_MAX_PAGES
#define KVP_PICK 2048            // page ids handed out through LDS; more go through scratch
// scratch: [0] copies, from KVP_COPIES on {source, target, positions, -} each, then the
// ids handed out, then where moved pages go
#define KVP_COPIES 16
#define KVP_PICKS (KVP_COPIES + 4 * (KVP_PAGES / 2))
#define KVP_MAP (KVP_PICKS + KVP_PAGES)
static_assert(KVP_MAP + KVP_PAGES == KVP_WORK_INTS && KVP_SEQS <= KVP_PAGES / 2, "a place for every copy, id and page");

// sums over the wave's lanes up to and with each
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);                  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, QASR_DPP_ROW_BCAST15, 0xA, 0xF, false);
    return v + __builtin_amdgcn_update_dpp(0, v, QASR_DPP_ROW_BCAST31, 0xC, 0xF, false);
}
// exclusive sums of N values over the block's threads, and their totals; every thread
// has to come, once for each `sums`
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&total)[N], int (*sums)[KVP_WAVES]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int x[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = wave_scan(v[i]);
        if (lane == 63) sums[i][w] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        // lane w' of each row of 16 holds wave w's sum: one more scan gives all that come before
        const int s = wave_scan(lane < KVP_WAVES ? sums[i][lane] : 0);
        total[i] = __builtin_amdgcn_readlane(s, KVP_WAVES - 1);
        v[i] = x[i] - v[i] + (w > 0 ? __shfl(s, w - 1, 64) : 0);
    }
}

__device__ __forceinline__ int kvp_held(int len, int shift) { return (len + (1 << shift) - 1) >> shift; }

// lanes that walk one sequence's entries together: a wave for few sequences, and so few for
// many that all sequences' loads are on their way at once
__device__ __forceinline__ int kvp_lanes(int n) {
    int lanes = 64;
    while (lanes > 4 && KVP_THREADS / lanes < n) lanes >>= 1;
    return lanes;
}

// entries [0, held) of a sequence's row, four of a lane on their way at a time
template <typename F>
__device__ __forceinline__ void kvp_entries(const int32_t *row, int held, int lane, int lanes, const F &f) {
    for (int s0 = lane; s0 < held; s0 += 4 * lanes) {
        int id[4];
#pragma unroll
        for (int u = 0; u < 4; u++) id[u] = s0 + u * lanes < held ? row[s0 + u * lanes] : -1;
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (s0 + u * lanes < held) f(s0 + u * lanes, id[u]);
    }
}

// A thread's part of a bitmap of nw words, in order of the threads: some words, or some bits of one.
struct KvpBits {
    int w0, words;
    uint32_t mask;
    __device__ __forceinline__ KvpBits(int nw) {
        const int t = threadIdx.x;
        int split = 1;                                   // threads a word
        while (split < 32 && nw * split * 2 <= KVP_THREADS) split *= 2;
        words = (nw + KVP_THREADS - 1) / KVP_THREADS;
        w0 = words > 1 ? t * words : t / split;
        words = w0 < nw ? min(words, nw - w0) : 0;
        mask = split == 1 ? ~0u : ((1u << 32 / split) - 1) << t % split * (32 / split);
    }
};

// bits past n_pages count as used
__device__ __forceinline__ uint32_t kvp_no_pages(int w, int n_pages) {
    return w * 32 + 32 <= n_pages ? 0u : w * 32 >= n_pages ? ~0u : ~((1u << (n_pages & 31)) - 1);
}

// One block: the new tables, and what has to be copied.  Bound by its own latency: a
// chain of loads (parent, entries) and a few passes over LDS; 5.1 us for 8 sequences, 9.3
// for 128.
//
// Who keeps a common last page is decided in a hash table of such pages: each sequence
// that holds one enters (positions in it, gets rows, -index), the largest stays.
__global__ __launch_bounds__(KVP_THREADS) void k_kvp_fork(KvpForkArgs a, int slots) {
    extern __shared__ uint32_t lds[];
    __shared__ int sums[3][KVP_WAVES], over;
    __shared__ unsigned long long all_need;
    const int t = threadIdx.x, n = a.n_out;
    const int n_pages = a.pools.n_pages, nw = (n_pages + 31) / 32, shift = a.pools.shift, page = 1 << shift, cap = a.table_ld << shift;
    uint32_t *used = lds, *full = used + nw;
    int *hash_id = reinterpret_cast<int *>(full + nw), *hash_key = hash_id + slots, *pick_l = hash_key + slots;
    int *len = pick_l + KVP_PICK, *par = len + n, *tail = par + n, *info = tail + n, *base = info + n, *rows_l = base + n;
    int *picks = a.work + KVP_PICKS, *copies = a.work + KVP_COPIES;
    // thread t has sequences t, t + 1024, .. until their entries are walked; all that is known of them goes out at once
    constexpr int PER = KVP_SEQS / KVP_THREADS;
    int p_of[PER], l_of[PER];
    int64_t r_of[PER][2];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int j = t + i * KVP_THREADS, jc = min(j, n - 1);
        p_of[i] = j;
        l_of[i] = 0;
        r_of[i][0] = 0;
        r_of[i][1] = a.max_rows;
        if (i > 0 && i * KVP_THREADS >= max(n, a.n_seq)) continue;
        if (n > 0 && a.parent) p_of[i] = a.parent[jc];
        if (a.n_seq > 0) l_of[i] = a.len[min(j, a.n_seq - 1)];
        if (n > 0 && a.row_start) {
            r_of[i][0] = a.row_start[jc];
            r_of[i][1] = a.row_start[jc + 1];
        }
    }
    if (t == 0) over = 0, all_need = 0;
    for (int i = t; i < nw; i += KVP_THREADS) {
        used[i] = kvp_no_pages(i, n_pages);
        full[i] = 0;
    }
    for (int i = t; i < slots; i += KVP_THREADS) {
        hash_id[i] = -1;
        hash_key[i] = 0;
    }
    static_assert(KVP_PICK >= KVP_SEQS, "the parents' lengths, before there are pages to hand out");
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (t + i * KVP_THREADS < a.n_seq) pick_l[t + i * KVP_THREADS] = l_of[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int j = t + i * KVP_THREADS, p = p_of[i], rows = (int)min(max(r_of[i][1] - r_of[i][0], (int64_t)0), a.max_rows);
        if (j >= n) break;
        const bool ok = (unsigned)p < (unsigned)a.n_seq;
        const int l = ok ? min(max(pick_l[p], 0), cap) : 0;
        const int held = kvp_held(l, shift), fresh = kvp_held(l + rows, shift) - held;
        len[j] = l;
        par[j] = ok ? p : 0;
        tail[j] = -1;
        info[j] = (l & (page - 1)) | (rows > 0 ? 256 : 0);
        base[j] = fresh;
        rows_l[j] = rows;
        if (held + fresh > a.table_ld) atomicAdd(&over, 1);
    }
    __syncthreads();
    // the entries that are taken over
    const int lanes = kvp_lanes(n), lane = t & (lanes - 1), g = t / lanes, groups = KVP_THREADS / lanes;
    for (int j = g; j < n; j += groups) {
        const int held = kvp_held(len[j], shift), last = (info[j] & 255) ? held - 1 : -1;
        int32_t *out = a.table_out + (int64_t)j * a.table_ld;
        kvp_entries(a.table + (int64_t)par[j] * a.table_ld, held, lane, lanes, [&](int s, int id) {
            const bool ok = (unsigned)id < (unsigned)n_pages;
            if (ok) {
                atomicOr(&used[id >> 5], 1u << (id & 31));
                if (s != last) atomicOr(&full[id >> 5], 1u << (id & 31));
            }
            if (s != last) out[s] = id;
            else if (ok) tail[j] = id;
        });
    }
    __syncthreads();
    // thread t has sequences 2 t and 2 t + 1 from here on
    int at_hash[PER], key[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int j = t * PER + i;
        const int p = j < n ? tail[j] : -1;
        at_hash[i] = -1;
        if (p < 0) continue;
        key[i] = (info[j] & 255) << 16 | (info[j] & 256) << 6 | (KVP_SEQS - j);
        int h = (int)((uint32_t)p * 2654435761u >> 16) & (slots - 1);
        while (true) {
            const int was = atomicCAS(&hash_id[h], -1, p);
            if (was == -1 || was == p) break;
            h = (h + 1) & (slots - 1);                       // ends: there are twice as many places as sequences
        }
        atomicMax(&hash_key[h], key[i]);
        at_hash[i] = h;
    }
    __syncthreads();
    int v[3] = {0, 0, 0}, total[3];
    const KvpBits mine(nw);
    long long want = 0;
    int copy[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int j = t * PER + i;
        copy[i] = 0;
        if (j >= n) continue;
        const int p = tail[j];
        if (at_hash[i] >= 0 && (info[j] & 256)) copy[i] = ((full[p >> 5] >> (p & 31)) & 1) || hash_key[at_hash[i]] != key[i];
        v[1] += copy[i];
        want += copy[i] + base[j];
    }
    if (want) atomicAdd(&all_need, (unsigned long long)want);
    // held to what is past any pool, so that the sums stay in 32 bits
    v[0] = (int)min(want, 1LL << 20);
    for (int i = 0; i < mine.words; i++) v[2] += __popc(~used[mine.w0 + i] & mine.mask);
    block_scan(v, total, sums);
    const int n_free = total[2], n_used = n_pages - n_free;
    const bool fail = over > 0 || total[0] > n_free;
    if (t == 0) {
        a.status[0] = over > 0 ? -over : fail ? (int)min((long long)all_need - n_free, 0x7fffffffLL) : 0;
        a.status[1] = fail ? n_used : n_used + total[0];
        a.work[0] = fail ? 0 : total[1];
    }
    if (fail) {
        for (int64_t i = t; i < (int64_t)n * a.table_ld; i += KVP_THREADS) a.table_out[i] = -1;
        for (int j = t; j < n; j += KVP_THREADS) a.pos_out[j] = a.len_out[j] = 0;
        return;
    }
    // places among the pages handed out: in order of the sequences
    int at = v[0], cp = v[1];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int j = t * PER + i;
        if (j >= n) continue;
        const int fresh = base[j];
        base[j] = at;
        at += copy[i] + fresh;
        if (copy[i]) info[j] |= 512 | cp++ << 10;
    }
    // the lowest free pages
    const bool in_lds = total[0] <= KVP_PICK;
    int rank = v[2];
    for (int i = 0; i < mine.words && rank < total[0]; i++) {
        for (uint32_t f = ~used[mine.w0 + i] & mine.mask; f && rank < total[0]; f &= f - 1, rank++) {
            const int id = (mine.w0 + i) * 32 + __builtin_ctz(f);
            if (in_lds) pick_l[rank] = id;
            else picks[rank] = id;
        }
    }
    __syncthreads();
    auto pick = [&](int r) { return in_lds ? pick_l[r] : picks[r]; };
    for (int j = g; j < n; j += groups) {
        const int l = len[j], held = kvp_held(l, shift), inf = info[j], c = (inf >> 9) & 1, rows = rows_l[j], last = tail[j];
        const int end = kvp_held(l + rows, shift), first = (inf & 255) ? held - 1 : held, b = base[j];
        int32_t *out = a.table_out + (int64_t)j * a.table_ld;
        for (int s = first + lane; s < a.table_ld; s += lanes) {
            int id = -1;
            if (s < held) id = c ? pick(b) : last >= 0 ? last : a.table[(int64_t)par[j] * a.table_ld + s];
            else if (s < end) id = pick(b + c + s - held);
            out[s] = id;
        }
        if (lane == 0) {
            a.pos_out[j] = l;
            a.len_out[j] = l + rows;
            if (c) *reinterpret_cast<int4 *>(copies + 4 * (inf >> 10)) = make_int4(last, pick(b), inf & 255, 0);
        }
    }
}

// One block: where pages go, and the tables with it.  Bound like the fork: 4.9 us.
__global__ __launch_bounds__(KVP_THREADS) void k_kvp_compact(KvpCompactArgs a) {
    extern __shared__ uint32_t lds[];
    __shared__ int sums[1][KVP_WAVES], sums2[2][KVP_WAVES];
    const int t = threadIdx.x;
    const int n_pages = a.pools.n_pages, nw = (n_pages + 31) / 32, shift = a.pools.shift, n = a.n_seq, cap = a.table_ld << shift;
    uint32_t *used = lds;
    int *held_l = reinterpret_cast<int *>(used + nw);
    int *copies = a.work + KVP_COPIES, *map = a.work + KVP_MAP;
    for (int i = t; i < nw; i += KVP_THREADS) used[i] = 0;
    for (int j = t; j < n; j += KVP_THREADS) held_l[j] = kvp_held(min(max(a.len[j], 0), cap), shift);
    __syncthreads();
    const int lanes = kvp_lanes(n), lane = t & (lanes - 1), g = t / lanes, groups = KVP_THREADS / lanes;
    for (int j = g; j < n; j += groups)
        kvp_entries(a.table + (int64_t)j * a.table_ld, held_l[j], lane, lanes, [&](int, int id) {
            if ((unsigned)id < (unsigned)n_pages) atomicOr(&used[id >> 5], 1u << (id & 31));
        });
    __syncthreads();
    const KvpBits mine(nw);
    const int w0 = mine.w0;
    int v1[1] = {0}, t1[1], v[2] = {0, 0}, total[2];
    for (int i = 0; i < mine.words; i++) v1[0] += __popc(used[w0 + i] & mine.mask);
    block_scan(v1, t1, sums);
    const int n_used = t1[0];
    // pages at n_used and behind that are held, and those before that are free: as many
    auto from_high = [&](int w) { return used[w] & kvp_no_pages(w, n_used) & mine.mask; };
    auto to_low = [&](int w) { return ~used[w] & ~kvp_no_pages(w, n_used) & mine.mask; };
    for (int i = 0; i < mine.words; i++) {
        v[0] += __popc(from_high(w0 + i));
        v[1] += __popc(to_low(w0 + i));
    }
    block_scan(v, total, sums2);
    int src = v[0], dst = v[1];
    const int n_moved = total[0];
    for (int i = 0; i < mine.words; i++) {
        for (uint32_t f = from_high(w0 + i); f; f &= f - 1) {
            copies[4 * src] = (w0 + i) * 32 + __builtin_ctz(f);
            copies[4 * src++ + 2] = 1 << shift;
        }
        for (uint32_t f = to_low(w0 + i); f; f &= f - 1) copies[4 * dst++ + 1] = (w0 + i) * 32 + __builtin_ctz(f);
    }
    if (t == 0) {
        a.status[0] = n_moved;
        a.status[1] = n_used;
        a.work[0] = n_moved;
    }
    __syncthreads();
    for (int i = t; i < n_moved; i += KVP_THREADS) map[copies[4 * i]] = copies[4 * i + 1];
    __syncthreads();
    for (int j = g; j < n; j += groups) {
        const int64_t row = (int64_t)j * a.table_ld;
        const int held = held_l[j];
        kvp_entries(a.table + row, held, lane, lanes, [&](int s, int id) { a.table_out[row + s] = id >= n_used && id < n_pages ? map[id] : id; });
        for (int s = held + lane; s < a.table_ld; s += lanes) a.table_out[row + s] = -1;
    }
}

// The copies of every pool: a block takes some heads of a page, and a page for each
// gridDim.z of them.  Only the positions that a page holds are moved; four 16-byte
// pieces a thread are on their way at a time, past the caches: what stands written in
// them is sent to memory when the launch ends (8 hypotheses, 20 MB read and written, plan
// and copies 24 -> 12 us).  Bound by memory: 900 pages of 2.5 MB 4.9 TB/s, as the plain copy.
__global__ __launch_bounds__(256) void k_kvp_copy(KvpPools p, const int *work, int per_block) {
    int4 c = *reinterpret_cast<const int4 *>(work + KVP_COPIES + 4 * (int64_t)blockIdx.z);   // along with the count
    const int count = work[0];
    const int h0 = blockIdx.x * per_block, heads = min(per_block, p.heads - h0);
    const int whole = p.units << p.shift;
    for (int64_t i = blockIdx.z; i < count; i += gridDim.z) {
        if (i != blockIdx.z) c = *reinterpret_cast<const int4 *>(work + KVP_COPIES + 4 * i);
        const unsigned per = (unsigned)c.z * p.units, total = per * heads;
        u32x4 *pool = reinterpret_cast<u32x4 *>(p.base + blockIdx.y * p.pool_stride);
        const u32x4 *src = pool + ((int64_t)c.x * p.heads + h0) * whole;
        u32x4 *dst = pool + ((int64_t)c.y * p.heads + h0) * whole;
        for (unsigned u = threadIdx.x; u < total; u += 4 * 256) {
            u32x4 v[4];
            unsigned at[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const unsigned x = u + e * 256, h = heads == 1 ? 0 : x / per;
                at[e] = x + h * (whole - per);
                if (x < total) v[e] = __builtin_nontemporal_load(src + at[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (u + e * 256 < total) __builtin_nontemporal_store(v[e], dst + at[e]);
        }
    }
}

static hipError_t launch_copies(const KvpPools &p, const int *work, int64_t most, hipStream_t st) {
    if (most <= 0) return hipSuccess;
    const int per_block = (int)std::min<int64_t>(p.heads, std::max<int64_t>(1, 1024 / ((int64_t)p.units << p.shift)));
    const unsigned x = (unsigned)((p.heads + per_block - 1) / per_block);
    // blocks past the copies that there turn out to be end at once
    const int64_t z = std::min<int64_t>({most, 65535, std::max<int64_t>(1, (1 << 20) / ((int64_t)x * p.n_pools))});
    hipLaunchKernelGGL(k_kvp_copy, dim3(x, (unsigned)p.n_pools, (unsigned)z), dim3(256), 0, st, p, work, per_block);
    return hipGetLastError();
}

hipError_t launch_kvp_fork(const KvpForkArgs &a, hipStream_t st) {
    if (a.pools.n_pages > KVP_PAGES || a.n_out > KVP_SEQS) return hipErrorInvalidValue;
    int slots = 64;
    while (slots < 2 * a.n_out) slots *= 2;
    const size_t lds = ((size_t)(a.pools.n_pages + 31) / 32 * 2 + 2 * (size_t)slots + 6 * (size_t)a.n_out + KVP_PICK) * 4;
    hipLaunchKernelGGL(k_kvp_fork, dim3(1), dim3(KVP_THREADS), lds, st, a, slots);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_copies(a.pools, a.work, a.max_rows > 0 ? a.n_out : 0, st);
}

hipError_t launch_kvp_compact(const KvpCompactArgs &a, hipStream_t st) {
    if (a.pools.n_pages > KVP_PAGES || a.n_seq > KVP_SEQS) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_kvp_compact, dim3(1), dim3(KVP_THREADS), ((size_t)(a.pools.n_pages + 31) / 32 + a.n_seq) * 4, st, a);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_copies(a.pools, a.work, std::min<int64_t>(a.pools.n_pages / 2, (int64_t)a.n_seq * a.table_ld), st);
}

// ---------------------------------------------------------------------------
// write
// ---------------------------------------------------------------------------

// Rows of K and V to their pages, 8 values a thread and step, past the caches.  Bound by
// memory (bf16 prompts, 51 MB read and written, 11.3 us, 4.5 TB/s), and for a row or two a
// sequence by the launch (5.0 us, 3.0 of them on the GPU).
template <bool BF16>
__global__ __launch_bounds__(256) void k_kvp_write(KvpWriteArgs a, int per_block) {
    const KvpSeqs &s = a.s;
    const int j = blockIdx.y;
    const KvpRows sq = kvp_rows(s, j);
    const int i0 = blockIdx.x * per_block, rows = min(sq.n - i0, per_block);
    const int half = s.Hkv * s.hd / 8, per_row = 2 * half;
    const int32_t *table = s.table + (int64_t)j * s.table_ld;
    const int cap = s.table_ld << s.shift;
    for (int64_t u = threadIdx.x; u < (int64_t)rows * per_row; u += 256) {
        const int i = i0 + (int)(u / per_row), w = (int)(u % per_row), is_v = w >= half, e = (w - is_v * half) * 8;
        const int p = sq.p0 + i;
        if ((unsigned)p >= (unsigned)cap) continue;
        const int id = table[p >> s.shift];
        if ((unsigned)id >= (unsigned)s.n_pages) continue;
        const int64_t from = (sq.r0 + i) * a.ld + e;
        const void *rows_in = is_v ? a.v : a.k;
        uint4 o;
        if (BF16) {
            const uint16_t *x = reinterpret_cast<const uint16_t *>(rows_in) + from;
            if (a.vec) o = *reinterpret_cast<const uint4 *>(x);
            else o = make_uint4(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16, x[4] | (uint32_t)x[5] << 16, x[6] | (uint32_t)x[7] << 16);
        } else {
            const float *x = reinterpret_cast<const float *>(rows_in) + from;
            f32x4 v[2];
            if (a.vec) {
                v[0] = reinterpret_cast<const f32x4 *>(x)[0];
                v[1] = reinterpret_cast<const f32x4 *>(x)[1];
            } else {
#pragma unroll
                for (int r = 0; r < 8; r++) v[r >> 2][r & 3] = x[r];
            }
            o = make_uint4(cvt_pk_bf16(v[0][0], v[0][1]), cvt_pk_bf16(v[0][2], v[0][3]), cvt_pk_bf16(v[1][0], v[1][1]), cvt_pk_bf16(v[1][2], v[1][3]));
        }
        uint16_t *to = (is_v ? a.vp : a.kp) + ((((int64_t)id * s.Hkv + e / s.hd) << s.shift) + (p & ((1 << s.shift) - 1))) * s.hd + e % s.hd;
        const u32x4 o4 = {o.x, o.y, o.z, o.w};
        __builtin_nontemporal_store(o4, reinterpret_cast<u32x4 *>(to));
    }
}

hipError_t launch_kvp_write(const KvpWriteArgs &a0, bool bf16, hipStream_t st) {
    KvpWriteArgs a = a0;
    if (a.s.hd % 8 != 0 || a.s.n_seq > 65535) return hipErrorInvalidValue;
    a.vec = (((uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0) && (a.ld * (bf16 ? 2 : 4)) % 16 == 0;
    const int per_block = 8;
    const dim3 grid((unsigned)((a.s.max_rows + per_block - 1) / per_block), (unsigned)a.s.n_seq);
    if (bf16) hipLaunchKernelGGL((k_kvp_write<true>), grid, dim3(256), 0, st, a, per_block);
    else hipLaunchKernelGGL((k_kvp_write<false>), grid, dim3(256), 0, st, a, per_block);
    return hipGetLastError();
}

}  // namespace qasr
