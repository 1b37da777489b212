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

#define KVP_THREADS 1024
#define KVP_PICK 2048            // page ids handed out through LDS; more go through scratch
// scratch: [0] copies, from KVP_COPIES on {source, target, positions, -} each, then the
// ids handed out, then where moved pages go
#define KVP_COPIES 16
#define KVP_PAGES QASR_KVP_MAX_PAGES
#define KVP_PICKS (KVP_COPIES + 4 * (KVP_PAGES / 2))
#define KVP_MAP (KVP_PICKS + KVP_PAGES)

// exclusive sums over the block's threads; every thread has to come.  Returns the
// sum before this thread, *total that of all.
__device__ __forceinline__ int block_scan(int v, int *sums, int *total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();                             // sums may still be read from the last call
    if (lane == 63) sums[w] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < KVP_THREADS / 64; i++) {
        const int s = sums[i];
        before += i < w ? s : 0;
        all += s;
    }
    *total = all;
    return before + x - v;
}

__device__ __forceinline__ int kvp_held(int len, int shift) { return (len + (1 << shift) - 1) >> shift; }

// Marks the pages of one sequence's entries [0, held); a last page that is not full
// only in `used`.  put(slot, id) sees every entry but that one, last(id) that one.
template <typename Put, typename Last>
__device__ __forceinline__ void kvp_mark(const int32_t *row, int held, bool part, int n_pages, uint32_t *used, uint32_t *full, int first,
                                         int id0, const Put &put, const Last &last) {
    const int lane = threadIdx.x & 63;
    for (int s = first + lane; s < held; s += 64) {
        const int id = s == lane ? id0 : row[s];
        const bool ok = (unsigned)id < (unsigned)n_pages, is_last = part && s == held - 1;
        if (ok) {
            atomicOr(&used[id >> 5], 1u << (id & 31));
            if (!is_last && full) atomicOr(&full[id >> 5], 1u << (id & 31));
        }
        if (is_last) last(ok ? id : -1);
        else put(s, id);
    }
}

// One block: the new tables, and what has to be copied.  Bound by its own latency: a
// chain of loads (parent, length, entries) and a few passes over LDS.
__global__ __launch_bounds__(KVP_THREADS) void k_kvp_fork(KvpForkArgs a) {
    extern __shared__ uint32_t lds[];
    __shared__ int sums[KVP_THREADS / 64], over;
    __shared__ unsigned long long all_need;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n_pages = a.pools.n_pages, nw = (n_pages + 31) / 32, shift = a.pools.shift, page = 1 << shift;
    const int n = a.n_out, cap = a.table_ld << shift;
    uint32_t *used = lds, *full = used + nw;
    int *len = reinterpret_cast<int *>(full + nw), *par = len + n, *tail = par + n, *info = tail + n, *base = info + n, *pick_l = base + n;
    int *picks = a.work + KVP_PICKS, *copies = a.work + KVP_COPIES;
    auto rows_of = [&](int j) -> int {
        if (!a.row_start) return (int)a.max_rows;
        return (int)min(max((int64_t)a.row_start[j + 1] - a.row_start[j], (int64_t)0), a.max_rows);
    };
    for (int i = t; i < 2 * nw; i += KVP_THREADS) used[i] = 0;
    if (t == 0) over = 0, all_need = 0;
    __syncthreads();
    for (int j = t; j < n; j += KVP_THREADS) {
        const int p = a.parent ? a.parent[j] : j;
        const bool ok = (unsigned)p < (unsigned)a.n_seq;
        const int l = ok ? min(max(a.len[p], 0), cap) : 0, rows = rows_of(j);
        const int held = kvp_held(l, shift), fresh = kvp_held(l + rows, shift) - held;
        len[j] = l;
        par[j] = ok ? p : 0;
        tail[j] = -1;
        info[j] = (l & (page - 1)) | (rows > 0 ? 256 : 0);
        base[j] = fresh;
        if (held + fresh > a.table_ld) atomicAdd(&over, 1);
    }
    __syncthreads();
    // the entries that are taken over; the first 64 of four sequences are on their way at a time
    for (int j0 = wave; j0 < n; j0 += 4 * (KVP_THREADS / 64)) {
        int id[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int j = j0 + u * (KVP_THREADS / 64);
            id[u] = j < n && lane < kvp_held(len[j], shift) ? a.table[(int64_t)par[j] * a.table_ld + lane] : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int j = j0 + u * (KVP_THREADS / 64);
            if (j >= n) break;
            int32_t *out = a.table_out + (int64_t)j * a.table_ld;
            kvp_mark(a.table + (int64_t)par[j] * a.table_ld, kvp_held(len[j], shift), (info[j] & 255) != 0, n_pages, used, full, 0, id[u],
                     [&](int s, int v) { out[s] = v; }, [&](int v) { tail[j] = v; });
        }
    }
    __syncthreads();
    // who needs a copy of its last page: those that do not go on in place
    for (int j = wave; j < n; j += KVP_THREADS / 64) {
        const int inf = info[j], p = tail[j], fill = inf & 255;
        if (p < 0 || !(inf & 256)) continue;
        bool copy = (full[p >> 5] >> (p & 31)) & 1;
        for (int i = lane; i < n && !copy; i += 64) {
            const int other = info[i];
            copy = tail[i] == p && ((other & 255) > fill || ((other & 255) == fill && (other & 256) && i < j));
        }
        if (__any(copy) && lane == 0) info[j] = inf | 512;
    }
    __syncthreads();
    // places among the pages handed out: in order of the sequences
    constexpr int PER = QASR_KVP_MAX_SEQ / KVP_THREADS;
    const int j0 = t * PER;
    long long want = 0;
    int cps = 0, total, n_copies, n_used;
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (j0 + i < n) {
            const int c = (info[j0 + i] >> 9) & 1;
            cps += c;
            want += c + base[j0 + i];
        }
    if (want) atomicAdd(&all_need, (unsigned long long)want);
    // held to what is past any pool, so that the sums stay in 32 bits
    int at = block_scan((int)min(want, 1LL << 20), sums, &total), cp = block_scan(cps, sums, &n_copies);
    const int per_w = (nw + KVP_THREADS - 1) / KVP_THREADS, w0 = t * per_w;
    int in_use = 0;
    for (int i = 0; i < per_w; i++) in_use += w0 + i < nw ? __popc(used[w0 + i]) : 0;
    block_scan(in_use, sums, &n_used);
    const bool fail = over > 0 || total > n_pages - n_used;
    if (t == 0) {
        a.status[0] = over > 0 ? -over : fail ? (int)min((long long)all_need - (n_pages - n_used), 0x7fffffffLL) : 0;
        a.status[1] = fail ? n_used : n_used + total;
        a.work[0] = fail ? 0 : n_copies;
    }
    if (fail) {
        for (int64_t i = t; i < (int64_t)n * a.table_ld; i += KVP_THREADS) a.table_out[i] = -1;
        for (int j = t; j < n; j += KVP_THREADS) a.pos_out[j] = a.len_out[j] = 0;
        return;
    }
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (j0 + i < n) {
            const int c = (info[j0 + i] >> 9) & 1, f = base[j0 + i];
            base[j0 + i] = at;
            if (c) {
                copies[4 * cp] = tail[j0 + i];
                copies[4 * cp + 2] = info[j0 + i] & 255;
                info[j0 + i] |= cp << 10;
            }
            at += c + f;
            cp += c;
        }
    // the lowest free pages
    const bool in_lds = total <= KVP_PICK;
    int free_here = 0, all_free;
    for (int i = 0; i < per_w; i++)
        if (w0 + i < nw) free_here += __popc(~used[w0 + i]);
    int rank = block_scan(free_here, sums, &all_free);           // bits past n_pages come last: never reached
    for (int i = 0; i < per_w && rank < total; i++) {
        if (w0 + i >= nw) break;
        uint32_t f = ~used[w0 + i];
        while (f && rank < total) {
            const int id = (w0 + i) * 32 + __builtin_ctz(f);
            f &= f - 1;
            if (in_lds) pick_l[rank] = id;
            else picks[rank] = id;
            rank++;
        }
    }
    __syncthreads();
    auto pick = [&](int r) { return in_lds ? pick_l[r] : picks[r]; };
    for (int j = wave; j < n; j += KVP_THREADS / 64) {
        const int l = len[j], held = kvp_held(l, shift), inf = info[j], c = (inf >> 9) & 1, rows = rows_of(j);
        const int end = kvp_held(l + rows, shift), first = (inf & 255) ? held - 1 : held, b = base[j];
        int32_t *out = a.table_out + (int64_t)j * a.table_ld;
        for (int s = first + lane; s < a.table_ld; s += 64) {
            int v = -1;
            if (s < held) v = c ? pick(b) : tail[j] >= 0 ? tail[j] : a.table[(int64_t)par[j] * a.table_ld + s];
            else if (s < end) v = pick(b + c + s - held);
            out[s] = v;
        }
        if (lane == 0) {
            a.pos_out[j] = l;
            a.len_out[j] = l + rows;
            if (c) copies[4 * (inf >> 10) + 1] = pick(b);
        }
    }
}

// One block: where pages go, and the tables with it.
__global__ __launch_bounds__(KVP_THREADS) void k_kvp_compact(KvpCompactArgs a) {
    extern __shared__ uint32_t lds[];
    __shared__ int sums[KVP_THREADS / 64];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n_pages = a.pools.n_pages, nw = (n_pages + 31) / 32, shift = a.pools.shift, n = a.n_seq, cap = a.table_ld << shift;
    uint32_t *used = lds;
    int *copies = a.work + KVP_COPIES, *map = a.work + KVP_MAP;
    for (int i = t; i < nw; i += KVP_THREADS) used[i] = 0;
    __syncthreads();
    auto held_of = [&](int j) { return kvp_held(min(max(a.len[j], 0), cap), shift); };
    for (int j = wave; j < n; j += KVP_THREADS / 64) {
        const int32_t *row = a.table + (int64_t)j * a.table_ld;
        const int held = held_of(j);
        kvp_mark(row, held, false, n_pages, used, nullptr, 0, lane < held ? row[lane] : -1, [](int, int) {}, [](int) {});
    }
    __syncthreads();
    const int per_w = (nw + KVP_THREADS - 1) / KVP_THREADS, w0 = t * per_w;
    int in_use = 0, n_used, n_moved, dummy;
    for (int i = 0; i < per_w; i++) in_use += w0 + i < nw ? __popc(used[w0 + i]) : 0;
    block_scan(in_use, sums, &n_used);
    // bits of word w whose page comes before n_used
    auto low = [&](int w) { return w * 32 + 32 <= n_used ? ~0u : w * 32 >= n_used ? 0u : (1u << (n_used & 31)) - 1; };
    int from = 0, to = 0;
    for (int i = 0; i < per_w; i++)
        if (w0 + i < nw) {
            from += __popc(used[w0 + i] & ~low(w0 + i));
            to += __popc(~used[w0 + i] & low(w0 + i));
        }
    int src = block_scan(from, sums, &n_moved), dst = block_scan(to, sums, &dummy);
    for (int i = 0; i < per_w; i++) {
        if (w0 + i >= nw) break;
        for (uint32_t f = used[w0 + i] & ~low(w0 + i); f; f &= f - 1) {
            copies[4 * src] = (w0 + i) * 32 + __builtin_ctz(f);
            copies[4 * src++ + 2] = 1 << shift;
        }
        for (uint32_t f = ~used[w0 + i] & low(w0 + i); f; f &= f - 1) copies[4 * dst++ + 1] = (w0 + i) * 32 + __builtin_ctz(f);
    }
    if (t == 0) {
        a.status[0] = n_moved;
        a.status[1] = n_used;
        a.work[0] = n_moved;
    }
    __syncthreads();
    for (int i = t; i < n_moved; i += KVP_THREADS) map[copies[4 * i]] = copies[4 * i + 1];
    __syncthreads();
    for (int j = wave; j < n; j += KVP_THREADS / 64) {
        const int held = held_of(j);
        for (int s = lane; s < a.table_ld; s += 64) {
            const int64_t at = (int64_t)j * a.table_ld + s;
            int id = -1;
            if (s < held) {
                id = a.table[at];
                if (id >= n_used && id < n_pages) id = map[id];
            }
            a.table_out[at] = id;
        }
    }
}

// The copies of every pool, in slices of a page; as many blocks as stay busy, each
// taking what is left over in turn.  Only the positions that a page holds are moved.
__global__ __launch_bounds__(256) void k_kvp_copy(KvpPools p, const int *work, int slices) {
    const int64_t items = (int64_t)work[0] * p.n_pools * slices;
    const int64_t page = ((int64_t)p.heads << p.shift) * p.units;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int slice = (int)(item % slices);
        const int64_t rest = item / slices, pool = rest % p.n_pools;
        const int *c = work + KVP_COPIES + 4 * (rest / p.n_pools);
        const int per = c[2] * p.units, total = per * p.heads, gap = (p.units << p.shift) - per;
        const uint4 *src = reinterpret_cast<const uint4 *>(p.base + pool * p.pool_stride) + c[0] * page;
        uint4 *dst = reinterpret_cast<uint4 *>(p.base + pool * p.pool_stride) + c[1] * page;
        const int lo = (int)((int64_t)total * slice / slices), hi = (int)((int64_t)total * (slice + 1) / slices);
        for (int u = lo + threadIdx.x; u < hi; u += 4 * 256) {
            uint4 v[4];
            int at[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int x = u + i * 256;
                at[i] = x + x / per * gap;
                if (x < hi) v[i] = src[at[i]];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (u + i * 256 < hi) dst[at[i]] = v[i];
        }
    }
}

static hipError_t launch_copies(const KvpPools &p, const int *work, int64_t most, hipStream_t st) {
    const int64_t bytes = ((int64_t)p.heads << p.shift) * p.units * 16;
    const int64_t slices = std::min<int64_t>(64, std::max<int64_t>(1, bytes / 16384));
    const int64_t blocks = std::min<int64_t>(4096, most * p.n_pools * slices);
    if (blocks > 0) hipLaunchKernelGGL(k_kvp_copy, dim3((unsigned)blocks), dim3(256), 0, st, p, work, (int)slices);
    return hipGetLastError();
}

hipError_t launch_kvp_fork(const KvpForkArgs &a, hipStream_t st) {
    if (a.pools.n_pages > KVP_PAGES || a.n_out > QASR_KVP_MAX_SEQ) return hipErrorInvalidValue;
    const size_t lds = ((size_t)(a.pools.n_pages + 31) / 32 * 2 + 5 * (size_t)a.n_out + KVP_PICK) * 4;
    hipLaunchKernelGGL(k_kvp_fork, dim3(1), dim3(KVP_THREADS), lds, st, a);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_copies(a.pools, a.work, a.max_rows > 0 ? a.n_out : 0, st);
}

hipError_t launch_kvp_compact(const KvpCompactArgs &a, hipStream_t st) {
    if (a.pools.n_pages > KVP_PAGES || a.n_seq > QASR_KVP_MAX_SEQ) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_kvp_compact, dim3(1), dim3(KVP_THREADS), (size_t)(a.pools.n_pages + 31) / 32 * 4, st, a);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_copies(a.pools, a.work, std::min<int64_t>(a.pools.n_pages / 2, (int64_t)a.n_seq * a.table_ld), st);
}

// ---------------------------------------------------------------------------
// write
// ---------------------------------------------------------------------------

// Rows of K and V to their pages, 8 values a thread and step; memory-bound, for a row
// or two a sequence one launch.
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
        *reinterpret_cast<uint4 *>(to) = o;
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
