// sequence_memory.hip -- copies of blocks and states (sequence_memory.h), and the tables of branching sequences: forks that
// share whole blocks by count, compaction of a pool, and the release of a table's blocks.
#include "sequence_memory.h"

#include <algorithm>
#include <atomic>
#include <mutex>
#include <new>
#include <numeric>
#include <unordered_map>

namespace nvllm {

bool stream_is_captured() {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    HIP_CHECK(hipStreamIsCapturing(rt().stream, &st));
    return st != hipStreamCaptureStatusNone;
}

// ------------------------------------------------------------------ the copy
// A program is a list of moves (slot, slot) that a thread makes for its own bytes of a slot, in every array alike: no thread
// touches another's bytes, so programs with different slots need no order, and a cycle of slots is one program with a value set
// aside (slot -1).  A slot is written after its last reading, so the readings of four moves are in flight before the first of
// their writes.  Moves that share a source read it once.  What is written is not kept in the caches, where it would drive out what is still
// to be read (369 MB of blocks: 76.4 us kept, 70.6 not; readings past the caches too: 66.6, but 11.4 us for 9.2 where all fits them).
// Bound by memory, 5.2 TB/s as a copy of 1 GiB, and by the launch and three trips to memory behind one another where there is
// little to copy.
constexpr int COPY_SETS = 6, COPY_INLINE = 200, COPY_FAN = 4, COPY_BATCH = 4;
struct CopySet {
    char* base;
    size_t stride;
    unsigned units;   // per slot
    int first;        // array
};
struct CopyArgs {
    CopySet sets[COPY_SETS];
    int n_programs;
    unsigned piece;               // of every slot, the launch's first
    const int* programs;          // null: the ints are right here
    int here[COPY_INLINE];        // [n_programs + 1] first moves, then moves (from, to)
};

template <typename U>
__device__ __forceinline__ void store_past_caches(U* p, const U& v) {
    typedef unsigned int q4_t __attribute__((ext_vector_type(4)));
    if constexpr (sizeof(U) == 16) __builtin_nontemporal_store(__builtin_bit_cast(q4_t, v), reinterpret_cast<q4_t*>(p));
    else __builtin_nontemporal_store(v, p);
}

template <typename U, int N, bool HERE>
__global__ __launch_bounds__(256) void k_copy_slots(CopyArgs a) {
    const int array = blockIdx.y, program = blockIdx.x % a.n_programs;
    const unsigned first = (a.piece + blockIdx.x / a.n_programs) * (256 * N) + threadIdx.x;
    CopySet set = a.sets[0];
#pragma unroll
    for (int i = 1; i < COPY_SETS; i++)   // (sets that are not there begin behind the last array)
        if (array >= a.sets[i].first) set = a.sets[i];
    if (first >= set.units) return;
    U* base = reinterpret_cast<U*>(set.base + (size_t)(array - set.first) * set.stride);
    auto number = [&](int i) { return __builtin_amdgcn_readfirstlane(HERE ? a.here[i] : a.programs[i]); };
    const int begin = number(program), end = number(program + 1), moves = a.n_programs + 1;
    U aside[N] = {};
    for (int m = begin; m < end; m += COPY_BATCH) {
        int from[COPY_BATCH], to[COPY_BATCH];
#pragma unroll
        for (int j = 0; j < COPY_BATCH; j++) {   // (behind the last move: the last one)
            from[j] = number(moves + 2 * min(m + j, end - 1));
            to[j] = number(moves + 2 * min(m + j, end - 1) + 1);
        }
        U v[COPY_BATCH][N] = {};
#pragma unroll
        for (int j = 0; j < COPY_BATCH; j++) {
            if (m + j >= end) break;
            if (from[j] < 0) {
#pragma unroll
                for (int i = 0; i < N; i++) v[j][i] = aside[i];
            } else if (j > 0 && from[j] == from[j - 1]) {
#pragma unroll
                for (int i = 0; i < N; i++) v[j][i] = v[j - 1][i];
            } else {
                const U* s = base + (size_t)from[j] * set.units;
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (first + 256 * i < set.units) v[j][i] = s[first + 256 * i];
            }
            if (to[j] < 0)
#pragma unroll
                for (int i = 0; i < N; i++) aside[i] = v[j][i];
        }
#pragma unroll
        for (int j = 0; j < COPY_BATCH; j++) {
            if (m + j >= end) break;
            if (to[j] < 0) continue;
            U* d = base + (size_t)to[j] * set.units;
#pragma unroll
            for (int i = 0; i < N; i++)
                if (first + 256 * i < set.units) store_past_caches(d + first + 256 * i, v[j][i]);
        }
    }
}

// The moves of a copy as programs: [n + 1] first moves, and the moves (from, to).
struct CopyPlan {
    std::vector<int> first, moves;
    int programs() const { return (int)first.size() - 1; }
    void add(int from, int to) {
        moves.push_back(from);
        moves.push_back(to);
    }
    void end() { first.push_back((int)moves.size() / 2); }
};
// Slots that meet are in one program, a slot is written after its last reading.  0 or a refusal.
static int plan_moves(const int* from, const int* to, int n, int n_slots, CopyPlan& plan) {
    // slots by number, or by their place among those that occur if they are few of many
    std::vector<int> slots;
    const bool dense = n_slots <= 16384 || n_slots / 8 <= n;
    for (int i = 0; i < n; i++) {
        if (from[i] < 0 || from[i] >= n_slots || to[i] < 0 || to[i] >= n_slots) return NVLLM_BAD_INDEX;
        if (dense) continue;
        slots.push_back(from[i]);
        slots.push_back(to[i]);
    }
    std::sort(slots.begin(), slots.end());
    slots.erase(std::unique(slots.begin(), slots.end()), slots.end());
    auto at = [&](int s) { return dense ? s : (int)(std::lower_bound(slots.begin(), slots.end(), s) - slots.begin()); };
    auto slot = [&](int k) { return dense ? k : slots[k]; };
    const int k = dense ? n_slots : (int)slots.size();
    std::vector<int> source((size_t)k, -1), uses((size_t)k, 0);
    std::vector<char> written((size_t)k, 0);
    int count = 0;
    for (int i = 0; i < n; i++) {
        const int d = at(to[i]), s = at(from[i]);
        if (written[d]) return NVLLM_BAD_INDEX;   // two values for one slot
        written[d] = 1;
        if (s == d) continue;
        source[d] = s;
        uses[s]++;
        count++;
    }
    plan.first.reserve((size_t)count + 1);
    plan.moves.reserve(2 * (size_t)count + 8);
    plan.first.push_back(0);
    bool apart = true;   // nobody reads what somebody writes
    for (int i = 0; i < n && apart; i++) apart = source[at(to[i])] < 0 || uses[at(to[i])] == 0;
    if (apart) {
        // a fan out of one source falls into programs of a few moves each
        std::vector<int> by_source((size_t)n), place((size_t)k, -1);
        int next = 0;
        for (int i = 0; i < n; i++) {
            const int d = at(to[i]), s = source[d];
            if (s < 0) continue;
            if (place[s] < 0) {
                place[s] = next;
                next += uses[s];
            }
            by_source[place[s]++] = d;
        }
        for (int i = 0, run = 0; i < next; i++) {
            plan.add(slot(source[by_source[i]]), slot(by_source[i]));
            run++;
            if (run == COPY_FAN || i + 1 == next || source[by_source[i + 1]] != source[by_source[i]]) {
                plan.end();
                run = 0;
            }
        }
        return 0;
    }
    std::vector<int> group((size_t)k), order, ready;   // order: pairs of places, -1: aside
    std::iota(group.begin(), group.end(), 0);
    auto root = [&](int x) {
        while (group[x] != x) x = group[x] = group[group[x]];
        return x;
    };
    for (int i = 0; i < n; i++) {
        const int d = at(to[i]);
        if (source[d] < 0) continue;
        group[root(d)] = root(source[d]);
        if (uses[d] == 0) ready.push_back(d);
    }
    while (!ready.empty()) {
        const int d = ready.back(), s = source[d];
        ready.pop_back();
        order.insert(order.end(), {s, d});
        source[d] = -1;
        if (--uses[s] == 0 && source[s] >= 0) ready.push_back(s);
    }
    for (int i = 0; i < n; i++) {   // what is left are cycles
        const int c = at(to[i]);
        if (source[c] < 0) continue;
        int d = c;
        order.insert(order.end(), {c, -1});
        while (source[d] != c) {
            order.insert(order.end(), {source[d], d});
            const int next = source[d];
            source[d] = -1;
            d = next;
        }
        order.insert(order.end(), {-1, d});
        source[d] = -1;
    }
    auto group_of = [&](size_t m) { return root(order[m + 1] >= 0 ? order[m + 1] : order[m]); };
    std::vector<int> size((size_t)k, 0), roots;
    for (size_t m = 0; m < order.size(); m += 2) {
        const int r = group_of(m);
        if (size[r]++ == 0) roots.push_back(r);
    }
    int next = 0;
    for (int r : roots) {
        const int had = size[r];
        size[r] = next;
        next += had;
        plan.first.push_back(next);
    }
    plan.moves.resize(order.size());
    for (size_t m = 0; m < order.size(); m += 2) {
        const size_t place = 2 * (size_t)size[group_of(m)]++;
        plan.moves[place] = order[m] < 0 ? -1 : slot(order[m]);
        plan.moves[place + 1] = order[m + 1] < 0 ? -1 : slot(order[m + 1]);
    }
    return 0;
}

constexpr long GRID_MOST = 0xffffffffL / 256;   // workgroups: a grid has fewer than 2^32 threads

template <typename U>
static void launch_copy(CopyArgs& a, unsigned most_units, int arrays, double bytes) {
    constexpr int N = 2;
    const long pieces = ((long)most_units + 256 * N - 1) / (256 * N), at_once = std::max(1L, std::min(pieces, GRID_MOST / a.n_programs));
    for (long p = 0; p < pieces; p += at_once) {
        a.piece = (unsigned)p;
        const long n = std::min(at_once, pieces - p);
        const dim3 grid((unsigned)(n * a.n_programs), arrays);
        ProfScope ps(PC_SLOT_COPY, bytes * n / pieces, 0);
        if (a.programs) NVLLM_LAUNCH((k_copy_slots<U, N, false>), grid, dim3(256), 0, a);
        else NVLLM_LAUNCH((k_copy_slots<U, N, true>), grid, dim3(256), 0, a);
    }
}

int copy_slots(const std::vector<SlotArrays>& arrays, int n_slots, const int* from, const int* to, int n) {
    CopyPlan plan;
    if (const int e = plan_moves(from, to, n, n_slots, plan)) return e;
    if (plan.moves.empty()) return 0;
    const size_t ints = plan.first.size() + plan.moves.size();
    size_t bits = 0;   // of every address and size
    for (const SlotArrays& s : arrays) {
        bits |= (size_t)s.base | s.slot_bytes | (s.count > 1 ? s.stride : 0);
        if (s.count < 0 || s.count > 65535) return NVLLM_BAD_SIZE;
    }
    const size_t unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
    for (const SlotArrays& s : arrays)
        if (s.slot_bytes / unit > 0x7fffffff) return NVLLM_BAD_SIZE;
    if (ints + 4 > staging_ints()) return NVLLM_BAD_SIZE;
    ensure_init();
    if (stream_is_captured()) return NVLLM_CAPTURED;
    CopyArgs a{};
    a.n_programs = plan.programs();
    const bool here = ints <= COPY_INLINE;
    int* dev = here ? nullptr : (int*)ws_try(WS_STEP, (ints + 4) * sizeof(int));
    if (!here && !dev) return NVLLM_NO_MEMORY;
    int* host = here ? a.here : pinned_ints((ints + 3) & ~(size_t)3);
    std::copy(plan.first.begin(), plan.first.end(), host);
    std::copy(plan.moves.begin(), plan.moves.end(), host + plan.first.size());
    if (!here) {
        launch_copy_ints(dev, host, ints);
        a.programs = dev;
    }
    for (size_t i = 0; i < arrays.size();) {
        int total = 0, sets = 0;
        unsigned most = 0;
        double part = 0;
        for (; i < arrays.size() && sets < COPY_SETS && total + arrays[i].count <= 65535; i++) {
            const SlotArrays& s = arrays[i];
            if (s.count == 0 || s.slot_bytes == 0) continue;
            a.sets[sets++] = CopySet{(char*)s.base, s.stride, (unsigned)(s.slot_bytes / unit), total};
            most = std::max(most, (unsigned)(s.slot_bytes / unit));
            part += 2.0 * n * (double)s.slot_bytes * s.count;
            total += s.count;
        }
        for (int j = sets; j < COPY_SETS; j++) a.sets[j] = CopySet{nullptr, 0, 0, 0x7fffffff};
        if (total == 0) continue;
        if (unit == 16) launch_copy<uint4>(a, most, total, part);
        else if (unit == 4) launch_copy<unsigned>(a, most, total, part);
        else launch_copy<unsigned char>(a, most, total, part);
    }
    return 0;
}

// ------------------------------------------------------------------ shared blocks
// Users of a block beside its first, per manager (by its free stack, which no other has).  Without forks there is no entry.  Threads that each keep a pool of their own meet in the
// map, not in an entry, which stays where it is when others come and go.
static std::mutex& shared_lock() {
    static std::mutex m;
    return m;
}
static std::unordered_map<const int*, std::vector<int>>& shared() {
    static std::unordered_map<const int*, std::vector<int>> m;
    return m;
}
static std::atomic<int> g_forked{0};   // entries: without one, as in programs that never fork, freeing a block takes no lock
static std::vector<int>* users_of(const KVCacheManager* mgr) {   // null: no forks
    if (g_forked.load() == 0) return nullptr;
    std::lock_guard<std::mutex> lock(shared_lock());
    const auto it = shared().find(mgr->free_block_indices);
    return it == shared().end() ? nullptr : &it->second;
}
static std::vector<int>* make_users(const KVCacheManager* mgr) {
    std::lock_guard<std::mutex> lock(shared_lock());
    std::vector<int>& users = shared()[mgr->free_block_indices];
    g_forked = (int)shared().size();
    if ((int)users.size() < mgr->num_blocks) users.resize((size_t)mgr->num_blocks, 0);
    return &users;
}
// users of a block beside its first, for reading and writing; null: none
static int* more_users(const KVCacheManager* mgr, int block) {
    std::vector<int>* u = users_of(mgr);
    return !u || block < 0 || block >= (int)u->size() || (*u)[block] == 0 ? nullptr : &(*u)[block];
}
bool drop_shared_block(const KVCacheManager* mgr, int block) {
    int* more = more_users(mgr, block);
    if (!more) return false;
    (*more)--;
    return true;
}
void forget_shared_blocks(const int* stack) {
    std::lock_guard<std::mutex> lock(shared_lock());
    shared().erase(stack);
    g_forked = (int)shared().size();
}

// which blocks lie on the free stack; empty: the stack is not one of this pool
static std::vector<char> free_blocks(const KVCacheManager* mgr) {
    std::vector<char> is_free((size_t)mgr->num_blocks, 0);
    if (mgr->free_blocks_count < 0 || mgr->free_blocks_count > mgr->num_blocks) return {};
    for (int i = 0; i < mgr->free_blocks_count; i++) {
        const int b = mgr->free_block_indices[i];
        if (b < 0 || b >= mgr->num_blocks || is_free[b]) return {};
        is_free[b] = 1;
    }
    return is_free;
}
// A table's release: how many blocks go back to the pool; a refusal for a table that names a block twice, or one that is free.  A shared block is
// in use; the free stack, which the caller may write too, is read for the others (a release of 33 blocks: 0.4 us beside 512 free ones, 2.0 beside
// 8,192).
static int blocks_to_free(const KVCacheManager* mgr, const BlockTable* table, const std::vector<int>* users) {
    const unsigned n = (unsigned)mgr->num_blocks;
    static thread_local std::vector<unsigned char> marks;   // all zeros between calls
    if (marks.size() < (size_t)n + 1) marks.resize((size_t)n + 1, 0);
    unsigned char* mark = marks.data();
    auto shared = [&](unsigned b) { return users && b < users->size() && (*users)[b] > 0; };
    int met = 0, back = 0;
    for (; met < table->num_blocks; met++) {
        const unsigned b = (unsigned)table->block_indices[met];
        if (b >= n || mark[b]) break;
        mark[b] = shared(b) ? 1 : 2;
        back += mark[b] - 1;
    }
    bool fits = met == table->num_blocks && mgr->free_blocks_count >= 0 && mgr->free_blocks_count <= mgr->num_blocks - back;
    if (fits && back > 0) {
        mark[n] = 2;   // (what is no block of the pool)
        unsigned char any = 0;
        for (int i = 0; i < mgr->free_blocks_count; i++) any |= mark[std::min((unsigned)mgr->free_block_indices[i], n)];
        mark[n] = 0;
        fits = any < 2;
    }
    while (met-- > 0) mark[table->block_indices[met]] = 0;
    return fits ? back : NVLLM_BAD_INDEX;
}
static bool usable(const KVCacheManager* mgr) { return mgr && mgr->free_block_indices && mgr->num_blocks > 0 && mgr->block_size > 0; }

}  // namespace nvllm

using namespace nvllm;

// Every entry point: no exception crosses it, nothing is changed when it refuses.
#define REFUSING(...)                  \
    try {                              \
        __VA_ARGS__                    \
    } catch (const std::bad_alloc&) {  \
        return NVLLM_NO_MEMORY;        \
    }

extern "C" {

int nvllm_copy_states(void* state, size_t slot_bytes, int n_layers, int n_slots, const int* from, const int* to, int n) {
    if (n < 0 || n_layers < 0 || n_slots < 0 || (n > 0 && (!state || !from || !to))) return NVLLM_BAD_ARGUMENT;
    if (n == 0 || n_layers == 0 || slot_bytes == 0) return 0;
    if (slot_bytes > ((size_t)1 << 46) / (size_t)std::max(1, n_slots)) return NVLLM_BAD_SIZE;
    REFUSING(return copy_slots({SlotArrays{state, slot_bytes, slot_bytes * n_slots, n_layers}}, n_slots, from, to, n);)
}

int nvllm_copy_blocks(KVCacheManager* mgr, const int* from, const int* to, int n) {
    if (!usable(mgr) || n < 0 || (n > 0 && (!from || !to))) return NVLLM_BAD_ARGUMENT;
    if (n == 0) return 0;
    REFUSING(
        const std::vector<SlotArrays> arrays = pool_arrays(mgr);
        if (arrays.empty()) return NVLLM_BAD_SIZE;
        return copy_slots(arrays, mgr->num_blocks, from, to, n);)
}

int nvllm_fork_tables(KVCacheManager* mgr, const BlockTable* from, int positions, BlockTable** to, int n) {
    if (!usable(mgr) || !from || positions < 0 || n < 0 || (n > 0 && !to)) return NVLLM_BAD_ARGUMENT;
    if (n == 0) return 0;
    REFUSING(
        const std::vector<SlotArrays> arrays = pool_arrays(mgr);
        if (arrays.empty()) return NVLLM_BAD_SIZE;
        const int whole = positions / mgr->block_size, tail = positions % mgr->block_size != 0;
        if (from->num_blocks < whole + tail || (whole + tail > 0 && !from->block_indices)) return NVLLM_BAD_INDEX;
        const std::vector<char> is_free = free_blocks(mgr);
        if (is_free.empty()) return NVLLM_BAD_INDEX;
        std::vector<char> seen((size_t)mgr->num_blocks, 0);
        for (int i = 0; i < whole + tail; i++) {
            const int b = from->block_indices[i];
            if (b < 0 || b >= mgr->num_blocks || is_free[b] || seen[b]) return NVLLM_BAD_INDEX;
            seen[b] = 1;
        }
        std::vector<BlockTable*> children(to, to + n);
        for (BlockTable* t : children)
            if (!t || t == from || (whole + tail > 0 && !t->block_indices)) return NVLLM_BAD_ARGUMENT;
        std::sort(children.begin(), children.end());
        if (std::adjacent_find(children.begin(), children.end()) != children.end()) return NVLLM_BAD_ARGUMENT;
        if (tail && mgr->free_blocks_count < n) return NVLLM_NO_BLOCKS;
        std::vector<int> source, target;
        if (tail) {
            source.assign((size_t)n, from->block_indices[whole]);
            for (int i = 0; i < n; i++) target.push_back(mgr->free_block_indices[mgr->free_blocks_count - 1 - i]);
        }
        std::vector<int>* users = nullptr;
        if (whole > 0) users = make_users(mgr);
        if (tail)
            if (const int e = copy_slots(arrays, mgr->num_blocks, source.data(), target.data(), n)) return e;
        // (nothing below fails)
        for (int i = 0; i < whole; i++) (*users)[from->block_indices[i]] += n;
        for (int i = 0; i < n; i++) {
            std::copy(from->block_indices, from->block_indices + whole, to[i]->block_indices);
            if (tail) to[i]->block_indices[whole] = alloc_block(mgr);
            to[i]->num_blocks = whole + tail;
        }
        return 0;)
}

int nvllm_block_users(const KVCacheManager* mgr, int block) {
    if (!usable(mgr) || block < 0 || block >= mgr->num_blocks) return NVLLM_BAD_ARGUMENT;
    for (int i = 0; i < mgr->free_blocks_count; i++)
        if (mgr->free_block_indices[i] == block) return 0;
    const int* more = more_users(mgr, block);
    return 1 + (more ? *more : 0);
}

int nvllm_free_table(KVCacheManager* mgr, BlockTable* table) {
    if (!usable(mgr) || !table || table->num_blocks < 0 || (table->num_blocks > 0 && !table->block_indices)) return NVLLM_BAD_ARGUMENT;
    if (table->num_blocks == 0) return 0;
    REFUSING(
        std::vector<int>* users = users_of(mgr);
        const int back = blocks_to_free(mgr, table, users);
        if (back < 0) return back;
        for (; table->num_blocks > 0; table->num_blocks--) {
            const int b = table->block_indices[table->num_blocks - 1];
            if (users && b < (int)users->size() && (*users)[b] > 0) (*users)[b]--;
            else mgr->free_block_indices[mgr->free_blocks_count++] = b;
        }
        return 0;)
}

int nvllm_compact_blocks(KVCacheManager* mgr, BlockTable** tables, int n) {
    if (!usable(mgr) || n < 0 || (n > 0 && !tables)) return NVLLM_BAD_ARGUMENT;
    REFUSING(
        const std::vector<SlotArrays> arrays = pool_arrays(mgr);
        if (arrays.empty()) return NVLLM_BAD_SIZE;
        std::vector<char> is_free = free_blocks(mgr);
        if (is_free.empty()) return NVLLM_BAD_INDEX;
        // how many of the given tables have a block: one that others use too stays where it is, like one that no table has
        std::vector<int> found((size_t)mgr->num_blocks, 0);
        std::vector<const BlockTable*> last((size_t)mgr->num_blocks, nullptr);   // (a table that names a block twice is one)
        std::vector<BlockTable*> all(tables, tables + n);
        std::sort(all.begin(), all.end());
        if (std::adjacent_find(all.begin(), all.end()) != all.end()) return NVLLM_BAD_ARGUMENT;
        for (const BlockTable* t : all) {
            if (!t || t->num_blocks < 0 || (t->num_blocks > 0 && !t->block_indices)) return NVLLM_BAD_ARGUMENT;
            for (int i = 0; i < t->num_blocks; i++) {
                const int b = t->block_indices[i];
                if (b < 0 || b >= mgr->num_blocks || is_free[b]) return NVLLM_BAD_INDEX;
                found[b] += last[b] != t;
                last[b] = t;
            }
        }
        const int used = mgr->num_blocks - mgr->free_blocks_count;
        std::vector<int>* users = users_of(mgr);
        if (users && (int)users->size() < mgr->num_blocks) users->resize((size_t)mgr->num_blocks, 0);
        std::vector<int> from, to, place((size_t)mgr->num_blocks);
        std::iota(place.begin(), place.end(), 0);
        int hole = 0;
        for (int b = used; b < mgr->num_blocks; b++) {
            if (is_free[b] || found[b] == 0 || (users && found[b] < 1 + (*users)[b])) continue;
            while (!is_free[hole]) hole++;   // (there are as many below `used` as blocks in use behind it)
            from.push_back(b);
            to.push_back(hole);
            place[b] = hole++;
        }
        if (!from.empty())
            if (const int e = copy_slots(arrays, mgr->num_blocks, from.data(), to.data(), (int)from.size())) return e;
        // (nothing below fails)
        for (size_t i = 0; i < from.size(); i++) {
            is_free[from[i]] = 1;
            is_free[to[i]] = 0;
            if (users) std::swap((*users)[from[i]], (*users)[to[i]]);
        }
        for (BlockTable* t : all)
            for (int i = 0; i < t->num_blocks; i++) t->block_indices[i] = place[t->block_indices[i]];
        int count = 0;
        for (int b = mgr->num_blocks - 1; b >= 0; b--)
            if (is_free[b]) mgr->free_block_indices[count++] = b;
        return (int)from.size();)
}

}  // extern "C"
