// extern "C" boundary of the paged cache: the page pool with its reference counts, and the calls on a batch of sequences.
// Host code only.
#include <hip/hip_runtime.h>

#include <cmath>
#include <new>
#include <vector>

#include "../../include/vfkv.h"
#include "api_internal.h"
#include "device_utils.h"
#include "paged.h"

using vfkv::fail;
using vfkv::hip_fail;

struct vfkv_pages {
    vfkv_pages_config cfg;
    uint32_t page_shift;
    uint64_t page_bytes, layer_bytes, bytes;   // one page of one layer, one layer, the whole buffer (one tensor)
    void* k;
    void* v;
    bool owns;
    int device;                                // where the buffers are; -1 without buffers
    std::vector<uint32_t> refs;                // per page; 0 = free
    std::vector<uint64_t> mark;                // per page: stamp of the last call that named it
    uint64_t stamp;
    uint32_t n_free, lowest;                   // no page below `lowest` is free
};

namespace {

#define VFKV_HIP(call)                                    \
    do {                                                  \
        hipError_t e_ = (call);                           \
        if (e_ != hipSuccess) return hip_fail(e_, #call); \
    } while (0)

inline hipStream_t S(vfkv_stream s) { return reinterpret_cast<hipStream_t>(s); }

// Nothing may be thrown across the C boundary: the host arrays of the pool are the only things that could.
template <typename F>
int guarded(const char* who, F&& f) {
    try {
        return f();
    } catch (...) {
        return fail(VFKV_ERR_HIP, "%s: host allocation failed", who);
    }
}

// The buffers' device must be the current one: work is enqueued there.
int check_device(int device, const char* who, const char* what) {
    int dev = -1;
    VFKV_HIP(hipGetDevice(&dev));
    if (dev != device) return fail(VFKV_ERR_INVALID_ARG, "%s: the %s is on device %d, the current device is %d", who, what, device, dev);
    return VFKV_OK;
}

int check_pages(const vfkv_pages* c, uint32_t layer, const char* who) {
    if (!c || !c->k || !c->v) return fail(VFKV_ERR_INVALID_ARG, "%s: cache has no buffers", who);
    if (layer >= c->cfg.n_layers) return fail(VFKV_ERR_INVALID_ARG, "%s: layer %u out of range", who, layer);
    return VFKV_OK;
}

// Sets *nothing when the batch has no rows.
int check_batch(const vfkv_pages* c, const vfkv_seq_batch* b, const char* who, vfkv::PagedSeqs* out, uint32_t* max_kv, bool* nothing) {
    if (!b) return fail(VFKV_ERR_INVALID_ARG, "%s: batch is NULL", who);
    *nothing = b->n_seqs == 0u || b->n_tokens == 0u;
    if (*nothing) return VFKV_OK;
    if (!b->page_table || !b->kv_lens) return fail(VFKV_ERR_INVALID_ARG, "%s: NULL page table or lengths", who);
    if ((((uintptr_t)b->page_table | (uintptr_t)b->kv_lens | (uintptr_t)b->q_offsets) & 3u) != 0u)
        return fail(VFKV_ERR_ALIGNMENT, "%s: the batch's arrays must be 4-byte aligned", who);
    if (b->n_seqs > vfkv::kPagedMaxSeqs) return fail(VFKV_ERR_UNSUPPORTED, "%s: %u sequences (at most %u in one call)", who, b->n_seqs, vfkv::kPagedMaxSeqs);
    if (b->table_stride == 0u) return fail(VFKV_ERR_INVALID_ARG, "%s: table_stride must be > 0", who);
    if (b->n_tokens >= 1u << 24) return fail(VFKV_ERR_UNSUPPORTED, "%s: %u tokens (less than 2^24 in one call)", who, b->n_tokens);
    if (!b->q_offsets && b->n_tokens != b->n_seqs)
        return fail(VFKV_ERR_INVALID_ARG, "%s: without q_offsets every sequence has one token (%u tokens, %u sequences)", who, b->n_tokens, b->n_seqs);
    const uint64_t held = (uint64_t)b->table_stride << c->page_shift;
    out->table = b->page_table; out->kv_lens = b->kv_lens; out->q_offsets = b->q_offsets;
    out->n_seqs = b->n_seqs; out->table_stride = b->table_stride; out->n_tokens = b->n_tokens;
    out->limit = held < vfkv::kPagedMaxLen ? (uint32_t)held : vfkv::kPagedMaxLen;
    *max_kv = b->max_kv_len != 0u && b->max_kv_len < out->limit ? b->max_kv_len : out->limit;
    return VFKV_OK;
}

vfkv::PagedSlab slab(const vfkv_pages* c, uint32_t layer) {
    vfkv::PagedSlab p;
    p.k = (const uint8_t*)c->k + layer * c->layer_bytes;
    p.v = (const uint8_t*)c->v + layer * c->layer_bytes;
    p.page_bytes = c->page_bytes;
    p.n_pages = c->cfg.n_pages; p.page_shift = c->page_shift; p.n_kv_heads = c->cfg.n_kv_heads; p.head_dim = c->cfg.head_dim;
    p.dtype = c->cfg.dtype;
    return p;
}

// A row stride in elements: 0 means contiguous rows, less than a row is an error.
int row_stride(uint32_t given, uint64_t row, const char* who, const char* what, uint64_t* out) {
    if (given != 0u && given < row)
        return fail(VFKV_ERR_INVALID_ARG, "%s: %s_stride %u is less than a row (%llu elements)", who, what, given, (unsigned long long)row);
    *out = given ? given : row;
    return VFKV_OK;
}

constexpr uint64_t kPrefillRows = 65536;       // partial rows a paged workspace has at least

int check_io(uint32_t io, const char* who) {
    if (io != VFKV_F32 && io != VFKV_F16) return fail(VFKV_ERR_INVALID_ARG, "%s: io_dtype %u (F32 and F16 are built)", who, io);
    return VFKV_OK;
}

int copy_pages(vfkv_pages* c, const uint32_t* src, const uint32_t* dst, const uint32_t* rows, uint32_t n, vfkv_stream stream) {
    vfkv::PagedCopyLaunch L;
    L.k = (uint8_t*)c->k; L.v = (uint8_t*)c->v;
    L.layer_bytes = c->layer_bytes; L.page_bytes = c->page_bytes;
    L.n_layers = c->cfg.n_layers; L.n_kv_heads = c->cfg.n_kv_heads; L.page_size = c->cfg.page_size;
    L.row_bytes = c->cfg.head_dim * vfkv::elem_size(c->cfg.dtype);
    for (uint32_t i = 0; i < n; i += vfkv::kCopyPairs) {
        L.n = n - i < vfkv::kCopyPairs ? n - i : vfkv::kCopyPairs;
        L.src = src + i; L.dst = dst + i; L.rows = rows ? rows + i : nullptr;
        VFKV_HIP(vfkv::launch_paged_copy(L, S(stream)));
    }
    return VFKV_OK;
}

// Takes the n lowest free pages (the caller has checked that there are n).
void take(vfkv_pages* c, uint32_t n, uint32_t* out) {
    uint32_t p = c->lowest;
    for (uint32_t i = 0; i < n; ++p)
        if (c->refs[p] == 0u) { c->refs[p] = 1u; out[i++] = p; }
    c->n_free -= n;
    if (n != 0u) c->lowest = p;
}

void drop(vfkv_pages* c, uint32_t page) {
    if (--c->refs[page] == 0u) {
        ++c->n_free;
        if (page < c->lowest) c->lowest = page;
    }
}

}  // namespace

extern "C" {

int vfkv_pages_create_external(const vfkv_pages_config* cfg, void* k_buffer, void* v_buffer, vfkv_pages** out) {
    if (!out) return fail(VFKV_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (!cfg) return fail(VFKV_ERR_INVALID_ARG, "pages config is NULL");
    if (cfg->dtype > VFKV_F8E4M3) return fail(VFKV_ERR_INVALID_ARG, "unknown kv dtype %u", cfg->dtype);
    if (cfg->n_layers == 0u || cfg->n_kv_heads == 0u || cfg->head_dim == 0u || cfg->n_pages == 0u)
        return fail(VFKV_ERR_INVALID_ARG, "pages: n_layers, n_kv_heads, head_dim and n_pages must be > 0");
    if (cfg->head_dim > 512u) return fail(VFKV_ERR_UNSUPPORTED, "pages: head_dim %u > 512", cfg->head_dim);
    if (cfg->n_layers > 32767u) return fail(VFKV_ERR_UNSUPPORTED, "pages: %u layers", cfg->n_layers);
    if (cfg->n_kv_heads > 16384u) return fail(VFKV_ERR_UNSUPPORTED, "pages: %u KV heads", cfg->n_kv_heads);
    const uint32_t ps = cfg->page_size;
    if (ps < 16u || ps > 256u || (ps & (ps - 1u)) != 0u)
        return fail(VFKV_ERR_INVALID_ARG, "pages: page_size must be 16, 32, 64, 128 or 256 (got %u)", ps);
    if ((uint64_t)cfg->n_pages * ps > 0x7FFFFFFFu)
        return fail(VFKV_ERR_OVERFLOW, "pages: n_pages * page_size (%llu) exceeds 2^31 - 1", (unsigned long long)cfg->n_pages * ps);
    if ((k_buffer == nullptr) != (v_buffer == nullptr)) return fail(VFKV_ERR_INVALID_ARG, "pages: one of the two buffers is NULL");
    if ((((uintptr_t)k_buffer | (uintptr_t)v_buffer) & 15u) != 0u)
        return fail(VFKV_ERR_ALIGNMENT, "pages: buffers must be 16-byte aligned");
    const uint64_t page_bytes = (uint64_t)cfg->n_kv_heads * ps * cfg->head_dim * vfkv::elem_size(cfg->dtype);   // < 2^34
    uint64_t layer_bytes, bytes;
    if (__builtin_mul_overflow(page_bytes, (uint64_t)cfg->n_pages, &layer_bytes) || __builtin_mul_overflow(layer_bytes, (uint64_t)cfg->n_layers, &bytes))
        return fail(VFKV_ERR_OVERFLOW, "pages: size overflow");
    return guarded("pages", [&]() -> int {
        vfkv_pages* c = new vfkv_pages();
        c->cfg = *cfg;
        c->page_shift = (uint32_t)__builtin_ctz(ps);
        c->page_bytes = page_bytes; c->layer_bytes = layer_bytes; c->bytes = bytes;
        c->k = k_buffer; c->v = v_buffer; c->owns = false; c->device = -1;
        c->stamp = 0u; c->n_free = cfg->n_pages; c->lowest = 0u;
        try {
            c->refs.assign(cfg->n_pages, 0u);
            c->mark.assign(cfg->n_pages, 0u);
        } catch (...) {
            delete c;
            throw;
        }
        if (k_buffer) {
            if (hipGetDevice(&c->device) != hipSuccess) c->device = -1;           // (no device: every compute call fails later)
            for (void* p : {k_buffer, v_buffer}) {
                hipPointerAttribute_t at;
                if (hipPointerGetAttributes(&at, p) != hipSuccess) {
                    (void)hipGetLastError();                                      // not a pointer the runtime knows: nothing to compare
                } else if (at.type == hipMemoryTypeDevice && at.device != c->device) {
                    const int there = at.device, here = c->device;
                    delete c;
                    return fail(VFKV_ERR_INVALID_ARG, "pages: a buffer is on device %d, the current device is %d", there, here);
                }
            }
        }
        *out = c;
        return VFKV_OK;
    });
}

int vfkv_pages_create(const vfkv_pages_config* cfg, vfkv_pages** out) {
    vfkv_pages* c = nullptr;
    const int rc = vfkv_pages_create_external(cfg, nullptr, nullptr, &c);
    if (out) *out = nullptr;
    if (rc != VFKV_OK) return rc;
    if (!out) { vfkv_pages_destroy(c); return fail(VFKV_ERR_INVALID_ARG, "out is NULL"); }
    hipError_t e = hipGetDevice(&c->device);
    if (e == hipSuccess) e = hipMalloc(&c->k, c->bytes);
    if (e == hipSuccess) {
        e = hipMalloc(&c->v, c->bytes);
        if (e != hipSuccess) { (void)hipFree(c->k); c->k = nullptr; }
    }
    if (e != hipSuccess) { delete c; return hip_fail(e, "hipMalloc(pages)"); }
    c->owns = true;
    *out = c;
    return VFKV_OK;
}

void vfkv_pages_destroy(vfkv_pages* c) {
    if (!c) return;
    if (c->owns) {
        if (c->k) (void)hipFree(c->k);
        if (c->v) (void)hipFree(c->v);
    }
    delete c;
}

void* vfkv_pages_k_ptr(const vfkv_pages* c) { return c ? c->k : nullptr; }
void* vfkv_pages_v_ptr(const vfkv_pages* c) { return c ? c->v : nullptr; }
uint64_t vfkv_pages_bytes_per_buffer(const vfkv_pages* c) { return c ? c->bytes : 0u; }
uint64_t vfkv_pages_offset_bytes(const vfkv_pages* c, uint32_t layer, uint32_t page) {
    return (c && layer < c->cfg.n_layers && page < c->cfg.n_pages) ? layer * c->layer_bytes + page * c->page_bytes : 0u;
}

// ---- page counting -------------------------------------------------------------------------------
uint32_t vfkv_pages_free_count(const vfkv_pages* c) { return c ? c->n_free : 0u; }
uint32_t vfkv_pages_refcount(const vfkv_pages* c, uint32_t page) { return (c && page < c->cfg.n_pages) ? c->refs[page] : 0u; }

int vfkv_pages_alloc(vfkv_pages* c, uint32_t n, uint32_t* pages_out) {
    if (!c) return fail(VFKV_ERR_INVALID_ARG, "pages_alloc: cache is NULL");
    if (n == 0u) return VFKV_OK;
    if (!pages_out) return fail(VFKV_ERR_INVALID_ARG, "pages_alloc: out is NULL");
    if (n > c->n_free) return fail(VFKV_ERR_WORKSPACE, "pages_alloc: %u pages wanted, %u free", n, c->n_free);
    take(c, n, pages_out);
    return VFKV_OK;
}

int vfkv_pages_retain(vfkv_pages* c, const uint32_t* pages, uint32_t n) {
    if (!c || (n != 0u && !pages)) return fail(VFKV_ERR_INVALID_ARG, "pages_retain: NULL argument");
    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t p = pages[i];
        if (p == VFKV_NO_PAGE) continue;
        if (p >= c->cfg.n_pages || c->refs[p] == 0u || c->refs[p] == UINT32_MAX) {
            for (uint32_t j = 0; j < i; ++j)
                if (pages[j] != VFKV_NO_PAGE) --c->refs[pages[j]];
            return fail(VFKV_ERR_INVALID_ARG, "pages_retain: page %u is not live", p);
        }
        ++c->refs[p];
    }
    return VFKV_OK;
}

int vfkv_pages_release(vfkv_pages* c, const uint32_t* pages, uint32_t n) {
    if (!c || (n != 0u && !pages)) return fail(VFKV_ERR_INVALID_ARG, "pages_release: NULL argument");
    // counts first, so that an error leaves everything as it was
    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t p = pages[i];
        if (p == VFKV_NO_PAGE) continue;
        if (p >= c->cfg.n_pages || c->refs[p] == 0u) {
            for (uint32_t j = 0; j < i; ++j)
                if (pages[j] != VFKV_NO_PAGE) ++c->refs[pages[j]];
            return fail(VFKV_ERR_INVALID_ARG, "pages_release: page %u is not live", p);
        }
        --c->refs[p];
    }
    const uint64_t stamp = ++c->stamp;
    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t p = pages[i];
        if (p == VFKV_NO_PAGE || c->refs[p] != 0u || c->mark[p] == stamp) continue;
        c->mark[p] = stamp;                    // a repeated entry is one free page
        ++c->n_free;
        if (p < c->lowest) c->lowest = p;
    }
    return VFKV_OK;
}

int vfkv_pages_copy(vfkv_pages* c, const uint32_t* src, const uint32_t* dst, const uint32_t* rows, uint32_t n, vfkv_stream stream) {
    int rc = check_pages(c, 0u, "pages_copy");
    if (rc != VFKV_OK) return rc;
    if (n == 0u) return VFKV_OK;
    if (!src || !dst) return fail(VFKV_ERR_INVALID_ARG, "pages_copy: NULL page list");
    const uint64_t stamp = ++c->stamp;
    for (uint32_t i = 0; i < n; ++i) {
        if (src[i] >= c->cfg.n_pages || dst[i] >= c->cfg.n_pages)
            return fail(VFKV_ERR_INVALID_ARG, "pages_copy: pair %u (%u -> %u) is outside the %u pages", i, src[i], dst[i], c->cfg.n_pages);
        if (rows && rows[i] > c->cfg.page_size)
            return fail(VFKV_ERR_INVALID_ARG, "pages_copy: %u rows of a page of %u", rows[i], c->cfg.page_size);
        if (c->mark[dst[i]] == stamp) return fail(VFKV_ERR_INVALID_ARG, "pages_copy: page %u is a destination twice", dst[i]);
        c->mark[dst[i]] = stamp;
    }
    for (uint32_t i = 0; i < n; ++i)
        if (c->mark[src[i]] == stamp) return fail(VFKV_ERR_INVALID_ARG, "pages_copy: page %u is a source and a destination", src[i]);
    if ((rc = check_device(c->device, "pages_copy", "cache")) != VFKV_OK) return rc;
    return copy_pages(c, src, dst, rows, n, stream);
}

int vfkv_pages_fork(vfkv_pages* c, const uint32_t* pages, uint32_t kv_len, uint32_t n_forks, uint32_t* pages_out, vfkv_stream stream) {
    if (!c) return fail(VFKV_ERR_INVALID_ARG, "pages_fork: cache is NULL");
    const uint32_t used = (uint32_t)(((uint64_t)kv_len + c->cfg.page_size - 1u) >> c->page_shift);
    if (used == 0u || n_forks == 0u) return VFKV_OK;
    if (!pages || !pages_out) return fail(VFKV_ERR_INVALID_ARG, "pages_fork: NULL page list");
    const uint32_t part = kv_len & (c->cfg.page_size - 1u);
    const bool own_last = part != 0u && pages[used - 1u] != VFKV_NO_PAGE;
    const uint32_t shared = own_last ? used - 1u : used;
    for (uint32_t i = 0; i < used; ++i) {
        const uint32_t p = pages[i];
        if (p == VFKV_NO_PAGE) continue;
        if (p >= c->cfg.n_pages || c->refs[p] == 0u) return fail(VFKV_ERR_INVALID_ARG, "pages_fork: page %u is not live", p);
        // (kv_len < 2^32, so a page repeated in the list adds at most used * n_forks references)
        if ((uint64_t)c->refs[p] + (uint64_t)used * n_forks > UINT32_MAX) return fail(VFKV_ERR_OVERFLOW, "pages_fork: too many references to page %u", p);
    }
    if (own_last && n_forks > c->n_free) return fail(VFKV_ERR_WORKSPACE, "pages_fork: %u pages wanted, %u free", n_forks, c->n_free);
    if (c->k && own_last) {
        const int rc = check_device(c->device, "pages_fork", "cache");
        if (rc != VFKV_OK) return rc;
    }
    return guarded("pages_fork", [&]() -> int {
        if (own_last) {
            std::vector<uint32_t> from(n_forks, pages[used - 1u]), fresh(n_forks), rows(n_forks, part);
            take(c, n_forks, fresh.data());
            if (c->k) {
                const int rc = copy_pages(c, from.data(), fresh.data(), rows.data(), n_forks, stream);
                if (rc != VFKV_OK) {
                    for (uint32_t p : fresh) drop(c, p);
                    return rc;
                }
            }
            for (uint32_t f = 0; f < n_forks; ++f) pages_out[(uint64_t)f * used + used - 1u] = fresh[f];
        }
        for (uint32_t f = 0; f < n_forks; ++f)
            for (uint32_t i = 0; i < shared; ++i) {
                pages_out[(uint64_t)f * used + i] = pages[i];
                if (pages[i] != VFKV_NO_PAGE) ++c->refs[pages[i]];
            }
        return VFKV_OK;
    });
}

int vfkv_pages_compact(vfkv_pages* c, uint32_t* new_ids_out, vfkv_stream stream) {
    if (!c || !new_ids_out) return fail(VFKV_ERR_INVALID_ARG, "pages_compact: NULL argument");
    const uint32_t n = c->cfg.n_pages, live = n - c->n_free;
    if (c->k) {
        const int rc = check_device(c->device, "pages_compact", "cache");
        if (rc != VFKV_OK) return rc;
    }
    return guarded("pages_compact", [&]() -> int {
        std::vector<uint32_t> src, dst;
        for (uint32_t p = live; p < n; ++p)
            if (c->refs[p] != 0u) src.push_back(p);
        dst.reserve(src.size());
        for (uint32_t p = 0; p < live; ++p)
            if (c->refs[p] == 0u) dst.push_back(p);      // as many as src: live pages outside [0, live) = free ones inside
        if (c->k) {
            const int rc = copy_pages(c, src.data(), dst.data(), nullptr, (uint32_t)src.size(), stream);
            if (rc != VFKV_OK) return rc;
        }
        for (uint32_t p = 0; p < n; ++p) new_ids_out[p] = c->refs[p] != 0u ? p : VFKV_NO_PAGE;
        for (size_t i = 0; i < src.size(); ++i) {
            new_ids_out[src[i]] = dst[i];
            c->refs[dst[i]] = c->refs[src[i]];
            c->refs[src[i]] = 0u;
        }
        c->lowest = live;
        return VFKV_OK;
    });
}

// ---- norm + rotation + append ----------------------------------------------------------------------
int vfkv_paged_qk_rope_kv_write(vfkv_pages* c, uint32_t layer, const vfkv_seq_batch* b, const vfkv_paged_rows* r,
                                const vfkv_mrope_params* p, vfkv_stream stream) {
    const char* const who = "paged_qk_rope_kv_write";
    int rc = check_pages(c, layer, who);
    if (rc != VFKV_OK) return rc;
    if (!r || !p) return fail(VFKV_ERR_INVALID_ARG, "%s: rows or params is NULL", who);
    vfkv::PagedWriteLaunch L = {};
    uint32_t max_kv = 0;
    bool nothing = false;
    if ((rc = check_batch(c, b, who, &L.s, &max_kv, &nothing)) != VFKV_OK) return rc;
    if ((rc = check_io(r->io_dtype, who)) != VFKV_OK) return rc;
    const uint32_t hd = c->cfg.head_dim, kvh = c->cfg.n_kv_heads;
    if (p->rope_mode != VFKV_ROPE_NORM && p->rope_mode != VFKV_ROPE_NEOX)
        return fail(VFKV_ERR_UNSUPPORTED, "%s: rope_mode %u (0 = NORM and 2 = NEOX are built)", who, p->rope_mode);
    if (p->rotary_dim % 2u != 0u || p->rotary_dim > hd)
        return fail(VFKV_ERR_INVALID_ARG, "%s: rotary_dim %u must be even and <= head_dim %u", who, p->rotary_dim, hd);
    if (p->n_axes == 0u || p->n_axes > 4u) return fail(VFKV_ERR_INVALID_ARG, "%s: n_axes %u (1 to 4)", who, p->n_axes);
    if (p->interleaved > 1u) return fail(VFKV_ERR_INVALID_ARG, "%s: interleaved must be 0 or 1", who);
    if (p->n_axes > 1u) {
        uint64_t sum = 0;
        for (uint32_t i = 0; i < p->n_axes; ++i) sum += p->section[i];
        if (sum != p->rotary_dim / 2u)
            return fail(VFKV_ERR_INVALID_ARG, "%s: the sections hold %llu pairs, rotary_dim %u has %u", who, (unsigned long long)sum,
                        p->rotary_dim, p->rotary_dim / 2u);
    }
    if (p->rotary_dim != 0u && (!(p->freq_base > 0.f) || !std::isfinite(p->freq_base) || !std::isfinite(p->freq_scale)))
        return fail(VFKV_ERR_INVALID_ARG, "%s: freq_base must be positive and finite, freq_scale finite", who);
    uint64_t q_row = 0;
    if (r->q) {
        if (r->n_heads == 0u) return fail(VFKV_ERR_INVALID_ARG, "%s: n_heads must be > 0", who);
        if (r->n_heads > 65536u) return fail(VFKV_ERR_UNSUPPORTED, "%s: %u heads", who, r->n_heads);
        if (!r->q_out) return fail(VFKV_ERR_INVALID_ARG, "%s: NULL q_out", who);
        q_row = (uint64_t)r->n_heads * hd;
    }
    if ((rc = row_stride(r->q_stride, q_row, who, "q", &L.q_stride)) != VFKV_OK) return rc;
    if ((rc = row_stride(r->q_out_stride, q_row, who, "q_out", &L.q_out_stride)) != VFKV_OK) return rc;
    if ((rc = row_stride(r->k_stride, (uint64_t)kvh * hd, who, "k", &L.k_stride)) != VFKV_OK) return rc;
    if ((rc = row_stride(r->v_stride, (uint64_t)kvh * hd, who, "v", &L.v_stride)) != VFKV_OK) return rc;
    if (r->q && r->q == r->q_out && L.q_stride != L.q_out_stride)
        return fail(VFKV_ERR_INVALID_ARG, "%s: in place, q and q_out must have the same stride", who);
    if (nothing) return VFKV_OK;
    if (!r->k || !r->v) return fail(VFKV_ERR_INVALID_ARG, "%s: NULL source", who);
    const uintptr_t io_mask = r->io_dtype == VFKV_F32 ? 3u : 1u;
    if ((((uintptr_t)r->q | (uintptr_t)r->q_out | (uintptr_t)r->k | (uintptr_t)r->v) & io_mask) != 0u ||
        (((uintptr_t)r->q_norm_weight | (uintptr_t)r->k_norm_weight | (uintptr_t)r->positions | (uintptr_t)r->freq_factors) & 3u) != 0u)
        return fail(VFKV_ERR_ALIGNMENT, "%s: a buffer is not aligned to its element size", who);
    if ((rc = check_device(c->device, who, "cache")) != VFKV_OK) return rc;
    L.c = slab(c, layer);
    L.q = r->q; L.q_weight = r->q_norm_weight; L.q_out = r->q_out;
    L.k = r->k; L.v = r->v; L.k_weight = r->k_norm_weight;
    L.positions = r->positions; L.freq_factors = r->freq_factors;
    L.n_heads = r->n_heads; L.io_f16 = r->io_dtype == VFKV_F16;
    L.mode = p->rope_mode; L.rotary_dim = p->rotary_dim; L.n_axes = p->n_axes; L.interleaved = p->interleaved;
    for (int i = 0; i < 4; ++i) L.section[i] = p->section[i];
    L.log2_step = p->rotary_dim ? -2.0 * std::log2((double)p->freq_base) / (double)p->rotary_dim : 0.0;
    L.freq_scale = p->freq_scale; L.attn_factor = p->attn_factor; L.eps = p->eps;
    VFKV_HIP(vfkv::launch_paged_write(L, S(stream)));
    return VFKV_OK;
}

// ---- attention -------------------------------------------------------------------------------------
int vfkv_paged_workspace_create(const vfkv_pages* c, uint32_t n_heads, vfkv_workspace** out) {
    if (!out) return fail(VFKV_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (!c) return fail(VFKV_ERR_INVALID_ARG, "paged_workspace: cache is NULL");
    if (n_heads == 0u || n_heads % c->cfg.n_kv_heads != 0u)
        return fail(VFKV_ERR_INVALID_ARG, "n_heads (%u) is not a multiple of n_kv_heads (%u)", n_heads, c->cfg.n_kv_heads);
    // rows of head_dim floats: two per head and workgroup of the decode launch, and room for the prefill's split over the keys
    const uint32_t slices = (n_heads / c->cfg.n_kv_heads + 7u) / 8u;
    uint64_t tiles = 2u * (uint64_t)vfkv::paged_decode_wgs(c->cfg.n_kv_heads * slices);
    if (tiles < kPrefillRows / n_heads) tiles = kPrefillRows / n_heads;
    return vfkv_workspace_create(n_heads, c->cfg.head_dim, (uint32_t)(tiles * 64u), out);
}

static int paged_attention(vfkv_pages* c, uint32_t layer, const vfkv_seq_batch* b, const vfkv_paged_attn_params* p, const void* q, void* o,
                           vfkv_workspace* ws, bool decode, vfkv_stream stream, const char* who) {
    int rc = check_pages(c, layer, who);
    if (rc != VFKV_OK) return rc;
    if (!p) return fail(VFKV_ERR_INVALID_ARG, "%s: params is NULL", who);
    vfkv::PagedAttnLaunch L;
    bool nothing = false;
    if ((rc = check_batch(c, b, who, &L.s, &L.max_kv, &nothing)) != VFKV_OK) return rc;
    if ((rc = check_io(p->io_dtype, who)) != VFKV_OK) return rc;
    const uint32_t hd = c->cfg.head_dim, kvh = c->cfg.n_kv_heads;
    if (p->n_heads == 0u || p->n_heads % kvh != 0u)
        return fail(VFKV_ERR_INVALID_ARG, "%s: n_heads (%u) is not a multiple of n_kv_heads (%u)", who, p->n_heads, kvh);
    if (p->n_heads > 65536u) return fail(VFKV_ERR_UNSUPPORTED, "%s: %u heads", who, p->n_heads);
    // (the kernels work with scale * log2 e and with the soft-cap's reciprocal: neither may leave the normal numbers)
    if (!(p->scale >= 1e-30f && p->scale <= 1e30f))
        return fail(VFKV_ERR_INVALID_ARG, "%s: scale must be between 1e-30 and 1e30 (got %g)", who, (double)p->scale);
    if (p->softcap != 0.f && !(p->softcap >= 1e-30f && p->softcap <= 1e30f))
        return fail(VFKV_ERR_INVALID_ARG, "%s: softcap must be 0 or between 1e-30 and 1e30 (got %g)", who, (double)p->softcap);
    if ((rc = row_stride(p->q_stride, (uint64_t)p->n_heads * hd, who, "q", &L.q_stride)) != VFKV_OK) return rc;
    if ((rc = row_stride(p->o_stride, (uint64_t)p->n_heads * hd, who, "o", &L.o_stride)) != VFKV_OK) return rc;
    if (decode && b->q_offsets) return fail(VFKV_ERR_INVALID_ARG, "%s: one token per sequence (q_offsets must be NULL)", who);
    vfkv::clear_note();
    if (nothing) return VFKV_OK;
    if (!q || !o) return fail(VFKV_ERR_INVALID_ARG, "%s: NULL buffer", who);
    if (q == o) return fail(VFKV_ERR_INVALID_ARG, "%s: o must not overlap q", who);
    if ((((uintptr_t)q | (uintptr_t)o) & (p->io_dtype == VFKV_F32 ? 3u : 1u)) != 0u)
        return fail(VFKV_ERR_ALIGNMENT, "%s: a buffer is not aligned to its element size", who);
    if ((uint64_t)b->n_tokens * p->n_heads > 1u << 30) return fail(VFKV_ERR_UNSUPPORTED, "%s: n_tokens * n_heads exceeds 2^30", who);
    if (ws && (ws->n_heads < p->n_heads || ws->head_dim < hd))
        return fail(VFKV_ERR_WORKSPACE, "%s: workspace built for %u heads x %u dims, need %u x %u", who, ws->n_heads, ws->head_dim, p->n_heads, hd);
    if (decode && !ws) return fail(VFKV_ERR_INVALID_ARG, "%s: workspace is NULL", who);
    if ((rc = check_device(c->device, who, "cache")) != VFKV_OK) return rc;
    L.c = slab(c, layer);
    L.q = q; L.o = o;
    L.n_heads = p->n_heads; L.window = p->window; L.n_sink = p->n_sink; L.io_f16 = p->io_dtype == VFKV_F16;
    L.scale = p->scale; L.softcap = p->softcap;
    if (ws) {
        if ((rc = check_device(ws->device, who, "workspace")) != VFKV_OK) return rc;
        L.scratch_out = ws->scratch_out; L.scratch_max = ws->scratch_max; L.scratch_sum = ws->scratch_sum;
        // (rows of this call's head_dim: the workspace may have been made for wider ones)
        L.scratch_rows = (uint64_t)ws->n_heads * ws->max_tiles;
    }
    const uint32_t per16 = p->io_dtype == VFKV_F32 ? 4u : 8u;
    const bool aligned = (((uintptr_t)q | (uintptr_t)o) & 15u) == 0u && L.q_stride % per16 == 0u && L.o_stride % per16 == 0u;
    const char* const why = hd % 16u != 0u ? "head_dim is not a multiple of 16"
                            : c->cfg.dtype == VFKV_F32 && hd > 256u ? "rows of F32 pages are wider than 256 elements"
                            : !aligned ? "q and o are not 16-byte aligned in every row" : nullptr;
    if (why) {
        VFKV_HIP(vfkv::launch_paged_generic(L, S(stream)));
        vfkv::set_note("%s: %s (kv dtype %u, head_dim %u): the call ran on the generic kernel, many times slower than the tiled kernels",
                       who, why, c->cfg.dtype, hd);
        return VFKV_OK;
    }
    VFKV_HIP(decode ? vfkv::launch_paged_decode(L, S(stream)) : vfkv::launch_paged_prefill(L, S(stream)));
    return VFKV_OK;
}

int vfkv_paged_decode_attention(vfkv_pages* c, uint32_t layer, const vfkv_seq_batch* b, const vfkv_paged_attn_params* p, const void* q,
                                void* o, vfkv_workspace* ws, vfkv_stream stream) {
    return paged_attention(c, layer, b, p, q, o, ws, true, stream, "paged_decode_attention");
}

int vfkv_paged_prefill_attention(vfkv_pages* c, uint32_t layer, const vfkv_seq_batch* b, const vfkv_paged_attn_params* p, const void* q,
                                 void* o, vfkv_workspace* ws, vfkv_stream stream) {
    return paged_attention(c, layer, b, p, q, o, ws, false, stream, "paged_prefill_attention");
}

}  // extern "C"
