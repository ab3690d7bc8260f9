// spans.h -- argument checks that the entry points of the serving and the prompt
// table share: the memory that a call's arguments cover, sizes and caps.
#pragma once
#include "extent.h"
#include "hip_context.h"

namespace lxh {

// the memory one argument covers
struct Span {
    const char* p = nullptr;
    size_t n = 0;
    bool out = false;
    bool meets(const Span& o) const { return n && o.n && p < o.p + o.n && o.p < p + n; }
};

// the arguments' memory: buffers large enough, aligned to their elements, and
// no output over another argument
struct Spans {
    Span s[12];
    int count = 0;
    bool ok = true;
    const void* add(LuxBackendBuffer* b, size_t skip, size_t bytes, size_t esz, bool out) {
        HipBuffer* h = B(b);
        if (!h || !holds(h->size, skip, bytes) || (bytes && reinterpret_cast<uintptr_t>(h->ptr) % esz)) {
            ok = false;
            return nullptr;
        }
        const char* p = static_cast<const char*>(h->ptr) + skip;
        s[count++] = Span{p, bytes, out};
        return bytes ? p : nullptr;
    }
    const void* in(LuxBackendBuffer* b, size_t skip, size_t bytes, size_t esz) { return add(b, skip, bytes, esz, false); }
    void* out(LuxBackendBuffer* b, size_t skip, size_t bytes, size_t esz) {
        return const_cast<void*>(add(b, skip, bytes, esz, true));
    }
    bool apart() const {
        for (int i = 0; i < count; i++)
            for (int j = 0; j < i; j++)
                if ((s[i].out || s[j].out) && s[i].meets(s[j])) return false;
        return true;
    }
};

// pages, table and slots that 31 bits hold
inline bool cache_ok(int kv_heads, int head_dim, int page_size, int num_pages) {
    return kv_heads > 0 && head_dim > 0 && page_size > 0 && num_pages >= 0;
}
inline bool rows_ok(int kv_heads, int page_size, int num_pages) {
    return (int64_t)num_pages * page_size < (1ll << 31) && (int64_t)num_pages * page_size * kv_heads < (1ll << 31);
}

// none, or a cap whose quotients and products with a score's factors stay in fp32
inline bool cap_ok(float c) { return c == 0.f || (c >= 0x1p-100f && c <= 0x1p100f); }

}  // namespace lxh
