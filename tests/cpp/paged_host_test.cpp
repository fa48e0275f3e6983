// Tests of the host code of packed tokens and caches in pages (csrc/paged_append.hip, csrc/decode_paged.hip) without a GPU: their objects, a HIP
// runtime that only keeps books (fake_hip.hpp), and what each launch was given.
//   paged_host_test NAME   runs one test, "ok" at its end
#include "fake_hip.hpp"

#include <cstdint>
#include <cstdio>
#include <string>
#include <vector>

#include "../../include/rt_attn.h"
#include "../../rustorch_amd/csrc/cache_paged.hpp"

static int g_failed = 0;
#define CHECK(cond)                                                     \
    do {                                                                \
        if (!(cond)) {                                                  \
            std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            ++g_failed;                                                 \
        }                                                               \
    } while (0)

namespace rt {
int ensure_device(rt_err_detail*) { return RT_OK; }
uint64_t next_launch_id() { return 256; }
}  // namespace rt

static std::vector<rt::PagedAppendParams> g_append;
static int g_decodes = 0, g_joins = 0;
static void note_launch(const std::string& name, dim3, void** args, hipStream_t) {
    if (name.find("paged_append") != std::string::npos) g_append.push_back(*(rt::PagedAppendParams*)args[0]);
    g_decodes += name.find("paged_decode_kernel") != std::string::npos;
    g_joins += name.find("paged_join_kernel") != std::string::npos;  // (where a prefix is read once)
}

// an address of its own for every buffer; none is looked into
static void* at(int i) { return (void*)((uintptr_t)(i + 1) << 40); }

struct Append {
    int32_t tokens = 4, batch = 2, heads = 4, n_kv = 2, n_pages = 8, page = 16, table_pages = 4, table_rows = 64, pos = 0;
    bool table = true, starts = false, positions = true;
    int call() const {
        return rt_qk_norm_rope_kv_append_paged_bf16(nullptr, at(0), at(1), n_kv ? at(2) : nullptr, nullptr, n_kv ? at(3) : nullptr, n_kv ? at(4) : nullptr, n_kv ? at(5) : nullptr,
                                                    (const int32_t*)(table ? at(6) : nullptr), (const int32_t*)(starts ? at(7) : nullptr), (const int32_t*)(positions ? at(8) : nullptr), pos, nullptr,
                                                    nullptr, 0, nullptr, nullptr, 1e-6f, (const float*)at(9), (const float*)at(10), table_rows, tokens, batch, heads, n_kv, 64, n_pages, page,
                                                    table_pages, nullptr);
    }
};

// ---- tests -----------------------------------------------------------------------------------------------------

// Where there are no kv heads there is no cache: a call without a page table has none that the kernel may read, whatever its width.
static void a_call_without_kv_heads_reads_no_table() {
    Append a;
    a.n_kv = 0;
    for (bool table : {false, true}) {
        a.table = table;
        g_append.clear();
        CHECK(a.call() == RT_OK && g_append.size() == 1);
        CHECK(g_append[0].table_pages == 0);
    }
    a.n_kv = 2;
    g_append.clear();
    CHECK(a.call() == RT_OK && g_append.size() == 1 && g_append[0].table_pages == 4 && g_append[0].page_table);
    a.table = false;
    CHECK(a.call() == RT_ERR_NULL_POINTER);
}

// Nor is a host position behind a page table that there is no use for.
static void a_call_without_kv_heads_has_no_last_row() {
    Append a;
    a.n_kv = a.table_pages = a.n_pages = 0;
    a.table = a.positions = false;
    for (bool starts : {true, false}) {
        a.starts = starts;
        a.pos = 0;
        g_append.clear();
        CHECK(a.call() == RT_OK && g_append.size() == 1);
        a.pos = 64;
        CHECK(a.call() == RT_ERR_ROPE_POSITION_OVERFLOW);
    }
    a.n_kv = 2;
    a.pos = 0;
    CHECK(a.call() == RT_ERR_KV_OVERFLOW);
}

// A prefix that the host gives is read once where that was measured to be shorter, on both sides of the rule; one on the device always.
static void a_prefix_is_read_once_where_that_is_shorter() {
    struct Case {
        int32_t heads, kv, dim, batch, shared;
        bool once;
    };
    for (const Case& c : {Case{16, 2, 256, 16, 4096, false}, Case{16, 2, 256, 8, 4096, false}, Case{8, 1, 256, 64, 1024, false}, Case{16, 16, 256, 4, 1024, false},
                          Case{16, 16, 256, 16, 1024, true}, Case{32, 8, 256, 16, 1024, true}, Case{32, 8, 256, 64, 1024, true}, Case{16, 2, 256, 64, 4096, true}, Case{32, 2, 128, 16, 4096, false},
                          Case{32, 2, 128, 32, 1024, false}, Case{28, 4, 128, 32, 1024, false}, Case{32, 8, 128, 64, 8192, true}, Case{16, 16, 64, 24, 1001, true}, Case{16, 16, 64, 8, 1024, false},
                          Case{32, 8, 128, 200, 63, false}, Case{32, 8, 128, 1, 30000, false}, Case{40, 1, 128, 64, 4096, true}}) {
        const int32_t columns = (c.shared + 512) / 16;
        const size_t need = rt_gqa_decode_paged_workspace_bytes(c.batch, c.heads, c.kv, c.dim, 16, columns);
        for (bool device : {false, true}) {
            g_decodes = g_joins = 0;
            CHECK(rt_gqa_decode_paged_bf16(nullptr, at(0), at(1), at(2), at(3), (const int32_t*)at(4), (const int32_t*)at(5), (const int32_t*)(device ? at(6) : nullptr), device ? 0 : c.shared,
                                           c.batch, c.heads, c.kv, c.dim, 64, 16, columns, at(7), need, nullptr) == RT_OK);
            const bool right = g_decodes == 1 && g_joins == (device || c.once ? 1 : 0);
            if (!right) std::printf("%d heads on %d of %d, %d behind %d\n", c.heads, c.kv, c.dim, c.batch, c.shared);
            CHECK(right);
        }
    }
}

int main(int argc, char** argv) {
    fake::on_launch() = note_launch;
    const std::map<std::string, std::function<void()>> tests = {
        {"a_call_without_kv_heads_reads_no_table", a_call_without_kv_heads_reads_no_table},
        {"a_call_without_kv_heads_has_no_last_row", a_call_without_kv_heads_has_no_last_row},
        {"a_prefix_is_read_once_where_that_is_shorter", a_prefix_is_read_once_where_that_is_shorter},
    };
    if (argc == 2 && tests.count(argv[1])) tests.at(argv[1])();
    else {
        for (auto& t : tests) std::printf("%s\n", t.first.c_str());
        return argc == 1 ? 0 : 2;
    }
    if (!g_failed) std::printf("ok\n");
    return g_failed ? 1 : 0;
}
