// Host logic of the 8-bit cache's calls (validation, planning, workspace sizes) under AddressSanitizer + UBSan; every call is
// rejected before a launch, so the program runs on a machine without a GPU.
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "fl_decode_attn.h"

static int checks = 0, failures = 0;
#define EXPECT(cond)                                                      \
    do {                                                                  \
        ++checks;                                                         \
        if (!(cond)) {                                                    \
            ++failures;                                                   \
            std::fprintf(stderr, "FAIL line %d: %s\n", __LINE__, #cond);  \
        }                                                                 \
    } while (0)

static void *at(uintptr_t p) { return reinterpret_cast<void *>(p); }

int main()
{
    for (int dtype = 0; dtype < 2; ++dtype)
        for (int D : {32, 64, 96, 128, 256, 512, 1024})
            for (int T : {32, 64, 128})
                for (int blocks : {1, 3, 65, 1000})
                    for (int B : {1, 3, 64})
                        for (int nsplit : {0, 1, 7, 1024}) {
                            fl_attn_desc d;
                            std::memset(&d, 0, sizeof d);
                            d.struct_size = sizeof d;
                            d.batch_size = B; d.head_num = 5; d.size_per_head = D; d.total_len = blocks * T; d.dtype = dtype; d.nsplit = nsplit;
                            size_t ws = 0, last = 0, r = 0, s = 0, t = 0;
                            for (int S : {1, 2, 33, 129, blocks * T}) {
                                if (S > d.total_len) continue;
                                EXPECT(fl_kv8_workspace_bytes(&d, T, S, &ws) == FL_ATTN_OK && ws % 256 == 0);
                                if (S != blocks * T || S > 129) EXPECT(ws >= last);
                                if (S <= 129) last = ws;
                            }
                            EXPECT(fl_kv8_workspace_bytes(&d, T, d.total_len + 1, &ws) == FL_ATTN_ERR_POSITION);
                            EXPECT(fl_kv8_cache_bytes(&d, T, &r, &s, &t) == FL_ATTN_OK && r == (size_t)B * 5 * blocks * T * D && s == (size_t)B * 5 * blocks * 4);

                            fl_kv8_cache c;
                            std::memset(&c, 0, sizeof c);
                            c.struct_size = sizeof c; c.block_len = T;
                            c.k = (int8_t *)at(0x10000000000); c.v = (int8_t *)at(0x20000000000);
                            c.k_scale = (float *)at(0x30000000000); c.v_scale = (float *)at(0x40000000000);
                            c.k_tail = at(0x50000000000); c.v_tail = at(0x60000000000); c.weights = (float *)at(0x70000000000);
                            fl_attn_io io;
                            std::memset(&io, 0, sizeof io);
                            io.struct_size = sizeof io;
                            io.q = io.k_new = io.v_new = at(0x1000);
                            io.freq_cis = (const float *)at(0x1000); io.out = (float *)at(0x1000);
                            io.start_pos = d.total_len; io.rope_row = -1; io.max_start_pos = -1;
                            EXPECT(fl_kv8_decode_forward(&d, &c, &io, nullptr, 0, nullptr) == FL_ATTN_ERR_POSITION);
                            EXPECT(fl_kv8_prefill_forward(&d, &c, &io, 1, nullptr, 0, nullptr) == FL_ATTN_ERR_POSITION);
                            io.start_pos = 0; // no workspace
                            EXPECT(fl_kv8_decode_forward(&d, &c, &io, nullptr, 0, nullptr) == FL_ATTN_ERR_WORKSPACE);
                            EXPECT(fl_kv8_prefill_forward(&d, &c, &io, 1, nullptr, 0, nullptr) == (D > 128 ? FL_ATTN_ERR_HEAD_DIM : FL_ATTN_ERR_WORKSPACE));
                            EXPECT(fl_kv8_read(&d, &c, 0, nullptr, at(0x1000), at(0x2000), nullptr) == FL_ATTN_ERR_POSITION);
                            fl_kv8_evict_args e;
                            std::memset(&e, 0, sizeof e);
                            e.struct_size = sizeof e;
                            e.keep_blocks = blocks + 1; e.kept = (int32_t *)at(0x80000000000); e.rows_out = (int32_t *)at(0x1000);
                            EXPECT(fl_kv8_evict(&d, &c, &c, &e, nullptr) == FL_ATTN_ERR_ARGUMENT);
                            e.keep_blocks = 1;
                            fl_kv8_cache to = c;
                            to.k = c.k + 16;
                            EXPECT(fl_kv8_evict(&d, &c, &to, &e, nullptr) == FL_ATTN_ERR_ARGUMENT);
                        }
    std::printf("%d checks, %d failures\n", checks, failures);
    return failures != 0;
}
