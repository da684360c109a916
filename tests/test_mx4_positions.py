"""Which tokens of the MXFP4 cache a row sees (ga_mx4_positions.hpp), as the kernels compute it in 32
bits, against the definition in 64 (CPU only): windows up to the largest int, more rows than tokens."""
import ctypes
import os
import subprocess

from gcnasm_amd import _lib

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gcnasm_amd",
                    "csrc")

CHECK = r"""
#include "ga_mx4_positions.hpp"
#include <stdio.h>
#include <algorithm>
typedef long long ll;
int main()
{
    const int lens[] = {0, 1, 3, 63, 64, 65, 500, 1 << 20, 0x7FFFF000};
    const int rows[] = {1, 2, 5, 9, 64, 700, 1 << 20};
    const int windows[] = {0, 1, 6, 64, 499, 1 << 30, 0x7FFFFFF0, 0x7FFFFFFE, 0x7FFFFFFF};
    ll bad = 0, checked = 0;
    for (int len : lens)
        for (int n : rows)
            for (int w : windows)
                for (int causal = w ? 1 : 0; causal < 2; causal++) {
                    const ll step = n > 1000 ? n / 7 : 1;
                    for (ll i0 = 0; i0 < n; i0 += step) {
                        const ll i1 = std::min<ll>(i0 + 15, n - 1);
                        const ga::Seen s(len, n, (int)i0, (int)i1, causal, w);
                        ll first = 1ll << 40, last = -1; // that some row of the block sees
                        for (ll i = i0; i <= i1; i++) {
                            const ll pos = (ll)len - n + i;
                            const ll hi = causal ? std::min<ll>(pos, len - 1) : len - 1;
                            const ll lo = w ? std::max<ll>(pos - w, -1) : -1;
                            const int got_hi = ga::last_seen((int)pos, len, causal);
                            const int got_lo = ga::before_first((int)pos, w);
                            if (hi > lo && hi >= 0) {
                                bad += got_hi != hi || got_lo != lo;
                                first = std::min(first, lo + 1);
                                last = std::max(last, hi);
                                bad += s.hi_min > hi || s.hi_max < hi || s.lo_min > lo ||
                                       s.lo_max < lo;
                            } else { // sees nothing
                                bad += got_hi > got_lo && got_hi >= 0;
                                bad += s.hi_min >= 0 && s.hi_min > s.lo_max && len > 0;
                            }
                            checked++;
                        }
                        // the tokens gone over are inside the sequence and hold all that is seen
                        bad += s.begin() < 0 || s.begin() % 64 || s.end() > len;
                        if (last >= 0)
                            bad += s.begin() > first || s.end() <= last;
                        else
                            bad += s.begin() < s.end();
                    }
                }
    // eviction: 16 waves' stretches of the tokens follow each other and end with the last one
    for (int n : {1, 2, 63, 64, 65, 1023, 1024, 1025, 8192, 8193, 65536, 65537, 100001, 0x7FFFEFFF,
                  0x7FFFF000}) {
        int at = 0;
        for (int part = 0; part < 16; part++) {
            const ga::Stretch s(n, part, 16);
            bad += s.lo != at || s.hi < s.lo || s.hi > n || s.rows != (s.hi - s.lo + 63) / 64;
            bad += s.rows > (n + 1023ll) / 1024;
            bad += s.rows && s.lo + 64ll * (s.rows - 1) + 63 > 0x7FFFFFFF;
            at = s.hi;
        }
        bad += at != n;
    }
    printf("%lld of %lld\n", bad, checked);
    return 0;
}
"""


def test_what_rows_see(tmp_path):
    src = tmp_path / "positions.cpp"
    src.write_text(CHECK)
    exe = str(tmp_path / "positions")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", CSRC, "-o", exe, str(src)], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    assert out[0] == "0" and int(out[2]) > 20000, out


def test_sizes_that_pass_the_positions_are_refused():
    """More tokens or rows than 32 bits can step over, before any device call."""
    l, r = _lib.lib(), ctypes.byref
    most, bad = 0x7FFFF000, 0x7FFFF001
    c = _lib.Mx4Cache(0x10000, 8, 2 * 8704, 2, 128, 64)
    a = _lib.Mx4AttentionArgs()
    e = _lib.Mx4EvictArgs()
    for n in ("q", "out", "lse", "table", "lens", "q_starts"):
        setattr(a, n, 0x10000)
    a.stride_q_row = a.stride_out_row = 4 * 128
    a.stride_q_head = a.stride_out_head = 128
    a.seqs, a.rows, a.heads, a.table_pages, a.max_q, a.max_len, a.causal = 3, 3, 4, 5, 1, 100, 1
    need = ctypes.c_size_t()
    assert l.ga_mx4_attention_weights_workspace_bytes(r(c), r(a), bad, r(need)) == _lib.GA_ERR_SHAPE
    assert l.ga_mx4_attention_weights(r(c), r(a), None, 0, 0, 0x1000, 8, 8, bad, None, 0,
                                      None) == _lib.GA_ERR_SHAPE
    a.rows = 0x3FFFFF00 // 4 + 1
    assert l.ga_mx4_attention(r(c), r(a), None, 0, None) == _lib.GA_ERR_SHAPE
    assert l.ga_mx4_attention_workspace_bytes(r(c), r(a), r(need)) == _lib.GA_ERR_SHAPE
    for n in ("table", "lens", "dst_table", "weights", "kept", "new_lens", "new_weights"):
        setattr(e, n, 0x10000)
    for e.width, e.new_width in ((bad, 100), (200, bad)):
        e.seqs, e.table_pages, e.dst_pages, e.keep, e.recent = 2, 4, 2, 100, 10
        assert l.ga_mx4_evict(r(c), r(e), None) == _lib.GA_ERR_SHAPE
    header = open(os.path.join(CSRC, "..", "..", "include", "gcnasm_amd.h")).read()
    assert "#define GA_MX4_MAX_TOKENS 0x%X" % most in header


def test_launches_of_too_many_threads_are_refused():
    """A launch takes fewer than 2^32 threads; what asks for more is refused before it."""
    l, r = _lib.lib(), ctypes.byref
    c = _lib.Mx4Cache(0x10000, 8, 16 * 8704, 16, 128, 64)
    # 2^24 tokens of 16 heads, 16 lanes a row of bf16, 32 of fp32: 2^32 and 2^33 threads
    for kind, tokens in ((1, 1 << 24), (0, 1 << 23)):
        assert l.ga_mx4_append(r(c), 0x1000, 0x1000, kind, tokens, 2048, 128, 2048, 128, 0x1000, 0,
                               None) == _lib.GA_ERR_SHAPE
    assert l.ga_mx4_read(r(c), 0x1000, 1 << 24, 0x1000, 0x1000, 0, None) == _lib.GA_ERR_SHAPE
    e = _lib.Mx4EvictArgs()
    for n in ("table", "lens", "dst_table", "weights", "kept", "new_lens", "new_weights"):
        setattr(e, n, 0x10000)
    # 1024 threads for each sequence's head to select; 256 for each 64 tokens of one to move
    for e.seqs, e.keep in ((1 << 18, 1), (1 << 10, 1 << 16)):
        e.table_pages, e.dst_pages, e.width, e.new_width = 4, 1 << 10, 200, e.keep
        assert l.ga_mx4_evict(r(c), r(e), None) == _lib.GA_ERR_SHAPE


def test_weights_of_no_rows_need_a_table():
    """Without rows the weights' kernel still goes over the tokens: a table that is not there is
    refused."""
    l, r = _lib.lib(), ctypes.byref
    c = _lib.Mx4Cache(0x10000, 8, 2 * 8704, 2, 128, 64)
    a = _lib.Mx4AttentionArgs()
    a.lens, a.q_starts = 0x10000, 0x10000
    a.seqs, a.rows, a.heads, a.table_pages, a.max_q, a.max_len, a.causal = 3, 0, 4, 5, 1, 100, 1
    assert l.ga_mx4_attention_weights(r(c), r(a), None, 0, 0, 0x1000, 8, 8, 8, None, 0,
                                      None) == _lib.GA_ERR_ARG
