"""A 4-bit cache on the device beside the oracle's on the host, and the calls
of the C ABI on it (ember_amd.capi).  GPU tests only."""

from __future__ import annotations

import numpy as np

import gpu_helpers as G
from ember_amd import capi
from ember_amd.capi import DeviceArray
from oracle import serving

U = 2.0 ** -24  # half a step of float32


class Bytes:
    """Device bytes, through the float buffers that the library hands out."""

    def __init__(self, a):
        self.shape, self.dtype = a.shape, a.dtype
        raw = np.ascontiguousarray(a).reshape(-1).view(np.uint8)
        self.n = raw.size
        words = np.zeros((self.n + 3) // 4 * 4 or 4, np.uint8)
        words[:self.n] = raw
        self.dev = DeviceArray.from_numpy(words.view(np.float32))

    @property
    def ptr(self):
        return self.dev.ptr

    def numpy(self):
        return self.dev.numpy().view(np.uint8)[:self.n].view(self.dtype).reshape(self.shape)


def ints(a):
    return None if a is None else Bytes(np.asarray(a, np.int32))


def ptr(x):
    return None if x is None else x.ptr


class Pair:
    """One cache twice: `host` is the oracle's, the rest is on the device.  Slots
    start as `fill` bytes in both (255: every scale is no number)."""

    def __init__(self, pages, heads, page_size, D, table, fill=255):
        self.host = serving.Cache(pages, heads, page_size, D, table)
        for a in (*self.host.codes, *self.host.scales):
            a.fill(fill)
        self.codes, self.scales = ([Bytes(a) for a in x] for x in (self.host.codes, self.host.scales))
        self.table = ints(self.host.table)
        self.view = capi.KVCacheView(self.codes[0].ptr, self.scales[0].ptr, self.codes[1].ptr, self.scales[1].ptr, self.table.ptr,
                                     pages, heads, page_size, D, *self.host.table.shape)

    def write(self, k, v, start=None, count=None, stride_pad=0):
        """Both caches; returns (device next, oracle next)."""
        B, T, H, D = k.shape
        G.say(f"kv_cache_write B={B} T={T} H={H} D={D} page={self.host.page_size}")
        row = H * D + stride_pad
        packed = np.full((2, B, T, row), G.SENTINEL, np.float32)
        packed[0, ..., :H * D], packed[1, ..., :H * D] = k.reshape(B, T, -1), v.reshape(B, T, -1)
        dev = [DeviceArray.from_numpy(x) for x in packed]
        s, n, nxt = ints(start), ints(count), ints(np.full(B, -7))
        rc = capi.lib().kv_cache_write(self.view, dev[0].ptr, dev[1].ptr, T, T * row, D, row, ptr(s), ptr(n), nxt.ptr)
        capi.check(rc, "kv_cache_write")
        return nxt.numpy(), self.host.write(k, v, start, count)

    def read(self, T, start=None, count=None):
        B, H, D = self.host.table.shape[0], self.host.heads, self.host.D
        G.say(f"kv_cache_read B={B} T={T} H={H} D={D} page={self.host.page_size}")
        out = [DeviceArray.from_numpy(np.full((B, T, H, D), G.SENTINEL)) for _ in range(2)]
        s, n = ints(start), ints(count)
        capi.check(capi.lib().kv_cache_read(self.view, out[0].ptr, out[1].ptr, T, T * H * D, D, H * D, ptr(s), ptr(n)), "kv_cache_read")
        return [x.numpy() for x in out]

    def attention(self, q, causal, scale=None, start=None, count=None, want_lse=True, head_major=False, log=None):
        """o (B, T, Hq, D) and lse; head_major lays q and o out as (B, Hq, T, D)."""
        B, T, Hq, D = q.shape
        scale = G.scale_for(D) if scale is None else scale
        G.say(f"kv_cache_attention B={B} T={T} Hq={Hq} H={self.host.heads} D={D} page={self.host.page_size} causal={causal}")
        lay = (lambda x: np.ascontiguousarray(x.transpose(0, 2, 1, 3))) if head_major else (lambda x: x)
        dq, o = DeviceArray.from_numpy(lay(q)), DeviceArray.from_numpy(np.full(lay(q).shape, G.SENTINEL))
        lse = DeviceArray.from_numpy(np.full((B, Hq, T), G.SENTINEL)) if want_lse else None
        st = (T * Hq * D, T * D, D) if head_major else (T * Hq * D, D, Hq * D)
        s, n = ints(start), ints(count)
        capi.launch_log_reset()
        rc = capi.lib().kv_cache_attention(self.view, dq.ptr, o.ptr, ptr(lse), T, Hq, scale, int(causal), *st, *st, ptr(s), ptr(n))
        if log is not None:
            log.extend(capi.launch_log())
        capi.check(rc, "kv_cache_attention")
        return lay(o.numpy()) if head_major else o.numpy(), None if lse is None else lse.numpy()

    def check_attention(self, q, causal, scale=None, start=None, count=None, **more):
        """Against the oracle.  A score is a sum of D products in fp32, scaled and
        shifted (D + 8 roundings of its largest partial sum, at most a whole
        step each on the matrix cores), so a weight is off by twice that (its
        own score and the sum's) and o by that and the roundings of its sum
        over the keys, all times sum p |v|; lse likewise."""
        D = q.shape[-1]
        scale = G.scale_for(D) if scale is None else scale
        o, lse = self.attention(q, causal, scale, start, count, **more)
        ro, rl, weight, reach = self.host.attention(q, causal, scale, start, count)
        keys = self.host.table.shape[1] * self.host.page_size
        off = 2 * U * (D + 8) * reach
        tol = (2 * off.transpose(0, 2, 1)[..., None] + 2 * U * (keys + 16)) * weight
        np.testing.assert_array_equal(np.isnan(o), np.isnan(ro))
        bad = ~np.isnan(ro) & ~(np.abs(o - ro) <= tol)
        assert not bad.any(), f"o: {bad.sum()} of {bad.size}, worst {np.nanmax(np.abs(o - ro))}"
        if lse is not None:
            same = (lse == rl) | (np.isnan(lse) & np.isnan(rl))
            near = np.abs(np.where(same, 0, lse) - np.where(same, 0, rl)) <= off + 2 * U * (np.where(np.isfinite(rl), np.abs(rl), 0) + keys + 16)
            assert (same | near).all()
        # Independent roundings of a few steps each, of scores up to about 8:
        # a relative 2-norm error of 64 half steps is far above them.
        fine = np.isfinite(ro)
        if fine.any() and np.linalg.norm(ro[fine]):
            assert np.linalg.norm((o - ro)[fine]) <= 64 * U * np.linalg.norm(ro[fine])
        return o, lse


def table(rng, B, places, spare=3):
    """A page table over strewn pages, and how many pages there are."""
    n = B * places + spare
    return rng.permutation(n)[:B * places].reshape(B, places).astype(np.int32), n
