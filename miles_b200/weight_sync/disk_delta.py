"""Disk-delta weight transfer: ship only what changed since the previous sync through a shared directory.

The trainer keeps a CPU snapshot of the last synced weights; per sync it writes, for every tensor, either
the byte-wise XOR against the snapshot or the new bytes (``--update-weight-delta-encoding xor|overwrite``),
compressed (zlib here; the reference uses zstd) into per-rank ``model-NNNNN-of-MMMMM.delta`` files plus an
index with ``version``, ``base_version``, ``encoding`` and a checksum per tensor; engines pull the index,
apply the delta to their weights and bump the version.  Reference:
miles/backends/megatron_utils/update_weight/update_weight_from_distributed/delta.py:32-378,
miles/utils/disk_delta.py:21-87.
"""
from __future__ import annotations

import hashlib
import json
import os
import zlib

import torch


def _bytes(t: torch.Tensor) -> bytes:
    return t.detach().contiguous().cpu().view(torch.uint8).numpy().tobytes()


def checksum(b: bytes, kind: str = "sha1") -> str:
    """Per-tensor checksum of a published delta. The reference's flag names xxh3-128 / blake3 / adler32
    (``--update-weight-delta-checksum``); xxhash and blake3 are not in this image, so the 128-bit kinds map to
    blake2b-128 from hashlib, ``adler32`` is zlib's."""
    if kind == "adler32":
        return f"{zlib.adler32(b) & 0xffffffff:08x}"
    if kind in ("blake2", "blake3", "xxh3-128"):
        return hashlib.blake2b(b, digest_size=16).hexdigest()
    return hashlib.sha1(b).hexdigest()


class DiskDeltaWriter:
    def __init__(self, directory: str, encoding: str = "xor", checksum_kind: str = "sha1", rank: int = 0, world: int = 1):
        assert encoding in ("xor", "overwrite")
        self.dir, self.encoding, self.ck = directory, encoding, checksum_kind
        self.rank, self.world = rank, world
        self.snapshot: dict = {}
        self.version = 0
        os.makedirs(directory, exist_ok=True)

    def write(self, named_tensors, version: int) -> dict:
        """Write the delta of ``named_tensors`` against the snapshot; returns this rank's index entry."""
        vdir = os.path.join(self.dir, f"v{version:08d}")
        os.makedirs(vdir, exist_ok=True)
        fname = f"model-{self.rank + 1:05d}-of-{self.world:05d}.delta"
        entries, blob, off = {}, bytearray(), 0
        raw_total = 0
        for name, t in named_tensors:
            new = _bytes(t)
            raw_total += len(new)
            old = self.snapshot.get(name)
            if self.encoding == "xor" and old is not None and len(old) == len(new):
                a = torch.frombuffer(bytearray(new), dtype=torch.uint8)
                b = torch.frombuffer(bytearray(old), dtype=torch.uint8)
                payload, enc = (a ^ b).numpy().tobytes(), "xor"
            else:
                payload, enc = new, "overwrite"
            comp = zlib.compress(payload, 1)
            entries[name] = {"offset": off, "nbytes": len(comp), "raw_nbytes": len(new), "encoding": enc,
                             "dtype": str(t.dtype).replace("torch.", ""), "shape": list(t.shape), "checksum": checksum(new, self.ck)}
            blob += comp
            off += len(comp)
            self.snapshot[name] = new
        tmp = os.path.join(vdir, fname + ".tmp")
        with open(tmp, "wb") as f:
            f.write(blob)
        os.replace(tmp, os.path.join(vdir, fname))
        idx = {"version": version, "base_version": self.version, "file": fname, "tensors": entries,
               "raw_bytes": raw_total, "compressed_bytes": off, "checksum_kind": self.ck}
        with open(os.path.join(vdir, f"index-{self.rank:05d}.json"), "w") as f:
            json.dump(idx, f)
        self.version = version
        return idx


class DiskDeltaReader:
    def __init__(self, directory: str):
        self.dir = directory
        self.version = 0

    def apply(self, version: int, params: dict, strict_base: bool = True) -> int:
        """Apply every rank's delta of ``version`` onto ``params`` (name -> tensor). Returns #tensors updated."""
        vdir = os.path.join(self.dir, f"v{version:08d}")
        n = 0
        for fn in sorted(os.listdir(vdir)):
            if not fn.startswith("index-"):
                continue
            idx = json.load(open(os.path.join(vdir, fn)))
            if strict_base and idx["base_version"] != self.version and any(e["encoding"] == "xor" for e in idx["tensors"].values()):
                raise RuntimeError(f"delta v{version} is based on v{idx['base_version']} but this engine holds v{self.version}")
            blob = open(os.path.join(vdir, idx["file"]), "rb").read()
            for name, e in idx["tensors"].items():
                if name not in params:
                    continue
                raw = zlib.decompress(blob[e["offset"]:e["offset"] + e["nbytes"]])
                dst = params[name]
                if e["encoding"] == "xor":
                    cur = torch.frombuffer(bytearray(_bytes(dst)), dtype=torch.uint8)
                    new = (cur ^ torch.frombuffer(bytearray(raw), dtype=torch.uint8)).numpy().tobytes()
                else:
                    new = raw
                if checksum(new, idx.get("checksum_kind", "sha1")) != e["checksum"]:
                    raise RuntimeError(f"checksum mismatch for {name} in delta v{version}")
                t = torch.frombuffer(bytearray(new), dtype=torch.uint8).view(getattr(torch, e["dtype"])).reshape(e["shape"])
                with torch.no_grad():
                    dst.copy_(t.to(dst.device))
                n += 1
        self.version = version
        return n


def apply_delta_dir(store, path: str) -> int:
    """Apply one published version directory (``.../v%08d``) to a parameter store; the store remembers the version
    it holds so that an XOR delta is only applied on top of its base."""
    path = path.rstrip("/")
    version = int(os.path.basename(path).lstrip("v"))
    reader = getattr(store, "_delta_reader", None)
    if reader is None or reader.dir != os.path.dirname(path):
        reader = DiskDeltaReader(os.path.dirname(path))
        store._delta_reader = reader
    return reader.apply(version, store.params)


class DiskDeltaUpdater:
    """Trainer side of ``--update-weight-transfer-mode disk-delta``: every weight update publishes a version directory
    of per-tensor deltas (``--update-weight-delta-encoding xor | overwrite``, checksummed with
    ``--update-weight-delta-checksum``) under ``--update-weight-disk-dir`` and tells each engine to pull it
    (``POST /pull_weights``). Engines that fall behind apply the versions in order. Reference:
    miles/backends/megatron_utils/update_weight/ (disk-delta transfer)."""

    def __init__(self, actor, handles: list, directory: str, encoding: str = "xor", checksum_kind: str = "xxh3-128"):
        self.actor, self.handles = actor, list(handles)
        self.writer = DiskDeltaWriter(directory, encoding=encoding, checksum_kind=checksum_kind, rank=actor.ps.rank,
                                      world=actor.ps.world_size)

    def update(self, requantize: str = "none") -> dict:
        """``requantize``: the block-scaled format that the engines serve from copies in."""
        import time

        import torch.distributed as dist

        t0 = time.perf_counter()
        version = self.actor.store.version
        idx = self.writer.write(((n, p) for n, p in self.actor.store.params.items()), version)
        if dist.is_initialized() and self.actor.ps.world_size > 1:
            dist.barrier()  # every rank's file is in place before an engine reads the directory
        vdir = os.path.join(self.writer.dir, f"v{version:08d}")
        futs = [h.post_async("/pull_weights", {"path": vdir, "weight_version": version}) for h in self.handles]
        for f in futs:
            f.result()
        if requantize != "none":
            for h in self.handles:
                h.post("/requantize_weights", {"format": requantize})
        dt = time.perf_counter() - t0
        return {"perf/update_weights_time": dt, "perf/update_weights_total_time": dt, "perf/update_weights_bytes": idx["compressed_bytes"],
                "perf/update_weights_raw_bytes": idx["raw_bytes"], "weight_version": version}
