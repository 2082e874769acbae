"""A matrix in microscaled 4-bit floats (MXFP4): 32 neighbours along a row share a scale 2^(byte - 127), a number is a sign and one of
0, 0.5, 1, 1.5, 2, 3, 4, 6.

``codes`` (uint8 ``[n, k / 2]``, of several experts ``[experts, n, k / 2]``) hold two numbers a byte, the earlier one in the low half.
``scales`` lie in runs of 1,024 bytes for 128 rows and 256 numbers of k, as the tensor cores read them: in a run two halves of four
blocks, in a half 16 bytes for each of 32 lanes, which are the four blocks of rows lane, lane + 32, lane + 64 and lane + 96.  Rows of a
run behind the matrix's last and blocks behind its last hold zeros (rows: anything, in matrices of a step's rows).  ``gated``: the
matrix is a gated unit's first product; of its gate rows and up rows, 16 gate rows and the 16 up rows of the same channels lie in turn.

The modelled project's 4-bit lanes keep int4 codes with a float scale a group (crates/runner/src/llama31_engine.rs:289-430).
"""
from __future__ import annotations

import torch

FP4_BLOCK = 32
_RUN_ROWS, _RUN_BLOCKS = 128, 8


class Fp4Matrix:
    """``shape`` is that of the numbers: (n, k), or (experts, n, k)."""

    __slots__ = ("_codes", "_scales", "shape", "gated", "device", "index", "codes_at", "scales_at", "_buffer", "_counters",
                 "_writes", "_known", "_streams", "_captured", "_settled")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, gated: bool = False):
        shape = tuple(int(s) for s in shape)
        n, k = shape[-2:] if len(shape) in (2, 3) else (0, 0)
        if n <= 0 or k <= 0 or k % FP4_BLOCK or min(shape) <= 0:
            raise ValueError(f"a 4-bit matrix has shape [n, k] or [experts, n, k] with k a multiple of {FP4_BLOCK}, not {shape}")
        if gated and n % (2 * FP4_BLOCK):
            raise ValueError(f"a gated unit has as many gate as up rows, a multiple of {FP4_BLOCK} of each; {n} rows in all")
        runs = (shape[0] if len(shape) == 3 else 1) * -(-n // _RUN_ROWS) * -(-k // (FP4_BLOCK * _RUN_BLOCKS))
        if codes.dtype != torch.uint8 or tuple(codes.shape) != shape[:-1] + (k // 2,) or not codes.is_contiguous():
            raise ValueError(f"codes must be contiguous uint8 {shape[:-1] + (k // 2,)}, are {codes.dtype} {tuple(codes.shape)}")
        if scales.dtype != torch.uint8 or tuple(scales.shape) != (runs, 1024) or not scales.is_contiguous() or scales.device != codes.device:
            raise ValueError(f"scales must be contiguous uint8 {(runs, 1024)} beside the codes, are {scales.dtype} {tuple(scales.shape)}")
        self._codes, self._scales, self.shape, self.gated, self._buffer, self._counters = codes, scales, shape, gated, None, None
        self._writes, self._known, self._settled = [0, False], None, None
        # where they are, for the kernels: the tensors stay what they are as long as the matrix lives
        self.device, self.index, self.codes_at, self.scales_at = codes.device, codes.get_device(), codes.data_ptr(), scales.data_ptr()
        if (self.codes_at | self.scales_at) % 16:
            raise ValueError("codes and scales must start on 16 bytes")

    @classmethod
    def empty(cls, *shape: int, device="cuda", gated: bool = False) -> "Fp4Matrix":
        """Zeros of ``shape``, for ``fp4_ops.quantize`` to fill."""
        if len(shape) not in (2, 3) or min(shape) <= 0 or shape[-1] % FP4_BLOCK:
            raise ValueError(f"a 4-bit matrix has shape [n, k] or [experts, n, k] with k a multiple of {FP4_BLOCK}, not {shape}")
        runs = (shape[0] if len(shape) == 3 else 1) * -(-shape[-2] // _RUN_ROWS) * -(-shape[-1] // (FP4_BLOCK * _RUN_BLOCKS))
        return cls(torch.zeros(shape[:-1] + (shape[-1] // 2,), dtype=torch.uint8, device=device),
                   torch.zeros((runs, 1024), dtype=torch.uint8, device=device), shape, gated)

    @classmethod
    def from_parts(cls, codes: torch.Tensor, scales: torch.Tensor, gated: bool = False) -> "Fp4Matrix":
        """From codes as above and scales in rows, uint8 ``[n, k / 32]`` (``[experts, n, k / 32]``), as model files hold them (255, a scale
        that is no number, is refused).  ``gated``: rows are the gate rows, then the up rows."""
        shape = tuple(codes.shape[:-1]) + (2 * codes.shape[-1],) if codes.dim() in (2, 3) else ()
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or not shape or shape[-1] % FP4_BLOCK \
                or tuple(scales.shape) != shape[:-1] + (shape[-1] // FP4_BLOCK,) or scales.device != codes.device:
            raise ValueError(f"codes uint8 [.., n, k / 2] and scales uint8 [.., n, k / {FP4_BLOCK}] on one device, are {codes.dtype} "
                             f"{tuple(codes.shape)} and {scales.dtype} {tuple(scales.shape)}")
        if bool((scales == 255).any()):
            raise ValueError("a scale of 255 is no number")
        if gated:
            codes, scales = (interleaved(t) for t in (codes, scales))
        n, blocks = scales.shape[-2:]
        s = scales.reshape(-1, n, blocks)
        s = torch.nn.functional.pad(s, (0, -blocks % _RUN_BLOCKS, 0, -n % _RUN_ROWS))
        # [experts, tile, 4, 32 lanes, k-block, half, 4] -> [experts, tile, k-block, half, lane, 4 rows, 4 blocks]
        s = s.view(s.shape[0], s.shape[1] // _RUN_ROWS, 4, 32, s.shape[2] // _RUN_BLOCKS, 2, 4).permute(0, 1, 4, 5, 3, 2, 6)
        return cls(codes.contiguous(), s.reshape(-1, 1024).contiguous(), shape, gated)

    def first_rows(self, n: int) -> "Fp4Matrix":
        """The first ``n`` rows, in the same memory."""
        if len(self.shape) != 2 or self.gated or not 0 < n <= self.shape[0]:
            raise ValueError(f"no first {n} rows of {self}")
        runs = -(-n // _RUN_ROWS) * -(-self.shape[1] // (FP4_BLOCK * _RUN_BLOCKS))
        m = Fp4Matrix(self.codes[:n], self.scales[:runs], (n, self.shape[1]))
        m._buffer = self._buffer
        m._writes, m._settled = self._writes, self._settled
        return m

    # A product may fetch its weights while the launch in front of it still runs, and such a launch sees for certain only what was written
    # before the launch in front of that one ended.  So the first product on a stream behind a write is launched behind everything; the
    # stream's next ones may read ahead.  Writes are counted: this package's (``written``), torch's by the tensors' versions.
    def written(self) -> None:
        """Said by whoever writes codes or scales other than through torch (``fp4_ops.quantize`` does), or in a capture: such a write comes
        again with every replay, so that products outside of graphs do not read ahead from then on."""
        self._writes[0] += 1
        if self.index >= 0 and torch.cuda.is_current_stream_capturing():
            self._writes[1] = True

    def _version(self):
        try:
            return self._writes[0] + self._codes._version + self._scales._version
        except RuntimeError:                                   # tensors of inference mode count no versions
            return None

    def reads_ahead(self, stream: int) -> bool:
        """Whether a product on this stream (its handle, the current one) may read the matrix ahead of its turn; that it is launched now
        is noted."""
        if self._writes[1] and not torch.cuda.is_current_stream_capturing():
            return False
        version = self._version()
        if version is None:                                    # what torch writes is not seen: only what was settled, and not written by a kernel since
            return self._settled == ("writes", self._writes[0])
        if version == self._settled:
            return True
        if version != self._known:
            self._known, self._streams, self._captured = version, set(), set()
        if stream in self._streams:
            return True
        # a captured launch orders nothing that runs outside its graph
        seen = self._captured if torch.cuda.is_current_stream_capturing() else self._streams
        if stream in seen:
            return True
        seen.add(stream)
        return False

    def settle(self) -> "Fp4Matrix":
        """Waits for the device, after which products on any stream may read the matrix ahead, until it is written again.  (Of tensors made
        in inference mode: until ``written`` is said.)"""
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)
        _ = self.codes, self.scales                            # (a step's rows make theirs when they are asked for)
        version = self._version()
        self._settled = ("writes", self._writes[0]) if version is None else version
        return self

    def plain_scales(self) -> torch.Tensor:
        """The scales in rows, uint8 ``[.., n, k / 32]`` (rows in the order that the codes have)."""
        n, k = self.shape[-2:]
        tiles, k_blocks = -(-n // _RUN_ROWS), -(-k // (FP4_BLOCK * _RUN_BLOCKS))
        s = self.scales.view(-1, tiles, k_blocks, 2, 32, 4, 4).permute(0, 1, 5, 4, 2, 3, 6)
        s = s.reshape(-1, tiles * _RUN_ROWS, k_blocks * _RUN_BLOCKS)[:, :n, : k // FP4_BLOCK]
        return s.reshape(self.shape[:-1] + (k // FP4_BLOCK,)).contiguous()

    @staticmethod
    def rows_layout(n: int, k: int):
        """(bytes of codes up to a whole 256, bytes of both) of a step's rows [n, k] in one buffer (:meth:`over_rows`)."""
        codes = (n * (k // 2) + 255) // 256 * 256
        return codes, codes + -(-n // _RUN_ROWS) * -(-k // (FP4_BLOCK * _RUN_BLOCKS)) * 1024

    @classmethod
    def over_rows(cls, buffer: torch.Tensor, n: int, k: int, codes: int) -> "Fp4Matrix":
        """A step's rows [n, k] at the start of an int8 ``buffer``: ``codes`` bytes of codes, then scales (:meth:`rows_layout`)."""
        m = cls.__new__(cls)
        m._codes = m._scales = m._counters = None          # made when somebody asks for them
        m._writes, m._known, m._settled = [0, False], None, None
        m.shape, m.gated, m._buffer, m.device, m.index = (n, k), False, buffer, buffer.device, buffer.get_device()
        m.codes_at = buffer.data_ptr()
        m.scales_at = m.codes_at + codes
        return m

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            n, k = self.shape
            self._codes = self._buffer[: n * (k // 2)].view(torch.uint8).view(n, k // 2)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            codes, both = self.rows_layout(*self.shape)
            self._scales = self._buffer[codes:both].view(torch.uint8).view(-1, 1024)
        return self._scales

    def bytes_held(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self) -> str:
        return f"Fp4Matrix({list(self.shape)}{', gated' if self.gated else ''}, {self.device})"


def interleaved(t: torch.Tensor) -> torch.Tensor:
    """Rows (the last but one dimension) that are a gated unit's gate rows, then its up rows: 16 of each in turn."""
    n = t.shape[-2]
    if n % 32:
        raise ValueError(f"{n} rows are not 16 gate and 16 up rows in turn")
    return t.unflatten(-2, (2, n // 32, 16)).transpose(-4, -3).flatten(-4, -2)
