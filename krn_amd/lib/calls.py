"""What the library's own operations share: a call is checked and marshalled once, then enqueued on the current stream
directly, for an event (`submit`), or again and again (`bind`), as a kernel's launcher does (runtime/api.py `Launcher`)."""

from collections.abc import Callable

from krn_amd.dtypes import Dtype
from krn_amd.runtime import roctx
from krn_amd.runtime.api import Bound, Launcher
from krn_amd.runtime.hip import HIPDevice, HIPEvent, HIPStream, HIPTensor


class Work:
    """One checked call: what it returns, what its launches read and write, and how it goes on a stream."""

    def __init__(self, name: str, device: HIPDevice, result: object, keep: tuple, run: Callable[[HIPStream], None]) -> None:
        self.name, self.device, self.result, self.keep, self.run = name, device, result, keep, run

    def enqueue(self) -> HIPStream:
        stream = self.device.launch_stream()
        if roctx.launch_ranges():
            with roctx.span(f"krn:{self.name}"):
                self.run(stream)
        else:
            self.run(stream)
        stream.note(self.name, self.keep)
        return stream


class LibraryCall(Launcher):
    """An operation of the library: calling it enqueues on the current stream and returns its result."""

    def __init__(self, check: Callable[..., Work]) -> None:
        self.check = check
        self.__doc__, self.__name__ = check.__doc__, check.__name__

    def __call__(self, *args, **kwargs):
        work = self.check(*args, **kwargs)
        work.enqueue()
        return work.result

    def submit(self, *args, **kwargs) -> HIPEvent:
        return self.check(*args, **kwargs).enqueue().record()

    def bind(self, *args, **kwargs) -> "LibraryBound":
        return LibraryBound(self, args, kwargs)


class LibraryBound(Bound):
    """A call with its arguments encoded; `result` is what it writes, allocated once when no `out` was given."""

    def __init__(self, call: LibraryCall, args: tuple, kwargs: dict) -> None:
        self.call = call
        self.rebind(*args, **kwargs)

    def rebind(self, *args, **kwargs) -> None:
        self.work = self.call.check(*args, **kwargs)

    @property
    def result(self):
        return self.work.result

    def __call__(self) -> None:
        self.work.enqueue()

    def submit(self) -> HIPEvent:
        return self.work.enqueue().record()


def tensor(value: object, what: str, rank: int, dtypes: tuple[Dtype, ...]) -> HIPTensor:
    """`value` if it is a device tensor of that rank and one of those element types."""
    if not isinstance(value, HIPTensor):
        raise TypeError(f"{what} is a device tensor, not {type(value).__name__}")
    if len(value.shape) != rank or value.dtype not in dtypes:
        raise ValueError(f"{what} has {rank} axes of {', '.join(map(str, dtypes))}, got {value.dtype}{list(value.shape)}")
    return value
