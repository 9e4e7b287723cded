"""mok: B200-native MoE-layer kernels behind the operator and functional surface of
cursor/mixture-of-kittens (`mok.ops`, `mok.functional`)."""
from . import functional, ops  # noqa: F401
from .functional import (  # noqa: F401
    MoKConfig, MoKForwardContext, MoKPackedContext, MoKRouterConfig, MoKRouting, MoKSchedule, MoKWorkspace)

__all__ = ["functional", "ops", "MoKConfig", "MoKForwardContext", "MoKPackedContext", "MoKRouterConfig", "MoKRouting", "MoKSchedule",
           "MoKWorkspace"]
