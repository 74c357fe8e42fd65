"""Operator packages (``tops.ops.gla``, ``tops.ops.simple_gla``, ``tops.ops.ssm``, ``tops.ops.rope``,
``tops.ops.common``)."""
