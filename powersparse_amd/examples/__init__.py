"""Small programs that use the framework as a user would."""
